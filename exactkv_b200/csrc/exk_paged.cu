// New tokens entering a paged cache (sm_100a): the packed queries, keys and
// values of a batch are rotated at their positions (queries and keys, after an
// optional RMS norm per head) and the keys and values stored in their
// sequences' pages, in bf16 pools or in the coded format.
//
// Token i of sequence b sits at position p = seq_lens[b] - n_b + i. With c, s
// the table's cosines and sines of p, channel j < 64 of a head x becomes
//   y_j = x_j c_j - x_{j+64} s_j,   y_{j+64} = x_{j+64} c_j + x_j s_j
// in fp32, every product and sum rounded by itself (no fma), then once to
// bf16: the stored bits do not depend on the path a token takes (one token at
// a time, a whole prompt, either pool). The norm is x rsqrt(mean x^2 + eps) w in fp32
// before the rotation, with no rounding between.
#include <algorithm>

#include "exk_device.cuh"
#include "exk_encode.cuh"
#include "exk_host.h"

namespace exk {

struct Append {
  exk_append t;
  // coded pools: [0] keys, [1] values
  uint8_t* sm[2];
  uint8_t* code[2];
  uint8_t* base[2];
  int32_t* rowmask[2];
  int32_t* rowoff[2];
  uint16_t* raw[2];
  int64_t cap[2];
  int32_t* cnt[2];
  int32_t tails;      // open pages per KV head that the raw pools hold
  uint8_t* counts;    // [2][items_pad] raw rows of every item (scratch)
  int32_t* base_cnt;  // [2] the pools' counters before this call (scratch)
  int32_t slots;      // page slots of the call (see page_slot)
  int32_t items;      // slots * Hkv
  int32_t items_pad;  // items rounded up to 16
  // bf16 pools
  uint16_t* pool[2];
  int32_t* status;
};

// Sequences whose end cu[b + 1] + b * step (each divided by div first) is at or
// before x: the index of the sequence that holds x when the ends are
// ascending. One round of independent loads for up to 32 sequences; called by
// a whole warp with the same x.
__device__ __forceinline__ int find_seq(const int32_t* cu, int B, int div, int step, int x, int lane) {
  int n = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int b = b0 + lane;
    const bool before = b < B && __ldg(cu + b + 1) / div + (b + 1) * step <= x;
    n += __popc(__ballot_sync(0xFFFFFFFFu, before));
  }
  return n;
}

struct Seq {
  int b, first, n, start;  // sequence, its first packed token, its tokens, its first position
};

__device__ __forceinline__ Seq load_seq(const exk_append& t, int b) {
  Seq s;
  s.b = b;
  s.first = t.cu_seqlens == nullptr ? b : __ldg(t.cu_seqlens + b);
  s.n = (t.cu_seqlens == nullptr ? b + 1 : __ldg(t.cu_seqlens + b + 1)) - s.first;
  if (s.first < 0 || s.n < 0 || s.first > t.N - s.n) s.n = 0;  // not a batch's bounds: nothing of it is read
  s.start = __ldg(t.seq_lens + b) - s.n;
  return s;
}

// A position that can be stored and rotated.
__device__ __forceinline__ bool position_ok(const exk_append& t, int pos) {
  return pos >= 0 && pos < t.rope_rows && pos < t.max_pages * kP;
}

// Pool page of page pg of sequence b, or -1 (reported).
__device__ __forceinline__ int pool_page(const Append& a, int b, int pg) {
  const int p = __ldg(a.t.block_table + static_cast<int64_t>(b) * a.t.max_pages + pg);
  if (p >= 0 && p < a.t.pool_pages) return p;
  set_status(a.status, EXK_S_PAGE_INDEX);
  return -1;
}

// ---------------------------------------------------------------- rotation

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// The pair (x_j, x_{j+64}) rotated.
__device__ __forceinline__ void rotate(float& lo, float& hi, float c, float s) {
  const float l = lo, h = hi;
  lo = __fsub_rn(__fmul_rn(l, c), __fmul_rn(h, s));
  hi = __fadd_rn(__fmul_rn(h, c), __fmul_rn(l, s));
}

// NW packed words of each half (channels c0 .. c0 + 2 NW - 1 and those + 64)
// of one head, held by LANES lanes of a group: normalised (w != nullptr) and
// rotated. cs: the position's row of the table.
template <int NW, int LANES>
__device__ __forceinline__ void norm_rotate(uint32_t (&lo)[NW], uint32_t (&hi)[NW], int c0, const uint16_t* w, float eps,
                                            const float (&c)[2 * NW], const float (&s)[2 * NW]) {
  float x[2 * NW], y[2 * NW];
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    x[2 * j] = bf_lo(lo[j]);
    x[2 * j + 1] = bf_hi(lo[j]);
    y[2 * j] = bf_lo(hi[j]);
    y[2 * j + 1] = bf_hi(hi[j]);
  }
  if (w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 2 * NW; ++j) ss += x[j] * x[j] + y[j] * y[j];
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
    const float r = rsqrtf(ss * (1.f / kD) + eps);
#pragma unroll
    for (int j = 0; j < 2 * NW; ++j) {
      x[j] = x[j] * r * __uint_as_float(static_cast<uint32_t>(__ldg(w + c0 + j)) << 16);
      y[j] = y[j] * r * __uint_as_float(static_cast<uint32_t>(__ldg(w + 64 + c0 + j)) << 16);
    }
  }
#pragma unroll
  for (int j = 0; j < 2 * NW; ++j) rotate(x[j], y[j], c[j], s[j]);
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    lo[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
    hi[j] = pack_bf16x2(y[2 * j], y[2 * j + 1]);
  }
}

__device__ __forceinline__ void load4(float* d, const float* s) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(s));
  d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w;
}

// ---------------------------------------------------------------- rows of a token

constexpr int kRowWarps = 8;
constexpr int kQuads = 2;  // groups of four heads one warp takes

// One warp: heads 4 * quad0 .. of one token (the queries' heads, then, with
// KV, the keys' and the values'), eight lanes to a head, 16 bytes of each half
// to a lane.
template <bool KV>
__device__ __forceinline__ void token_rows(const Append& a, int64_t work, int lane) {
  const exk_append& t = a.t;
  const int heads = t.Hq + (KV ? 2 * t.Hkv : 0);
  const int per_token = (heads + 4 * kQuads - 1) / (4 * kQuads);
  const int tok = static_cast<int>(work / per_token);
  if (tok >= t.N) return;
  const int h0 = static_cast<int>(work % per_token) * (4 * kQuads) + (lane >> 3);
  const int b = t.cu_seqlens == nullptr ? tok : find_seq(t.cu_seqlens, t.B, 1, 0, tok, lane);
  if (b >= t.B) return;  // behind the last sequence
  const Seq s = load_seq(t, b);
  if (s.n <= 0) return;
  const int pos = s.start + tok - s.first;
  const bool ok = position_ok(t, pos);
  const int c0 = 8 * (lane & 7);
  float c[8], sn[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = sn[j] = 0.f;
  int64_t row = -1;
  if (ok) {
    const float* cs = t.cos_sin + static_cast<int64_t>(pos) * kD + c0;
    load4(c, cs);
    load4(c + 4, cs + 4);
    load4(sn, cs + 64);
    load4(sn + 4, cs + 68);
    if (KV) {
      const int page = pool_page(a, b, pos / kP);
      if (page >= 0) row = static_cast<int64_t>(page) * kP + pos % kP;
    }
  } else {
    set_status(a.status, EXK_S_POSITION);
  }
  uint32_t lo[kQuads][4], hi[kQuads][4];
#pragma unroll
  for (int u = 0; u < kQuads; ++u) {
    const int h = h0 + 4 * u;
    const uint16_t* src = nullptr;
    if (h < t.Hq)
      src = t.q + tok * t.q_st + h * t.q_sh;
    else if (KV && h < t.Hq + t.Hkv)
      src = t.k + tok * t.k_st + (h - t.Hq) * t.k_sh;
    else if (KV && h < heads)
      src = t.v + tok * t.v_st + (h - t.Hq - t.Hkv) * t.v_sh;
    uint4 l = make_uint4(0, 0, 0, 0), g = l;
    if (src != nullptr) {
      l = *reinterpret_cast<const uint4*>(src + c0);
      g = *reinterpret_cast<const uint4*>(src + 64 + c0);
    }
    lo[u][0] = l.x; lo[u][1] = l.y; lo[u][2] = l.z; lo[u][3] = l.w;
    hi[u][0] = g.x; hi[u][1] = g.y; hi[u][2] = g.z; hi[u][3] = g.w;
  }
#pragma unroll
  for (int u = 0; u < kQuads; ++u) {
    const int h = h0 + 4 * u;
    if (h - (lane >> 3) >= heads) break;  // whole warp
    // a warp's four heads may be of two kinds: every lane runs the same
    // shuffles, and a value head keeps what it loaded
    const bool value = KV && h >= t.Hq + t.Hkv;
    uint32_t rl[4], rh[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      rl[j] = lo[u][j];
      rh[j] = hi[u][j];
    }
    if (t.q_norm != nullptr || t.k_norm != nullptr) {
      // both norms or none (checked on the host)
      norm_rotate<4, 8>(rl, rh, c0, h < t.Hq ? t.q_norm : t.k_norm, t.eps, c, sn);
    } else {
      norm_rotate<4, 8>(rl, rh, c0, nullptr, 0.f, c, sn);
    }
    uint16_t* dst = nullptr;
    if (h < t.Hq)
      dst = t.q_out + tok * t.o_st + h * t.o_sh;
    else if (KV && row >= 0 && h < heads)
      dst = a.pool[value ? 1 : 0] + (row * t.Hkv + (h - t.Hq - (value ? t.Hkv : 0))) * kD;
    if (dst == nullptr) continue;
    if (value) {
      *reinterpret_cast<uint4*>(dst + c0) = make_uint4(lo[u][0], lo[u][1], lo[u][2], lo[u][3]);
      *reinterpret_cast<uint4*>(dst + 64 + c0) = make_uint4(hi[u][0], hi[u][1], hi[u][2], hi[u][3]);
    } else {
      *reinterpret_cast<uint4*>(dst + c0) = make_uint4(rl[0], rl[1], rl[2], rl[3]);
      *reinterpret_cast<uint4*>(dst + 64 + c0) = make_uint4(rh[0], rh[1], rh[2], rh[3]);
    }
  }
}

__global__ void __launch_bounds__(kRowWarps * 32) append_bf16_kernel(const __grid_constant__ Append a) {
  token_rows<true>(a, static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5), threadIdx.x & 31);
}

// ---------------------------------------------------------------- coded pools
//
// Work items are (page slot, KV head) of the keys and of the values. Sequence
// b's touched pages take slots cu[b] / 16 + 2b, + 1, ...: n tokens touch at
// most (n + 30) / 16 pages, which never reaches sequence b + 1's first slot,
// so the map needs no prefix sum over the batch; slots left over are empty.
// With one token per sequence (cu_seqlens null) slot b is sequence b's.
// append_encode_kernel gives every item a warp: a page that the call completes
// is encoded, with its raw-row count left in `counts`; a page that stays open
// gets its new rows in the sequence's tail rows. append_place_kernel turns the
// counts into raw-pool slots in (sequence, page, head) order and copies the
// escaped rows. A call that completes a page whose earlier rows are in the
// tail and leaves another page open writes the latter's rows in the second
// kernel, by the warp that has copied the former's escaped rows.

struct Item {
  Seq s;
  int h, pg, pool;     // KV head, page of the sequence, its page in the pool (-1: nothing to do)
  int slot;            // tail slot of the sequence
  bool full;           // the call completes the page
  bool later;          // open, and written by append_place_kernel
};

__device__ __forceinline__ int last_page(const Seq& s) { return (s.start + s.n - 1) / kP; }

__device__ __forceinline__ bool tail_of(const Append& a, int b, int& slot) {
  slot = a.t.slots == nullptr ? b : __ldg(a.t.slots + b);
  if (slot >= 0 && slot < a.tails) return true;
  set_status(a.status, EXK_S_POSITION);
  return false;
}

// Item `item` of the call (whole warp); pool = -1 where there is nothing to do.
__device__ __forceinline__ Item load_item(const Append& a, int item, int lane) {
  const exk_append& t = a.t;
  Item it;
  it.h = item % t.Hkv;
  const int slot = item / t.Hkv;
  it.pool = -1;
  it.full = it.later = false;
  const int b = t.cu_seqlens == nullptr ? slot : find_seq(t.cu_seqlens, t.B, kP, 2, slot, lane);
  if (b >= t.B) return it;
  it.s = load_seq(t, b);
  if (it.s.n <= 0) return it;
  if (!position_ok(t, it.s.start) || !position_ok(t, it.s.start + it.s.n - 1)) {
    set_status(a.status, EXK_S_POSITION);
    return it;
  }
  it.pg = it.s.start / kP + (t.cu_seqlens == nullptr ? 0 : slot - (it.s.first / kP + 2 * b));
  if (it.pg > last_page(it.s) || !tail_of(a, b, it.slot)) return it;
  it.full = (it.pg + 1) * kP <= it.s.start + it.s.n;
  it.later = !it.full && it.pg * kP > it.s.start && it.s.start % kP != 0;
  it.pool = pool_page(a, b, it.pg);
  return it;
}

// The lane's channels (4q.. and 64 + 4q..) of packed token tok, KV head h, as
// the cache holds them: keys (which = 0) normalised and rotated at pos.
__device__ __forceinline__ void cache_row(const Append& a, int which, int tok, int h, int pos, int q, uint32_t (&w)[4]) {
  const exk_append& t = a.t;
  const uint16_t* src = which == 0 ? t.k + tok * t.k_st + h * t.k_sh : t.v + tok * t.v_st + h * t.v_sh;
  const uint2 lo = *reinterpret_cast<const uint2*>(src + 4 * q);
  const uint2 hi = *reinterpret_cast<const uint2*>(src + 64 + 4 * q);
  uint32_t l[2] = {lo.x, lo.y}, g[2] = {hi.x, hi.y};
  if (which == 0) {
    float c[4], s[4];
    const float* cs = t.cos_sin + static_cast<int64_t>(pos) * kD + 4 * q;
    load4(c, cs);
    load4(s, cs + 64);
    norm_rotate<2, 16>(l, g, 4 * q, t.k_norm, t.eps, c, s);
  }
  w[0] = l[0]; w[1] = l[1]; w[2] = g[0]; w[3] = g[1];
}

__device__ __forceinline__ uint16_t* tail_row(const Append& a, int which, int slot, int h, int r) {
  return a.raw[which] + (a.cap[which] + (static_cast<int64_t>(slot) * a.t.Hkv + h) * kP + r) * kD;
}

__device__ __forceinline__ void store_quads(uint16_t* d, int q, const uint32_t (&w)[4]) {
  *reinterpret_cast<uint2*>(d + 4 * q) = make_uint2(w[0], w[1]);
  *reinterpret_cast<uint2*>(d + 64 + 4 * q) = make_uint2(w[2], w[3]);
}

// The new rows of an open page into the sequence's tail rows, and the page's
// entry: all rows raw, at the tail rows.
__device__ __forceinline__ void write_open(const Append& a, const Item& it, int which, int lane) {
  const int q = lane & 15, th = lane >> 4;
  const int end = it.s.start + it.s.n;
  // two rows at a time, one per half warp; the norm's shuffles need every lane
  for (int r = max(0, it.s.start - it.pg * kP) & ~1; it.pg * kP + r < end; r += 2) {
    const int pos = it.pg * kP + r + th;
    const bool mine = pos >= it.s.start && pos < end;
    const int at = min(max(pos, it.s.start), end - 1);
    uint32_t w[4];
    cache_row(a, which, it.s.first + at - it.s.start, it.h, at, q, w);
    if (mine) store_quads(tail_row(a, which, it.slot, it.h, r + th), q, w);
  }
  if (lane == 0) {
    const int64_t page = static_cast<int64_t>(it.pool) * a.t.Hkv + it.h;
    a.rowmask[which][page] = 0xFFFF;
    a.rowoff[which][page] = static_cast<int32_t>(a.cap[which] + (static_cast<int64_t>(it.slot) * a.t.Hkv + it.h) * kP);
  }
}

// Blocks below `enc_blocks`: the items; the others rotate the queries.
__global__ void __launch_bounds__(kRowWarps * 32) append_encode_kernel(const __grid_constant__ Append a, int enc_blocks) {
  allow_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (static_cast<int>(blockIdx.x) >= enc_blocks) {
    token_rows<false>(a, static_cast<int64_t>(blockIdx.x - enc_blocks) * kRowWarps + warp, lane);
    return;
  }
  if (blockIdx.x == 0 && threadIdx.x < 2) a.base_cnt[threadIdx.x] = *a.cnt[threadIdx.x];
  const int work = blockIdx.x * kRowWarps + warp;
  if (work >= 2 * a.items) return;
  const int which = work >= a.items ? 1 : 0, item = work - which * a.items;
  const Item it = load_item(a, item, lane);
  uint32_t rm = 0u;
  if (it.pool >= 0 && it.full) {
    const int q = lane & 15, th = lane >> 4;
    uint32_t w[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pos = it.pg * kP + 8 * th + i;
      // (rows of the page that this call does not bring come from the tail)
      const int at = max(pos, it.s.start);
      cache_row(a, which, it.s.first + at - it.s.start, it.h, at, q, w[i]);
      if (pos < it.s.start) {
        const uint16_t* tr = tail_row(a, which, it.slot, it.h, 8 * th + i);
        const uint2 lo = *reinterpret_cast<const uint2*>(tr + 4 * q), hi = *reinterpret_cast<const uint2*>(tr + 64 + 4 * q);
        w[i][0] = lo.x; w[i][1] = lo.y; w[i][2] = hi.x; w[i][3] = hi.y;
      }
    }
    const int64_t page = static_cast<int64_t>(it.pool) * a.t.Hkv + it.h;
    const int64_t row = static_cast<int64_t>(it.pool) * kP * a.t.Hkv + it.h;
    rm = encode_rows(w, lane, a.sm[which] + row * kD, static_cast<int64_t>(a.t.Hkv) * kD, a.code[which] + row * (kD / 2),
                     static_cast<int64_t>(a.t.Hkv) * (kD / 2), a.base[which] + page * kD);
    if (lane == 0) a.rowmask[which][page] = static_cast<int32_t>(rm);
  } else if (it.pool >= 0 && !it.later) {
    write_open(a, it, which, lane);
  }
  if (lane == 0) a.counts[static_cast<int64_t>(which) * a.items_pad + item] = static_cast<uint8_t>(__popc(rm));
}

constexpr int kPlaceItems = 256;  // items of one CTA of append_place_kernel, one per thread

// blockIdx.y: keys, values. The CTA adds up the counts of all items before its
// own (bytes: 65,536 items are 16 loads of 16 bytes per thread), scans its
// own, writes the offsets and copies the escaped rows.
__global__ void __launch_bounds__(kPlaceItems) append_place_kernel(const __grid_constant__ Append a) {
  __shared__ int s_warp[kPlaceItems / 32], s_before[kPlaceItems / 32];
  __shared__ int s_off[kPlaceItems];
  after_prior();
  const int which = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint8_t* counts = a.counts + static_cast<int64_t>(which) * a.items_pad;
  const int i0 = blockIdx.x * kPlaceItems, mine = i0 + threadIdx.x;
  int before = 0;
  for (int i = threadIdx.x; i < i0 / 16; i += kPlaceItems) {
    const uint4 v = reinterpret_cast<const uint4*>(counts)[i];
    before = __dp4a(v.x, 0x01010101u, static_cast<uint32_t>(before));
    before = __dp4a(v.y, 0x01010101u, static_cast<uint32_t>(before));
    before = __dp4a(v.z, 0x01010101u, static_cast<uint32_t>(before));
    before = __dp4a(v.w, 0x01010101u, static_cast<uint32_t>(before));
  }
  const int n = mine < a.items ? counts[mine] : 0;
  int incl = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xFFFFFFFFu, incl, d);
    if (lane >= d) incl += y;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) before += __shfl_xor_sync(0xFFFFFFFFu, before, d);
  if (lane == 31) s_warp[warp] = incl;
  if (lane == 0) s_before[warp] = before;
  __syncthreads();
  int off = a.base_cnt[which] + incl - n, total = 0;
  for (int w = 0; w < kPlaceItems / 32; ++w) {
    off += s_before[w];
    if (w < warp) off += s_warp[w];
    total += s_before[w] + s_warp[w];
  }
  s_off[threadIdx.x] = off;
  // (may exceed the capacity: the caller grows the pool before it calls)
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *a.cnt[which] = a.base_cnt[which] + total;
  __syncthreads();
  const int q = lane & 15, th = lane >> 4;
  for (int i = warp; i < kPlaceItems && i0 + i < a.items; i += kPlaceItems / 32) {
    Item it = load_item(a, i0 + i, lane);
    if (it.pool < 0 || !it.full) continue;
    const int64_t page = static_cast<int64_t>(it.pool) * a.t.Hkv + it.h;
    if (lane == 0) a.rowoff[which][page] = s_off[i];
    uint32_t rm = static_cast<uint32_t>(a.rowmask[which][page]) & 0xFFFFu;
    int64_t ridx = s_off[i];
    for (; rm != 0u; rm &= rm - 1u, ++ridx) {
      if (ridx < 0 || ridx >= a.cap[which]) continue;
      const int r = __ffs(rm) - 1, pos = it.pg * kP + r;
      const int at = max(pos, it.s.start);
      uint32_t w[4];
      cache_row(a, which, it.s.first + at - it.s.start, it.h, at, q, w);
      if (pos < it.s.start) {
        const uint16_t* tr = tail_row(a, which, it.slot, it.h, r);
        const uint2 lo = *reinterpret_cast<const uint2*>(tr + 4 * q), hi = *reinterpret_cast<const uint2*>(tr + 64 + 4 * q);
        w[0] = lo.x; w[1] = lo.y; w[2] = hi.x; w[3] = hi.y;
      }
      if (th == 0) store_quads(a.raw[which] + ridx * kD, q, w);
    }
    const int last = last_page(it.s);
    if (it.pg == it.s.start / kP && it.s.start % kP != 0 && last > it.pg && (last + 1) * kP > it.s.start + it.s.n) {
      it.pg = last;
      it.pool = pool_page(a, it.s.b, last);
      __syncwarp();  // every lane has read the tail rows
      if (it.pool >= 0) write_open(a, it, which, lane);
    }
  }
}

}  // namespace exk

using namespace exk;

namespace {

int check_append(const exk_append* t) {
  if (t == nullptr) return EXK_EARG;
  if (t->q == nullptr || t->k == nullptr || t->v == nullptr || t->q_out == nullptr || t->cos_sin == nullptr ||
      t->seq_lens == nullptr || t->block_table == nullptr || (t->q_norm == nullptr) != (t->k_norm == nullptr))
    return EXK_EARG;
  if (t->N < 0 || t->B <= 0 || t->Hq <= 0 || t->Hkv <= 0 || t->Hq % t->Hkv != 0 || t->rope_rows <= 0 ||
      t->max_pages <= 0 || t->max_pages > (1 << 26) || t->pool_pages <= 0)
    return EXK_EARG;
  if (t->cu_seqlens == nullptr && t->N != t->B) return EXK_EARG;
  if (t->N > (1 << 28) || t->B > (1 << 24) || t->Hq > 4096) return EXK_EARG;
  if (!aligned16(t->q) || !aligned16(t->k) || !aligned16(t->v) || !aligned16(t->q_out) || !aligned16(t->cos_sin))
    return EXK_EALIGN;
  for (int64_t s : {t->q_st, t->q_sh, t->k_st, t->k_sh, t->v_st, t->v_sh, t->o_st, t->o_sh})
    if (s % 8 != 0) return EXK_EALIGN;
  return 0;
}

int64_t row_blocks(const exk_append& t, int heads) {
  const int64_t work = static_cast<int64_t>(t.N) * ((heads + 4 * kQuads - 1) / (4 * kQuads));
  return (work + kRowWarps - 1) / kRowWarps;
}

int64_t page_slots(const exk_append& t) {
  return t.cu_seqlens == nullptr ? t.B : t.N / kP + 2 * static_cast<int64_t>(t.B);
}

}  // namespace

extern "C" int exk_rope_append_bf16(const exk_append* t, uint16_t* k_pool, uint16_t* v_pool, int32_t* status, int device,
                                    void* stream) {
  int r = check_append(t);
  if (r != 0) return r;
  if (k_pool == nullptr || v_pool == nullptr) return EXK_EARG;
  if (!aligned16(k_pool) || !aligned16(v_pool)) return EXK_EALIGN;
  if (t->N == 0) return 0;
  const int64_t blocks = row_blocks(*t, t->Hq + 2 * t->Hkv);
  if (blocks >= (int64_t{1} << 31)) return EXK_EARG;
  DeviceScope scope;
  if ((r = use_device(device, nullptr)) != 0) return r;
  Append a = {};
  a.t = *t;
  a.pool[0] = k_pool;
  a.pool[1] = v_pool;
  a.status = status;
  append_bf16_kernel<<<static_cast<unsigned>(blocks), kRowWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return launch_status();
}

extern "C" int64_t exk_rope_append_scratch(int N, int B, int Hkv, int packed) {
  if (N < 0 || B <= 0 || Hkv <= 0) return EXK_EARG;
  const int64_t items = (packed ? N / kP + 2 * static_cast<int64_t>(B) : B) * Hkv;
  return 2 * ((items + 15) / 16 * 16) + 16;
}

extern "C" int exk_rope_append_compressed(const exk_append* t, const exk_cview* k, int64_t k_cap, int32_t* k_cnt,
                                          const exk_cview* v, int64_t v_cap, int32_t* v_cnt, void* scratch,
                                          int64_t scratch_bytes, int32_t* status, int device, void* stream) {
  int r = check_append(t);
  if (r != 0) return r;
  if (k == nullptr || v == nullptr || k_cnt == nullptr || v_cnt == nullptr || scratch == nullptr) return EXK_EARG;
  const exk_cview* c[2] = {k, v};
  const int64_t cap[2] = {k_cap, v_cap};
  int32_t* cnt[2] = {k_cnt, v_cnt};
  const int64_t items = page_slots(*t) * t->Hkv;
  if (items > (int64_t{1} << 29)) return EXK_EARG;
  Append a = {};
  a.t = *t;
  int64_t tails = int64_t{1} << 24;
  for (int i = 0; i < 2; ++i) {
    if (c[i]->sm == nullptr || c[i]->code == nullptr || c[i]->base == nullptr || c[i]->rowmask == nullptr ||
        c[i]->rowoff == nullptr || c[i]->raw == nullptr || cap[i] < 0 || c[i]->raw_rows < cap[i] ||
        c[i]->raw_rows >= (int64_t{1} << 31))
      return EXK_EARG;
    if (!aligned16(c[i]->sm) || !aligned16(c[i]->code) || !aligned16(c[i]->base) || !aligned16(c[i]->raw))
      return EXK_EALIGN;
    tails = std::min(tails, (c[i]->raw_rows - cap[i]) / (static_cast<int64_t>(t->Hkv) * kP));
    a.sm[i] = const_cast<uint8_t*>(c[i]->sm);
    a.code[i] = const_cast<uint8_t*>(c[i]->code);
    a.base[i] = const_cast<uint8_t*>(c[i]->base);
    a.rowmask[i] = const_cast<int32_t*>(c[i]->rowmask);
    a.rowoff[i] = const_cast<int32_t*>(c[i]->rowoff);
    a.raw[i] = const_cast<uint16_t*>(c[i]->raw);
    a.cap[i] = cap[i];
    a.cnt[i] = cnt[i];
  }
  if (tails < (t->slots == nullptr ? t->B : 1)) return EXK_EARG;  // an open page for every sequence
  if (!aligned16(scratch)) return EXK_EALIGN;
  if (scratch_bytes < exk_rope_append_scratch(t->N, t->B, t->Hkv, t->cu_seqlens != nullptr)) return EXK_EARG;
  if (t->N == 0) return 0;
  DeviceScope scope;
  if ((r = use_device(device, nullptr)) != 0) return r;
  a.tails = static_cast<int32_t>(tails);
  a.slots = static_cast<int32_t>(page_slots(*t));
  a.items = static_cast<int32_t>(items);
  a.items_pad = static_cast<int32_t>((items + 15) / 16 * 16);
  a.base_cnt = static_cast<int32_t*>(scratch);
  a.counts = static_cast<uint8_t*>(scratch) + 16;
  a.status = status;
  const int64_t enc = (2 * items + kRowWarps - 1) / kRowWarps;
  const int64_t blocks = enc + row_blocks(*t, t->Hq);
  if (blocks >= (int64_t{1} << 31)) return EXK_EARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  append_encode_kernel<<<static_cast<unsigned>(blocks), kRowWarps * 32, 0, st>>>(a, static_cast<int>(enc));
  if ((r = launch_status()) != 0) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((items + kPlaceItems - 1) / kPlaceItems), 2);
  cfg.blockDim = dim3(kPlaceItems);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, append_place_kernel, a);
  if (e == cudaSuccess) return 0;
  (void)cudaGetLastError();
  return static_cast<int>(e);
}
