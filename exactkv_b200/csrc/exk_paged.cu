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
//
// Long calls are bound by memory: 11,016 tokens of 32 + 8 + 8 heads into bf16 pages
// take 44.4 us (276 MB, 6.2 TB/s; with the norm 49 us), 9,529 of 28 + 4 + 4 into
// coded pages 36 us (14 the encoding, 22 the queries, the raw rows' places beside
// them; 39 us a call with its launches); a step of 64 sequences 3 us, of 32 into coded
// pages 9 us.
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
  int64_t cap[2], raw_rows[2];
  int32_t* cnt[2];
  int32_t tails;      // open pages per KV head that the raw pools hold
  uint8_t* counts;    // [2][items_pad] raw rows of every item, and its flags (scratch)
  int2* pages;        // [items] where the item completed its page: its entry of the page arrays, its sequence (scratch)
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

// -0 that the compiler does not know: x y + (-0) is the rounded product, kept
// from being fused with the sum that follows (a packed product and a packed sum,
// both .rn, come out as one packed fma).
static __constant__ float c_minus_zero = -0.f;

// Cosines and sines of 2 NW consecutive channels, as pairs; sines negated too:
// l c - h s is formed as l c + h (-s), the same bits, so that two channels at a
// time are rotated by packed products and sums.
template <int NW>
struct Turn {
  F2 c[NW], s[NW], ns[NW];
};

__device__ __forceinline__ float4 ldg4(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }

// Channels c0 .. c0 + 2 NW - 1 of the table's row `cs`.
template <int NW>
__device__ __forceinline__ void load_turn(const float* cs, int c0, Turn<NW>& t) {
#pragma unroll
  for (int j = 0; j < NW; j += 2) {
    const float4 c = ldg4(cs + c0 + 2 * j), s = ldg4(cs + 64 + c0 + 2 * j);
    t.c[j] = f2(c.x, c.y);
    t.c[j + 1] = f2(c.z, c.w);
    t.s[j] = f2(s.x, s.y);
    t.s[j + 1] = f2(s.z, s.w);
    t.ns[j] = f2(-s.x, -s.y);
    t.ns[j + 1] = f2(-s.z, -s.w);
  }
}

// One head held by a group of lanes, NW packed words of each half (channels c0 ..
// c0 + 2 NW - 1 and those + 64) to a lane: this lane's part of its sum of squares.
// Every path adds in one order, whatever its lanes hold: channels 4i .. 4i + 3 and
// those + 64 first (i = 0 .. 15), then i with i ^ 1, i ^ 8, i ^ 4 and i ^ 2.
template <int NW>
__device__ __forceinline__ float squares(const uint32_t (&lo)[NW], const uint32_t (&hi)[NW]) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NW; i += 2) {
    F2 ss = f2(0.f, 0.f);
#pragma unroll
    for (int j = i; j < i + 2; ++j) {
      const F2 x = f2_bf16(lo[j]), y = f2_bf16(hi[j]);
      ss = fma2(y, y, fma2(x, x, ss));
    }
    float s0, s1;
    split2(ss, s0, s1);
    sum = i == 0 ? s0 + s1 : sum + (s0 + s1);
  }
  return sum;
}

// 1 / sqrt(mean square + eps) of a head's sum of squares.
__device__ __forceinline__ float norm_factor(float sum, float eps) { return rsqrtf(fmaf(sum, 1.f / kD, eps)); }

// The head rotated, after the norm by weight w where NORM: r = 1 / sqrt(mean square + eps).
template <int NW, bool NORM>
__device__ __forceinline__ void norm_rotate(uint32_t (&lo)[NW], uint32_t (&hi)[NW], int c0, const uint16_t* w, float r,
                                            const Turn<NW>& t) {
  F2 x[NW], y[NW];
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    x[j] = f2_bf16(lo[j]);
    y[j] = f2_bf16(hi[j]);
  }
  if constexpr (NORM) {
    const F2 rr = f2(r, r);
#pragma unroll
    for (int j = 0; j < NW; j += 2) {
      const uint2 a = __ldg(reinterpret_cast<const uint2*>(w + c0 + 2 * j));
      const uint2 b = __ldg(reinterpret_cast<const uint2*>(w + 64 + c0 + 2 * j));
      x[j] = mul2(mul2(x[j], rr), f2_bf16(a.x));
      x[j + 1] = mul2(mul2(x[j + 1], rr), f2_bf16(a.y));
      y[j] = mul2(mul2(y[j], rr), f2_bf16(b.x));
      y[j + 1] = mul2(mul2(y[j + 1], rr), f2_bf16(b.y));
    }
  }
  const float mz = c_minus_zero;
  const F2 z = f2(mz, mz);
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    lo[j] = bf16_f2(add2(fma2(x[j], t.c[j], z), fma2(y[j], t.ns[j], z)));
    hi[j] = bf16_f2(add2(fma2(y[j], t.c[j], z), fma2(x[j], t.s[j], z)));
  }
}

// ---------------------------------------------------------------- rows of a token

constexpr int kRowWarps = 4;
// Groups of four heads that a warp has in flight at once: four with 124 registers
// (11,016 tokens of 48 heads: 44.3 us, 6.2 TB/s; two: 49.0 us); the norm's
// shuffles make two with more warps better (50.3 us; four: 61.4 us).
template <bool NORM>
constexpr int kQuads = NORM ? 2 : 4;

// One warp: `steps` times 4 * kQuads heads of one token (the queries' heads,
// then, with KV, the keys' and the values'), eight lanes to a head, 16 bytes of
// each half to a lane. The first heads are loaded before the token's sequence
// is looked up, and every step's while the step before is rotated.
template <bool KV, bool NORM>
__device__ __forceinline__ void token_rows(const Append& a, int64_t work, int steps, int lane) {
  constexpr int Q = kQuads<NORM>;
  const exk_append& t = a.t;
  const int heads = t.Hq + (KV ? 2 * t.Hkv : 0);
  const int per_token = (heads + 4 * Q * steps - 1) / (4 * Q * steps);
  const int tok = static_cast<int>(work / per_token);
  if (tok >= t.N) return;
  int base = static_cast<int>(work % per_token) * (4 * Q * steps);
  const int sub = lane >> 3, c0 = 8 * (lane & 7);
  uint4 lo[Q], hi[Q];
  auto load = [&](int from) {
#pragma unroll
    for (int u = 0; u < Q; ++u) {
      const int h = from + 4 * u + sub;
      const uint16_t* src = nullptr;
      if (h < t.Hq)
        src = t.q + tok * t.q_st + h * t.q_sh;
      else if (KV && h < t.Hq + t.Hkv)
        src = t.k + tok * t.k_st + (h - t.Hq) * t.k_sh;
      else if (KV && h < heads)
        src = t.v + tok * t.v_st + (h - t.Hq - t.Hkv) * t.v_sh;
      lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
      if (src != nullptr) {
        lo[u] = *reinterpret_cast<const uint4*>(src + c0);
        hi[u] = *reinterpret_cast<const uint4*>(src + 64 + c0);
      }
    }
  };
  load(base);
  const int b = t.cu_seqlens == nullptr ? tok : find_seq(t.cu_seqlens, t.B, 1, 0, tok, lane);
  if (b >= t.B) return;  // behind the last sequence
  const Seq s = load_seq(t, b);
  if (tok < s.first || tok - s.first >= s.n) return;  // (rows before the first sequence)
  const int pos = s.start + tok - s.first;
  const bool ok = position_ok(t, pos);
  Turn<4> turn;
  int64_t row = -1;
  load_turn(t.cos_sin + static_cast<int64_t>(ok ? pos : 0) * kD, c0, turn);
  if (!ok) {
    set_status(a.status, EXK_S_POSITION);
  } else if (KV) {
    const int page = pool_page(a, b, pos / kP);
    if (page >= 0) row = static_cast<int64_t>(page) * kP + pos % kP;
  }
  for (; steps > 0 && base < heads; --steps, base += 4 * Q) {
    uint32_t l[Q][4], g[Q][4];
    float r[Q];
#pragma unroll
    for (int u = 0; u < Q; ++u) {
      l[u][0] = lo[u].x; l[u][1] = lo[u].y; l[u][2] = lo[u].z; l[u][3] = lo[u].w;
      g[u][0] = hi[u].x; g[u][1] = hi[u].y; g[u][2] = hi[u].z; g[u][3] = hi[u].w;
      r[u] = 0.f;
    }
    if (steps > 1) load(base + 4 * Q);
    if constexpr (NORM) {  // every quad's sums together: their shuffles do not wait on one another
#pragma unroll
      for (int u = 0; u < Q; ++u) r[u] = squares<4>(l[u], g[u]);
#pragma unroll
      for (int d = 4; d > 0; d >>= 1) {
#pragma unroll
        for (int u = 0; u < Q; ++u) r[u] += __shfl_xor_sync(0xFFFFFFFFu, r[u], d);
      }
#pragma unroll
      for (int u = 0; u < Q; ++u) r[u] = norm_factor(r[u], t.eps);
    }
#pragma unroll
    for (int u = 0; u < Q; ++u) {
      const int h = base + 4 * u + sub;
      uint16_t* dst = nullptr;
      if (h < t.Hq + (KV ? t.Hkv : 0)) {
        norm_rotate<4, NORM>(l[u], g[u], c0, h < t.Hq ? t.q_norm : t.k_norm, r[u], turn);
        if (h < t.Hq)
          dst = t.q_out + tok * t.o_st + h * t.o_sh;
        else if (row >= 0)
          dst = a.pool[0] + (row * t.Hkv + (h - t.Hq)) * kD;
        if (!ok) {  // (queries alone get here)
#pragma unroll
          for (int j = 0; j < 4; ++j) l[u][j] = g[u][j] = 0u;
        }
      } else if (KV && h < heads && row >= 0) {
        dst = a.pool[1] + (row * t.Hkv + (h - t.Hq - t.Hkv)) * kD;
      }
      if (dst == nullptr) continue;
      *reinterpret_cast<uint4*>(dst + c0) = make_uint4(l[u][0], l[u][1], l[u][2], l[u][3]);
      *reinterpret_cast<uint4*>(dst + 64 + c0) = make_uint4(g[u][0], g[u][1], g[u][2], g[u][3]);
    }
  }
}

template <bool NORM>
__global__ void __launch_bounds__(kRowWarps * 32) append_bf16_kernel(const __grid_constant__ Append a, int steps) {
  token_rows<true, NORM>(a, static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5), steps, threadIdx.x & 31);
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

// In an item's count byte: the call completed the page; the item's warp in the
// second kernel also writes the sequence's open page.
constexpr int kItemFull = 0x20, kItemOpens = 0x40, kItemRows = 0x1F;

// rowoff of a page whose raw rows do not all have a slot below the capacity: no
// row's index (rowoff + rank) is one, so readers report the page. The slots behind
// the capacity are other sequences' open pages.
constexpr int kNoRoom = -kP;

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
  // (before the first page: offsets that do not ascend, whose slots are not the sequence's)
  if (it.pg < it.s.start / kP || it.pg > last_page(it.s) || !tail_of(a, b, it.slot)) return it;
  it.full = (it.pg + 1) * kP <= it.s.start + it.s.n;
  // (where the first page's entry is bad nothing of that page is read or written, and
  // the open one need not wait for it)
  it.later = !it.full && it.pg * kP > it.s.start && it.s.start % kP != 0 && pool_page(a, b, it.s.start / kP) >= 0;
  it.pool = pool_page(a, b, it.pg);
  return it;
}

// `it` completes its sequence's first page, whose earlier rows are in the tail,
// and the sequence's last page stays open: that one is written after `it`.
__device__ __forceinline__ bool opens_later(const Item& it) {
  const int last = last_page(it.s);
  return it.pg == it.s.start / kP && it.s.start % kP != 0 && last > it.pg && (last + 1) * kP > it.s.start + it.s.n;
}

// The lane's channels (4q.. and 64 + 4q..) of packed token tok, KV head h: keys
// (which = 0) or values.
__device__ __forceinline__ void load_quads(const Append& a, int which, int tok, int h, int q, uint32_t (&w)[4]) {
  const exk_append& t = a.t;
  const uint16_t* src = which == 0 ? t.k + tok * t.k_st + h * t.k_sh : t.v + tok * t.v_st + h * t.v_sh;
  const uint2 lo = *reinterpret_cast<const uint2*>(src + 4 * q);
  const uint2 hi = *reinterpret_cast<const uint2*>(src + 64 + 4 * q);
  w[0] = lo.x; w[1] = lo.y; w[2] = hi.x; w[3] = hi.y;
}

// They as the cache holds them: keys normalised and rotated at pos (whole warp).
template <bool NORM>
__device__ __forceinline__ void cache_form(const Append& a, int which, int pos, int q, uint32_t (&w)[4]) {
  if (which != 0) return;
  uint32_t l[2] = {w[0], w[1]}, g[2] = {w[2], w[3]};
  Turn<2> turn;
  load_turn(a.t.cos_sin + static_cast<int64_t>(pos) * kD, 4 * q, turn);
  float r = 0.f;
  if constexpr (NORM) {
    r = squares<2>(l, g);
#pragma unroll
    for (int d : {1, 8, 4, 2}) r += __shfl_xor_sync(0xFFFFFFFFu, r, d);
    r = norm_factor(r, a.t.eps);
  }
  norm_rotate<2, NORM>(l, g, 4 * q, a.t.k_norm, r, turn);
  w[0] = l[0]; w[1] = l[1]; w[2] = g[0]; w[3] = g[1];
}

__device__ __forceinline__ uint16_t* tail_row(const Append& a, int which, int slot, int h, int r) {
  return a.raw[which] + (a.cap[which] + (static_cast<int64_t>(slot) * a.t.Hkv + h) * kP + r) * kD;
}

__device__ __forceinline__ void load_tail(const Append& a, int which, int slot, int h, int r, int q, uint32_t (&w)[4]) {
  const uint16_t* s = tail_row(a, which, slot, h, r);
  const uint2 lo = *reinterpret_cast<const uint2*>(s + 4 * q), hi = *reinterpret_cast<const uint2*>(s + 64 + 4 * q);
  w[0] = lo.x; w[1] = lo.y; w[2] = hi.x; w[3] = hi.y;
}

__device__ __forceinline__ void store_quads(uint16_t* d, int q, const uint32_t (&w)[4]) {
  *reinterpret_cast<uint2*>(d + 4 * q) = make_uint2(w[0], w[1]);
  *reinterpret_cast<uint2*>(d + 64 + 4 * q) = make_uint2(w[2], w[3]);
}

// The new rows of an open page into the sequence's tail rows, and the page's
// entry: all rows raw, at the tail rows.
template <bool NORM>
__device__ __forceinline__ void write_open(const Append& a, const Item& it, int which, int lane) {
  const int q = lane & 15, th = lane >> 4;
  const int first = it.s.start - it.pg * kP, end = it.s.start + it.s.n - it.pg * kP;  // new rows of the page
  uint32_t w[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 8 * th + i;
    w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0u;
    if (r >= first && r < end) load_quads(a, which, it.s.first + r - first, it.h, q, w[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 8 * th + i;
    const bool mine = r >= first && r < end;
    if (!__any_sync(0xFFFFFFFFu, mine)) continue;
    cache_form<NORM>(a, which, it.pg * kP + min(r, end - 1), q, w[i]);
    if (mine) store_quads(tail_row(a, which, it.slot, it.h, r), q, w[i]);
  }
  if (lane == 0) {
    const int64_t page = static_cast<int64_t>(it.pool) * a.t.Hkv + it.h;
    a.rowmask[which][page] = 0xFFFF;
    a.rowoff[which][page] = static_cast<int32_t>(a.cap[which] + (static_cast<int64_t>(it.slot) * a.t.Hkv + it.h) * kP);
  }
}

template <bool NORM>
__global__ void __launch_bounds__(kRowWarps * 32) append_encode_kernel(const __grid_constant__ Append a) {
  allow_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
    for (int i = 0; i < 8; ++i) {  // (rows of the page that this call does not bring come from the tail, as they are)
      const int pos = it.pg * kP + 8 * th + i;
      if (pos >= it.s.start)
        load_quads(a, which, it.s.first + pos - it.s.start, it.h, q, w[i]);
      else
        load_tail(a, which, it.slot, it.h, 8 * th + i, q, w[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pos = it.pg * kP + 8 * th + i;
      uint32_t f[4] = {w[i][0], w[i][1], w[i][2], w[i][3]};
      cache_form<NORM>(a, which, pos, q, f);
      if (pos >= it.s.start) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i][j] = f[j];
      }
    }
    const int64_t page = static_cast<int64_t>(it.pool) * a.t.Hkv + it.h;
    const int64_t row = static_cast<int64_t>(it.pool) * kP * a.t.Hkv + it.h;
    rm = encode_rows(w, lane, a.sm[which] + row * kD, static_cast<int64_t>(a.t.Hkv) * kD, a.code[which] + row * (kD / 2),
                     static_cast<int64_t>(a.t.Hkv) * (kD / 2), a.base[which] + page * kD);
    if (lane == 0) a.rowmask[which][page] = static_cast<int32_t>(rm);
  } else if (it.pool >= 0 && !it.later) {
    write_open<NORM>(a, it, which, lane);
  }
  if (lane == 0) {
    const bool full = it.pool >= 0 && it.full;
    a.counts[static_cast<int64_t>(which) * a.items_pad + item] =
        static_cast<uint8_t>(__popc(rm) + (full ? kItemFull + (opens_later(it) ? kItemOpens : 0) : 0));
    if (which == 0 && full) a.pages[item] = make_int2(it.pool * a.t.Hkv + it.h, it.s.b);
  }
}

constexpr int kPlaceItems = 64;     // items of one CTA of append_place_kernel
constexpr int kPlaceThreads = 256;  // eight warps, eight items each

// Blocks below 2 * chunks place a chunk of items, keys and values in turn: the CTA
// adds up the counts of all items before its own (bytes: 65,536 items are 16 loads
// of 16 bytes per thread), scans its own, writes the offsets and copies the
// escaped rows. That is a chain of look-ups with little to move, so the other
// blocks rotate the queries beside it, and start without waiting for the first
// kernel (9,529 tokens: 36 us; rotated in the first kernel 44 us).
template <bool NORM>
__global__ void __launch_bounds__(kPlaceThreads) append_place_kernel(const __grid_constant__ Append a, int chunks, int steps) {
  __shared__ int s_before[kPlaceThreads / 32];
  __shared__ int s_count[kPlaceItems], s_off[kPlaceItems];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (static_cast<int>(blockIdx.x) >= 2 * chunks) {
    token_rows<false, NORM>(a, static_cast<int64_t>(blockIdx.x - 2 * chunks) * (kPlaceThreads / 32) + warp, steps, lane);
    return;
  }
  after_prior();
  const int which = blockIdx.x & 1, chunk = blockIdx.x >> 1;
  const uint8_t* counts = a.counts + static_cast<int64_t>(which) * a.items_pad;
  const int i0 = chunk * kPlaceItems, mine = i0 + threadIdx.x;
  const int count = threadIdx.x < kPlaceItems && mine < a.items ? counts[mine] : 0;
  const int2 page = threadIdx.x < kPlaceItems && (count & kItemFull) ? a.pages[mine] : make_int2(0, 0);
  int before = 0;
  for (int i = threadIdx.x; i < i0 / 16; i += kPlaceThreads) {
    const uint4 v = reinterpret_cast<const uint4*>(counts)[i];
    before = __dp4a(v.x & 0x1F1F1F1Fu, 0x01010101u, static_cast<uint32_t>(before));
    before = __dp4a(v.y & 0x1F1F1F1Fu, 0x01010101u, static_cast<uint32_t>(before));
    before = __dp4a(v.z & 0x1F1F1F1Fu, 0x01010101u, static_cast<uint32_t>(before));
    before = __dp4a(v.w & 0x1F1F1F1Fu, 0x01010101u, static_cast<uint32_t>(before));
  }
  before = __reduce_add_sync(0xFFFFFFFFu, before);
  if (lane == 0) s_before[warp] = before;
  if (threadIdx.x < kPlaceItems) s_count[threadIdx.x] = count;
  __syncthreads();
  if (threadIdx.x < kPlaceItems) {
    int off = a.base_cnt[which], total = 0;
    for (int w = 0; w < kPlaceThreads / 32; ++w) off += s_before[w];
    for (int i = 0; i < kPlaceItems; ++i) {
      const int n = s_count[i] & kItemRows;
      off += i < threadIdx.x ? n : 0;
      total += i >= threadIdx.x ? n : 0;
    }
    s_off[threadIdx.x] = off;
    if (count & kItemFull) {
      const int n = count & kItemRows;
      a.rowoff[which][page.x] = n > 0 && static_cast<int64_t>(off) + n > a.cap[which] ? kNoRoom : off;
    }
    // (may exceed the capacity: the caller grows the pool before it calls)
    if (chunk == chunks - 1 && threadIdx.x == 0) *a.cnt[which] = off + total;
  }
  __syncthreads();
  const int q = lane & 15, th = lane >> 4;
  // the warp's eight items, every eighth of the CTA's (a sequence's heads, which
  // have their open pages to write at once, go to different warps): those with
  // escaped rows or an open page
  constexpr int warps = kPlaceThreads / 32;
  const int flags = lane < kPlaceItems / warps ? s_count[warps * lane + warp] : 0;
  for (uint32_t todo = __ballot_sync(0xFFFFFFFFu, (flags & (kItemRows | kItemOpens)) != 0); todo != 0u; todo &= todo - 1u) {
    const int i = warps * (__ffs(todo) - 1) + warp, item = i0 + i;
    const int2 at = a.pages[item];
    Item it;
    it.s = load_seq(a.t, at.y);
    it.h = item % a.t.Hkv;
    it.pg = it.s.start / kP + (a.t.cu_seqlens == nullptr ? 0 : item / a.t.Hkv - (it.s.first / kP + 2 * at.y));
    it.slot = a.t.slots == nullptr ? at.y : __ldg(a.t.slots + at.y);
    uint32_t rm = static_cast<uint32_t>(a.rowmask[which][at.x]) & 0xFFFFu;
    int64_t ridx = s_off[i];
    for (; rm != 0u; rm &= rm - 1u, ++ridx) {
      if (ridx < 0 || ridx >= a.cap[which]) continue;
      const int r = __ffs(rm) - 1, pos = it.pg * kP + r;
      uint32_t w[4];
      if (pos < it.s.start) {
        load_tail(a, which, it.slot, it.h, r, q, w);
      } else {
        load_quads(a, which, it.s.first + pos - it.s.start, it.h, q, w);
        cache_form<NORM>(a, which, pos, q, w);
      }
      if (th == 0) store_quads(a.raw[which] + ridx * kD, q, w);
    }
    if (s_count[i] & kItemOpens) {
      it.pg = last_page(it.s);
      it.pool = pool_page(a, at.y, it.pg);
      __syncwarp();  // every lane has read the tail rows
      if (it.pool >= 0) write_open<NORM>(a, it, which, lane);
    }
  }
}

// ---------------------------------------------------------------- sequences cut back
//
// A sequence whose length was taken back (drafts that were not accepted) may end
// inside a page that was completed: its rows are coded, and the tail rows, where the
// next append looks for the page's earlier rows, hold a later page's. A warp per
// (sequence, KV head) of the keys and of the values: the page's remaining rows,
// decoded (all loaded before the first is), go to the tail rows, and the page is
// open again. Pages that are open, and ends of whole pages, are left alone: the look
// is all that most calls cost (64 sequences of 8 heads: 2.2 us; all reopened 4.0).

__global__ void __launch_bounds__(kRowWarps * 32) reopen_kernel(const __grid_constant__ Append a) {
  const exk_append& t = a.t;
  const int lane = threadIdx.x & 31, q = lane & 15, th = lane >> 4;
  const int work = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (work >= 2 * a.items) return;
  const int which = work >= a.items ? 1 : 0, item = work - which * a.items;
  const int b = item / t.Hkv, h = item % t.Hkv, len = __ldg(t.seq_lens + b), held = len % kP;
  if (len <= 0 || held == 0) return;
  if (len > t.max_pages * kP) {
    set_status(a.status, EXK_S_POSITION);
    return;
  }
  int slot;
  if (!tail_of(a, b, slot)) return;
  const int pool = pool_page(a, b, len / kP);
  if (pool < 0) return;
  const int64_t page = static_cast<int64_t>(pool) * t.Hkv + h;
  const int64_t tail = a.cap[which] + (static_cast<int64_t>(slot) * t.Hkv + h) * kP;
  const uint32_t rm = static_cast<uint32_t>(a.rowmask[which][page]) & 0xFFFFu;
  const int32_t ro = a.rowoff[which][page];
  if (rm == 0xFFFFu && ro == tail) return;
  const int n = min(held - 8 * th, 8);
  const uint32_t bl = *reinterpret_cast<const uint32_t*>(a.base[which] + page * kD + 4 * q);
  const uint32_t bh = *reinterpret_cast<const uint32_t*>(a.base[which] + page * kD + 64 + 4 * q);
  uint32_t w[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 8 * th + i;
    const int64_t row = (static_cast<int64_t>(pool) * kP + r) * t.Hkv + h;
    const int64_t ridx = static_cast<int64_t>(ro) + __popc(rm & ((1u << r) - 1u));
    w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0u;
    if (i >= n) continue;
    if (((rm >> r) & 1u) == 0u) {
      w[i][0] = *reinterpret_cast<const uint32_t*>(a.sm[which] + row * kD + 4 * q);
      w[i][1] = *reinterpret_cast<const uint32_t*>(a.sm[which] + row * kD + 64 + 4 * q);
      w[i][2] = *reinterpret_cast<const uint32_t*>(a.code[which] + row * (kD / 2) + 4 * q);
    } else if (ridx >= 0 && ridx < a.raw_rows[which]) {
      const uint16_t* src = a.raw[which] + ridx * kD;
      const uint2 lo = *reinterpret_cast<const uint2*>(src + 4 * q), hi = *reinterpret_cast<const uint2*>(src + 64 + 4 * q);
      w[i][0] = lo.x; w[i][1] = lo.y; w[i][2] = hi.x; w[i][3] = hi.y;
    } else {
      set_status(a.status, EXK_S_RAW_INDEX);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= n) break;
    if (((rm >> (8 * th + i)) & 1u) == 0u) {
      const uint32_t sl = w[i][0], sh = w[i][1], cw = w[i][2];
      dec4(sl, lo_nibbles(cw), bl & 0x7F7F7F7Fu, bl, w[i][0], w[i][1]);
      dec4(sh, hi_nibbles(cw), bh & 0x7F7F7F7Fu, bh, w[i][2], w[i][3]);
    }
    store_quads(tail_row(a, which, slot, h, 8 * th + i), q, w[i]);
  }
  if (lane == 0) {
    a.rowmask[which][page] = 0xFFFF;
    a.rowoff[which][page] = static_cast<int32_t>(tail);
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
      t->max_pages <= 0 || t->max_pages > (1 << 26) || t->pool_pages <= 0 ||
      static_cast<int64_t>(t->pool_pages) * t->Hkv >= (int64_t{1} << 31))
    return EXK_EARG;
  if (t->cu_seqlens == nullptr && t->N != t->B) return EXK_EARG;
  if (t->N > (1 << 28) || t->B > (1 << 24) || t->Hq > 4096) return EXK_EARG;
  if (!aligned16(t->q) || !aligned16(t->k) || !aligned16(t->v) || !aligned16(t->q_out) || !aligned16(t->cos_sin))
    return EXK_EALIGN;
  for (const uint16_t* w : {t->q_norm, t->k_norm})  // read 8 bytes at a time
    if ((reinterpret_cast<uintptr_t>(w) & 7u) != 0) return EXK_EALIGN;
  for (int64_t s : {t->q_st, t->q_sh, t->k_st, t->k_sh, t->v_st, t->v_sh, t->o_st, t->o_sh})
    if (s % 8 != 0) return EXK_EALIGN;
  return 0;
}

// Steps of a warp of token_rows: one while the warps do not fill the GPU about
// twice (short calls, where latency counts), else a whole token, so that the
// look-up is paid once (11,016 tokens of 48 heads, two groups in flight: 50 us; one step
// a warp: 68 us).
int row_steps(const exk_append& t, int heads, int sms) {
  const int quads = t.q_norm != nullptr ? kQuads<true> : kQuads<false>;
  const int steps = (heads + 4 * quads - 1) / (4 * quads);
  return static_cast<int64_t>(t.N) * steps > int64_t{48} * sms ? steps : 1;
}

int64_t row_blocks(const exk_append& t, int heads, int steps, int warps) {
  const int quads = t.q_norm != nullptr ? kQuads<true> : kQuads<false>;
  const int64_t work = static_cast<int64_t>(t.N) * ((heads + 4 * quads * steps - 1) / (4 * quads * steps));
  return (work + warps - 1) / warps;
}

// The pools of a call whose a.t is set, checked.
int coded_pools(Append& a, const exk_cview* k, int64_t k_cap, const exk_cview* v, int64_t v_cap) {
  if (k->sm == v->sm || k->raw == v->raw) return EXK_EARG;  // keys and values have pools of their own
  const exk_cview* c[2] = {k, v};
  const int64_t cap[2] = {k_cap, v_cap};
  int64_t tails = int64_t{1} << 24;
  for (int i = 0; i < 2; ++i) {
    if (c[i]->sm == nullptr || c[i]->code == nullptr || c[i]->base == nullptr || c[i]->rowmask == nullptr ||
        c[i]->rowoff == nullptr || c[i]->raw == nullptr || cap[i] < 0 || c[i]->raw_rows < cap[i] ||
        c[i]->raw_rows >= (int64_t{1} << 31))
      return EXK_EARG;
    if (!aligned16(c[i]->sm) || !aligned16(c[i]->code) || !aligned16(c[i]->base) || !aligned16(c[i]->raw))
      return EXK_EALIGN;
    tails = std::min(tails, (c[i]->raw_rows - cap[i]) / (static_cast<int64_t>(a.t.Hkv) * kP));
    a.sm[i] = const_cast<uint8_t*>(c[i]->sm);
    a.code[i] = const_cast<uint8_t*>(c[i]->code);
    a.base[i] = const_cast<uint8_t*>(c[i]->base);
    a.rowmask[i] = const_cast<int32_t*>(c[i]->rowmask);
    a.rowoff[i] = const_cast<int32_t*>(c[i]->rowoff);
    a.raw[i] = const_cast<uint16_t*>(c[i]->raw);
    a.cap[i] = cap[i];
    a.raw_rows[i] = c[i]->raw_rows;
  }
  if (tails < (a.t.slots == nullptr ? a.t.B : 1)) return EXK_EARG;  // an open page for every sequence
  a.tails = static_cast<int32_t>(tails);
  return 0;
}

int64_t page_slots(const exk_append& t) {
  return t.cu_seqlens == nullptr ? t.B : t.N / kP + 2 * static_cast<int64_t>(t.B);
}

}  // namespace

static_assert(sizeof(exk_append) == 184, "the Python binding packs these bytes");

extern "C" int exk_rope_append_bf16(const exk_append* t, uint16_t* k_pool, uint16_t* v_pool, int32_t* status, int device,
                                    void* stream) {
  int r = check_append(t);
  if (r != 0) return r;
  if (k_pool == nullptr || v_pool == nullptr || k_pool == v_pool) return EXK_EARG;
  if (!aligned16(k_pool) || !aligned16(v_pool)) return EXK_EALIGN;
  if (t->N == 0) return 0;
  DeviceScope scope;
  int sms = 0;
  if ((r = use_device(device, &sms)) != 0) return r;
  const int heads = t->Hq + 2 * t->Hkv, steps = row_steps(*t, heads, sms);
  const int64_t blocks = row_blocks(*t, heads, steps, kRowWarps);
  if (blocks >= (int64_t{1} << 31)) return EXK_EARG;
  Append a = {};
  a.t = *t;
  a.pool[0] = k_pool;
  a.pool[1] = v_pool;
  a.status = status;
  const auto kernel = t->q_norm != nullptr ? append_bf16_kernel<true> : append_bf16_kernel<false>;
  kernel<<<static_cast<unsigned>(blocks), kRowWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(a, steps);
  return launch_status();
}

extern "C" int64_t exk_rope_append_scratch(int N, int B, int Hkv, int packed) {
  if (N < 0 || B <= 0 || Hkv <= 0) return EXK_EARG;
  const int64_t items = (packed ? N / kP + 2 * static_cast<int64_t>(B) : B) * Hkv;
  return 16 + 2 * ((items + 15) / 16 * 16) + 8 * items;
}

extern "C" int exk_rope_append_compressed(const exk_append* t, const exk_cview* k, int64_t k_cap, int32_t* k_cnt,
                                          const exk_cview* v, int64_t v_cap, int32_t* v_cnt, void* scratch,
                                          int64_t scratch_bytes, int32_t* status, int device, void* stream) {
  int r = check_append(t);
  if (r != 0) return r;
  if (k == nullptr || v == nullptr || k_cnt == nullptr || v_cnt == nullptr || scratch == nullptr) return EXK_EARG;
  if (k_cnt == v_cnt) return EXK_EARG;
  const int64_t items = page_slots(*t) * t->Hkv;
  if (items > (int64_t{1} << 29)) return EXK_EARG;
  Append a = {};
  a.t = *t;
  if ((r = coded_pools(a, k, k_cap, v, v_cap)) != 0) return r;
  a.cnt[0] = k_cnt;
  a.cnt[1] = v_cnt;
  if (!aligned16(scratch)) return EXK_EALIGN;
  if (scratch_bytes < exk_rope_append_scratch(t->N, t->B, t->Hkv, t->cu_seqlens != nullptr)) return EXK_EARG;
  if (t->N == 0) return 0;
  DeviceScope scope;
  int sms = 0;
  if ((r = use_device(device, &sms)) != 0) return r;
  a.slots = static_cast<int32_t>(page_slots(*t));
  a.items = static_cast<int32_t>(items);
  a.items_pad = static_cast<int32_t>((items + 15) / 16 * 16);
  a.base_cnt = static_cast<int32_t*>(scratch);
  a.counts = static_cast<uint8_t*>(scratch) + 16;
  a.pages = reinterpret_cast<int2*>(a.counts + 2 * static_cast<int64_t>(a.items_pad));
  a.status = status;
  const int64_t enc = (2 * items + kRowWarps - 1) / kRowWarps;
  const int64_t chunks = (items + kPlaceItems - 1) / kPlaceItems;
  const int steps = row_steps(*t, t->Hq, sms);
  const int64_t blocks = 2 * chunks + row_blocks(*t, t->Hq, steps, kPlaceThreads / 32);
  if (blocks >= (int64_t{1} << 31)) return EXK_EARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool norm = t->q_norm != nullptr;
  const auto encode = norm ? append_encode_kernel<true> : append_encode_kernel<false>;
  encode<<<static_cast<unsigned>(enc), kRowWarps * 32, 0, st>>>(a);
  if ((r = launch_status()) != 0) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kPlaceThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, norm ? append_place_kernel<true> : append_place_kernel<false>, a,
                                           static_cast<int>(chunks), steps);
  if (e == cudaSuccess) return 0;
  (void)cudaGetLastError();
  return static_cast<int>(e);
}

extern "C" int exk_reopen_pages(const int32_t* block_table, int B, int max_pages, int pool_pages, int Hkv,
                                const int32_t* seq_lens, const int32_t* slots, const exk_cview* k, int64_t k_cap,
                                const exk_cview* v, int64_t v_cap, int32_t* status, int device, void* stream) {
  if (block_table == nullptr || seq_lens == nullptr || k == nullptr || v == nullptr || B <= 0 || B > (1 << 24) ||
      max_pages <= 0 || max_pages > (1 << 26) || pool_pages <= 0 || Hkv <= 0 || Hkv > 4096 ||
      static_cast<int64_t>(pool_pages) * Hkv >= (int64_t{1} << 31) || static_cast<int64_t>(B) * Hkv > (int64_t{1} << 29))
    return EXK_EARG;
  Append a = {};
  a.t.block_table = block_table;
  a.t.seq_lens = seq_lens;
  a.t.slots = slots;
  a.t.B = B;
  a.t.Hkv = Hkv;
  a.t.max_pages = max_pages;
  a.t.pool_pages = pool_pages;
  int r = coded_pools(a, k, k_cap, v, v_cap);
  if (r != 0) return r;
  a.items = B * Hkv;
  a.status = status;
  DeviceScope scope;
  if ((r = use_device(device, nullptr)) != 0) return r;
  const unsigned blocks = static_cast<unsigned>((2 * static_cast<int64_t>(a.items) + kRowWarps - 1) / kRowWarps);
  reopen_kernel<<<blocks, kRowWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return launch_status();
}
