// Causal attention of many query tokens per sequence (sm_100a): packed prompts
// over their own keys, or a prompt's chunk over the pages of a paged cache.
//
// Query i of a sequence of n queries and L keys sees keys j <= i + L - n:
//   o_i = sum_j softmax_j(q_i k_j / sqrt(128)) v_j ,  0 where it sees none.
//
// An item of work is 256 rows of one KV head's group: a row is a (token, query
// head of the group) pair, so the G = Hq / Hkv heads that share keys share the
// item's key tiles, and 256 / G consecutive tokens keep the diagonal narrow. The
// item streams tiles of 128 keys from the diagonal down: S = Q K^T (tcgen05,
// K-major operands in shared memory, S in TMEM), one thread per row for the running
// maximum, P = 2^(s - m) in bf16 back into TMEM over S, O += P V (P from TMEM, V
// MN-major as the TMA left it). Two 128-row tiles alternate, so the tensor
// core works on one while the other's softmax runs: two S and two O tiles are all
// of TMEM's 512 columns. 148 persistent CTAs, one to an SM (232 KB of shared
// memory), take items as they come; while one item's rows are written out the
// next one's first tiles run.
//
// A key tile costs 2,048 cycles of products and 2,048 of exponentials (16 a cycle)
// for its 256 rows; a tile's chain (S out of TMEM 60 cycles, maximum 400,
// exponentials 1,350, then P V's rest, the next S and the hand-overs 1,150) sets
// a period of about 3,000, 66 % of the tensor pipe, at the 1.6 GHz that the power
// limit leaves. One prompt of 16,384 tokens, 32 heads over 8: 1,676 us after a pause
// (1,312 TFLOP/s), 1,952 us in a loop under the power limit; 4,096: 133 and 145 us; 16
// prompts of 73 to 1,988 tokens, 28 over 4: 192 and 217 us.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "exk_device.cuh"
#include "exk_encode.cuh"
#include "exk_host.h"

namespace exk {

namespace {

constexpr int kTile = 128;                 // rows of a query tile, keys of a key tile
constexpr int kHalf = kTile * 128;         // bytes of one operand half: 128 rows x 64 channels bf16
constexpr int kOperand = 2 * kHalf;        // one operand tile
constexpr int kSlots = 4;                  // key/value ring: K, V, K, V, ...
// Warps 0-3, 4-7: softmax of the two query tiles; 8-11: output; 12: MMA; 13: TMA;
// 14: values of masked tiles; 15: schedule. The register split adds up to
// the launch's 512 threads x 128.
constexpr int kPrefillThreads = 512;
constexpr int kMmaWarp = 12, kTmaWarp = 13, kValueWarp = 14;
constexpr int kReaders = 15;               // warps that read the schedule
constexpr int kRegsSoftmax = 176, kRegsOutput = 96, kRegsOther = 64;
constexpr float kRescale = 8.f;            // a row's maximum may grow by 2^8 before O is rescaled

struct PrefillArgs {
  const int32_t* cu_q;
  const int32_t* cu_k;         // packed keys, or null
  const int32_t* lens;         // keys of each sequence where cu_k is null
  const int32_t* block_table;  // pages of the keys, or null: sequence b's rows start at b * k_stride
  int k_stride;
  const uint16_t* v;           // the values again, for non-finite ones under a mask
  int64_t v_st, v_sh;
  uint16_t* out;
  int64_t o_st, o_sh;
  float* po;                   // partials [N * Hq, ns, 128], [N * Hq, ns] (ns > 1)
  float* pm;
  float* pl;
  int32_t* status;
  int N, Nk, B, Hq, Hkv, G, tpt;  // tpt: tokens of a query tile
  int max_pages, pool_pages, ns, slots;
  uint64_t by_block;           // divides by the tokens of a block (divide())
  float scale;                 // log2(e) / sqrt(128)
};

struct PrefillMaps {
  CUtensorMap q, k, v;
};

// ---------------------------------------------------------------- tcgen05

__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One lane of a converged warp, the same each time. The tensor core's operands
// are uniform registers: issued under a plain lane test, each product took
// about 120 cycles of moves (1,050 for eight against 512 that they run).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}

// Arrives on `bar` when every tcgen05 operation this thread issued before has completed.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}

// D[tmem] (+)= A[smem] B[smem]; both bf16, fp32 accumulation.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem].
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// 32 columns of the calling warp's 32 lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
      "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Shared-memory operand descriptors, 128-byte swizzle, tiles as TMA leaves
// them: 128-byte rows (64 channels), eight rows to a 1024-byte swizzle block.
// K-major (Q, K: the contraction runs along the row): groups of eight rows
// 1024 bytes apart; 16 channels are 32 bytes further. MN-major (V: the
// contraction runs down the rows): the second half of the channels kHalf
// bytes on, the next eight keys 1024; 16 keys are 2048 bytes further.
constexpr uint64_t kDescBase = (uint64_t{1} << 46) | (uint64_t{2} << 61);
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t addr) {
  return kDescBase | (uint64_t{1024 >> 4} << 32) | (uint64_t{1} << 16) | ((addr & 0x3FFFF) >> 4);
}
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t addr) {
  return kDescBase | (uint64_t{1024 >> 4} << 32) | (uint64_t{kHalf >> 4} << 16) | ((addr & 0x3FFFF) >> 4);
}
// fp32 D, bf16 A and B, M = N = 128; bit 16: B is MN-major.
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((kTile / 8) << 17) | ((kTile / 16) << 24);
constexpr uint32_t kIdescMN = kIdesc | (1u << 16);

// ---------------------------------------------------------------- one item of work

// Asks for a block of the grid that has not started: this CTA then does its
// work in its place. The answer (16 bytes) arrives on `bar`.
__device__ __forceinline__ void steal_block(void* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_addr(answer)),
               "r"(smem_addr(bar))
               : "memory");
}
// The block taken, or (-1, 0): none was left.
__device__ __forceinline__ int2 stolen_block(const void* answer) {
  int2 at;
  asm volatile(
      "{\n .reg .b128 h;\n .reg .pred p;\n ld.shared.b128 h, [%2];\n mov.b32 %0, -1;\n mov.b32 %1, 0;\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::y.b32.b128 %1, h;\n}"
      : "=r"(at.x), "=r"(at.y)
      : "r"(smem_addr(answer))
      : "memory");
  return at;
}

struct Work {
  int valid;        // 0: no more work
  int b, hk, split;
  int first, n;     // the sequence's first packed query, its queries
  int L, krow;      // its keys, its first key row (not paged)
  int tok0, tiles;  // first token of the rows; query tiles in use: 1 or 2
  int keys;         // keys that the last row sees
  int nt, t1;       // key tiles of this split: t1 - 1 down to t1 - nt
  int low;          // keys that every row sees
  int masked;       // the first of the tiles, in which some row does not see some key
};

// x / T for 0 <= x < 2^28, T <= 256, with m = 2^36 / T + 1.
__device__ __forceinline__ int divide(int x, uint64_t m) { return static_cast<int>((static_cast<uint64_t>(x) * m) >> 36); }

// The batch as the scheduling warp holds it when it has at most 32 sequences: lane b
// sequence b's queries and keys, its 256-row blocks, and the blocks of the
// sequences with more keys (they come first: the calls' last blocks are then short
// ones). With more sequences nothing of this is used.
struct Batch {
  int first, n, L, krow, blocks, before;
};

// Sequence b's queries and keys; n = 0 where its bounds are not a batch's.
__device__ __forceinline__ void load_seq(const PrefillArgs& a, int b, Batch& s) {
  s.first = __ldg(a.cu_q + b);
  s.n = __ldg(a.cu_q + b + 1) - s.first;
  if (s.first < 0 || s.n < 0 || s.first > a.N - s.n) s.n = 0;
  if (a.cu_k != nullptr) {
    s.krow = __ldg(a.cu_k + b);
    s.L = __ldg(a.cu_k + b + 1) - s.krow;
    if (s.krow < 0 || s.L < 0 || s.krow > a.Nk - s.L) s.L = s.krow = 0;
  } else {
    s.krow = b * a.k_stride;
    const int most = a.block_table != nullptr ? a.max_pages * kP : a.k_stride, L = __ldg(a.lens + b);
    if (L > most && s.n > 0) set_status(a.status, EXK_S_POSITION);  // keys past the table or the workspace are not seen
    s.L = max(0, min(L, most));
  }
}

__device__ __forceinline__ Batch load_batch(const PrefillArgs& a, int lane) {
  Batch s = {0, 0, -1, 0, 0, 0};
  if (a.B > 32) return s;
  if (lane < a.B) load_seq(a, lane, s);
  s.blocks = divide(s.n + 2 * a.tpt - 1, a.by_block);
#pragma unroll 1
  for (int b = 0; b < a.B; ++b) {
    const int L = __shfl_sync(0xFFFFFFFFu, s.L, b), blocks = __shfl_sync(0xFFFFFFFFu, s.blocks, b);
    if (L > s.L || (L == s.L && b < lane)) s.before += blocks;
  }
  return s;
}

// Offsets of a batch: 0 <= cu[0] <= .. <= cu[B] <= most. By a whole warp, one answer.
__device__ __forceinline__ bool ascending(const int32_t* cu, int B, int most, int lane) {
  bool ok = __ldg(cu) >= 0 && __ldg(cu + B) <= most;
  for (int b = lane; b < B; b += 32) ok = ok && __ldg(cu + b) <= __ldg(cu + b + 1);
  return __all_sync(0xFFFFFFFFu, ok);
}

// Block (x, y) of the grid: (KV head, split) and 256-row block of T = 2 tpt tokens,
// a sequence's blocks with long rows of keys first. With more than 32 sequences,
// b's blocks take slots cu[b] / T + b, + 1, ...: n tokens need at most (n + T - 1) /
// T, which never reaches sequence b + 1's first slot, so the map needs no
// prefix sum. False for a block left over. By a whole warp.
__device__ __forceinline__ bool load_work(const PrefillArgs& a, const Batch& batch, int2 block, int lane, Work& w) {
  if (block.x < 0) return false;
  const int T = 2 * a.tpt;
  w.split = 0;
  w.hk = block.x;
  if (a.ns > 1) {
    w.hk = block.x / a.ns;
    w.split = block.x - w.hk * a.ns;
  }
  if (a.B <= 32) {
    const uint32_t mine = __ballot_sync(0xFFFFFFFFu, block.y >= batch.before && block.y < batch.before + batch.blocks);
    if (mine == 0u) return false;
    w.b = __ffs(mine) - 1;
    w.first = __shfl_sync(0xFFFFFFFFu, batch.first, w.b);
    w.n = __shfl_sync(0xFFFFFFFFu, batch.n, w.b);
    w.L = __shfl_sync(0xFFFFFFFFu, batch.L, w.b);
    w.krow = __shfl_sync(0xFFFFFFFFu, batch.krow, w.b);
    w.tok0 = (__shfl_sync(0xFFFFFFFFu, batch.before + batch.blocks, w.b) - 1 - block.y) * T;
  } else {
    const int slot = a.slots - 1 - block.y;
    w.b = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const bool before = b0 + lane < a.B && divide(__ldg(a.cu_q + b0 + lane + 1), a.by_block) + b0 + lane + 1 <= slot;
      w.b += __popc(__ballot_sync(0xFFFFFFFFu, before));
    }
    if (w.b >= a.B) return false;
    Batch s;
    load_seq(a, w.b, s);
    w.first = s.first;
    w.n = s.n;
    w.L = s.L;
    w.krow = s.krow;
    w.tok0 = (slot - (divide(w.first, a.by_block) + w.b)) * T;
    if (w.tok0 < 0 || w.tok0 >= w.n) return false;
  }
  w.valid = 1;
  w.tiles = w.n - w.tok0 > a.tpt ? 2 : 1;
  w.keys = max(0, w.L - w.n + min(w.tok0 + T, w.n));
  const int all = (w.keys + kTile - 1) / kTile;
  const int per = a.ns > 1 ? (all + a.ns - 1) / a.ns : all;
  const int t0 = min(all, w.split * per);
  w.t1 = min(all, t0 + per);
  w.nt = w.t1 - t0;
  // tile j holds a key past the first row's last one when (j + 1) * 128 > low
  w.low = max(0, w.L - w.n + w.tok0 + 1);
  w.masked = min(w.nt, max(0, w.t1 - w.low / kTile));
  return true;
}

// Waits that end: after about two seconds, or at once when another role gave up.
// The cycle counter rather than %globaltimer keeps the loop small: this
// kernel's roles share the instruction cache, and at the change of an item all
// of them run code that the main loop does not.
constexpr uint32_t kWaitCycles = 3500000000u;  // 1.8 s at 1.965 GHz
__device__ __forceinline__ uint32_t cycles() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%clock;" : "=r"(t));
  return t;
}
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* stop) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t t0 = cycles();
  while (!mbar_try_wait(bar, parity)) {
    if (cycles() - t0 > kWaitCycles) *stop = 1;
    if (*stop != 0) return false;
  }
  return true;
}

// bar_wait by a whole warp, with one answer for all lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* stop) {
  return __all_sync(0xFFFFFFFFu, bar_wait(bar, parity, stop));
}

// Bits 15 and 31: the half's exponent field is all ones.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
}

// f += the values of v [32] that are not finite.
__device__ __forceinline__ void add_not_finite(float (&f)[32], const uint4* v) {
  uint32_t any = 0u;
#pragma unroll 1
  for (int i = 0; i < 4; ++i) any |= not_finite(v[i].x) | not_finite(v[i].y) | not_finite(v[i].z) | not_finite(v[i].w);
  if (any == 0u) return;
  const uint16_t* h = reinterpret_cast<const uint16_t*>(v);
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if ((h[i] & 0x7F80) == 0x7F80) f[i] += __uint_as_float(static_cast<uint32_t>(h[i]) << 16);
}

struct __align__(16) Bars {
  uint4 answer;
  uint64_t q_full[2], q_empty[2], kv_full[kSlots], kv_empty[kSlots], v_ok[kSlots], s_full[2], p_most[2], p_full[2], o_full[2], o_empty[2];
  uint64_t l_full[2], l_empty[2];
  uint64_t work_full[2], work_empty[2], block, want;
  Work work[2];
  float l[2][kTile];  // the rows' sums at the end of an item
  uint32_t tmem;
  int stop, bad;
};

constexpr int kStage = 4 * 2 * 32 * 128;
constexpr int kPrefillSmem = 2 * kOperand + kSlots * kOperand + kStage + static_cast<int>(sizeof(Bars)) + 1024;
static_assert(kPrefillSmem <= 227 * 1024, "one CTA's shared memory");

// The softmax threads' side of one item: query tile x, a row per thread; rt: the
// row's token in the tile. s_phase, o_phase: tiles of S taken and items ended so
// far.
__device__ __forceinline__ void softmax_item(const PrefillArgs& a, const Work& w, Bars* bars, uint32_t tmem, int x, int rt,
                                             uint32_t& s_phase, uint32_t& o_phase, volatile int* stop) {
  const int warp = threadIdx.x >> 5, r = threadIdx.x & 127;
  const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
  const uint32_t ts = tmem + lanes + x * kTile, to = tmem + lanes + 2 * kTile + x * kTile;
  const int tok = w.tok0 + x * a.tpt + rt;
  const bool valid = r < a.G * a.tpt && tok < w.n;
  const int lim = valid ? w.L - w.n + tok : w.keys - 1;  // last key the row sees
  const int nt = w.nt;
  float m = -INFINITY, l = 0.f;
  for (int it = 0; it < nt; ++it) {
    if (!warp_wait(&bars->s_full[x], s_phase & 1, stop)) break;
    ++s_phase;
    tc_fence_after();
    uint32_t s[kTile];
#pragma unroll
    for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, s + 32 * c);
    tc_wait_ld();
    if (it < w.masked) {
      // columns past the last key that the row sees; groups of 32 that every row
      // of the warp sees are left alone
      const int seen = lim - (w.t1 - 1 - it) * kTile;
      const int least = __reduce_min_sync(0xFFFFFFFFu, seen);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (least >= 32 * c + 31) continue;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (32 * c + i > seen) s[32 * c + i] = 0xFF800000u;
      }
    }
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < kTile; i += 2)
      mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
    const float top = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * a.scale;
    // The maximum follows by steps of 2^kRescale at least: P stays below
    // 2^kRescale, and O is rarely rescaled. Every lane decides by its own row
    // alone, so a row's bits do not depend on its neighbours.
    const bool grown = valid && top > m + kRescale;
    if (it == 0) {
      m = top;
    } else if (__any_sync(0xFFFFFFFFu, grown)) {
      // S is complete, so the tensor core has finished O += P V of the tile before
      const float f = grown ? ex2(m - top) : 1.f;
      l *= f;
      m = grown ? top : m;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        tmem_ld32(to + 32 * c, o);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tmem_st32(to + 32 * c, o);
      }
    }
    const float off = m == -INFINITY ? 0.f : -m;
    const F2 scale2 = f2(a.scale, a.scale), off2 = f2(off, off);
    F2 sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int e = 32 * c + 2 * i;
        float p0, p1;
        split2(fma2(f2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale2, off2), p0, p1);
        p0 = ex2(p0);
        p1 = ex2(p1);
        sum[i & 1] = add2(sum[i & 1], f2(p0, p1));
        p[i] = pack_bf16x2(p0, p1);
      }
      tmem_st16(ts + 16 * c, p);
      if (c == 2) {  // three quarters: the product may start
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(&bars->p_most[x]);
      }
    }
    float l0, l1;
    split2(add2(sum[0], sum[1]), l0, l1);
    l += l0 + l1;
    tc_wait_st();
    tc_fence_before();
    mbar_arrive(&bars->p_full[x]);
  }
  if (nt > 0 && warp_wait(&bars->l_empty[x], (o_phase & 1) ^ 1, stop)) {
    bars->l[x][r] = l;
    mbar_arrive(&bars->l_full[x]);
    if (a.ns > 1 && valid) {
      const int64_t at = (static_cast<int64_t>(w.first + tok) * a.Hq + w.hk * a.G + r - rt * a.G) * a.ns + w.split;
      a.pm[at] = m;
      a.pl[at] = l;
    }
  }
  if (nt > 0) ++o_phase;
}

// The output warps' side of query tile x: row r = TMEM lane, thread r of the four warps.
__device__ __forceinline__ void output_item(const PrefillArgs& a, const Work& w, Bars* bars, uint4* stage, uint32_t tmem, int x, int rt,
                                            uint32_t& o_phase, volatile int* stop) {
  const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, r = threadIdx.x & 127;
  const uint32_t to = tmem + (static_cast<uint32_t>(warp) << 21) + 2 * kTile + x * kTile;
  const int g = r - rt * a.G, tok = w.tok0 + x * a.tpt + rt;
  const bool valid = r < a.G * a.tpt && tok < w.n;
  const int lim = w.L - w.n + tok;
  const int h = w.hk * a.G + g;
  const int64_t row = static_cast<int64_t>(w.first + tok) * a.Hq + h;
  bool have = false;
  float l = 0.f;
  if (w.nt > 0) {
    have = warp_wait(&bars->l_full[x], (o_phase >> x) & 1, stop);
    if (have) {
      l = bars->l[x][r];
      mbar_arrive(&bars->l_empty[x]);
    }
    have = have && warp_wait(&bars->o_full[x], (o_phase >> x) & 1, stop);
    o_phase ^= 1u << x;
    tc_fence_after();
  }
  if (a.ns > 1 && valid && w.nt == 0) {
    a.pm[row * a.ns + w.split] = -INFINITY;
    a.pl[row * a.ns + w.split] = 0.f;
  }
  // (a NaN sum makes the row NaN; a row without keys becomes 0)
  const float inv = a.ns > 1 ? 1.f : (l == 0.f ? 0.f : 1.f / l);
  const bool bad = *const_cast<volatile int*>(&bars->bad) != 0;
  // The row's place; null: not written (no row, or a split without keys).
  uint64_t dst = 0;
  if (valid && a.ns == 1)
    dst = reinterpret_cast<uint64_t>(a.out + static_cast<int64_t>(w.first + tok) * a.o_st + h * a.o_sh);
  if (valid && a.ns > 1 && have) dst = reinterpret_cast<uint64_t>(a.po + (row * a.ns + w.split) * kD);
  // 128 bytes of every row at a time go through shared memory, 16-byte pieces
  // swizzled by row, so that eight lanes write a whole line: stored by the rows'
  // own threads, 16 bytes a row, the tile took 6,000 cycles.
  uint4* mine = stage + warp * 512;
  auto flush = [&](int part) {
#pragma unroll 4
    for (int i = 0; i < 8; ++i) {
      const int from = 4 * i + (lane >> 3);
      const uint64_t d = __shfl_sync(0xFFFFFFFFu, dst, from);
      const uint4 v = mine[(part & 1) * 256 + from * 8 + ((lane & 7) ^ (from & 7))];
      if (d != 0) reinterpret_cast<uint4*>(d + 128 * part)[lane & 7] = v;
    }
  };
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t o[32];
    if (have) {
      tmem_ld32(to + 32 * c, o);
      tc_wait_ld();
    }
    float f[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = l == 0.f ? 0.f : __uint_as_float(o[i]) * inv;
    if (bad && valid) {
      // a masked tile held values that are not finite: they were left out of
      // the product and reach the rows that see them here, whatever their weight (it is
      // above 0 in the formula; where it underflows, a product gives NaN instead of
      // infinity: not finite either way)
#pragma unroll 1
      for (int t = max(w.low, (w.t1 - w.nt) * kTile); t < min(w.t1 * kTile, lim + 1); ++t) {
        int64_t vrow = static_cast<int64_t>(w.krow) + t;
        if (a.block_table != nullptr) {
          const int pg = __ldg(a.block_table + static_cast<int64_t>(w.b) * a.max_pages + t / kP);
          if (pg < 0 || pg >= a.pool_pages) continue;
          vrow = static_cast<int64_t>(pg) * kP + t % kP;
        }
        add_not_finite(f, reinterpret_cast<const uint4*>(a.v + vrow * a.v_st + w.hk * a.v_sh + 32 * c));
      }
    }
    if (a.ns > 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        mine[(c & 1) * 256 + lane * 8 + (i ^ (lane & 7))] =
            make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                       __float_as_uint(f[4 * i + 3]));
      __syncwarp();
      flush(c);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mine[(c >> 1) * 256 + lane * 8 + ((4 * (c & 1) + i) ^ (lane & 7))] =
            make_uint4(pack_bf16x2(f[8 * i], f[8 * i + 1]), pack_bf16x2(f[8 * i + 2], f[8 * i + 3]),
                       pack_bf16x2(f[8 * i + 4], f[8 * i + 5]), pack_bf16x2(f[8 * i + 6], f[8 * i + 7]));
    }
  }
  if (have) {  // the next item may write O
    tc_fence_before();
    mbar_arrive(&bars->o_empty[x]);
  }
  if (a.ns == 1) {
    __syncwarp();
#pragma unroll 1
    for (int part = 0; part < 2; ++part) flush(part);
  }
  __syncwarp();
}

// One CTA per SM, which takes blocks of the grid as they come (longest first):
// while one item's rows are written out, the next one's operands are loaded and
// its first S is computed.
__global__ void __launch_bounds__(kPrefillThreads, 1)
    prefill_kernel(const __grid_constant__ PrefillArgs a, const __grid_constant__ PrefillMaps maps) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* sq = smem;
  uint8_t* ring = smem + 2 * kOperand;
  uint4* stage = reinterpret_cast<uint4*>(ring + kSlots * kOperand);  // 2 x 32 rows of 128 bytes for each output warp
  Bars* bars = reinterpret_cast<Bars*>(ring + kSlots * kOperand + kStage);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int* stop = &bars->stop;

  allow_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->q_full[i], 1);
      mbar_init(&bars->q_empty[i], 1);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_most[i], kTile);
      mbar_init(&bars->p_full[i], kTile);
      mbar_init(&bars->o_full[i], 1);
      mbar_init(&bars->work_full[i], 1);
      mbar_init(&bars->work_empty[i], kReaders);
      mbar_init(&bars->o_empty[i], kTile);
      mbar_init(&bars->l_full[i], kTile);
      mbar_init(&bars->l_empty[i], kTile);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&bars->kv_full[i], 1);
      mbar_init(&bars->kv_empty[i], 1 + (i & 1));  // V entries (odd): the products and the value warp
      mbar_init(&bars->v_ok[i], 32);
    }
    mbar_init(&bars->block, 1);
    mbar_init(&bars->want, 1);
    bars->stop = bars->bad = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) tmem_alloc(&bars->tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  // Work number `k` of this CTA, as the scheduling warp left it: false at the end.
  uint32_t k = 0;
  auto next_work = [&](Work& w) {
    const int i = k & 1;
    const bool ok = warp_wait(&bars->work_full[i], (k >> 1) & 1, stop);
    w = bars->work[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->work_empty[i]);
    ++k;
    return ok && w.valid != 0;
  };

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int x = warp >> 2, rt = (threadIdx.x & 127) / a.G;
    uint32_t s_phase = 0, o_phase = 0;
    Work w;
    while (next_work(w))
      if (x < w.tiles) softmax_item(a, w, bars, tmem, x, rt, s_phase, o_phase, stop);
  } else if (warp < kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOutput));
    const int rt = (threadIdx.x & 127) / a.G;
    uint32_t o_phase = 0;
    // (a warp that waits for the first rows anyway)
    if (warp == 8 && blockIdx.x == 0 && blockIdx.y == 0 &&
        !(ascending(a.cu_q, a.B, a.N, lane) && (a.cu_k == nullptr || ascending(a.cu_k, a.B, a.Nk, lane))))
      set_status(a.status, EXK_S_POSITION);
    Work w;
    while (next_work(w))
      for (int x = 0; x < w.tiles; ++x) output_item(a, w, bars, stage, tmem, x, rt, o_phase, stop);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == kMmaWarp) {
      // ---- MMA: K of an item's tile `it` is ring entry e + 2 it, V the one after
      const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
      const uint64_t dq = desc_kmajor(smem_addr(sq)), dk = desc_kmajor(smem_addr(ring)), dv = desc_mnmajor(smem_addr(ring));
      uint32_t e = 0, q_phase = 0, p_phase = 0, o_phase = 3, ok_phase = 0;  // bit x (or slot): the parity to wait for next
      // S of query tile x from the K in `slot`; `last`: the item's last use of Q
      auto qk = [&](int x, uint32_t slot, bool last) {
        if (elect_one()) {
          const uint64_t a0 = dq + x * (kOperand >> 4), b0 = dk + slot * (kOperand >> 4);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint64_t off = ((c >> 2) * kHalf + (c & 3) * 32) >> 4;
            mma_ss(tm + x * kTile, a0 + off, b0 + off, kIdesc, c > 0);
          }
          tc_commit(&bars->s_full[x]);
          if (last) tc_commit(&bars->q_empty[x]);
        }
        __syncwarp();
      };
      Work w;
      while (next_work(w)) {
        const int nt = __shfl_sync(0xFFFFFFFFu, w.nt, 0), tiles = __shfl_sync(0xFFFFFFFFu, w.tiles, 0);
        const int masked = __shfl_sync(0xFFFFFFFFu, w.masked, 0);
        if (nt == 0) continue;
        bool ok = warp_wait(&bars->kv_full[e % kSlots], (e / kSlots) & 1, stop);
        for (int x = 0; x < tiles && ok; ++x) {
          ok = warp_wait(&bars->q_full[x], (q_phase >> x) & 1, stop);
          q_phase ^= 1u << x;
          tc_fence_after();
          if (ok) qk(x, e % kSlots, nt == 1);
        }
        if (ok && elect_one()) tc_commit(&bars->kv_empty[e % kSlots]);
        for (int it = 0; it < nt && ok; ++it) {
          const uint32_t ve = e + 2 * it + 1, ke = ve + 1, vs = ve % kSlots, ks = ke % kSlots;
          if (it < masked) {
            ok = warp_wait(&bars->v_ok[vs], (ok_phase >> vs) & 1, stop);
            ok_phase ^= 1u << vs;
          } else {
            ok = warp_wait(&bars->kv_full[vs], (ve / kSlots) & 1, stop);
          }
          for (int x = 0; x < tiles && ok; ++x) {
            // P comes in two parts, 96 keys and 32: the first part's product runs
            // beside the last exponentials
            const uint64_t b0 = dv + vs * (kOperand >> 4);
            const uint32_t d = tm + 2 * kTile + x * kTile, p0 = tm + x * kTile;
            if (it == 0) {  // the item before has been read out of O
              ok = warp_wait(&bars->o_empty[x], (o_phase >> x) & 1, stop);
              o_phase ^= 1u << x;
            }
            ok = ok && warp_wait(&bars->p_most[x], (p_phase >> x) & 1, stop);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int c = 0; c < 6; ++c) mma_ts(d, p0 + 8 * c, b0 + c * (2048 >> 4), kIdescMN, it > 0 || c > 0);
            }
            __syncwarp();
            ok = warp_wait(&bars->p_full[x], (p_phase >> x) & 1, stop);
            p_phase ^= 1u << x;
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int c = 6; c < 8; ++c) mma_ts(d, p0 + 8 * c, b0 + c * (2048 >> 4), kIdescMN, 1);
              if (x == tiles - 1) tc_commit(&bars->kv_empty[vs]);
              if (it == nt - 1) tc_commit(&bars->o_full[x]);
            }
            __syncwarp();
            if (it < nt - 1) {
              if (x == 0) ok = warp_wait(&bars->kv_full[ks], (ke / kSlots) & 1, stop);
              if (ok) qk(x, ks, it == nt - 2);
            }
          }
          if (ok && it < nt - 1 && elect_one()) tc_commit(&bars->kv_empty[ks]);
        }
        e += 2 * nt;
        if (!ok) break;
      }
    } else if (warp == kTmaWarp) {
      // ---- TMA: an item's first K, its queries, its V, K, V, ...
      const uint32_t tile_bytes = 2 * 64 * 2 * a.G * a.tpt;
      uint32_t e = 0, q_phase = 3;
      if (elect_one()) {
        prefetch_tmap(&maps.q);
        prefetch_tmap(&maps.k);
        prefetch_tmap(&maps.v);
      }
      after_prior();  // unpack_kernel's rows; the other warps read none of them before they land here
      Work w;
      while (next_work(w)) {
        bool ok = true;
        for (int i = 0; i < 2 * w.nt && ok; ++i, ++e) {
          const uint32_t slot = e % kSlots;
          const int j = w.t1 - 1 - i / 2;
          ok = warp_wait(&bars->kv_empty[slot], ((e / kSlots) & 1) ^ 1, stop);
          if (!ok) break;
          const CUtensorMap* map = (i & 1) == 0 ? &maps.k : &maps.v;
          uint8_t* dst = ring + slot * kOperand;
          uint64_t* full = &bars->kv_full[slot];
          if (a.block_table == nullptr) {
            if (elect_one()) {
              mbar_arrive_expect_tx(full, kOperand);
              tma_load_4d(dst, map, 0, w.hk, w.krow + j * kTile, 0, full);
            }
          } else {
            // a lane looks each page up; pages past the keys are not loaded (their
            // columns are masked). One lane issues the copies: issued by sixteen
            // lanes side by side they are taken one by one all the same, and
            // slower.
            const int pages = min(kTile / kP, (w.keys - j * kTile + kP - 1) / kP);
            int row = 0;
            if (lane < pages) {
              const int page = __ldg(a.block_table + static_cast<int64_t>(w.b) * a.max_pages + j * (kTile / kP) + lane);
              if (page >= 0 && page < a.pool_pages) {
                row = page * kP;
              } else {
                set_status(a.status, EXK_S_PAGE_INDEX);
                row = a.pool_pages * kP;  // outside the map: zeros
              }
            }
            const int hk = __shfl_sync(0xFFFFFFFFu, w.hk, 0), n = __shfl_sync(0xFFFFFFFFu, pages, 0);
            if (elect_one()) mbar_arrive_expect_tx(full, n * (2 * 64 * 2 * kP));
            __syncwarp();
#pragma unroll
            for (int pg = 0; pg < kTile / kP; ++pg) {
              const int at = __shfl_sync(0xFFFFFFFFu, row, pg);
              if (pg < n && elect_one()) {
                tma_load_4d(dst + pg * (kP * 128), map, 0, hk, at, 0, full);
                tma_load_4d(dst + kHalf + pg * (kP * 128), map, 0, hk, at, 1, full);
              }
            }
          }
          __syncwarp();
          for (int x = 0; i == 0 && x < w.tiles && ok; ++x) {
            ok = warp_wait(&bars->q_empty[x], (q_phase >> x) & 1, stop);
            q_phase ^= 1u << x;
            if (ok && elect_one()) {
              mbar_arrive_expect_tx(&bars->q_full[x], tile_bytes);
              // (rows that do not fill the tile leave a gap between its halves)
              for (int c = 0; c < (a.G * a.tpt == kTile ? 1 : 2); ++c)
                tma_load_4d(sq + x * kOperand + c * kHalf, &maps.q, 0, w.hk * a.G, w.first + w.tok0 + x * a.tpt, c,
                            &bars->q_full[x]);
            }
            __syncwarp();
          }
        }
        if (!ok) break;
        if (lane == 0) mbar_arrive(&bars->want);
      }
    } else if (warp == kValueWarp) {
      // ---- values of masked tiles: rows past the last key become zeros, and so do
      // values that are not finite and that some row does not see (0 x inf is NaN). Only
      // such rows are looked at, up to 64 of 128 with four heads to a group: a look
      // at every piece by itself held the products up for 8,000 cycles an item.
      uint32_t e = 0;
      Work w;
      while (next_work(w)) {
        bool ok = true;
        for (int it = 0; it < w.nt && ok; ++it) {
          // (every tile, and the ring waits for this warp: a wait on a phase of a
          // barrier that may be two phases ahead or behind would not be one)
          const uint32_t ve = e + 2 * it + 1, vs = ve % kSlots;
          ok = warp_wait(&bars->kv_full[vs], (ve / kSlots) & 1, stop);
          if (!ok) break;
          if (it >= w.masked) {
            if (lane == 0) mbar_arrive(&bars->kv_empty[vs]);
            continue;
          }
          // the tile's rows [open, end): keys that some of the item's rows see and some do not
          const int base = (w.t1 - 1 - it) * kTile;
          const int open = max(0, w.low - base), end = min(kTile, w.keys - base);
          uint4* v = reinterpret_cast<uint4*>(ring + vs * kOperand);
          const int n = 8 * max(0, end - open);  // pieces of one half
          auto piece = [&](int i) { return i < n ? 8 * open + i : kHalf / 16 + 8 * open + i - n; };
          bool bad = false;
          // six pieces in flight at once; what is found is cleared in a second look.
          // (w + w drops the sign and leaves the exponent on top of each half.)
          for (int i0 = lane; i0 < 2 * n; i0 += 6 * 32) {
            uint4 u[6];
#pragma unroll
            for (int c = 0; c < 6; ++c) u[c] = i0 + 32 * c < 2 * n ? v[piece(i0 + 32 * c)] : make_uint4(0, 0, 0, 0);
            uint32_t m0 = 0u, m1 = 0u;
#pragma unroll
            for (int c = 0; c < 6; ++c) {
              m0 = max_u16x2(max_u16x2(m0, u[c].x + u[c].x), u[c].y + u[c].y);
              m1 = max_u16x2(max_u16x2(m1, u[c].z + u[c].z), u[c].w + u[c].w);
            }
            m0 = max_u16x2(m0, m1);
            if ((m0 & 0xFFFFu) < 0xFF00u && (m0 >> 16) < 0xFF00u) continue;
            bad = true;
#pragma unroll 1
            for (int i = i0; i < min(2 * n, i0 + 6 * 32); i += 32) {
              uint4 x = v[piece(i)];
              x.x &= ~((not_finite(x.x) >> 15) * 0xFFFFu);
              x.y &= ~((not_finite(x.y) >> 15) * 0xFFFFu);
              x.z &= ~((not_finite(x.z) >> 15) * 0xFFFFu);
              x.w &= ~((not_finite(x.w) >> 15) * 0xFFFFu);
              v[piece(i)] = x;
            }
          }
          for (int i = 8 * end + lane; i < 8 * kTile; i += 32) v[i] = v[kHalf / 16 + i] = make_uint4(0, 0, 0, 0);
          // (kept for the CTA's later items: they then look for such values too)
          if (bad) *const_cast<volatile int*>(&bars->bad) = 1;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          mbar_arrive(&bars->v_ok[vs]);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->kv_empty[vs]);
        }
        e += 2 * w.nt;
        if (!ok) break;
      }
    } else {
      // ---- schedule: this CTA's own block, then blocks that have not started. The
      // next is asked for when the last copies of an item are under way, about two
      // key tiles before it ends: asked for sooner, a CTA with a long item would hold
      // back another that an idle one could start (4096 tokens: 174 us for 150).
      const Batch batch = load_batch(a, lane);
      int2 item = make_int2(blockIdx.x, blockIdx.y);
      uint32_t asked = 0, wanted = 0;
      Work w;
      while (true) {
        const bool some = load_work(a, batch, item, lane, w);
        if (!some) w.valid = 0;
        if (some || item.x < 0) {
          if (!warp_wait(&bars->work_empty[k & 1], ((k >> 1) & 1) ^ 1, stop)) break;
          if (lane == 0) {
            bars->work[k & 1] = w;
            mbar_arrive(&bars->work_full[k & 1]);
          }
          ++k;
          if (item.x < 0) break;
          if (!warp_wait(&bars->want, wanted++ & 1, stop)) break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->block, 16);
          steal_block(&bars->answer, &bars->block);
        }
        if (!warp_wait(&bars->block, asked++ & 1, stop)) break;
        item = stolen_block(&bars->answer);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
    }
  }
  __syncthreads();
  if (*stop != 0) {
    // a wait ran out: what is in flight (copies of at most 192 KB, products of a
    // tile) ends long before this pause does, and nothing more is issued
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 2000000) {
    }
    if (threadIdx.x == 0) set_status(a.status, EXK_S_FULL_TIMEOUT);
    __syncthreads();
  }
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

// Partials of ns splits of each row: out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M),
// 0 for a row without keys; rows of no sequence are left alone. One warp per
// row; a lane holds the weights of splits lane and lane + 32, and eight splits'
// o are loaded before they are added, in split order.
constexpr int kMaxSplits = 64;

__global__ void __launch_bounds__(256) prefill_merge_kernel(const __grid_constant__ PrefillArgs a) {
  after_prior();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= static_cast<int64_t>(a.N) * a.Hq) return;
  const int tok = static_cast<int>(row / a.Hq);
  // (offsets that are no batch's may name rows whose partials nothing wrote)
  if (tok < __ldg(a.cu_q) || tok >= __ldg(a.cu_q + a.B) || !ascending(a.cu_q, a.B, a.N, lane)) return;
  float m[2], l[2], f[2];
  float M = -INFINITY, den = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool in = lane + 32 * i < a.ns;
    m[i] = in ? a.pm[row * a.ns + lane + 32 * i] : -INFINITY;
    l[i] = in ? a.pl[row * a.ns + lane + 32 * i] : 0.f;
    M = fmaxf(M, m[i]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, d));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[i] = m[i] == -INFINITY ? (l[i] == 0.f ? 0.f : 1.f) : ex2(m[i] - M);  // (no key of the row: its o was not written)
    den += f[i] * l[i];
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) den += __shfl_xor_sync(0xFFFFFFFFu, den, d);
  // Splits that saw a key of the row. (A weight of 0 does not leave one out: its o may be
  // infinite or NaN, and 0 times that is NaN, as it is without splits.)
  uint32_t saw[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) saw[i] = __ballot_sync(0xFFFFFFFFu, m[i] != -INFINITY || l[i] != 0.f);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* o = reinterpret_cast<const float4*>(a.po + row * a.ns * kD) + lane;
  for (int s0 = 0; s0 < a.ns; s0 += 8) {
    float4 v[8];
    float g[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      g[u] = __shfl_sync(0xFFFFFFFFu, s0 < 32 ? f[0] : f[1], (s0 + u) & 31);
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (((s0 < 32 ? saw[0] : saw[1]) >> ((s0 + u) & 31)) & 1u) v[u] = o[(s0 + u) * (kD / 4)];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      acc.x += g[u] * v[u].x;
      acc.y += g[u] * v[u].y;
      acc.z += g[u] * v[u].z;
      acc.w += g[u] * v[u].w;
    }
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;
  uint16_t* d = a.out + tok * a.o_st + (row % a.Hq) * a.o_sh;
  reinterpret_cast<uint2*>(d)[lane] =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

// Coded pages of the sequences into bf16 rows b * k_stride + position: the
// pages' keys (blockIdx.y 0) and values (1), a warp per (page, KV head). Nothing
// of a sequence that has no queries in the call.
struct Unpack {
  exk_cview c[2];
  uint16_t* out[2];
  const int32_t* cu_q;
  const int32_t* block_table;
  const int32_t* lens;
  int32_t* status;
  int64_t k_stride;
  int B, Hkv, max_pages, pool_pages, pages;  // pages: k_stride / 16
};

// The attention is launched as its programmatic dependent: set up where SMs run
// out of pages, it loads keys once all are written (131 MB of 16 sequences: 97 us
// to 93 us for both).
// Eight lanes to a row, 8 bytes of sm's halves and of code to a lane; all rows
// of the page are loaded before the first is decoded.
__global__ void __launch_bounds__(256) unpack_kernel(const __grid_constant__ Unpack u) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t ph = static_cast<int64_t>(blockIdx.x) * 8 + warp;
  const int h = static_cast<int>(ph % u.Hkv);
  const int pg = static_cast<int>((ph / u.Hkv) % u.pages);
  const int64_t b = ph / (static_cast<int64_t>(u.Hkv) * u.pages);
  allow_dependents();
  if (b >= u.B) return;
  const int L = min(__ldg(u.lens + b), static_cast<int>(u.k_stride)) - pg * kP;  // rows of the page that are wanted
  if (L <= 0 || __ldg(u.cu_q + b + 1) <= __ldg(u.cu_q + b)) return;
  const int pool = __ldg(u.block_table + b * u.max_pages + pg);
  const exk_cview& v = u.c[blockIdx.y];
  const int c = lane & 7, r4 = lane >> 3;
  uint16_t* out = u.out[blockIdx.y] + ((b * u.k_stride + static_cast<int64_t>(pg) * kP + r4) * u.Hkv + h) * kD + 8 * c;
  const int64_t step = static_cast<int64_t>(4) * u.Hkv * kD;
  if (pool < 0 || pool >= u.pool_pages) {
    set_status(u.status, EXK_S_PAGE_INDEX);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (4 * s + r4 < L) {
        uint4* o = reinterpret_cast<uint4*>(out + s * step);
        o[0] = o[8] = make_uint4(0, 0, 0, 0);
      }
    return;
  }
  const int64_t page = static_cast<int64_t>(pool) * u.Hkv + h;
  const int64_t token = (static_cast<int64_t>(pool) * kP + r4) * u.Hkv + h;
  const uint32_t rm = static_cast<uint32_t>(__ldg(v.rowmask + page)) & 0xFFFFu;
  const int32_t ro = __ldg(v.rowoff + page);
  const uint2 bl = __ldg(reinterpret_cast<const uint2*>(v.base + page * kD + 8 * c));
  const uint2 bh = __ldg(reinterpret_cast<const uint2*>(v.base + page * kD + 64 + 8 * c));
  uint2 sl[4], sh[4], cw[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int64_t at = token + static_cast<int64_t>(4) * s * u.Hkv;
    sl[s] = __ldg(reinterpret_cast<const uint2*>(v.sm + at * kD + 8 * c));
    sh[s] = __ldg(reinterpret_cast<const uint2*>(v.sm + at * kD + 64 + 8 * c));
    cw[s] = __ldg(reinterpret_cast<const uint2*>(v.code + at * (kD / 2) + 8 * c));
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int row = 4 * s + r4;
    if (row >= L) break;
    uint4 lo, hi;
    if ((rm >> row) & 1u) {
      const int64_t ridx = static_cast<int64_t>(ro) + __popc(rm & ((1u << row) - 1u));
      lo = hi = make_uint4(0, 0, 0, 0);
      if (ridx >= 0 && ridx < v.raw_rows) {
        const uint4* p = reinterpret_cast<const uint4*>(v.raw + ridx * kD + 8 * c);
        lo = __ldg(p);
        hi = __ldg(p + 8);
      } else {
        set_status(u.status, EXK_S_RAW_INDEX);
      }
    } else {
      dec4(sl[s].x, lo_nibbles(cw[s].x), bl.x & 0x7F7F7F7Fu, bl.x, lo.x, lo.y);
      dec4(sl[s].y, lo_nibbles(cw[s].y), bl.y & 0x7F7F7F7Fu, bl.y, lo.z, lo.w);
      dec4(sh[s].x, hi_nibbles(cw[s].x), bh.x & 0x7F7F7F7Fu, bh.x, hi.x, hi.y);
      dec4(sh[s].y, hi_nibbles(cw[s].y), bh.y & 0x7F7F7F7Fu, bh.y, hi.z, hi.w);
    }
    uint4* o = reinterpret_cast<uint4*>(out + s * step);
    o[0] = lo;
    o[8] = hi;
  }
}

// ---------------------------------------------------------------- host

int64_t prefill_slots(int N, int B, int G) { return N / (2 * (kTile / G)) + static_cast<int64_t>(B); }

int check_prefill(const exk_prefill* p) {
  if (p == nullptr || p->q == nullptr || p->out == nullptr || p->cu_q == nullptr) return EXK_EARG;
  if (p->N < 0 || p->B <= 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv != 0 || p->ns < 1 || p->ns > kMaxSplits ||
      p->N > (1 << 28) || p->B > (1 << 24) || p->Hq > 4096)
    return EXK_EARG;
  if (p->Hq / p->Hkv > 16) return EXK_EHEADS;
  if (prefill_slots(p->N, p->B, p->Hq / p->Hkv) > 65535) return EXK_EARG;  // the grid's second dimension
  if (p->ns > 1 && (p->po == nullptr || p->pm == nullptr || p->pl == nullptr)) return EXK_EARG;
  if (!aligned16(p->q) || !aligned16(p->out) || !aligned16(p->po)) return EXK_EALIGN;
  for (int64_t s : {p->q_st, p->q_sh, p->o_st, p->o_sh})
    if (s % 8 != 0) return EXK_EALIGN;
  if (p->q_st <= 0 || p->q_sh <= 0) return EXK_EARG;
  return 0;
}

// Rows [rows, heads, 128] with element strides as (64 channels, heads, rows, halves):
// a box of `tokens` rows of `heads_box` heads lands as one or two halves of
// [tokens][heads_box] 128-byte rows.
int make_rows_map(CUtensorMap* map, const uint16_t* p, int64_t rows, int heads, int64_t st, int64_t sh, int heads_box,
                  int tokens, int halves) {
  const uint64_t dims[4] = {kD / 2, static_cast<uint64_t>(heads), static_cast<uint64_t>(rows), 2};
  const uint64_t strides[3] = {static_cast<uint64_t>(sh) * 2, static_cast<uint64_t>(st) * 2, kD};
  const uint32_t box[4] = {kD / 2, static_cast<uint32_t>(heads_box), static_cast<uint32_t>(tokens),
                           static_cast<uint32_t>(halves)};
  return make_tmap(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Lets the kernel have its shared memory, once per device (the current one).
int allow_smem(int device) {
  static std::atomic<uint64_t> done{0};
  if (done.load(std::memory_order_acquire) >> device & 1) return 0;
  const cudaError_t e = cudaFuncSetAttribute(prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPrefillSmem);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return static_cast<int>(e);
  }
  done.fetch_or(uint64_t{1} << device, std::memory_order_release);
  return 0;
}

int launch_prefill(const exk_prefill* p, PrefillArgs& a, const uint16_t* k, int64_t k_st, int64_t k_sh, const uint16_t* v,
                   int64_t v_st, int64_t v_sh, int64_t key_rows, int key_box, int32_t* status, int device, cudaStream_t st,
                   bool unpacked) {
  if (!aligned16(k) || !aligned16(v)) return EXK_EALIGN;
  for (int64_t s : {k_st, k_sh, v_st, v_sh}) {
    if (s % 8 != 0) return EXK_EALIGN;
    if (s <= 0) return EXK_EARG;
  }
  a.cu_q = p->cu_q;
  a.v = v;
  a.v_st = v_st;
  a.v_sh = v_sh;
  a.out = p->out;
  a.o_st = p->o_st;
  a.o_sh = p->o_sh;
  a.po = p->po;
  a.pm = p->pm;
  a.pl = p->pl;
  a.status = status;
  a.N = p->N;
  a.B = p->B;
  a.Hq = p->Hq;
  a.Hkv = p->Hkv;
  a.G = p->Hq / p->Hkv;
  a.tpt = kTile / a.G;
  a.ns = p->ns;
  a.scale = p->qk_scale;
  const int64_t slots = prefill_slots(p->N, p->B, a.G);
  const dim3 grid(static_cast<unsigned>(p->Hkv * p->ns), static_cast<unsigned>(slots));
  a.by_block = (uint64_t{1} << 36) / static_cast<uint64_t>(2 * a.tpt) + 1;
  a.slots = static_cast<int>(slots);
  PrefillMaps maps;
  const int halves = key_box == kTile ? 2 : 1;  // a page's halves lie apart in the tile
  int r;
  if ((r = make_rows_map(&maps.q, p->q, p->N, p->Hq, p->q_st, p->q_sh, a.G, a.tpt, a.G * a.tpt == kTile ? 2 : 1)) != 0) return r;
  if ((r = make_rows_map(&maps.k, k, key_rows, p->Hkv, k_st, k_sh, 1, key_box, halves)) != 0) return r;
  if ((r = make_rows_map(&maps.v, v, key_rows, p->Hkv, v_st, v_sh, 1, key_box, halves)) != 0) return r;
  if ((r = allow_smem(device)) != 0) return r;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kPrefillThreads);
  cfg.dynamicSmemBytes = kPrefillSmem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = unpacked ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, prefill_kernel, a, maps);
  if (e == cudaSuccess && p->ns > 1) {
    const int64_t rows = static_cast<int64_t>(p->N) * p->Hq;
    cfg.gridDim = dim3(static_cast<unsigned>((rows + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, prefill_merge_kernel, a);
  }
  if (e == cudaSuccess) return 0;
  (void)cudaGetLastError();
  return static_cast<int>(e);
}

}  // namespace

}  // namespace exk

using namespace exk;

static_assert(sizeof(exk_prefill) == 104, "the Python binding packs these bytes");

extern "C" int exk_prefill_splits(int N, int B, int Hq, int Hkv, int64_t max_keys, int num_sms) {
  if (N < 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || max_keys < 0 || num_sms <= 0) return EXK_EARG;
  if (Hq / Hkv > 16) return EXK_EHEADS;
  const int64_t items = prefill_slots(N, B, Hq / Hkv) * Hkv;
  const int64_t tiles = (max_keys + kTile - 1) / kTile;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(tiles / 4, kMaxSplits));  // four key tiles to a split at least
  if (items == 0 || items >= 4 * static_cast<int64_t>(num_sms)) return 1;
  const double row_bytes = static_cast<double>(N) * Hq * (kD + 2) * 4;  // of one split's partials
  if (B > 1) {
    // The lengths are on the device: the queries are taken as spread evenly over the
    // sequences and the mean length as 0.6 of the longest. A call takes as long as its
    // longest block or an SM's share (1.8 us a key tile, 4 us a block), and the
    // partials' traffic and merge. Over 39 shapes (1 to 1,000 queries on 300 to
    // 28,000 keys, 2 to 64 sequences, packed prompts) within 2 % of the best number
    // of splits in the mean: 3 sequences of 150 tokens over 4,000 to 15,000 keys 120 us,
    // unsplit 243; 4 of 168 to 484 over 2,600 to 7,500 unsplit 137 us, two splits 150.
    // (Splits for the longest sequences alone, cut to an SM's share on the device,
    // measured slower: the latter 153 us.)
    const double each = static_cast<double>(N) / B, block = 2. * (kTile / (Hq / Hkv));
    const double blocks = B * std::ceil(each / block) * Hkv;
    const double mean = std::max(1., (0.6 * static_cast<double>(max_keys) - 0.5 * each) / kTile);
    double best = 0.;
    int64_t choice = 1;
    for (int64_t ns = 1; ns <= most; ++ns) {
      double us = std::max(1.8 * static_cast<double>((tiles + ns - 1) / ns) + 4., blocks * (1.8 * mean + 4. * ns) / num_sms);
      if (ns > 1) us += 6. + 4. * row_bytes * ns / 6.5e6;
      if (ns == 1 || us < best) {
        best = us;
        choice = ns;
      }
    }
    return static_cast<int>(choice);
  }
  // One sequence: its blocks see max_keys - N keys of context and up to N more. The
  // estimate counts waves of blocks (1.8 us a key tile, 4 us a block) where the
  // context outweighs the blocks' differences, else the longest block or an SM's
  // share, and the partials' traffic. (2,048 tokens over 32,768 keys, 28 heads to 4:
  // 228 blocks, three splits 848 us, unsplit 900 us.)
  const double context = static_cast<double>(std::max<int64_t>(0, max_keys - N));
  double best = 0.;
  int64_t choice = 1;
  for (int64_t ns = 1; ns <= most; ++ns) {
    const double longest = 1.8 * static_cast<double>((tiles + ns - 1) / ns) + 4.;
    const double waves = static_cast<double>((items * ns + num_sms - 1) / num_sms);
    const double share = static_cast<double>(items) * (1.8 * (context + 0.5 * N) / kTile + 4. * ns) / num_sms;
    double us = context > N ? waves * longest : std::max(longest, share);
    if (ns > 1) us += 4. + 2. * row_bytes * ns / 6.5e6;
    if (ns == 1 || us < best) {
      best = us;
      choice = ns;
    }
  }
  return static_cast<int>(choice);
}

extern "C" int exk_attention_prefill(const exk_prefill* p, const uint16_t* k, int64_t k_st, int64_t k_sh,
                                     const uint16_t* v, int64_t v_st, int64_t v_sh, int Nk, const int32_t* cu_k,
                                     int32_t* status, int device, void* stream) {
  int r = check_prefill(p);
  if (r != 0) return r;
  if (k == nullptr || v == nullptr || cu_k == nullptr || Nk <= 0 || Nk > (1 << 30)) return EXK_EARG;
  if (p->N == 0) return 0;
  DeviceScope scope;
  if ((r = use_device(device, nullptr)) != 0) return r;
  PrefillArgs a = {};
  a.cu_k = cu_k;
  a.Nk = Nk;
  return launch_prefill(p, a, k, k_st, k_sh, v, v_st, v_sh, Nk, kTile, status, device, static_cast<cudaStream_t>(stream),
                        false);
}

extern "C" int exk_attention_prefill_paged(const exk_prefill* p, const uint16_t* k, const uint16_t* v, int pool_pages,
                                           const int32_t* block_table, int max_pages, const int32_t* seq_lens,
                                           int32_t* status, int device, void* stream) {
  int r = check_prefill(p);
  if (r != 0) return r;
  if (k == nullptr || v == nullptr || block_table == nullptr || seq_lens == nullptr || pool_pages <= 0 ||
      pool_pages >= (1 << 26) || max_pages <= 0 || max_pages >= (1 << 26))
    return EXK_EARG;
  if (p->N == 0) return 0;
  DeviceScope scope;
  if ((r = use_device(device, nullptr)) != 0) return r;
  PrefillArgs a = {};
  a.lens = seq_lens;
  a.block_table = block_table;
  a.max_pages = max_pages;
  a.pool_pages = pool_pages;
  const int64_t st = static_cast<int64_t>(p->Hkv) * kD;
  return launch_prefill(p, a, k, st, kD, v, st, kD, static_cast<int64_t>(pool_pages) * kP, kP, status, device,
                        static_cast<cudaStream_t>(stream), false);
}

extern "C" int exk_attention_prefill_paged_compressed(const exk_prefill* p, const exk_cview* k, const exk_cview* v,
                                                      int pool_pages, const int32_t* block_table, int max_pages,
                                                      const int32_t* seq_lens, uint16_t* k_rows, uint16_t* v_rows,
                                                      int max_len, int32_t* status, int device, void* stream) {
  int r = check_prefill(p);
  if (r != 0) return r;
  if (k == nullptr || v == nullptr || block_table == nullptr || seq_lens == nullptr || k_rows == nullptr ||
      v_rows == nullptr || pool_pages <= 0 || pool_pages >= (1 << 26) || max_pages <= 0 || max_pages >= (1 << 26) ||
      max_len <= 0 || max_len % kP != 0 || max_len > max_pages * kP)
    return EXK_EARG;
  const int64_t rows = static_cast<int64_t>(p->B) * max_len;
  if (rows > (int64_t{1} << 30)) return EXK_EARG;
  for (const exk_cview* c : {k, v}) {
    if (c->sm == nullptr || c->code == nullptr || c->base == nullptr || c->rowmask == nullptr || c->rowoff == nullptr ||
        c->raw == nullptr || c->raw_rows < 0)
      return EXK_EARG;
    if (!aligned16(c->sm) || !aligned16(c->code) || !aligned16(c->base) || !aligned16(c->raw)) return EXK_EALIGN;
  }
  if (!aligned16(k_rows) || !aligned16(v_rows)) return EXK_EALIGN;
  if (p->N == 0) return 0;
  DeviceScope scope;
  if ((r = use_device(device, nullptr)) != 0) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Unpack u = {};
  u.c[0] = *k;
  u.c[1] = *v;
  u.out[0] = k_rows;
  u.out[1] = v_rows;
  u.cu_q = p->cu_q;
  u.block_table = block_table;
  u.lens = seq_lens;
  u.status = status;
  u.k_stride = max_len;
  u.B = p->B;
  u.Hkv = p->Hkv;
  u.max_pages = max_pages;
  u.pool_pages = pool_pages;
  u.pages = max_len / kP;
  const int64_t blocks = (rows / kP * p->Hkv + 7) / 8;
  if (blocks >= (int64_t{1} << 31)) return EXK_EARG;
  unpack_kernel<<<dim3(static_cast<unsigned>(blocks), 2), 256, 0, st>>>(u);
  if ((r = launch_status()) != 0) return r;
  PrefillArgs a = {};
  a.lens = seq_lens;
  a.k_stride = max_len;
  const int64_t st_e = static_cast<int64_t>(p->Hkv) * kD;
  return launch_prefill(p, a, k_rows, st_e, kD, v_rows, st_e, kD, rows, kTile, status, device, st, true);
}
