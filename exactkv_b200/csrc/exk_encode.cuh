// Pieces shared by the encoder kernels (exk_codec.cu, exk_paged.cu): launch
// chaining and the 16-bit-lane arithmetic of the page encoder.
#pragma once

#include "exk_device.cuh"

namespace exk {

// The kernels after the first of a call are programmatic dependents of the
// kernel before them on the stream (launch_after): they may become resident
// while it runs its last wave, which hides their launch latency, and wait in
// after_prior() until it has completed and its writes are visible (a no-op
// after an ordinary launch). allow_dependents() lets them be scheduled.
__device__ __forceinline__ void after_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_dependents() {
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Constants the compiler cannot see (2^25, 2^24, 1, 2), so that shifts and
// lane-wise adds of the encoder become multiplies on the FMA pipe: the encoder
// keeps the ALU pipe busy. A lane-wise add is a plain 32-bit add when neither
// 16-bit lane can carry into the next: the lanes then hold 0x8000 + e - b.
static __constant__ uint32_t c_fma[5] = {1u << 25, 1u << 24, 1u, 2u, 16u};

__device__ __forceinline__ uint32_t mulhi(uint32_t x, uint32_t k) {
  uint32_t d;
  asm("mul.hi.u32 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(k));
  return d;
}
__device__ __forceinline__ uint32_t mad_lo(uint32_t x, uint32_t k, uint32_t y) {
  uint32_t d;
  asm("mad.lo.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(k), "r"(y));
  return d;
}

// Two 16-bit lanes per word (PTX integer SIMD; add wraps within each lane).
__device__ __forceinline__ uint32_t max_u16x2(uint32_t x, uint32_t y) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
  return d;
}
__device__ __forceinline__ uint32_t min_u16x2(uint32_t x, uint32_t y) {
  uint32_t d;
  asm("min.u16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
  return d;
}
__device__ __forceinline__ uint32_t max_s16x2(uint32_t x, uint32_t y) {
  uint32_t d;
  asm("max.s16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
  return d;
}
__device__ __forceinline__ uint32_t add_u16x2(uint32_t x, uint32_t y) {
  uint32_t d;
  asm("add.u16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
  return d;
}

// One (page, KV head) of the encoder with its rows in registers: lane (q =
// lane % 16, th = lane / 16) passes w[i] = rows 8th + i as bf16 pairs (4q, 4q+1),
// (4q+2, 4q+3), (64+4q, ..), (64+4q+2, ..). Writes the base bytes at `base`
// and row r's bytes at sm + r * sm_row and code + r * code_row (bytes), and
// returns the page's rowmask in every lane. The same per-value rules as
// encode_kernel (base b = max(emax - 15, 0), zero group zm, code e - b, escape
// e < b + zm or b >= 128), so the bytes are the same.
__device__ __forceinline__ uint32_t encode_rows(const uint32_t (&w)[8][4], int lane, uint8_t* sm, int64_t sm_row,
                                                uint8_t* code, int64_t code_row, uint8_t* base) {
  const int q = lane & 15, th = lane >> 4;
  const uint32_t k25 = c_fma[0], k24 = c_fma[1], k1 = c_fma[2], k2 = c_fma[3], k16 = c_fma[4];
  uint32_t emax2[4], emin2[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    emax2[j] = 0u;
    emin2[j] = 0xFFFFFFFFu;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t e2 = mad_lo(w[i][j], k2, 0u);
      emax2[j] = max_u16x2(emax2[j], e2);
      emin2[j] = min_u16x2(emin2[j], e2);
    }
  }
  uint32_t byte2[4], cb2[4], czb2[4], escany = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    emax2[j] = max_u16x2(emax2[j], __shfl_xor_sync(0xFFFFFFFFu, emax2[j], 16));
    emin2[j] = min_u16x2(emin2[j], __shfl_xor_sync(0xFFFFFFFFu, emin2[j], 16));
    const uint32_t e2 = (emax2[j] >> 8) & 0x00FF00FFu;
    const uint32_t z2 = (emin2[j] >> 8) & 0x00FF00FFu;
    const uint32_t b2 = max_s16x2(add_u16x2(e2, 0xFFF1FFF1u), 0u);
    const uint32_t zm2 = (min_u16x2(z2, 0x00010001u) ^ 0x00010001u) & min_u16x2(b2, 0x00010001u);
    byte2[j] = min_u16x2(add_u16x2(b2, zm2 << 7), 0x00FF00FFu);
    cb2[j] = 0x80008000u - (j < 2 ? b2 : b2 << 4);
    czb2[j] = 0x80008000u - (b2 + zm2);
    escany |= b2 & 0xFF80FF80u;
  }
  if (th == 0) {
    *reinterpret_cast<uint32_t*>(base + 4 * q) = prmt(byte2[0], byte2[1], 0x6420u);
    *reinterpret_cast<uint32_t*>(base + 64 + 4 * q) = prmt(byte2[2], byte2[3], 0x6420u);
  }
  uint32_t escw = escany != 0u ? 0x00FF00FFu : 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t code2[4], x[4], escacc = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t e2 = mulhi(w[i][j], k25) & 0x00FF00FFu;
      code2[j] = max_u16x2(mad_lo(e2, j < 2 ? k1 : k16, cb2[j]), 0x80008000u);
      escacc |= ~mad_lo(e2, k1, czb2[j]) & mad_lo(e2, k1, 0x7FFF7FFFu);
      x[j] = (mulhi(w[i][j], k24) & 0x00800080u) | (w[i][j] & 0xFF7FFF7Fu);
    }
    uint8_t* srow = sm + (th * 8 + i) * sm_row;
    *reinterpret_cast<uint32_t*>(srow + 4 * q) = prmt(x[0], x[1], 0x6420u);
    *reinterpret_cast<uint32_t*>(srow + 64 + 4 * q) = prmt(x[2], x[3], 0x6420u);
    *reinterpret_cast<uint32_t*>(code + (th * 8 + i) * code_row + 4 * q) =
        prmt(code2[0] | code2[2], code2[1] | code2[3], 0x6420u);
    escw |= (escacc >> (15 - i)) & (0x00010001u << i);
  }
  const uint32_t escrow = (escw | (escw >> 16)) & 0xFFu;
  return __reduce_or_sync(0xFFFFFFFFu, escrow << (8 * th));
}

}  // namespace exk
