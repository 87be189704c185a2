// Device helpers of the 8-bit paged cache: its layout, codes and scales, and the
// checked view of a call's sequence (kv8.cu, kv8_attention.cu, kv8_prompts.cu).
#pragma once

#include "common.cuh"
#include "lowbit.h"

namespace mmc {

__device__ __forceinline__ size_t kv8_slab(const Kv8Args& c, int page, int kv, int h) {
  return (((size_t)page * c.layers + c.layer) * 2 + kv) * c.nkv + h;  // x 64 * hd codes, x 4 scales
}

// ---------------------------------------------------------------- scales and codes

// Smallest power of two s with amax <= 448 s: amax = f * 2^x with f in [1, 2),
// and 448 = 1.75 * 2^8. NaN for a block that holds an infinity or a NaN.
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax) & 0x7fffffffu;
  if (u >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const int e = int(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(uint32_t(max(e, -126) + 127) << 23);
}
// 1 / s of a power of two in [2^-126, 2^120]
__device__ __forceinline__ float pow2_inverse(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint8_t to_e4m3(float x) { return uint8_t(to_e4m3x2(x, 0.f)); }
// two e4m3 codes (low byte first) to fp16: exact
__device__ __forceinline__ uint32_t e4m3x2_half2(uint32_t two) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(uint16_t(two)));
  return d;
}
__device__ __forceinline__ float from_e4m3(uint8_t c) {
  const uint32_t h2 = e4m3x2_half2(c);
  return __half2float(__ushort_as_half(uint16_t(h2)));
}

// ---------------------------------------------------------------- attention

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoScore = -3.0e38f;  // the running maximum of a row that has seen nothing
constexpr int kKv8PromptRows = 128;   // rows of a CTA of the kernel for long runs

__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  const __half2 d = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The kernel for long runs: a.tiles of kKv8PromptRows rows a sequence and kv head
cudaError_t launch_kv8_prompts(const Kv8AttnArgs& a, int hd, cudaStream_t s);
cudaError_t kv8_prompts_init_attributes();

// ---------------------------------------------------------------- a call's sequences

struct Kv8Seq {
  int slot, first, n, pos0;  // n: rows of the sequence (0: none, or refused)
  bool refused;
};
// The sequence's rows and positions, checked: everything later indexes within them.
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Args& c, int max_ctx, int seq, bool report) {
  Kv8Seq s{-1, 0, 0, 0, false};
  const int slot = c.slots[seq];  // (with the rows, not behind them)
  s.first = c.row_start ? c.row_start[seq] : seq;
  const int last = c.row_start ? c.row_start[seq + 1] : seq + 1;
  int e = 0;
  if (s.first < 0 || last > c.rows || last < s.first || last - s.first > c.max_new) {
    e = kDevBadRows;
  } else {
    s.n = last - s.first;
    s.slot = slot;
    if (s.slot >= c.max_seqs) {
      e = kDevBadSlot;
    } else if (s.slot >= 0) {
      s.pos0 = c.seq_pos[s.slot];
      const int64_t end = (int64_t)s.pos0 + s.n;
      if (s.pos0 < 0 || end > max_ctx || end > (int64_t)c.max_pages * kPageTokens) e = kDevContextLimit;
    }
  }
  if (e != 0) {
    if (report) set_error(c.err, e);
    s.n = 0;
    s.refused = true;
  }
  return s;
}

}  // namespace mmc
