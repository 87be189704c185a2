// Projections with weights in 4 bits: y[b][n] = sum_k (c[n][k] - z[n][k / G]) s[n][k / G] x[b][k].
#include "common.cuh"
#include "lowbit.h"

namespace mmc {
namespace {

constexpr int kW4Warps = 8;

// The code c in 0..15 sits in the low mantissa bits of 1024 (or, four bits up,
// of 1024 as 16 c): 1024 + c and 1024 + 16 c are exact in fp16, and so are the
// differences below.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) { return (a & mask) | bits; }
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
  const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 d =
      __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&d);
}
// eight codes of one word less z: pairs of columns (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ void codes_less(uint32_t w, uint32_t z1024, uint32_t z64, uint32_t (&h)[4]) {
  const uint32_t sixteenth = 0x2c002c00u;  // 1/16
  h[0] = h2_sub(and_or(w, 0x000f000fu, 0x64006400u), z1024);
  h[1] = h2_fma(and_or(w, 0x00f000f0u, 0x64006400u), sixteenth, z64);  // (1024 + 16 c) / 16 - (64 + z)
  w >>= 8;
  h[2] = h2_sub(and_or(w, 0x000f000fu, 0x64006400u), z1024);
  h[3] = h2_fma(and_or(w, 0x00f000f0u, 0x64006400u), sixteenth, z64);
}

// One CTA: 16 weight rows x 8 NT batch rows; the warps take the groups of
// columns in turn and their sums are joined in order. m16n8k16 with the weight
// rows on M: the codes less the zero point are exact in fp16, each group's sum
// is taken in fp32 and then scaled.
template <int NT>
__global__ void __launch_bounds__(kW4Warps * 32) w4_projection_kernel(const W4Args a) {
  __shared__ float part[kW4Warps][NT][32][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, b0 = blockIdx.y * 8 * NT;
  const int groups = a.K / a.group;
  const int rA = min(n0 + g, a.N - 1), rB = min(n0 + g + 8, a.N - 1);
  float acc[NT][4] = {};
  for (int gr = warp; gr < groups; gr += kW4Warps) {
    const float sA = __half2float(a.scales[(size_t)rA * groups + gr]), sB = __half2float(a.scales[(size_t)rB * groups + gr]);
    const uint32_t zA = a.zeros ? a.zeros[(size_t)rA * groups + gr] : 8u, zB = a.zeros ? a.zeros[(size_t)rB * groups + gr] : 8u;
    const __half hA = __float2half_rn(1024.f + float(zA)), hB = __float2half_rn(1024.f + float(zB));
    const __half lA = __float2half_rn(-64.f - float(zA)), lB = __float2half_rn(-64.f - float(zB));
    const __half2 hA2 = __half2half2(hA), hB2 = __half2half2(hB), lA2 = __half2half2(lA), lB2 = __half2half2(lB);
    float d[NT][4] = {};
    for (int k = gr * a.group; k < (gr + 1) * a.group; k += 32) {
      const uint32_t wA = *reinterpret_cast<const uint32_t*>(a.codes + (size_t)rA * (a.K / 2) + k / 2 + 4 * t);
      const uint32_t wB = *reinterpret_cast<const uint32_t*>(a.codes + (size_t)rB * (a.K / 2) + k / 2 + 4 * t);
      uint32_t hA4[4], hB4[4];
      codes_less(wA, *reinterpret_cast<const uint32_t*>(&hA2), *reinterpret_cast<const uint32_t*>(&lA2), hA4);
      codes_less(wB, *reinterpret_cast<const uint32_t*>(&hB2), *reinterpret_cast<const uint32_t*>(&lB2), hB4);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int b = b0 + nt * 8 + g;
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (b < a.B) x = *reinterpret_cast<const uint4*>(a.x + (size_t)b * a.K + k + 8 * t);
        // columns 0..7 into the codes' order of pairs
        mma16816(d[nt], hA4[0], hB4[0], hA4[1], hB4[1], __byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632));
        mma16816(d[nt], hA4[2], hB4[2], hA4[3], hB4[3], __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[nt][e] += (e < 2 ? sA : sB) * d[nt][e];
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[warp][nt][lane][e] = acc[nt][e];
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 128; i += kW4Warps * 32) {
    const int b = i / 16, r = i % 16;  // batch row and weight row in the tile
    const int nt = b / 8, ln = (r % 8) * 4 + (b % 8) / 2, e = (r / 8) * 2 + (b & 1);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kW4Warps; ++w) sum += part[w][nt][ln][e];
    if (b0 + b < a.B && n0 + r < a.N) a.y[(size_t)(b0 + b) * a.N + n0 + r] = sum;
  }
}

template <int NT>
cudaError_t launch_nt(const W4Args& a, cudaStream_t s) {
  w4_projection_kernel<NT><<<dim3((a.N + 15) / 16, (a.B + 8 * NT - 1) / (8 * NT)), kW4Warps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_w4_projection(const W4Args& a, int sms, cudaStream_t s) {
  return a.B <= 8 ? launch_nt<1>(a, s) : a.B <= 16 ? launch_nt<2>(a, s) : launch_nt<4>(a, s);
}

cudaError_t w4_init_attributes() { return cudaSuccess; }

}  // namespace mmc
