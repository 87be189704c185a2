// Projections with weights in 4 bits: y[b][n] = sum_k (c[n][k] - z[n][k / G]) s[n][k / G] x[b][k].
//
// A CTA takes BM weight rows and 8 NT batch rows. Tensor copies stream the codes
// and x through a ring; eight warps (WM down the rows, WK along the columns, 128
// columns of each stage a warp) take them from there: codes by ldmatrix, less
// their zero point in fp16 (exact), m16n8k16 with the weight rows on M, each
// group's sum in fp32, then scaled. The warps' and, where a cluster shares the
// columns, the CTAs' sums are joined in a fixed order.
//   Few batch rows are bound by HBM; the codes' way to fp16 (nine instructions a
// word of eight) is what keeps the warps busy, so the rows of x are cheap up to
// eight. With more, the matrix instructions are (8.9 cycles each of a quarter of
// an SM).
#include "common.cuh"
#include "lowbit.h"

namespace mmc {
namespace {

constexpr int kW4Warps = 8;
constexpr int kW4Threads = kW4Warps * 32;
constexpr int kW4Part = 128;                     // columns of a stage that one warp takes

template <int NT>
struct W4Cfg {
  static constexpr int MT = 2;                                   // 16-row tiles of a warp
  static constexpr int WM = NT == 1 ? 1 : NT == 2 ? 2 : 4;       // warps down the rows
  static constexpr int WK = kW4Warps / WM;                       // warps along the columns
  static constexpr int BM = 16 * MT * WM, KC = kW4Part * WK;     // rows of a CTA, columns of a stage
  static constexpr int W_BYTES = BM * KC / 2, X_BYTES = 8 * NT * KC * 2, STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = NT <= 2 ? 3 : 4;
  static constexpr int CTAS = NT <= 2 ? 2 : 1;                   // of an SM
  static constexpr int JOIN = (WK + 1) * BM * 8 * NT * 4;
  static constexpr int RING = STAGE * STAGES > JOIN ? STAGE * STAGES : JOIN;
  static constexpr int SMEM = 1024 + RING + 2 * STAGES * 8;
};

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
  const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 d =
      __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&d);
}
// Eight codes of one word less z, as pairs of columns (0, 4), (1, 5), (2, 6),
// (3, 7). A code in the low mantissa bits of 1024 is 1024 + c, four bits up
// 1024 + 16 c: exact, and so are the differences. z1024: 1024 + z, z64: -(64 + z).
__device__ __forceinline__ void codes_less(uint32_t w, uint32_t z1024, uint32_t z64, uint32_t (&h)[4]) {
  constexpr uint32_t sixteenth = 0x2c002c00u, low = 0x000f000fu, high = 0x00f000f0u, k1024 = 0x64006400u;
  h[0] = h2_sub((w & low) | k1024, z1024);
  h[1] = h2_fma((w & high) | k1024, sixteenth, z64);
  w >>= 8;
  h[2] = h2_sub((w & low) | k1024, z1024);
  h[3] = h2_fma((w & high) | k1024, sixteenth, z64);
}
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// A wait that a copy or a warp of this CTA ends; after two seconds it gives up
// and the call's outputs become NaN (there is no error word to set).
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, nullptr); }

template <int NT, int GROUP>
__global__ void __launch_bounds__(kW4Threads, W4Cfg<NT>::CTAS)
    w4_projection_kernel(const W4Args a, int parts, const __grid_constant__ CUtensorMap wmap,
                         const __grid_constant__ CUtensorMap xmap) {
  using C = W4Cfg<NT>;
  constexpr int MT = C::MT, GP = kW4Part / GROUP;  // groups of a warp's columns in a stage
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::RING);
  uint64_t* empty = full + C::STAGES;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int n0 = blockIdx.x / parts * C::BM, b0 = blockIdx.y * 8 * NT;
  const int all = (a.K + C::KC - 1) / C::KC, per = (all + parts - 1) / parts;
  const int s0 = min(all, int(rank) * per), s1 = min(all, s0 + per);  // this CTA's stages of columns
  if (tid < C::STAGES) {
    mbar_init(full + tid, 1);
    mbar_init(empty + tid, kW4Warps);
  }
  fence_mbar_init();
  __syncthreads();
  bool ok = true;
  float acc[MT][NT][4] = {};
  const int wm = warp % C::WM, wk = warp / C::WM;
  // thread 0 starts the copies of this CTA's i-th stage
  auto fill = [&](int i) {
    const int s = s0 + i, st = i % C::STAGES;
    const uint32_t dst = smem_u32(smem + st * C::STAGE);
    mbar_arrive_expect_tx(full + st, C::STAGE);
#pragma unroll
    for (int j = 0; j < C::KC / 256; ++j) load_2d(dst + j * C::BM * 128, &wmap, s * (C::KC / 2) + j * 128, n0, full + st);
#pragma unroll
    for (int j = 0; j < C::KC / 64; ++j)
      load_2d(dst + C::W_BYTES + j * 8 * NT * 128, &xmap, s * C::KC + j * 64, b0, full + st);
  };
  int filled = min(C::STAGES, s1 - s0);
  if (tid == 0)
    for (int i = 0; i < filled; ++i) fill(i);
  {
    const int groups = a.K / GROUP;
    // this lane's rows, n0 + wm * 32 + g + 8 r, and (of a stage's GP groups of this warp) group t
    const int row0 = n0 + wm * 16 * MT + g;
    auto fetch = [&](int s, uint32_t (&sc)[2 * MT], uint32_t (&z)[2 * MT]) {
      const int gr = s * (C::KC / GROUP) + wk * GP + (t % GP);
      const bool in = s < s1 && gr < groups;
#pragma unroll
      for (int r = 0; r < 2 * MT; ++r) {
        const bool here = in && row0 + 8 * r < a.N;
        const size_t at = (size_t)(row0 + 8 * r) * groups + gr;
        sc[r] = here ? __half_as_ushort(a.scales[at]) : 0u;
        z[r] = here && a.zeros ? a.zeros[at] : 8u;
      }
    };
    uint32_t sc[2 * MT], z[2 * MT];
    fetch(s0, sc, z);
    // ldmatrix: row `lane` of the warp's 32, 16-byte chunk 4 (wk & 1) + c of its 128-byte row
    const uint32_t w_at = (wk >> 1) * C::BM * 128 + (wm * 32 + lane) * 128;
    // x: batch row 8 nt + xr is column g of the n-tile, so that the eight lanes of a 16-byte read's phase fall on all banks
    // of the swizzled rows
    const int xr = (g & 1) * 4 + (g >> 1);
    const uint32_t x_at = C::W_BYTES + wk * 2 * (8 * NT * 128) + xr * 128 + ((t ^ (xr & 3)) << 4);
    for (int s = s0; s < s1; ++s) {
      const int i = s - s0, st = i % C::STAGES;
      uint32_t sc1[2 * MT], z1[2 * MT];
      fetch(s + 1, sc1, z1);
      ok = __all_sync(0xffffffffu, ok && wait(full + st, (i / C::STAGES) & 1));
      if (!ok) break;
      if (tid == 0 && i > 0 && i - 1 + C::STAGES < s1 - s0) {  // the stage before this one, once all warps have left it
        ok = wait(empty + (i - 1) % C::STAGES, ((i - 1) / C::STAGES) & 1);
        if (ok) fill(filled++);
      }
      const uint8_t* base = smem + st * C::STAGE;
      const uint32_t base_u = smem_u32(base);
      float d[MT][NT][4];
#pragma unroll
      for (int c = 0; c < kW4Part / 32; ++c) {
        if (c % (GROUP / 32) == 0) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) d[mt][nt][0] = d[mt][nt][1] = d[mt][nt][2] = d[mt][nt][3] = 0.f;
        }
        const int gi = c / (GROUP / 32);  // group of the stage's GP
        uint32_t w[4], h[2 * MT][4];
        ldsm_x4(base_u + w_at + (((4 * (wk & 1) + c) ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) {
          const uint32_t zr = GP == 1 ? z[r] : __shfl_sync(0xffffffffu, z[r], (lane & ~3) + gi);
          const uint32_t z1024 = (0x6400u + zr) * 0x10001u;
          codes_less(w[r], z1024, h2_sub(0x63806380u, z1024), h[r]);  // 960 - (1024 + z)
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 x = *reinterpret_cast<const uint4*>(
              base + ((x_at + (c >> 1) * (8 * NT * 128) + nt * 1024) ^ (((xr & 4) ^ (4 * (c & 1))) << 4)));
          // columns 0..7 into the codes' order of pairs
          const uint32_t p04 = __byte_perm(x.x, x.z, 0x5410), p15 = __byte_perm(x.x, x.z, 0x7632);
          const uint32_t p26 = __byte_perm(x.y, x.w, 0x5410), p37 = __byte_perm(x.y, x.w, 0x7632);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16816(d[mt][nt], h[2 * mt][0], h[2 * mt + 1][0], h[2 * mt][1], h[2 * mt + 1][1], p04, p15);
            mma16816(d[mt][nt], h[2 * mt][2], h[2 * mt + 1][2], h[2 * mt][3], h[2 * mt + 1][3], p26, p37);
          }
        }
        if ((c + 1) % (GROUP / 32) == 0) {
#pragma unroll
          for (int r = 0; r < 2 * MT; ++r) {
            const uint32_t sr = GP == 1 ? sc[r] : __shfl_sync(0xffffffffu, sc[r], (lane & ~3) + gi);
            const float f = __half2float(__ushort_as_half(uint16_t(sr)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float* dst = acc[r >> 1][nt] + 2 * (r & 1);
              const float* src = d[r >> 1][nt] + 2 * (r & 1);
              dst[0] += f * src[0];
              dst[1] += f * src[1];
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
#pragma unroll
      for (int r = 0; r < 2 * MT; ++r) {
        sc[r] = sc1[r];
        z[r] = z1[r];
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[mt][nt][0] = acc[mt][nt][1] = acc[mt][nt][2] = acc[mt][nt][3] = __uint_as_float(0x7fc00000u);
  }
  // a CTA whose wait ran out still has copies on their way into the ring: wait for them (again with a limit)
  if (!__syncthreads_and(ok)) {
    if (tid == 0)
      for (int i = max(0, filled - C::STAGES); i < filled; ++i) wait(full + i % C::STAGES, (i / C::STAGES) & 1);
    __syncthreads();
  }
  // ---- join the warps along the columns: [wk][batch row][BM]
  float* part = reinterpret_cast<float*>(smem);
  float* joined = part + C::WK * 8 * NT * C::BM;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e)  // columns 2 t and 2 t + 1 are batch rows t and t + 4
        part[(wk * 8 * NT + nt * 8 + t + 4 * (e & 1)) * C::BM + wm * 16 * MT + mt * 16 + g + 8 * (e >> 1)] = acc[mt][nt][e];
  __syncthreads();
  const int nb = min(8 * NT, a.B - b0);
  for (int i = tid; i < nb * C::BM; i += kW4Threads) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < C::WK; ++k) sum += part[k * 8 * NT * C::BM + i];
    const int n = n0 + i % C::BM;
    if (parts > 1) joined[i] = sum;
    else if (n < a.N) a.y[(size_t)(b0 + i / C::BM) * a.N + n] = sum;
  }
  if (parts == 1) return;
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const uint32_t joined_u = smem_u32(joined);
  for (int i = rank * kW4Threads + tid; i < nb * C::BM; i += parts * kW4Threads) {
    float sum = 0.f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      uint32_t at;
      float v;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(joined_u + 4 * i), "r"(p));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
      sum += v;
    }
    const int n = n0 + i % C::BM;
    if (n < a.N) a.y[(size_t)(b0 + i / C::BM) * a.N + n] = sum;
  }
  __syncwarp();  // no CTA leaves while another reads its shared memory
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

template <int NT, int GROUP>
cudaError_t launch(const W4Args& a, int sms, cudaStream_t s) {
  using C = W4Cfg<NT>;
  const EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  CUtensorMap wmap, xmap;
  {  // codes [N][K / 2] bytes, boxes of 128 bytes x BM rows, 128-byte swizzle
    const cuuint64_t dims[2] = {cuuint64_t(a.K / 2), cuuint64_t(a.N)}, strides[1] = {cuuint64_t(a.K / 2)};
    const cuuint32_t box[2] = {128, C::BM}, one[2] = {1, 1};
    if (fn(&wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(a.codes), dims, strides, box, one,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  {  // x [B][K] fp16, boxes of 64 columns x 8 NT rows, 128-byte swizzle
    const cuuint64_t dims[2] = {cuuint64_t(a.K), cuuint64_t(a.B)}, strides[1] = {cuuint64_t(a.K) * 2};
    const cuuint32_t box[2] = {64, 8 * NT}, one[2] = {1, 1};
    if (fn(&xmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<__half*>(a.x), dims, strides, box, one,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  const int64_t tiles = (int64_t)((a.N + C::BM - 1) / C::BM) * ((a.B + 8 * NT - 1) / (8 * NT));
  const int stages = (a.K + C::KC - 1) / C::KC;
  int parts = 1;  // CTAs that share the columns: while they find places, and two stages each
  while (parts < 8 && tiles * parts * 2 <= (int64_t)sms * C::CTAS && stages >= 4 * parts) parts *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.N + C::BM - 1) / C::BM * parts, (a.B + 8 * NT - 1) / (8 * NT));
  cfg.blockDim = dim3(kW4Threads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, w4_projection_kernel<NT, GROUP>, a, parts, wmap, xmap);
}

template <int NT>
cudaError_t launch_nt(const W4Args& a, int sms, cudaStream_t s) {
  return a.group == 32 ? launch<NT, 32>(a, sms, s) : a.group == 64 ? launch<NT, 64>(a, sms, s) : launch<NT, 128>(a, sms, s);
}

template <int NT>
cudaError_t attrs() {
  for (const cudaError_t e : {set_kernel_smem(w4_projection_kernel<NT, 32>, W4Cfg<NT>::SMEM),
                              set_kernel_smem(w4_projection_kernel<NT, 64>, W4Cfg<NT>::SMEM),
                              set_kernel_smem(w4_projection_kernel<NT, 128>, W4Cfg<NT>::SMEM)})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_w4_projection(const W4Args& a, int sms, cudaStream_t s) {
  const int nt = (a.B + 7) / 8;
  return nt == 1   ? launch_nt<1>(a, sms, s)
         : nt == 2 ? launch_nt<2>(a, sms, s)
         : nt == 3 ? launch_nt<3>(a, sms, s)
         : nt == 4 ? launch_nt<4>(a, sms, s)
                   : launch_nt<8>(a, sms, s);
}

cudaError_t w4_init_attributes() {
  for (const cudaError_t e : {attrs<1>(), attrs<2>(), attrs<3>(), attrs<4>(), attrs<8>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

}  // namespace mmc
