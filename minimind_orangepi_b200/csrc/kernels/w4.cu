// Projections with weights in 4 bits: y[b][n] = sum_k (c[n][k] - z[n][k / G]) s[n][k / G] x[b][k].
//
// A CTA takes BM weight rows and 8 NT batch rows. Tensor copies stream the codes
// and x through a ring; the warps (WM down the rows, WK along the columns, 128
// columns of each stage a warp) take them from there: codes by ldmatrix, less
// their zero point in fp16 (exact), m16n8k16 with the weight rows on M, each
// group's sum in fp32, then scaled. The warps' and, where a cluster shares the
// columns, the CTAs' sums are joined in a fixed order.
//   Up to eight batch rows the codes are all that counts in bytes, and their way to
// fp16 (nine instructions a word of eight) in instructions, so further rows of x are
// cheap (8192 x 8192, group 64 with zero points: one row 15.7 us, eight 16.1). What
// bounds it is latency: the schedulers issue in 51 % of the cycles with 7 warps each,
// which wait for loads, for the half-rate pipe where they unpack at the same time,
// and for x to be laid out; 768 x 768 takes 2.9 us, 16384 x 8192 20.2 of a floor of
// 10.6 (29 with x from L1 and unpacking by two instructions more), with zero points
// in groups of 32 and eight rows 31. With more rows the same warps unpack and
// multiply, and the matrix instructions (8.9 cycles each of a quarter of an SM) lead
// from some 32 rows on: 8192 x 8192, group 128: 16 rows 16.4 us, 24 rows 19.5, 64
// rows 38.6; above, the codes are read and unpacked again for each 64 rows (group 64
// with zero points: 64 rows 44, 256 rows 147, 2048 rows 1020). The scales by a load
// of each lane's own had taken a third of the time, hence their asynchronous copies. Tried: refilling a stage two turns after its last
// reader instead of one (the same), shorter stages (slower).
#include "common.cuh"
#include "lowbit.h"

#include <algorithm>

namespace mmc {
namespace {

constexpr int kW4Part = 128;                     // columns of a stage that one warp takes

template <int NT>
struct W4Cfg {
  static constexpr int WARPS = NT == 8 ? 8 : 16, THREADS = WARPS * 32;
  static constexpr int MT = 2;                                   // 16-row tiles of a warp
  static constexpr int WM = 4;                                   // warps down the rows
  static constexpr int WK = WARPS / WM;                          // warps along the columns
  static constexpr int BM = 16 * MT * WM, KC = kW4Part * WK;     // rows of a CTA, columns of a stage
  static constexpr int W_BYTES = BM * KC / 2, X_BYTES = 8 * NT * KC * 2, STAGE = W_BYTES + X_BYTES;
  static constexpr int SC_BYTES = BM * (KC / 32) * 3;            // scales and zero points of the smallest groups
  static constexpr int STAGES = 216 * 1024 / (STAGE + SC_BYTES);
  static constexpr int JOIN = (WK + 1) * BM * 8 * NT * 4;
  static constexpr int RING = STAGE * STAGES > JOIN ? STAGE * STAGES : JOIN;
  static constexpr int SMEM = 1024 + RING + STAGES * SC_BYTES + 2 * STAGES * 8;
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
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {  // (a & mask) | bits, one instruction
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(mask), "r"(bits));
  return d;
}
__device__ __forceinline__ void codes_less(uint32_t w, uint32_t z1024, uint32_t z64, uint32_t (&h)[4]) {
  constexpr uint32_t sixteenth = 0x2c002c00u, low = 0x000f000fu, high = 0x00f000f0u, k1024 = 0x64006400u;
  h[0] = h2_sub(and_or(w, low, k1024), z1024);
  h[1] = h2_fma(and_or(w, high, k1024), sixteenth, z64);
  w >>= 8;
  h[2] = h2_sub(and_or(w, low, k1024), z1024);
  h[3] = h2_fma(and_or(w, high, k1024), sixteenth, z64);
}
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// One row's scales (and zero points) of a stage, groups gr0 .. gr0 + gps - 1, by
// one thread: asynchronous copies as wide as the addresses allow, which arrive at
// `bar` when they are done; groups behind the last one read as 0. An odd number
// of groups a row leaves halves that such copies cannot take.
template <bool ZEROS>
__device__ __forceinline__ void copy_scales(const W4Args& a, uint8_t* sc, uint8_t* z, int row, int groups, int gr0, int gps,
                                            uint64_t* bar) {
  const size_t at = (size_t)row * groups + gr0;
  const int have = min(max(groups - gr0, 0), gps);
  auto copy = [&](uint8_t* dst, const uint8_t* src, int bytes, int valid, uint32_t align) {
    if (align % 16 == 0) {
      for (int o = 0; o < bytes; o += 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + o)),
                     "l"(valid > o ? src + o : reinterpret_cast<const uint8_t*>(a.codes)), "r"(min(max(valid - o, 0), 16))
                     : "memory");
    } else if (align % 4 == 0) {
      for (int o = 0; o < bytes; o += 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst + o)),
                     "l"(valid > o ? src + o : reinterpret_cast<const uint8_t*>(a.codes)), "r"(min(max(valid - o, 0), 4))
                     : "memory");
    } else {
      for (int o = 0; o < bytes; ++o) dst[o] = o < valid ? src[o] : 0;
    }
    return align % 4 == 0;
  };
  const uint8_t* s = reinterpret_cast<const uint8_t*>(a.scales);
  bool async = copy(sc, s + 2 * at, 2 * gps, 2 * have, uint32_t(reinterpret_cast<uintptr_t>(s)) | 2 * groups | 2 * gps);
  if constexpr (ZEROS)
    async &= copy(z, a.zeros + at, gps, have, uint32_t(reinterpret_cast<uintptr_t>(a.zeros)) | groups | gps);
  if (async) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
  } else {
    cp_async_wait_all();
    mbar_arrive(bar);
  }
}
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// A wait that a copy or a warp of this CTA ends; after two seconds it gives up
// and the call's outputs become NaN (there is no error word to set).
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, nullptr); }

template <int NT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(W4Cfg<NT>::THREADS, 1)
    w4_projection_kernel(const W4Args a, int parts, const __grid_constant__ CUtensorMap wmap,
                         const __grid_constant__ CUtensorMap xmap) {
  using C = W4Cfg<NT>;
  constexpr int MT = C::MT, CHUNKS = kW4Part / 32;
  constexpr int CG = GROUP / 32, GP = kW4Part / GROUP;  // 32-column chunks of a group, groups of a warp's part
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* scales = smem + C::RING;  // [stage][BM][GPS] fp16, [BM][GPS] bytes
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + C::STAGES * C::SC_BYTES);
  uint64_t* empty = full + C::STAGES;
  constexpr int GPS = C::KC / GROUP;  // groups of a stage
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int n0 = blockIdx.x / parts * C::BM, b0 = blockIdx.y * 8 * NT;
  const int all = (a.K + C::KC - 1) / C::KC, per = (all + parts - 1) / parts;
  const int s0 = min(all, int(rank) * per), n_st = min(all, s0 + per) - s0;  // this CTA's stages of columns
  if (tid < C::STAGES) {
    mbar_init(full + tid, 1 + C::BM);
    mbar_init(empty + tid, C::WARPS);
  }
  fence_mbar_init();
  __syncthreads();
  // the first BM threads start the copies of this CTA's i-th stage: thread 0 codes and x, each its row's scales
  const int groups = a.K / GROUP;
  auto fill = [&](int i) {
    const int s = s0 + i, st = i % C::STAGES;
    if (tid == 0) {
      const uint32_t dst = smem_u32(smem + st * C::STAGE);
      mbar_arrive_expect_tx(full + st, C::STAGE);
#pragma unroll
      for (int j = 0; j < C::KC / 256; ++j) load_2d(dst + j * C::BM * 128, &wmap, s * (C::KC / 2) + j * 128, n0, full + st);
#pragma unroll
      for (int j = 0; j < C::KC / 64; ++j)
        load_2d(dst + C::W_BYTES + j * 8 * NT * 128, &xmap, s * C::KC + j * 64, b0, full + st);
    }
    uint8_t* sc = scales + st * C::SC_BYTES;
    copy_scales<ZEROS>(a, sc + tid * GPS * 2, sc + C::BM * GPS * 2 + tid * GPS, min(n0 + tid, a.N - 1), groups, s * GPS, GPS, full + st);
  };
  int filled = min(C::STAGES, n_st);
  if (tid < C::BM)
    for (int i = 0; i < filled; ++i) fill(i);

  const int wm = warp % C::WM, wk = warp / C::WM;
  // this lane's weight rows of the CTA's are 32 wm + g + 8 r (behind N: the last one's scales, not stored)
  const int sc_at = (wm * 32 + g) * GPS + wk * GP;
  // Batch row 8 nt + xr is column g of an n-tile, so that the eight lanes of a 16-byte read's phase fall on all banks of the
  // swizzled rows.
  const int xr = (g & 1) * 4 + (g >> 1);
  const uint32_t x_at = C::W_BYTES + wk * 2 * (8 * NT * 128) + xr * 128 + ((t ^ (xr & 3)) << 4);
  // ldmatrix: row `lane` of the warp's 32, 16-byte chunk 4 (wk & 1) + c of its 128-byte row
  const uint32_t w_at = (wk >> 1) * C::BM * 128 + (wm * 32 + lane) * 128;
  const uint32_t w_swz = ((4 * (wk & 1)) ^ (lane & 7)) << 4;

  bool ok = true;
  float acc[MT][NT][4] = {};
  int st = 0;
  uint32_t parity = 0;
#pragma unroll 1
  for (int i = 0; i < n_st; ++i) {
    ok = __all_sync(0xffffffffu, ok && wait(full + st, parity));
    if (!ok) break;
    if (tid < C::BM && i > 0 && filled < n_st) {  // the stage before this one, once all warps have left it
      ok = wait(empty + (st == 0 ? C::STAGES - 1 : st - 1), st == 0 ? parity ^ 1 : parity);
      if (ok) fill(filled++);
    }
    const __half* sc_st = reinterpret_cast<const __half*>(scales + st * C::SC_BYTES) + sc_at;
    const uint8_t* z_st = scales + st * C::SC_BYTES + C::BM * GPS * 2 + sc_at;
    const uint8_t* base = smem + st * C::STAGE;
    const uint32_t base_w = smem_u32(base) + w_at;
    uint32_t z1024[2 * MT], z64[2 * MT];
    float d[MT][NT][4];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (c % CG == 0) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) d[mt][nt][0] = d[mt][nt][1] = d[mt][nt][2] = d[mt][nt][3] = 0.f;
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) {
          if constexpr (ZEROS) {
            z1024[r] = (0x6400u + z_st[8 * r * GPS + c / CG]) * 0x10001u;
            z64[r] = h2_sub(0x63806380u, z1024[r]);  // 960 - (1024 + z)
          } else {
            z1024[r] = 0x64086408u;  // 1032
            z64[r] = 0xd480d480u;    // -72
          }
        }
      }
      uint32_t w[4], h[2 * MT][4];
      ldsm_x4(base_w + (w_swz ^ (c << 4)), w[0], w[1], w[2], w[3]);
#pragma unroll
      for (int r = 0; r < 2 * MT; ++r) codes_less(w[r], z1024[r], z64[r], h[r]);
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
      if ((c + 1) % CG == 0) {
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) {
          const float f = __half2float(sc_st[8 * r * GPS + c / CG]);
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
    st = st + 1 == C::STAGES ? 0 : st + 1;
    parity ^= st == 0 ? 1u : 0u;
  }
  ok = __all_sync(0xffffffffu, ok);
  if (!ok)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[mt][nt][0] = acc[mt][nt][1] = acc[mt][nt][2] = acc[mt][nt][3] = __uint_as_float(0x7fc00000u);
  cp_async_wait_all();
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
  for (int i = tid; i < nb * C::BM; i += C::THREADS) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < C::WK; ++k) sum += part[k * 8 * NT * C::BM + i];
    const int n = n0 + i % C::BM;
    if (parts > 1) joined[i] = sum;
    else if (n < a.N) a.y[(size_t)(b0 + i / C::BM) * a.N + n] = sum;
  }
  if (parts == 1) return;
  cluster_barrier();
  const uint32_t joined_u = smem_u32(joined);
  for (int i = rank * C::THREADS + tid; i < nb * C::BM; i += parts * C::THREADS) {
    float sum = 0.f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) sum += ld_cluster(joined_u + 4 * i, p);
    const int n = n0 + i % C::BM;
    if (n < a.N) a.y[(size_t)(b0 + i / C::BM) * a.N + n] = sum;
  }
  cluster_barrier();  // no CTA leaves while another reads its shared memory
}

// Up to eight batch rows: bound by HBM, so each SM gets one CTA with an even share
// of the 16-row tiles, one pass over the columns and one join at its end. WM warps
// down the rows and WK along the columns, PART columns of each stage a warp. With
// so few rows the instructions that take the codes to the tensor core count: x is
// laid out once in shared memory in the codes' order of pairs (XS), where it has
// room, and read from L1 or L2 otherwise.
struct W4RowsPlan {
  int wm, wk, stages, parts, per;  // parts: CTAs of a cluster that share the columns, `per` stages each
  int ring;                        // bytes of the stages with their scales
};
constexpr int kW4RowsWarps = 16, kW4RowsMoreWarps = 28;
constexpr int kW4RowsSmem = 224 * 1024, kW4RowsHead = 1024;  // barriers, alignment
constexpr int kW4RowsX = 96 * 1024;                          // most of x in shared memory

// D = A * B (no sum goes in)
__device__ __forceinline__ void mma16816_zero(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

template <int PART, int GROUP, bool ZEROS, bool XS, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 1)
    w4_rows_kernel(const W4Args a, const W4RowsPlan p, const __grid_constant__ CUtensorMap wmap) {
  constexpr int SUBS = PART / 128, CG = GROUP / 32, SG = 128 / GROUP;  // runs of 128 columns, chunks of a group, groups of a run
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full[32], empty[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int rows = 16 * p.wm, kc = PART * p.wk, stage_bytes = rows * kc / 2, gps = kc / GROUP;
  const int sc_bytes = rows * gps * (ZEROS ? 3 : 2);  // of a stage: [rows][gps] fp16, [rows][gps] bytes
  uint8_t* scales = smem + p.stages * stage_bytes;
  const int n0 = blockIdx.x / p.parts * rows;
  const int all = (a.K + kc - 1) / kc;
  const int s0 = min(all, int(rank) * p.per), n_st = min(all, s0 + p.per) - s0;
  if (tid < p.stages) {
    mbar_init(full + tid, 1 + rows);
    mbar_init(empty + tid, p.wm * p.wk);
  }
  fence_mbar_init();
  __syncthreads();
  // the first `rows` threads start a stage's copies: thread 0 the codes, each its row's scales
  const int groups = a.K / GROUP;
  int filled = 0;
  auto fill = [&](int st) {
    if (tid == 0) {
      const uint32_t dst = smem_u32(smem + st * stage_bytes);
      mbar_arrive_expect_tx(full + st, stage_bytes);
      for (int j = 0; j < kc / 256; ++j)
        load_2d(dst + j * rows * 128, &wmap, (s0 + filled) * (kc / 2) + j * 128, n0, full + st);
    }
    uint8_t* sc = scales + st * sc_bytes;
    copy_scales<ZEROS>(a, sc + tid * gps * 2, sc + rows * gps * 2 + tid * gps, min(n0 + tid, a.N - 1), groups, (s0 + filled) * gps,
                       gps, full + st);
    ++filled;
  };
  if (tid < rows)
    while (filled < min(p.stages, n_st)) fill(filled);

  const int wm = warp % p.wm, wk = warp / p.wm;
  const int xr = min((g & 1) * 4 + (g >> 1), a.B - 1);  // the batch row that is column g (as above); behind the batch: the last, not stored
  const uint32_t pitch = p.per * kc * 2 + 16;           // of a row of x in shared memory: rows r and r + 4 half the banks apart
  uint8_t* xsm = smem + p.ring;  // (behind the scales)
  if constexpr (XS) {
    const int cols = n_st * kc / 8;
    for (int b = 0; b < a.B; ++b)
      for (int c0 = tid; c0 < cols; c0 += 4 * blockDim.x) {
        uint4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = c0 + u * blockDim.x;
          x[u] = c < cols && s0 * kc + 8 * c < a.K ? *reinterpret_cast<const uint4*>(a.x + (size_t)b * a.K + s0 * kc + 8 * c)
                                                   : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = c0 + u * blockDim.x;
          if (c < cols)
            *reinterpret_cast<uint4*>(xsm + b * pitch + 16 * c) =
                make_uint4(__byte_perm(x[u].x, x[u].z, 0x5410), __byte_perm(x[u].x, x[u].z, 0x7632),
                           __byte_perm(x[u].y, x[u].w, 0x5410), __byte_perm(x[u].y, x[u].w, 0x7632));
        }
      }
  }
  // ldmatrix: row (lane & 15) of the warp's 16, 16-byte chunks c and c + 1 of its part
  const uint32_t w_lane = (wk * PART >> 8) * rows * 128 + (wm * 16 + (lane & 15)) * 128 +
                          ((((lane >> 4) ^ (lane & 7)) << 4) ^ ((wk * PART & 128) >> 1));
  const uint8_t* x_lane = xsm + xr * pitch + wk * PART * 2 + 16 * t;
  const __half* xrow = a.x + (size_t)xr * a.K + 8 * t;
  uint4 xs[XS ? 1 : 4];
  // this lane's weight rows of the CTA's are 16 wm + g + 8 r (behind N: the last one's scales, not stored)
  const int sc_at = (wm * 16 + g) * gps + wk * (PART / GROUP);
  int k = s0 * kc + wk * PART;  // this warp's first column of the stage
  if constexpr (!XS) {
#pragma unroll
    for (int c = 0; c < 4; ++c) xs[c] = k + 32 * c < a.K ? *reinterpret_cast<const uint4*>(xrow + k + 32 * c) : make_uint4(0u, 0u, 0u, 0u);
  }
  if constexpr (XS) __syncthreads();
  bool ok = true;
  int st = 0;
  uint32_t parity = 0;
  float acc[4] = {};
#pragma unroll 1
  for (int i = 0; i < n_st; ++i) {
    ok = __all_sync(0xffffffffu, ok && wait(full + st, parity));
    if (!ok) break;
    if (tid < rows && i > 0 && filled < n_st) {  // the stage before this one, once all warps have left it
      const int before = st == 0 ? p.stages - 1 : st - 1;
      ok = wait(empty + before, st == 0 ? parity ^ 1 : parity);
      if (ok) fill(before);
    }
    const uint32_t w_st = smem_u32(smem) + st * stage_bytes + w_lane;
    const __half* sc_st = reinterpret_cast<const __half*>(scales + st * sc_bytes) + sc_at;
    const uint8_t* z_st = scales + st * sc_bytes + rows * gps * 2 + sc_at;
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
      const uint32_t w_at = PART == 128 ? w_st : (w_st + (sub >> 1) * rows * 128) ^ ((sub & 1) << 6);
      uint32_t z1024[2], z64[2], w[4];
      float d[4], e[4];  // two chains of products
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = sub * SG + c / CG;  // group of the part
        if (c % CG == 0) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (ZEROS) {
              z1024[r] = (0x6400u + z_st[8 * r * gps + j]) * 0x10001u;
              z64[r] = h2_sub(0x63806380u, z1024[r]);  // 960 - (1024 + z)
            } else {
              z1024[r] = 0x64086408u;  // 1032
              z64[r] = 0xd480d480u;    // -72
            }
          }
        }
        if (c % 2 == 0) ldsm_x4(w_at ^ (c << 4), w[0], w[1], w[2], w[3]);
        uint32_t h0[4], h1[4];
        codes_less(w[2 * (c & 1)], z1024[0], z64[0], h0);
        codes_less(w[2 * (c & 1) + 1], z1024[1], z64[1], h1);
        uint4 x;
        if constexpr (XS) {
          x = *reinterpret_cast<const uint4*>(x_lane + sub * 256 + c * 64);
        } else {
          const uint4 y = xs[c];
          x = make_uint4(__byte_perm(y.x, y.z, 0x5410), __byte_perm(y.x, y.z, 0x7632), __byte_perm(y.y, y.w, 0x5410),
                         __byte_perm(y.y, y.w, 0x7632));
        }
        if (c % CG == 0) {
          mma16816_zero(d, h0[0], h1[0], h0[1], h1[1], x.x, x.y);
          mma16816_zero(e, h0[2], h1[2], h0[3], h1[3], x.z, x.w);
        } else {
          mma16816(d, h0[0], h1[0], h0[1], h1[1], x.x, x.y);
          mma16816(e, h0[2], h1[2], h0[3], h1[3], x.z, x.w);
        }
        if constexpr (!XS) {
          const int kn = k + (sub + 1 < SUBS ? 128 * (sub + 1) : kc) + 32 * c;  // the next run's chunk
          xs[c] = kn < a.K ? *reinterpret_cast<const uint4*>(xrow + kn) : make_uint4(0u, 0u, 0u, 0u);
        }
        if ((c + 1) % CG == 0) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float f = __half2float(sc_st[8 * r * gps + j]);
            acc[2 * r] += f * (d[2 * r] + e[2 * r]);
            acc[2 * r + 1] += f * (d[2 * r + 1] + e[2 * r + 1]);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + st);
    k += kc;
    x_lane += 2 * kc;
    st = st + 1 == p.stages ? 0 : st + 1;
    parity ^= st == 0 ? 1u : 0u;
  }
  cp_async_wait_all();
  // after a wait that ran out: outputs are NaN, and no copy may be on its way when the CTA goes on (waits have a limit)
  if (!__syncthreads_and(ok)) {
    acc[0] = acc[1] = acc[2] = acc[3] = __uint_as_float(0x7fc00000u);
    if (tid == 0)
      for (int i = max(0, filled - p.stages); i < filled; ++i) wait(full + i % p.stages, (i / p.stages) & 1);
    __syncthreads();
  }
  // ---- join the warps along the columns, then the cluster's CTAs
  float4* part = reinterpret_cast<float4*>(smem);                              // [wk][wm][lane]
  float* joined = reinterpret_cast<float*>(part + p.wm * p.wk * 32);           // [wm][lane][4]
  part[warp * 32 + lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  auto store = [&](int i, float sum) {  // value e of lane l of row tile i / 128
    const int l = (i >> 2) & 31, e = i & 3;
    const int n = n0 + (i >> 7) * 16 + (l >> 2) + 8 * (e >> 1), b = (l & 3) + 4 * (e & 1);
    if (n < a.N && b < a.B) a.y[(size_t)b * a.N + n] = sum;
  };
  const float* src = reinterpret_cast<const float*>(part);
  for (int i = tid; i < p.wm * 128; i += blockDim.x) {
    float sum = 0.f;
    for (int w = 0; w < p.wk; ++w) sum += src[w * p.wm * 128 + i];
    if (p.parts > 1) joined[i] = sum;
    else store(i, sum);
  }
  if (p.parts == 1) return;
  cluster_barrier();
  const uint32_t joined_u = smem_u32(joined);
  for (int i = rank * blockDim.x + tid; i < p.wm * 128; i += p.parts * blockDim.x) {
    float sum = 0.f;
#pragma unroll 4
    for (int r = 0; r < p.parts; ++r) sum += ld_cluster(joined_u + 4 * i, r);
    store(i, sum);
  }
  cluster_barrier();  // no CTA leaves while another reads its shared memory
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

// codes [N][K / 2] bytes, boxes of 128 bytes x `rows`; x [B][K] fp16, boxes of 64 columns x `rows`; 128-byte swizzle
cudaError_t make_map(CUtensorMap* m, CUtensorMapDataType type, const void* base, int64_t cols, int64_t rows, int64_t pitch,
                     int box_cols, int box_rows) {
  const EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)}, strides[1] = {cuuint64_t(pitch)};
  const cuuint32_t box[2] = {cuuint32_t(box_cols), cuuint32_t(box_rows)}, one[2] = {1, 1};
  const CUresult r = fn(m, type, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int PART, int GROUP, bool ZEROS, bool XS, int WARPS = kW4RowsWarps>
cudaError_t launch_rows_x(const W4Args& a, const W4RowsPlan& p, int ctas, cudaStream_t s) {
  CUtensorMap wmap;
  const cudaError_t e = make_map(&wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.codes, a.K / 2, a.N, a.K / 2, 128, 16 * p.wm);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas * p.parts);
  cfg.blockDim = dim3(32 * p.wm * p.wk);
  cfg.dynamicSmemBytes = kW4RowsSmem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = p.parts > 1 ? 1 : 0;  // (a cluster of one costs a launch some 0.3 us)
  return cudaLaunchKernelEx(&cfg, w4_rows_kernel<PART, GROUP, ZEROS, XS, WARPS>, a, p, wmap);
}

template <int PART, int GROUP, bool ZEROS>
cudaError_t launch_rows(const W4Args& a, int sms, cudaStream_t s) {
  const int tiles = (a.N + 15) / 16, k_parts = (a.K + PART - 1) / PART;
  W4RowsPlan p;
  int ctas = 0;
  bool xs = false;
  auto plan = [&](int warps) {
    // one round of the SMs where sixteen warps' tiles are enough, the other warps along the columns
    p.wm = std::min(PART == 128 ? 8 : 16, (tiles + sms - 1) / sms);
    p.wk = std::max(1, std::min(warps / p.wm, k_parts));
    if (PART == 128) p.wk = std::max(2, p.wk & ~1);  // (boxes of 256 columns)
    ctas = (tiles + p.wm - 1) / p.wm;
    const int all = (k_parts + p.wk - 1) / p.wk;
    p.parts = 1;  // while the SMs are not full, CTAs share the columns
    while (p.parts < 8 && ctas * p.parts * 2 <= sms && all >= 2 * p.parts) p.parts *= 2;
    p.per = (all + p.parts - 1) / p.parts;
    const int64_t x_bytes = (int64_t)a.B * ((int64_t)p.per * PART * p.wk * 2 + 16);
    xs = PART > 128 && x_bytes <= kW4RowsX;
    const int stage = 16 * p.wm * PART * p.wk / 2 + 16 * p.wm * (PART * p.wk / GROUP) * (ZEROS ? 3 : 2);
    p.stages = int(std::min<int64_t>(32, (kW4RowsSmem - kW4RowsHead - (xs ? x_bytes : 0)) / stage));
    p.ring = p.stages * stage;
  };
  plan(kW4RowsWarps);
  if constexpr (PART == 256) {
    // More warps hide the unpacking's latency where x is in shared memory (without it they lack registers) and they divide
    // the columns about as evenly. Microseconds with 16 warps at most and with 28: 16384 x 8192, one row, 22.4 and 19.8; 6144
    // x 4096, one row, 8.2 and 7.7; 12288 x 4096, eight rows, groups of 32 with zero points, 17.5 and 15.9; but 8192 x 8192,
    // one row, 13.4 and 14.9 (32 runs of columns for 4 warps a row tile or 7).
    const int few = (k_parts + p.wk - 1) / p.wk * p.wk, warps = p.wm * p.wk;
    const W4RowsPlan p16 = p;
    const int ctas16 = ctas;
    const bool xs16 = xs;
    plan(kW4RowsMoreWarps);
    const int more = (k_parts + p.wk - 1) / p.wk * p.wk;
    if (xs && p.stages >= 2 && p.wm * p.wk > warps && more * 20 <= few * 21)
      return launch_rows_x<PART, GROUP, ZEROS, true, kW4RowsMoreWarps>(a, p, ctas, s);
    p = p16;
    ctas = ctas16;
    if (xs16) return launch_rows_x<PART, GROUP, ZEROS, true>(a, p, ctas, s);
  }
  return launch_rows_x<PART, GROUP, ZEROS, false>(a, p, ctas, s);
}

template <int NT, int GROUP, bool ZEROS>
cudaError_t launch(const W4Args& a, int sms, cudaStream_t s) {
  if constexpr (NT == 1) {
    return a.K >= 2048 ? launch_rows<256, GROUP, ZEROS>(a, sms, s) : launch_rows<128, GROUP, ZEROS>(a, sms, s);
  } else {
  using C = W4Cfg<NT>;
  CUtensorMap wmap, xmap;
  cudaError_t e = make_map(&wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.codes, a.K / 2, a.N, a.K / 2, 128, C::BM);
  if (e == cudaSuccess)
    e = make_map(&xmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.x, a.K, a.B, (int64_t)a.K * 2, 64, 8 * NT);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (int64_t)((a.N + C::BM - 1) / C::BM) * ((a.B + 8 * NT - 1) / (8 * NT));
  const int stages = (a.K + C::KC - 1) / C::KC;
  int parts = 1;  // CTAs that share the columns: while they find places, and two stages each
  while (parts < 8 && tiles * parts * 2 <= sms && stages >= 4 * parts) parts *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.N + C::BM - 1) / C::BM * parts, (a.B + 8 * NT - 1) / (8 * NT));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, w4_projection_kernel<NT, GROUP, ZEROS>, a, parts, wmap, xmap);
  }
}

template <int NT, int GROUP>
cudaError_t launch_group(const W4Args& a, int sms, cudaStream_t s) {
  return a.zeros ? launch<NT, GROUP, true>(a, sms, s) : launch<NT, GROUP, false>(a, sms, s);
}
template <int NT>
cudaError_t launch_nt(const W4Args& a, int sms, cudaStream_t s) {
  return a.group == 32   ? launch_group<NT, 32>(a, sms, s)
         : a.group == 64 ? launch_group<NT, 64>(a, sms, s)
                         : launch_group<NT, 128>(a, sms, s);
}

template <int NT, int GROUP, bool ZEROS>
cudaError_t attrs_kernel() {
  if constexpr (NT == 1) {
    for (const cudaError_t e : {set_kernel_smem(w4_rows_kernel<128, GROUP, ZEROS, false, kW4RowsWarps>, kW4RowsSmem),
                                set_kernel_smem(w4_rows_kernel<256, GROUP, ZEROS, false, kW4RowsWarps>, kW4RowsSmem),
                                set_kernel_smem(w4_rows_kernel<256, GROUP, ZEROS, true, kW4RowsWarps>, kW4RowsSmem),
                                set_kernel_smem(w4_rows_kernel<256, GROUP, ZEROS, true, kW4RowsMoreWarps>, kW4RowsSmem)})
      if (e != cudaSuccess) return e;
    return cudaSuccess;
  } else {
    return set_kernel_smem(w4_projection_kernel<NT, GROUP, ZEROS>, W4Cfg<NT>::SMEM);
  }
}
template <int NT, int GROUP>
cudaError_t attrs_group() {
  const cudaError_t e = attrs_kernel<NT, GROUP, false>();
  return e != cudaSuccess ? e : attrs_kernel<NT, GROUP, true>();
}
template <int NT>
cudaError_t attrs() {
  for (const cudaError_t e : {attrs_group<NT, 32>(), attrs_group<NT, 64>(), attrs_group<NT, 128>()})
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
