// Append and attention over a paged KV cache in 8 bits.
//
// Cache: e4m3 codes [n_pages][layers][2 (K, V)][nkv][64][hd], rows in plain
// order, and one fp32 scale for each 16 positions of a page, kv head and K or V
// ([n_pages][layers][2][nkv][4]); a value is code * scale. Scales are powers of
// two, the smallest 2^e (e >= -126) with amax <= 448 * 2^e: e4m3 is a floating
// format, so a power of two costs no precision, and when a later position needs
// a larger scale the block's older codes go over to it exactly (but for those
// that become subnormal, which round once more).
#include "common.cuh"
#include "lowbit.h"

#include <algorithm>

namespace mmc {
namespace {

constexpr int kAppendThreads = 128;
constexpr int kAttnWarps = 4;  // warp w reads block w of each page
constexpr int kTileRows = 16;  // (new position, q head) rows of one CTA: the M of m16n8k16
constexpr float kLog2e = 1.4426950408889634f;

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
__device__ __forceinline__ uint8_t to_e4m3(float x) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(0.f), "f"(x));
  return uint8_t(d);
}
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

// ---------------------------------------------------------------- append

// One CTA per row. Its warps take the row's q heads (RMSNorm, rotation, fp16),
// and where the row is the first of this call in its block of 16 positions, the
// block's K and V of each kv head: one warp holds the block's new rows in
// registers, finds their largest magnitude, takes the older codes over to the
// new scale if it grew, and writes the new codes. A block has one owner, so no
// atomics and no order that could change the result.
template <int HD>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const Kv8AppendArgs a) {
  constexpr int HALF = HD / 2;
  constexpr int PP = (HALF + 31) / 32;  // (d, d + HALF) pairs of a lane
  const Kv8Args& c = a.c;
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ int s_seq, s_twice;
  if (tid == 0) {
    s_seq = -1;
    s_twice = 0;
  }
  __syncthreads();
  if (c.row_start == nullptr) {
    if (tid == 0) s_seq = row < c.n_seqs ? row : -1;
  } else {
    for (int i = tid; i < c.n_seqs; i += kAppendThreads)
      if (c.row_start[i] <= row && row < c.row_start[i + 1]) s_seq = i;
  }
  __syncthreads();
  const int seq = s_seq;
  if (seq < 0) return;  // a row behind the last sequence
  const int slot = c.slots[seq];
  if (slot < 0) return;  // an unused sequence
  const int first = c.row_start ? c.row_start[seq] : seq;
  const int last = c.row_start ? c.row_start[seq + 1] : seq + 1;
  if (slot >= c.max_seqs) {
    if (tid == 0) set_error(c.err, kDevBadSlot);
    return;
  }
  if (first < 0 || last > c.rows || last - first > c.max_new) {
    if (tid == 0) set_error(c.err, kDevBadRows);
    return;
  }
  for (int i = tid; i < c.n_seqs; i += kAppendThreads)
    if (i != seq && c.slots[i] == slot && (c.row_start == nullptr || c.row_start[i] < c.row_start[i + 1])) s_twice = 1;
  __syncthreads();
  if (s_twice) {
    if (tid == 0) set_error(c.err, kDevSlotTwice);
    return;
  }
  const int pos0 = c.seq_pos[slot];
  if (pos0 < 0 || (int64_t)pos0 + (last - first) > (int64_t)c.max_pages * kPageTokens) {
    if (tid == 0) set_error(c.err, kDevContextLimit);
    return;
  }
  if (pos0 + (last - first) > a.max_pos) {
    if (tid == 0) set_error(c.err, kDevPositionLimit);
    return;
  }
  const int pos = pos0 + (row - first);
  const int heads = c.nq + 2 * c.nkv;

  // norm and rotation of one head of row r at position p: x[i][0] is element lane + 32 i, x[i][1] its partner
  auto turned = [&](int r, int head, const float* w, int p, float (&x)[PP][2]) {
    const float* src = a.qkv + ((size_t)r * heads + head) * HD;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const int d = lane + 32 * i;
      x[i][0] = d < HALF ? src[d] : 0.f;
      x[i][1] = d < HALF ? src[d + HALF] : 0.f;
      ss += x[i][0] * x[i][0] + x[i][1] * x[i][1];
    }
    float rs = 1.f;
    if (w != nullptr) rs = 1.0f / sqrtf(warp_sum(ss) / float(HD) + a.eps);
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const int d = lane + 32 * i;
      if (d >= HALF) continue;
      const float u = w ? x[i][0] * rs * w[d] : x[i][0], v = w ? x[i][1] * rs * w[d + HALF] : x[i][1];
      const float co = a.rope_cos[(size_t)p * HALF + d], si = a.rope_sin[(size_t)p * HALF + d];
      x[i][0] = u * co - v * si;
      x[i][1] = v * co + u * si;
    }
  };

  for (int h = warp; h < c.nq; h += kAppendThreads / 32) {
    float x[PP][2];
    turned(row, h, a.q_norm, pos, x);
    __half* dst = a.q + ((size_t)row * c.nq + h) * HD;
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const int d = lane + 32 * i;
      if (d < HALF) {
        dst[d] = __float2half_rn(x[i][0]);
        dst[d + HALF] = __float2half_rn(x[i][1]);
      }
    }
  }

  // the first row of this call in its block writes the block
  if (row != first && pos % kKv8Block != 0) return;
  const int page = c.table[(size_t)slot * c.max_pages + pos / kPageTokens];
  if (page < 0 || page >= c.n_pages) {
    if (tid == 0) set_error(c.err, kDevNoPage);
    return;
  }
  const int r0 = pos % kPageTokens, blk = r0 / kKv8Block, older = pos % kKv8Block;
  const int n = min(kKv8Block - older, last - row);
  for (int u = warp; u < 2 * c.nkv; u += kAppendThreads / 32) {
    const int kv = u / c.nkv, h = u % c.nkv;
    const size_t slab = kv8_slab(c, page, kv, h);
    uint8_t* codes = c.codes + slab * (kPageTokens * HD);
    float* scale = c.scales + slab * kKv8BlocksPerPage + blk;
    float x[kKv8Block][PP][2];
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < kKv8Block; ++j) {
      if (j >= n) break;
      if (kv == 0) {
        turned(row + j, c.nq + h, a.k_norm, pos + j, x[j]);
      } else {
        const float* src = a.qkv + ((size_t)(row + j) * heads + c.nq + c.nkv + h) * HD;
#pragma unroll
        for (int i = 0; i < PP; ++i) {
          const int d = lane + 32 * i;
          x[j][i][0] = d < HALF ? src[d] : 0.f;
          x[j][i][1] = d < HALF ? src[d + HALF] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < PP; ++i) amax = max_nan(amax, max_nan(fabsf(x[j][i][0]), fabsf(x[j][i][1])));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float s = pow2_scale(amax);
    const float had = older > 0 ? *scale : 0.f;
    if (older > 0) s = max_nan(s, had);
    if (older > 0 && s > had) {  // (false where s is NaN: a block that is lost keeps its codes)
      for (int e = lane; e < older * HD; e += 32) {
        uint8_t* p = codes + (size_t)(blk * kKv8Block) * HD + e;
        *p = to_e4m3(from_e4m3(*p) * (had / s));
      }
    }
    const bool lost = s != s;
    const float inv = lost ? 0.f : pow2_inverse(s);
#pragma unroll
    for (int j = 0; j < kKv8Block; ++j) {
      if (j >= n) break;
      uint8_t* dst = codes + (size_t)(r0 + j) * HD;
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        const int d = lane + 32 * i;
        if (d < HALF) {
          dst[d] = lost ? 0 : to_e4m3(x[j][i][0] * inv);
          dst[d + HALF] = lost ? 0 : to_e4m3(x[j][i][1] * inv);
        }
      }
    }
    __syncwarp();
    if (lane == 0) *scale = s;
  }
}

// ---------------------------------------------------------------- attention

struct Kv8Seq {
  int slot, first, n, pos0;  // n: rows of the sequence (0: none, or refused)
  bool refused;
};
// The sequence's rows and positions, checked: everything later indexes within them.
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Args& c, int max_ctx, int seq, bool report) {
  Kv8Seq s{-1, 0, 0, 0, false};
  s.first = c.row_start ? c.row_start[seq] : seq;
  const int last = c.row_start ? c.row_start[seq + 1] : seq + 1;
  int e = 0;
  if (s.first < 0 || last > c.rows || last < s.first || last - s.first > c.max_new) {
    e = kDevBadRows;
  } else {
    s.n = last - s.first;
    s.slot = c.slots[seq];
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

template <int HD>
struct Kv8Cfg {
  static constexpr int KC = HD / 16;                          // 16-wide steps of a head
  static constexpr int PITCH = HD == 16 ? 16 : HD + 16;       // odd multiple of 16 bytes: ldmatrix without bank conflicts
  static constexpr int STAGE = 2 * kKv8Block * PITCH + 16;    // K rows, V rows, two scales
  static constexpr int STAGES = 4;
  static constexpr int RING = kAttnWarps * STAGES * STAGE;
  static constexpr int MERGE = kAttnWarps * kTileRows * (HD + 2) * 4;
  static constexpr int SMEM = RING > MERGE ? RING : MERGE;
};

// One CTA: up to 16 rows (new position, q head of the group) of one sequence and
// kv head, over one part of the sequence's pages. Each warp streams its own
// blocks of 16 positions (block w of every page) through a ring of its own, so
// the loop has no CTA barrier: S = Q K^T and O += P V on m16n8k16 with the rows
// on M, running maximum and sum in registers. The four warps' states are joined
// in shared memory in a fixed order; with several parts the joined states go to
// `part` and kv8_merge_kernel joins them, again in order.
template <int HD>
__global__ void __launch_bounds__(kAttnWarps * 32) kv8_attention_kernel(const Kv8AttnArgs a) {
  using C = Kv8Cfg<HD>;
  extern __shared__ __align__(16) uint8_t smem[];
  const Kv8Args& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits, h = blockIdx.y, seq = blockIdx.z;
  const int rep = c.nq / c.nkv;
  const Kv8Seq sq = kv8_seq(c, a.max_ctx, seq, tid == 0);
  const int fr0 = tile * kTileRows, n_fr = min(kTileRows, sq.n * rep - fr0);  // this tile's rows
  if (n_fr <= 0) return;
  if (sq.slot < 0) {  // an unused sequence: its rows attend nothing
    if (split == 0)
      for (int e = tid; e < n_fr * HD; e += kAttnWarps * 32) {
        const int fr = fr0 + e / HD;
        a.out[((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD + e % HD] = __float2half_rn(0.f);
      }
    return;
  }
  // the last position that rows g and g + 8 see, and the tile's pages
  const int fA = fr0 + g, fB = fr0 + g + 8;
  const int limA = sq.pos0 + (g < n_fr ? fA / rep : 0), limB = sq.pos0 + (g + 8 < n_fr ? fB / rep : 0);
  const int lim_lo = sq.pos0 + fr0 / rep, lim_hi = sq.pos0 + (fr0 + n_fr - 1) / rep;
  const int end = sq.pos0 + sq.n;  // positions written
  const int pages = lim_hi / kPageTokens + 1;
  const int per = (pages + a.splits - 1) / a.splits;
  const int p0 = min(pages, split * per), p1 = min(pages, p0 + per);

  uint32_t qf[C::KC][4];  // A fragments: lane (g, t) holds columns 16 c + 4 t .. + 3 of rows g and g + 8
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) {
    uint2 x = make_uint2(0u, 0u), y = x;
    if (g < n_fr)
      x = *reinterpret_cast<const uint2*>(a.q + ((size_t)(sq.first + fA / rep) * c.nq + h * rep + fA % rep) * HD + 16 * kc + 4 * t);
    if (g + 8 < n_fr)
      y = *reinterpret_cast<const uint2*>(a.q + ((size_t)(sq.first + fB / rep) * c.nq + h * rep + fB % rep) * HD + 16 * kc + 4 * t);
    qf[kc][0] = x.x;
    qf[kc][1] = y.x;
    qf[kc][2] = x.y;
    qf[kc][3] = y.y;
  }
  const float sl2 = kLog2e / sqrtf(float(HD));

  uint8_t* ring = smem + (size_t)warp * C::STAGES * C::STAGE;
  const int* row_table = c.table + (size_t)sq.slot * c.max_pages;
  // pages whose block `warp` starts within the tile's positions
  const int n_it = max(0, (p1 < pages ? p1 : (p1 > p0 && (p1 - 1) * kPageTokens + warp * kKv8Block > lim_hi ? p1 - 1 : p1)) - p0);
  int ids = -1;  // page ids of 32 iterations, one a lane
  auto load = [&](int it) {
    if (it % 32 == 0) ids = p0 + it + lane < p1 ? row_table[p0 + it + lane] : -1;
    const int page = __shfl_sync(0xffffffffu, ids, it % 32);
    if (page >= 0 && page < c.n_pages) {
      uint8_t* st = ring + (it % C::STAGES) * C::STAGE;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const size_t slab = kv8_slab(c, page, kv, h);
        const uint8_t* src = c.codes + slab * (kPageTokens * HD) + (size_t)warp * kKv8Block * HD;
#pragma unroll
        for (int i = lane; i < HD; i += 32)
          cp_async16(st + kv * kKv8Block * C::PITCH + (i / C::KC) * C::PITCH + (i % C::KC) * 16, src + i * 16);
        if (lane == kv)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(st + 2 * kKv8Block * C::PITCH + 4 * kv)),
                       "l"(c.scales + slab * kKv8BlocksPerPage + warp)
                       : "memory");
      }
    } else if (lane == 0) {
      set_error(c.err, kDevNoPage);
    }
    return page >= 0 && page < c.n_pages;
  };

  uint32_t have = 0;  // bit s: stage s holds a page
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) {
    if (i < n_it) have |= uint32_t(load(i)) << i;
    cp_async_commit();
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[C::KC][2][4];
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc)
#pragma unroll
    for (int j = 0; j < 8; ++j) o[kc][j / 4][j % 4] = 0.f;

  for (int it = 0; it < n_it; ++it) {
    cp_async_wait<C::STAGES - 2>();
    __syncwarp();
    {
      const int nx = it + C::STAGES - 1, s = nx % C::STAGES;
      have &= ~(1u << s);
      if (nx < n_it) have |= uint32_t(load(nx)) << s;
      cp_async_commit();
    }
    const uint8_t* st = ring + (it % C::STAGES) * C::STAGE;
    const bool ok = (have >> (it % C::STAGES)) & 1;
    if (!ok) continue;  // (uniform in the warp) a page that is missing: reported, left out
    const uint32_t kb = smem_u32(st), vb = kb + kKv8Block * C::PITCH;
    const float* sc2 = reinterpret_cast<const float*>(st + 2 * kKv8Block * C::PITCH);
    const float ks = sc2[0] * sl2, vs = sc2[1];
    const int tok0 = (p0 + it) * kPageTokens + warp * kKv8Block;

    float sc[2][4] = {};
#pragma unroll
    for (int kc = 0; kc < C::KC; kc += 2) {
      // matrices: positions 0-7 | 8-15 of columns 16 kc .., then of 16 (kc + 1) ..
      uint32_t r[4];
      const int mi = lane >> 3, col = kc + (mi >> 1) < C::KC ? kc + (mi >> 1) : kc;
      ldsm_x4(kb + ((mi & 1) * 8 + (lane & 7)) * C::PITCH + col * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (kc + x >= C::KC) break;
#pragma unroll
        for (int n = 0; n < 2; ++n)
          mma16816(sc[n], qf[kc + x][0], qf[kc + x][1], qf[kc + x][2], qf[kc + x][3], e4m3x2_half2(r[2 * x + n]),
                   e4m3x2_half2(r[2 * x + n] >> 16));
      }
    }
    const bool edge = tok0 + kKv8Block - 1 > lim_lo;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[n][e] *= ks;
        if (edge && tok0 + 8 * n + 2 * t + (e & 1) > (e < 2 ? limA : limB)) sc[n][e] = -INFINITY;
      }
    float alpha[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[r], mx);
      const float base = mn == -INFINITY ? 0.f : mn;  // nothing seen yet
      alpha[r] = exp2f(m[r] - base);
      m[r] = mn;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 2 * r; e < 2 * r + 2; ++e) {
          sc[n][e] = exp2f(sc[n][e] - base);
          sum += sc[n][e];
        }
      l[r] = l[r] * alpha[r] + sum;
    }
    const uint32_t pa0 = pack_half2(sc[0][0], sc[0][1]), pa1 = pack_half2(sc[0][2], sc[0][3]);
    const uint32_t pa2 = pack_half2(sc[1][0], sc[1][1]), pa3 = pack_half2(sc[1][2], sc[1][3]);
    // codes behind the last position are whatever the page held: 0 x NaN would spoil the sum
    const int left = end - tok0;
    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
    if (left < kKv8Block) {
      keep0 = (2 * t < left ? 0xffffu : 0u) | (2 * t + 1 < left ? 0xffff0000u : 0u);
      keep1 = (2 * t + 8 < left ? 0xffffu : 0u) | (2 * t + 9 < left ? 0xffff0000u : 0u);
    }
#pragma unroll
    for (int kc = 0; kc < C::KC; kc += 2) {
      uint32_t r[4];
      const int mi = lane >> 3, col = kc + (mi >> 1) < C::KC ? kc + (mi >> 1) : kc;
      ldsm_x4_t(vb + ((mi & 1) * 8 + (lane & 7)) * C::PITCH + col * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (kc + x >= C::KC) break;
        // lane (g, t): columns 2 g, 2 g + 1 of positions 2 t, 2 t + 1 -> the pair of positions of each column
        const uint32_t u0 = __byte_perm(r[2 * x] & keep0, 0, 0x3120), u1 = __byte_perm(r[2 * x + 1] & keep1, 0, 0x3120);
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          float d[4] = {};
          mma16816(d, pa0, pa1, pa2, pa3, e4m3x2_half2(odd ? u0 >> 16 : u0), e4m3x2_half2(odd ? u1 >> 16 : u1));
#pragma unroll
          for (int e = 0; e < 4; ++e) o[kc + x][odd][e] = o[kc + x][odd][e] * alpha[e >> 1] + vs * d[e];
        }
      }
    }
  }
  cp_async_wait<0>();
  // ---- join the warps
  __syncthreads();
  float* wo = reinterpret_cast<float*>(smem);                 // [warp][16][HD]
  float* wml = wo + kAttnWarps * kTileRows * HD;              // [warp][16][2]
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float sum = l[r];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    const int row = warp * kTileRows + g + 8 * r;
    if (t == 0) {
      wml[2 * row] = m[r];
      wml[2 * row + 1] = sum;
    }
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc)
      *reinterpret_cast<float4*>(wo + (size_t)row * HD + 16 * kc + 4 * t) =
          make_float4(o[kc][0][2 * r], o[kc][1][2 * r], o[kc][0][2 * r + 1], o[kc][1][2 * r + 1]);
  }
  __syncthreads();
  const int tile_rows = min(kTileRows, c.max_new * rep);
  const int tiles = (c.max_new * rep + kTileRows - 1) / kTileRows;
  for (int e = tid; e < n_fr * HD; e += kAttnWarps * 32) {
    const int r = e / HD, d = e % HD;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) mx = fmaxf(mx, wml[2 * (w * kTileRows + r)]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, val = 0.f;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      const float f = exp2f(wml[2 * (w * kTileRows + r)] - base);
      sum += f * wml[2 * (w * kTileRows + r) + 1];
      val += f * wo[(size_t)(w * kTileRows + r) * HD + d];
    }
    if (a.splits == 1) {
      const int fr = fr0 + r;
      a.out[((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD + d] =
          __float2half_rn(sum > 0.f || sum != sum ? val / sum : 0.f);
    } else {
      float* p = a.part + ((((size_t)seq * tiles + tile) * c.nkv + h) * a.splits + split) * tile_rows * (HD + 2);
      p[(size_t)r * HD + d] = val;
      if (d == 0) {
        p[(size_t)tile_rows * HD + 2 * r] = mx;
        p[(size_t)tile_rows * HD + 2 * r + 1] = sum;
      }
    }
  }
}

// Joins the parts' states of one tile: one CTA per (tile, kv head, sequence).
template <int HD>
__global__ void __launch_bounds__(128) kv8_merge_kernel(const Kv8AttnArgs a) {
  const Kv8Args& c = a.c;
  const int tile = blockIdx.x, h = blockIdx.y, seq = blockIdx.z, rep = c.nq / c.nkv;
  const Kv8Seq sq = kv8_seq(c, a.max_ctx, seq, false);
  const int fr0 = tile * kTileRows, n_fr = min(kTileRows, sq.n * rep - fr0);
  if (n_fr <= 0 || sq.slot < 0) return;
  const int tile_rows = min(kTileRows, c.max_new * rep);
  const float* base_p = a.part + (((size_t)seq * gridDim.x + tile) * c.nkv + h) * a.splits * tile_rows * (HD + 2);
  const size_t stride = (size_t)tile_rows * (HD + 2);
  for (int e = threadIdx.x; e < n_fr * HD; e += 128) {
    const int r = e / HD, d = e % HD;
    float mx = -INFINITY;
    for (int s = 0; s < a.splits; ++s) mx = fmaxf(mx, base_p[s * stride + (size_t)tile_rows * HD + 2 * r]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, val = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      const float f = exp2f(base_p[s * stride + (size_t)tile_rows * HD + 2 * r] - base);
      sum += f * base_p[s * stride + (size_t)tile_rows * HD + 2 * r + 1];
      val += f * base_p[s * stride + (size_t)r * HD + d];
    }
    const int fr = fr0 + r;
    a.out[((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD + d] =
        __float2half_rn(sum > 0.f || sum != sum ? val / sum : 0.f);
  }
}

int tiles_of(int max_new, int nq, int nkv) { return (max_new * (nq / nkv) + kTileRows - 1) / kTileRows; }

template <int HD>
cudaError_t attention_hd(const Kv8AttnArgs& a, cudaStream_t s) {
  const int tiles = tiles_of(a.c.max_new, a.c.nq, a.c.nkv);
  kv8_attention_kernel<HD><<<dim3(tiles * a.splits, a.c.nkv, a.c.n_seqs), kAttnWarps * 32, Kv8Cfg<HD>::SMEM, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && a.splits > 1) {
    kv8_merge_kernel<HD><<<dim3(tiles, a.c.nkv, a.c.n_seqs), 128, 0, s>>>(a);
    e = cudaGetLastError();
  }
  return e;
}

template <int HD>
cudaError_t append_hd(const Kv8AppendArgs& a, cudaStream_t s) {
  kv8_append_kernel<HD><<<a.c.rows, kAppendThreads, 0, s>>>(a);
  return cudaGetLastError();
}

template <int HD>
cudaError_t attr_hd() {
  return set_kernel_smem(kv8_attention_kernel<HD>, Kv8Cfg<HD>::SMEM);
}

}  // namespace

int kv8_plan_splits(int n_seqs, int max_new, int nq, int nkv, int max_ctx, int sms) {
  const int64_t items = (int64_t)n_seqs * nkv * tiles_of(max_new, nq, nkv);
  const int64_t pages = (max_ctx + kPageTokens - 1) / kPageTokens;
  const int64_t want = (4 * (int64_t)sms + items - 1) / items;
  return int(std::max<int64_t>(1, std::min<int64_t>(want, (pages + 3) / 4)));
}

size_t kv8_part_floats(int n_seqs, int max_new, int nq, int nkv, int hd, int splits) {
  if (splits <= 1) return 0;
  const int rep = nq / nkv;
  const size_t tile_rows = size_t(std::min<int64_t>(kTileRows, (int64_t)max_new * rep));
  return (size_t)n_seqs * tiles_of(max_new, nq, nkv) * nkv * splits * tile_rows * (hd + 2);
}

#define MMC_BY_HD(fn, ...)                                                                                          \
  (hd == 16 ? fn<16>(__VA_ARGS__) : hd == 32 ? fn<32>(__VA_ARGS__) : hd == 64 ? fn<64>(__VA_ARGS__)                 \
   : hd == 96 ? fn<96>(__VA_ARGS__) : hd == 128 ? fn<128>(__VA_ARGS__) : cudaErrorInvalidValue)

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, int hd, cudaStream_t s) { return MMC_BY_HD(append_hd, a, s); }
cudaError_t launch_kv8_attention(const Kv8AttnArgs& a, int hd, cudaStream_t s) {
  return MMC_BY_HD(attention_hd, a, s);
}
cudaError_t kv8_init_attributes() {
  for (int hd : {16, 32, 64, 96, 128}) {
    const cudaError_t e = MMC_BY_HD(attr_hd);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace mmc
