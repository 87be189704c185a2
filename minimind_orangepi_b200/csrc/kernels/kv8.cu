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

constexpr int kAppendThreads = 256;
constexpr int kAttnWarps = 4;  // warp w reads block w of each page
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

// ---------------------------------------------------------------- append

// One CTA per window of `window` rows. A head's row is held by hd / 8 lanes, four
// elements of each half a lane, so that a lane has both ends of its rotations and
// loads and stores are 16, 8 (fp16 q) and 4 (codes) bytes wide. The q heads
// (RMSNorm, rotation, fp16) are dealt to the warps. Then, for each row that is the
// first of this call in its block of 16 positions, the CTA takes the whole block,
// four of its K and V heads at a time: the new rows stay in registers while their
// largest magnitudes go through shared memory, older codes go over to the new
// scale if it grew, and the new codes are written. With at most kStepRows rows a
// sequence (STEP) a window is one row and each K or V head one warp's, without
// barriers. A block has one owner, so no atomics on the cache and no order that
// could change the result.
//   Bound by HBM with many rows (the raw projections are four times the bytes of
// all that is written); with few, by the chain of loads slot -> position -> page
// -> old scale, so the projections are loaded before it.
constexpr int kWindow = 8, kStepRows = 8;

template <int HD, bool STEP>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const Kv8AppendArgs a) {
  constexpr int window = STEP ? 1 : kWindow;
  constexpr int HALF = HD / 2, LPH = HD / 8;                                    // lanes of a head's row
  constexpr int GL = LPH <= 2 ? 2 : LPH <= 4 ? 4 : LPH <= 8 ? 8 : 16;           // lanes of a group
  constexpr int HPW = 32 / GL, BATCH = STEP ? 1 : 4;                                    // heads of a warp at once, and of a unit
  constexpr int WARPS = kAppendThreads / 32;
  const Kv8Args& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane / GL, gl = lane % GL;
  const bool in = gl < LPH;
  const int d0 = 4 * (in ? gl : 0);
  const int row0 = blockIdx.x * window, nrows = min(window, c.rows - row0);
  const int heads = c.nq + 2 * c.nkv;
  __shared__ int s_seq[kWindow], s_slot[kWindow], s_first[kWindow], s_last[kWindow], s_twice[kWindow];
  __shared__ int s_pos[kWindow];   // position, -1: not of any sequence, unused or refused
  __shared__ int s_lead[kWindow];  // rows that own a block
  __shared__ int s_leads;

  struct Row8 {
    float4 lo, hi;  // elements d0 .. + 3 of the first and of the second half
  };
  auto load = [&](int row, int head) {
    Row8 x{make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    if (in) {
      const float* src = a.qkv + ((size_t)row * heads + head) * HD + d0;
      x.lo = *reinterpret_cast<const float4*>(src);
      x.hi = *reinterpret_cast<const float4*>(src + HALF);
    }
    return x;
  };
  // the q units of a window: BATCH * HPW heads of a row; the first is loaded ahead of everything else
  const int per_row = (c.nq + BATCH * HPW - 1) / (BATCH * HPW), q_units = nrows * per_row;
  Row8 x[BATCH];
  auto load_unit = [&](int u) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b)
      x[b] = load(row0 + u / per_row, min((u % per_row * BATCH + b) * HPW + grp, c.nq - 1));
  };
  if (warp < q_units) load_unit(warp);
  // STEP: K and V heads, one a warp, from the last warp on
  constexpr int ITS = (kStepRows + HPW - 1) / HPW;
  Row8 v[STEP ? ITS : 1];
  const int kv_first = WARPS - 1 - warp;
  if constexpr (STEP) {
    if (c.max_new == 1 && kv_first < 2 * c.nkv) v[0] = load(row0, c.nq + kv_first);
  }

  // ---- which sequence each row of the window belongs to, and whether its slot appears twice
  if (tid < window) {
    s_seq[tid] = -1;
    s_slot[tid] = -1;
    s_twice[tid] = 0;
  }
  if (tid == 0) s_leads = 0;
  __syncthreads();
  int my_slot = -1;  // of sequence tid (the first round of the loop)
  bool my_rows = false;
  for (int i = tid; i < c.n_seqs; i += kAppendThreads) {
    const int b = c.row_start ? c.row_start[i] : i, e = c.row_start ? c.row_start[i + 1] : i + 1, slot = c.slots[i];
    if (i == tid) {
      my_slot = slot;
      my_rows = b < e;
    }
    for (int r = max(b, row0); r < min(e, row0 + nrows); ++r) {
      s_seq[r - row0] = i;
      s_slot[r - row0] = slot;
      s_first[r - row0] = b;
      s_last[r - row0] = e;
    }
  }
  __syncthreads();
  for (int i = tid; i < c.n_seqs; i += kAppendThreads) {
    const int slot = i == tid ? my_slot : c.slots[i];
    if (slot < 0) continue;
    for (int r = 0; r < nrows; ++r)
      if (s_slot[r] == slot && s_seq[r] != i && (i == tid ? my_rows : c.row_start == nullptr || c.row_start[i] < c.row_start[i + 1]))
        s_twice[r] = 1;
  }
  int pos0 = 0;
  const int slot = tid < nrows ? s_slot[tid] : -1;
  if (slot >= 0 && slot < c.max_seqs) pos0 = c.seq_pos[slot];
  __syncthreads();
  if (tid < nrows) {
    int pos = -1, e = 0;
    if (s_seq[tid] >= 0 && slot >= 0) {
      const int first = s_first[tid], last = s_last[tid];
      if (slot >= c.max_seqs) e = kDevBadSlot;
      else if (first < 0 || last > c.rows || last - first > c.max_new) e = kDevBadRows;
      else if (s_twice[tid]) e = kDevSlotTwice;
      else if (pos0 < 0 || (int64_t)pos0 + (last - first) > (int64_t)c.max_pages * kPageTokens) e = kDevContextLimit;
      else if (pos0 + (last - first) > a.max_pos) e = kDevPositionLimit;
      else pos = pos0 + (row0 + tid - first);
      if (e != 0) set_error(c.err, e);
    }
    s_pos[tid] = pos;
    // the first row of this call in its block writes the block
    if (pos >= 0 && (row0 + tid == s_first[tid] || pos % kKv8Block == 0)) s_lead[atomicAdd(&s_leads, 1)] = tid;
  }
  __syncthreads();

  auto weights = [&](const float* w) {  // of a norm
    Row8 v{};
    if (w != nullptr) {
      v.lo = *reinterpret_cast<const float4*>(w + d0);
      v.hi = *reinterpret_cast<const float4*>(w + d0 + HALF);
    }
    return v;
  };
  auto angles = [&](int p) {  // cosines, sines
    return Row8{*reinterpret_cast<const float4*>(a.rope_cos + (size_t)p * HALF + d0),
                *reinterpret_cast<const float4*>(a.rope_sin + (size_t)p * HALF + d0)};
  };
  auto norm = [&](Row8& v, const Row8& w) {
    float ss = v.lo.x * v.lo.x + v.lo.y * v.lo.y + v.lo.z * v.lo.z + v.lo.w * v.lo.w + v.hi.x * v.hi.x + v.hi.y * v.hi.y +
               v.hi.z * v.hi.z + v.hi.w * v.hi.w;
#pragma unroll
    for (int o = GL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float rs = 1.0f / sqrtf(ss / float(HD) + a.eps);
    v.lo = make_float4(v.lo.x * rs * w.lo.x, v.lo.y * rs * w.lo.y, v.lo.z * rs * w.lo.z, v.lo.w * rs * w.lo.w);
    v.hi = make_float4(v.hi.x * rs * w.hi.x, v.hi.y * rs * w.hi.y, v.hi.z * rs * w.hi.z, v.hi.w * rs * w.hi.w);
  };
  auto turn = [&](Row8& v, const Row8& cs) {
    const Row8 u = v;
    v.lo = make_float4(u.lo.x * cs.lo.x - u.hi.x * cs.hi.x, u.lo.y * cs.lo.y - u.hi.y * cs.hi.y,
                       u.lo.z * cs.lo.z - u.hi.z * cs.hi.z, u.lo.w * cs.lo.w - u.hi.w * cs.hi.w);
    v.hi = make_float4(u.hi.x * cs.lo.x + u.lo.x * cs.hi.x, u.hi.y * cs.lo.y + u.lo.y * cs.hi.y,
                       u.hi.z * cs.lo.z + u.lo.z * cs.hi.z, u.hi.w * cs.lo.w + u.lo.w * cs.hi.w);
  };

  {
    const Row8 w = weights(a.q_norm);
    for (int u = warp; u < q_units; u += WARPS) {
      if (u != warp) load_unit(u);
      const int r = u / per_row, pos = s_pos[r];
      if (pos < 0) continue;  // (uniform in the warp)
      const Row8 cs = angles(pos);
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int h = (u % per_row * BATCH + b) * HPW + grp;
        if (a.q_norm != nullptr) norm(x[b], w);
        turn(x[b], cs);
        if (in && h < c.nq) {
          __half* dst = a.q + ((size_t)(row0 + r) * c.nq + h) * HD + d0;
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack_half2(x[b].lo.x, x[b].lo.y), pack_half2(x[b].lo.z, x[b].lo.w));
          *reinterpret_cast<uint2*>(dst + HALF) =
              make_uint2(pack_half2(x[b].hi.x, x[b].hi.y), pack_half2(x[b].hi.z, x[b].hi.w));
        }
      }
    }
  }

  const int leads = s_leads;
  // a block's codes: older ones over to a larger scale, by `threads` threads; four new ones
  auto regrow = [&](uint8_t* block, int older, float f, int thread, int threads) {
    for (int e = thread; e < older * HD / 4; e += threads) {
      uint32_t* p = reinterpret_cast<uint32_t*>(block) + e;
      const uint32_t was = *p;
      uint32_t now = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) now |= uint32_t(to_e4m3(from_e4m3(uint8_t(was >> 8 * k)) * f)) << 8 * k;
      *p = now;
    }
  };
  auto four = [&](const float4& f, float inv) {
    return uint32_t(to_e4m3x2(f.x * inv, f.y * inv)) | uint32_t(to_e4m3x2(f.z * inv, f.w * inv)) << 16;
  };
  auto largest = [&](const Row8& f) {
    const float lo = max_nan(max_nan(fabsf(f.lo.x), fabsf(f.lo.y)), max_nan(fabsf(f.lo.z), fabsf(f.lo.w)));
    const float hi = max_nan(max_nan(fabsf(f.hi.x), fabsf(f.hi.y)), max_nan(fabsf(f.hi.z), fabsf(f.hi.w)));
    return max_nan(lo, hi);
  };
  if constexpr (STEP) {
    if (leads == 0) return;
    const int pos = s_pos[0], r0 = pos % kPageTokens, blk = r0 / kKv8Block;
    const int older = row0 == s_first[0] ? pos % kKv8Block : 0, n = min(kKv8Block - older, s_last[0] - row0);
    const int page = c.table[(size_t)s_slot[0] * c.max_pages + pos / kPageTokens];
    const Row8 w = weights(a.k_norm);
    for (int u = kv_first; u < 2 * c.nkv; u += WARPS) {
      if (c.max_new > 1 || u != kv_first) {
#pragma unroll
        for (int i = 0; i < ITS; ++i)
          if (i * HPW < n) v[i] = load(row0 + min(i * HPW + grp, n - 1), c.nq + u);
      }
      if (page < 0 || page >= c.n_pages) {
        if (lane == 0) set_error(c.err, kDevNoPage);
        break;
      }
      const size_t slab = kv8_slab(c, page, u / c.nkv, u % c.nkv);
      uint8_t* codes = c.codes + slab * (kPageTokens * HD);
      float* scale = c.scales + slab * kKv8BlocksPerPage + blk;
      const float had = older > 0 ? *scale : 0.f;
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < ITS; ++i) {
        if (i * HPW >= n) break;
        if (u < c.nkv) {
          if (a.k_norm != nullptr) norm(v[i], w);
          turn(v[i], angles(pos + min(i * HPW + grp, n - 1)));
        }
        if (in) amax = max_nan(amax, largest(v[i]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      float s = pow2_scale(amax);
      if (older > 0) s = max_nan(s, had);
      if (older > 0 && s > had)  // (false where s is NaN: a block that is lost keeps its codes)
        regrow(codes + blk * kKv8Block * HD, older, had / s, lane, 32);
      const bool lost = s != s;
      const float inv = lost ? 0.f : pow2_inverse(s);
#pragma unroll
      for (int i = 0; i < ITS; ++i) {
        const int j = i * HPW + grp;
        if (j < n && in) {
          uint8_t* dst = codes + (size_t)(r0 + j) * HD + d0;
          *reinterpret_cast<uint32_t*>(dst) = lost ? 0u : four(v[i].lo, inv);
          *reinterpret_cast<uint32_t*>(dst + HALF) = lost ? 0u : four(v[i].hi, inv);
        }
      }
      __syncwarp();
      if (lane == 0) *scale = s;
    }
    return;
  }
  __shared__ float s_amax[2][BATCH][WARPS];
  int turns = 0;  // of the two buffers of s_amax
  for (int li = 0; li < leads; ++li) {
    const int lead = s_lead[li], row = row0 + lead, pos = s_pos[lead];
    const int r0 = pos % kPageTokens, blk = r0 / kKv8Block, older = row == s_first[lead] ? pos % kKv8Block : 0;
    const int n = min(kKv8Block - older, s_last[lead] - row);
    const int page = c.table[(size_t)s_slot[lead] * c.max_pages + pos / kPageTokens];
    const int j = warp * HPW + grp;  // this group's row of the new ones
    const bool mine = in && j < n;
    const Row8 w = weights(a.k_norm), cs = angles(pos + min(j, n - 1));
    if (page < 0 || page >= c.n_pages) {  // (uniform in the CTA)
      if (tid == 0) set_error(c.err, kDevNoPage);
      continue;
    }
    for (int u0 = 0; u0 < 2 * c.nkv; u0 += BATCH, turns ^= 1) {  // units: K of each kv head, then V
      Row8 v[BATCH];
      float had[BATCH];
      const int m = min(BATCH, 2 * c.nkv - u0);
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int u = u0 + min(b, m - 1);
        v[b] = load(row + min(j, n - 1), c.nq + u);
        had[b] = older > 0 ? c.scales[kv8_slab(c, page, u / c.nkv, u % c.nkv) * kKv8BlocksPerPage + blk] : 0.f;
      }
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        if (u0 + b < c.nkv) {
          if (a.k_norm != nullptr) norm(v[b], w);
          turn(v[b], cs);
        }
        float amax = mine ? largest(v[b]) : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (lane == 0) s_amax[turns][b][warp] = amax;
      }
      __syncthreads();  // (every thread has read the old scales, too)
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        if (b >= m) break;
        const int u = u0 + b;
        const size_t slab = kv8_slab(c, page, u / c.nkv, u % c.nkv);
        uint8_t* codes = c.codes + slab * (kPageTokens * HD);
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) amax = max_nan(amax, s_amax[turns][b][k]);
        float s = pow2_scale(amax);
        if (older > 0) s = max_nan(s, had[b]);
        if (older > 0 && s > had[b])  // (false where s is NaN: a block that is lost keeps its codes)
          regrow(codes + blk * kKv8Block * HD, older, had[b] / s, tid, kAppendThreads);
        const bool lost = s != s;
        const float inv = lost ? 0.f : pow2_inverse(s);
        if (mine) {
          uint8_t* dst = codes + (size_t)(r0 + j) * HD + d0;
          *reinterpret_cast<uint32_t*>(dst) = lost ? 0u : four(v[b].lo, inv);
          *reinterpret_cast<uint32_t*>(dst + HALF) = lost ? 0u : four(v[b].hi, inv);
        }
        if (tid == b) c.scales[slab * kKv8BlocksPerPage + blk] = s;
      }
    }
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
  static constexpr int STAGES = 3;
  static constexpr int RING = kAttnWarps * STAGES * STAGE;
  static constexpr int smem(int rows) {
    const int merge = kAttnWarps * rows * (HD + 2) * 4;
    return RING > merge ? RING : merge;
  }
};

// CTAs of an SM that the registers are bounded for
constexpr int kv8_ctas(int hd, int nt) { return nt == 1 ? (hd <= 96 ? 5 : 4) : nt == 2 ? 3 : 2; }

constexpr float kNoScore = -3.0e38f;  // the running maximum of a row that has seen nothing

__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  const __half2 d = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One CTA: up to 8 NT rows (new position, q head of the group) of one sequence
// and kv head, over one part of `split_pages` pages. Each warp streams its own
// blocks of 16 positions (block w of every page) through a ring of its own, so
// the loop has no CTA barrier. On m16n8k16 the 16 positions are M and the rows
// are N: S^T = K Q^T and O^T += V^T P^T, so K and V are taken from e4m3 to fp16
// (exact) once for all rows, and a group of up to 8 q heads fills N.
//   Softmax: p = 2^(s - m), where m follows the largest score only when one
// exceeds it by more than 8 (p stays below 2^8, far within fp16, at the same
// relative precision), so most blocks need one vote and no reduction; the sums
// stay in each lane until the end.
//   V's scales are powers of two: with vref the largest so far, p * (scale /
// vref) is exact in fp16 down to scale = vref / 64, and O stays in units of
// vref. A block whose scale lies further off takes a second accumulator.
// The four warps' states are joined in shared memory in a fixed order; with
// several parts the joined states go to `part` and kv8_merge_kernel joins them,
// again in order.
template <int HD, int NT>
__global__ void __launch_bounds__(kAttnWarps * 32, kv8_ctas(HD, NT)) kv8_attention_kernel(const Kv8AttnArgs a) {
  using C = Kv8Cfg<HD>;
  constexpr int ROWS = 8 * NT;
  constexpr int CH = (HD + 31) / 32;  // 16-byte chunks a lane copies of a block's K, and of its V
  extern __shared__ __align__(16) uint8_t smem[];
  const Kv8Args& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  // later tiles of a sequence see more positions: first
  const int split = blockIdx.x % a.splits, tile = gridDim.x / a.splits - 1 - blockIdx.x / a.splits;
  const int h = blockIdx.y, seq = blockIdx.z;
  const int rep = c.nq / c.nkv;
  const int p0 = split * a.split_pages;
  // the first page ids need only the slot: with the sequence's position, not after it
  const int slot = c.slots[seq];
  const int* row_table = c.table + (size_t)(slot >= 0 && slot < c.max_seqs ? slot : 0) * c.max_pages;
  int ids = p0 + lane < c.max_pages ? row_table[p0 + lane] : -1;  // page ids of 32 iterations, one a lane
  const Kv8Seq sq = kv8_seq(c, a.max_ctx, seq, tid == 0);
  const int fr0 = tile * ROWS, n_fr = min(ROWS, sq.n * rep - fr0);  // this tile's rows
  if (n_fr <= 0) return;
  if (sq.slot < 0) {  // an unused sequence: its rows attend nothing
    if (split == 0)
      for (int e = tid; e < n_fr * HD; e += kAttnWarps * 32) {
        const int fr = fr0 + e / HD;
        a.out[((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD + e % HD] = __float2half_rn(0.f);
      }
    return;
  }
  const int lim_lo = sq.pos0 + fr0 / rep, lim_hi = sq.pos0 + (fr0 + n_fr - 1) / rep;  // last positions seen
  const int end = sq.pos0 + sq.n;                                                     // positions written
  const int pages = lim_hi / kPageTokens + 1;
  if (p0 >= pages) return;
  const int p1 = min(pages, p0 + a.split_pages);
  // pages whose block `warp` starts within the tile's positions
  const int n_it = p1 - p0 - ((p1 - 1) * kPageTokens + warp * kKv8Block > lim_hi ? 1 : 0);

  uint8_t* ring = smem + (size_t)warp * C::STAGES * C::STAGE;
  const uint32_t ring_u = smem_u32(ring);
  uint32_t dst[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) dst[i] = ring_u + ((lane + 32 * i) / C::KC) * C::PITCH + ((lane + 32 * i) % C::KC) * 16;
  const size_t page_slabs = (size_t)c.layers * 2 * c.nkv;
  const size_t my_slab = (size_t)c.layer * 2 * c.nkv + h;  // K; V is nkv further
  const uint8_t* src0 = c.codes + my_slab * (kPageTokens * HD) + warp * kKv8Block * HD + lane * 16;
  const float* sc0 = c.scales + (my_slab + (lane & 1) * c.nkv) * kKv8BlocksPerPage + warp;
  const size_t v_off = (size_t)c.nkv * kPageTokens * HD;
  auto load = [&](int it, int stage) {
    if (it != 0 && it % 32 == 0) ids = p0 + it + lane < p1 ? row_table[p0 + it + lane] : -1;
    const int page = __shfl_sync(0xffffffffu, ids, it & 31);
    const bool ok = unsigned(page) < unsigned(c.n_pages);
    if (ok) {
      const uint8_t* src = src0 + page * (page_slabs * (kPageTokens * HD));
      const uint32_t st = stage * C::STAGE;
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (HD % 32 == 0 || lane + 32 * i < HD) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst[i] + st), "l"(src + 512 * i) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst[i] + st + kKv8Block * C::PITCH),
                       "l"(src + v_off + 512 * i)
                       : "memory");
        }
      if (lane < 2)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(ring_u + st + 2 * kKv8Block * C::PITCH + 4 * lane),
                     "l"(sc0 + page * (page_slabs * kKv8BlocksPerPage))
                     : "memory");
    } else if (lane == 0) {
      set_error(c.err, kDevNoPage);
    }
    return ok;
  };

  uint32_t have = 0;  // bit s: stage s holds a page
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) {
    if (i < n_it) have |= uint32_t(load(i, i)) << i;
    cp_async_commit();
  }

  uint32_t qf[NT][C::KC][2];  // B fragments: lane (g, t) holds columns 16 kc + 4 t .. + 3 of row g
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int fr = fr0 + nt * 8 + g;
    const bool in = nt * 8 + g < n_fr;
    const __half* src = a.q + ((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD + 4 * t;
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) {
      uint2 x = make_uint2(0u, 0u);
      if (in) x = *reinterpret_cast<const uint2*>(src + 16 * kc);
      qf[nt][kc][0] = x.x;
      qf[nt][kc][1] = x.y;
    }
  }
  const float sl2 = kLog2e / sqrtf(float(HD));

  // lane (g, t): rows 2 t and 2 t + 1 of each n-tile, positions g and g + 8 of the block
  float m[NT][2], l[NT][2], o[NT][C::KC][4];
  int eref = 0;  // exponent field of vref; 0: no block yet
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = kNoScore;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) o[nt][kc][0] = o[nt][kc][1] = o[nt][kc][2] = o[nt][kc][3] = 0.f;
  }
  const int mat = lane >> 3;
  const uint32_t lds = ring_u + ((mat & 1) * 8 + (lane & 7)) * C::PITCH + (C::KC > 1 ? (mat >> 1) * 16 : 0);

  int stage = 0, fill = C::STAGES - 1;
  for (int it = 0; it < n_it; ++it) {
    cp_async_wait<C::STAGES - 2>();
    __syncwarp();
    have &= ~(1u << fill);
    if (it + C::STAGES - 1 < n_it) have |= uint32_t(load(it + C::STAGES - 1, fill)) << fill;
    cp_async_commit();
    const int st = stage;
    fill = stage;
    stage = stage + 1 == C::STAGES ? 0 : stage + 1;
    if (!((have >> st) & 1)) continue;  // (uniform in the warp) a page that is missing: reported, left out
    const uint32_t kb = lds + st * C::STAGE, vb = kb + kKv8Block * C::PITCH;
    const float* sc2 = reinterpret_cast<const float*>(ring + st * C::STAGE + 2 * kKv8Block * C::PITCH);
    const float ks = sc2[0] * sl2, vs = sc2[1];
    const int tok0 = (p0 + it) * kPageTokens + warp * kKv8Block;
    if (end - tok0 < kKv8Block) {
      // codes behind the last position are whatever the page held: 0 x NaN would spoil the sum
      uint8_t* v = ring + st * C::STAGE + (kKv8Block + end - tok0) * C::PITCH;
      for (int i = lane; i < (kKv8Block - (end - tok0)) * (C::PITCH / 16); i += 32)
        *reinterpret_cast<uint4*>(v + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
    }

    float s[NT][4], s2[NT][4];  // two chains of sums
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
#pragma unroll
    for (int kc = 0; kc < C::KC; kc += 2) {
      // matrices: positions 0-7 | 8-15 of columns 16 kc .., then of 16 (kc + 1) ..
      uint32_t r[4];
      ldsm_x4(kb + kc * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (kc + x >= C::KC) break;
        const uint32_t a0 = e4m3x2_half2(r[2 * x]), a2 = e4m3x2_half2(r[2 * x] >> 16);
        const uint32_t a1 = e4m3x2_half2(r[2 * x + 1]), a3 = e4m3x2_half2(r[2 * x + 1] >> 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816(x == 0 ? s[nt] : s2[nt], a0, a1, a2, a3, qf[nt][kc + x][0], qf[nt][kc + x][1]);
      }
    }
    bool above = false;
    const bool edge = tok0 + kKv8Block - 1 > lim_lo;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = (s[nt][e] + s2[nt][e]) * ks;
      if (edge) {
        // (a position that is not seen has no score, whatever its codes and scale are)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int seen = sq.pos0 + (fr0 + min(nt * 8 + 2 * t + r, n_fr - 1)) / rep - tok0 - g;
          if (seen < 0) s[nt][r] = -INFINITY;
          if (seen < 8) s[nt][2 + r] = -INFINITY;
        }
      }
      above |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] + 8.f || fmaxf(s[nt][1], s[nt][3]) > m[nt][1] + 8.f;
    }
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float mx = fmaxf(s[nt][r], s[nt][2 + r]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          mx = fmaxf(mx, m[nt][r]);  // (the same in the row's eight lanes)
          const float f = ex2(m[nt][r] - mx);
          m[nt][r] = mx;
          l[nt][r] *= f;
#pragma unroll
          for (int kc = 0; kc < C::KC; ++kc) {
            o[nt][kc][r] *= f;
            o[nt][kc][2 + r] *= f;
          }
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[nt][e] = ex2(s[nt][e] - m[nt][e & 1]);
        l[nt][e & 1] += s[nt][e];
      }
      pb[nt][0] = movmatrix_t(pack_half2(s[nt][0], s[nt][1]));
      pb[nt][1] = movmatrix_t(pack_half2(s[nt][2], s[nt][3]));
    }
    // exponents: 1 .. 247; 255 where the block is lost (NaN)
    const int ev = __float_as_uint(vs) >> 23 & 255;
    bool far = false;
    if (ev != eref) {
      if (eref == 0 && ev != 255) {
        eref = ev;
      } else if (ev > eref && ev - eref <= 20) {
        const float f = __uint_as_float(uint32_t(127 + eref - ev) << 23);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int kc = 0; kc < C::KC; ++kc)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][kc][e] *= f;
        eref = ev;
      } else if (ev < eref && eref - ev <= 6) {
        const uint32_t f = uint32_t(15 + ev - eref) * 0x04000400u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pb[nt][0] = h2_mul(pb[nt][0], f);
          pb[nt][1] = h2_mul(pb[nt][1], f);
        }
      } else {
        far = true;
      }
    }
    // vs / vref where it is not within P: a power of two (at most 2^127), or NaN
    const float ffar = ev == 255 ? vs : ev < eref ? exp2f(float(ev - eref)) : exp2f(float(min(ev - eref, 127)));
#pragma unroll
    for (int kc = 0; kc < C::KC; kc += 2) {
      uint32_t r[4];
      ldsm_x4_t(vb + kc * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (kc + x >= C::KC) break;
        // lane (g, t): columns 2 g, 2 g + 1 of positions 2 t, 2 t + 1 -> the pair of positions of each column; the even
        // columns are rows 0-7 of M, the odd ones rows 8-15
        const uint32_t u0 = __byte_perm(r[2 * x], 0, 0x3120), u1 = __byte_perm(r[2 * x + 1], 0, 0x3120);
        const uint32_t a0 = e4m3x2_half2(u0), a1 = e4m3x2_half2(u0 >> 16);
        const uint32_t a2 = e4m3x2_half2(u1), a3 = e4m3x2_half2(u1 >> 16);
        if (!far) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][kc + x], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float d[4] = {};
            mma16816(d, a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              // (a scale that is NaN is nothing to a row that sees none of the block)
              const bool sees = tok0 <= sq.pos0 + (fr0 + min(nt * 8 + 2 * t + (e & 1), n_fr - 1)) / rep;
              o[nt][kc + x][e] += sees ? ffar * d[e] : 0.f;
            }
          }
        }
      }
    }
  }
  cp_async_wait<0>();
  pdl_launch_dependents();
  // ---- join the warps
  __syncthreads();
  const float vref = __uint_as_float(uint32_t(eref) << 23);
  float* wo = reinterpret_cast<float*>(smem);            // [warp][ROWS][HD]
  float* wml = wo + kAttnWarps * ROWS * HD;              // [warp][ROWS][2]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float sum = l[nt][r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int row = warp * ROWS + nt * 8 + 2 * t + r;
      if (g == 0) {
        wml[2 * row] = m[nt][r];
        wml[2 * row + 1] = sum;
      }
#pragma unroll
      for (int kc = 0; kc < C::KC; ++kc)
        *reinterpret_cast<float2*>(wo + (size_t)row * HD + 16 * kc + 2 * g) =
            make_float2(o[nt][kc][r] * vref, o[nt][kc][2 + r] * vref);
    }
  __syncthreads();
  const int tile_rows = min(ROWS, c.max_new * rep);
  const int tiles = gridDim.x / a.splits;
  const bool alone = pages <= a.split_pages;  // the sequence's only part: nothing to merge
  for (int e = tid; e < n_fr * HD; e += kAttnWarps * 32) {
    const int r = e / HD, d = e % HD;
    float mx = kNoScore;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) mx = fmaxf(mx, wml[2 * (w * ROWS + r)]);
    float sum = 0.f, val = 0.f;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      const float f = ex2(wml[2 * (w * ROWS + r)] - mx);
      sum += f * wml[2 * (w * ROWS + r) + 1];
      val += f * wo[(size_t)(w * ROWS + r) * HD + d];
    }
    if (alone) {
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

// Joins the parts' states of a row, in order: WPR warps per row, each taking a
// run of the parts with their loads in flight together. Bound by two dependent
// trips to L2 (the parts' maxima and sums, then their values).
template <int HD, int NT, int WPR>
__global__ void __launch_bounds__(128) kv8_merge_kernel(const Kv8AttnArgs a) {
  constexpr int ROWS = 8 * NT, RPC = 4 / WPR, PER = (HD + 31) / 32, UN = 8;
  const Kv8Args& c = a.c;
  const int rep = c.nq / c.nkv, tile_rows = min(ROWS, c.max_new * rep);
  const int tiles = (c.max_new * rep + ROWS - 1) / ROWS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y, seq = blockIdx.z;
  const int fr = blockIdx.x * RPC + warp / WPR, sub = warp % WPR;  // (new position, q head) row, part of its parts
  __shared__ float s_val[WPR > 1 ? WPR : 1][HD], s_ml[WPR > 1 ? WPR : 1][2];
  pdl_wait();
  const Kv8Seq sq = kv8_seq(c, a.max_ctx, seq, false);
  // parts of this row's tile; a tile with one part has written its output
  const int last_row = min((fr / ROWS + 1) * ROWS, sq.n * rep) - 1;
  const int parts = (sq.pos0 + last_row / rep) / kPageTokens / a.split_pages + 1;
  const bool in = fr < sq.n * rep && sq.slot >= 0 && parts > 1;
  if (WPR == 1 && !in) return;
  const size_t stride = (size_t)tile_rows * (HD + 2);
  const float* base = a.part + (((size_t)seq * tiles + fr / ROWS) * c.nkv + h) * a.splits * stride;
  const float* ml = base + (size_t)tile_rows * HD + 2 * (fr % ROWS);
  const int per = (parts + WPR - 1) / WPR, s0 = min(parts, sub * per), s1 = min(parts, s0 + per);
  float mx = kNoScore, sum = 0.f, val[PER] = {};
  if (in) {
    for (int s = s0 + lane; s < s1; s += 32) mx = fmaxf(mx, ml[s * stride]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    for (int sb = s0; sb < s1; sb += UN) {
      float f[UN], l[UN], v[UN][PER];
#pragma unroll
      for (int j = 0; j < UN; ++j) {
        const bool ok = sb + j < s1;
        const size_t at = (size_t)(ok ? sb + j : s0) * stride;
        f[j] = ok ? ml[at] : -INFINITY;
        l[j] = ml[at + 1];
#pragma unroll
        for (int i = 0; i < PER; ++i) v[j][i] = lane + 32 * i < HD ? base[at + (size_t)(fr % ROWS) * HD + lane + 32 * i] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < UN; ++j) {
        if (sb + j >= s1) break;
        const float w = ex2(f[j] - mx);
        sum += w * l[j];
#pragma unroll
        for (int i = 0; i < PER; ++i) val[i] += w * v[j][i];
      }
    }
  }
  if (WPR > 1) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < HD) s_val[sub][lane + 32 * i] = val[i];
    if (lane == 0) {
      s_ml[sub][0] = mx;
      s_ml[sub][1] = sum;
    }
    __syncthreads();
    if (sub != 0 || !in) return;
    mx = kNoScore;
#pragma unroll
    for (int w = 0; w < WPR; ++w) mx = fmaxf(mx, s_ml[w][0]);
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) val[i] = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) {
      const float f = ex2(s_ml[w][0] - mx);
      sum += f * s_ml[w][1];
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < HD) val[i] += f * s_val[w][lane + 32 * i];
    }
  }
  __half* dst = a.out + ((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 32 * i < HD) dst[lane + 32 * i] = __float2half_rn(sum > 0.f || sum != sum ? val[i] / sum : 0.f);
}

// rows of a tile in eights: one, two or four n-tiles, no more than the call's rows of a kv head fill
int tile_nt(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }
int tile_rows_of(int max_new, int nq, int nkv) { return 8 * tile_nt((int64_t)max_new * (nq / nkv)); }
int tiles_of(int max_new, int nq, int nkv) {
  const int r = tile_rows_of(max_new, nq, nkv);
  return int(((int64_t)max_new * (nq / nkv) + r - 1) / r);
}

template <int HD, int NT>
cudaError_t attention_nt(const Kv8AttnArgs& a, cudaStream_t s) {
  const int tiles = tiles_of(a.c.max_new, a.c.nq, a.c.nkv);
  kv8_attention_kernel<HD, NT>
      <<<dim3(tiles * a.splits, a.c.nkv, a.c.n_seqs), kAttnWarps * 32, Kv8Cfg<HD>::smem(8 * NT), s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && a.splits > 1) {
    cudaLaunchAttribute attr[1];  // its launch overlaps the end of the attention kernel
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    const int rows = a.c.max_new * (a.c.nq / a.c.nkv), wpr = a.splits > 8 ? 4 : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((rows * wpr + 3) / 4, a.c.nkv, a.c.n_seqs);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = wpr == 4 ? cudaLaunchKernelEx(&cfg, kv8_merge_kernel<HD, NT, 4>, a)
                 : cudaLaunchKernelEx(&cfg, kv8_merge_kernel<HD, NT, 1>, a);
  }
  return e;
}
template <int HD>
cudaError_t attention_hd(const Kv8AttnArgs& a, cudaStream_t s) {
  const int nt = tile_nt((int64_t)a.c.max_new * (a.c.nq / a.c.nkv));
  return nt == 1 ? attention_nt<HD, 1>(a, s) : nt == 2 ? attention_nt<HD, 2>(a, s) : attention_nt<HD, 4>(a, s);
}

template <int HD>
cudaError_t append_hd(const Kv8AppendArgs& a, cudaStream_t s) {
  if (a.c.max_new <= kStepRows)
    kv8_append_kernel<HD, true><<<a.c.rows, kAppendThreads, 0, s>>>(a);
  else
    kv8_append_kernel<HD, false><<<(a.c.rows + kWindow - 1) / kWindow, kAppendThreads, 0, s>>>(a);
  return cudaGetLastError();
}

template <int HD>
cudaError_t attr_hd() {
  const cudaError_t e1 = set_kernel_smem(kv8_attention_kernel<HD, 1>, Kv8Cfg<HD>::smem(8));
  const cudaError_t e2 = set_kernel_smem(kv8_attention_kernel<HD, 2>, Kv8Cfg<HD>::smem(16));
  const cudaError_t e4 = set_kernel_smem(kv8_attention_kernel<HD, 4>, Kv8Cfg<HD>::smem(32));
  return e1 != cudaSuccess ? e1 : e2 != cudaSuccess ? e2 : e4;
}

}  // namespace

Kv8Plan kv8_plan(int n_seqs, int max_new, int nq, int nkv, int hd, int max_ctx, int sms) {
  const int64_t rows = (int64_t)max_new * (nq / nkv);
  const int64_t items = (int64_t)n_seqs * nkv * tiles_of(max_new, nq, nkv);
  const int64_t pages = ((int64_t)max_ctx + kPageTokens - 1) / kPageTokens;
  const int64_t places = (int64_t)sms * kv8_ctas(hd, tile_nt(rows));  // CTAs on the GPU at once
  // one round of the places where that leaves parts of less than 8 pages, otherwise three, so that ragged lengths even out
  int64_t sp = (items * pages + places - 1) / places;
  if (sp > 8) sp = std::max<int64_t>(8, (sp + 2) / 3);
  sp = std::max<int64_t>(4, std::min(sp, pages));
  Kv8Plan p;
  p.split_pages = int(sp);
  p.splits = int((pages + sp - 1) / sp);
  if (p.splits > 1)
    p.part_floats = (size_t)items * p.splits * std::min<int64_t>(tile_rows_of(max_new, nq, nkv), rows) * (hd + 2);
  return p;
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
