// Append to a paged KV cache in 8 bits (kv8_attention.cu reads it).
//
// Cache: e4m3 codes [n_pages][layers][2 (K, V)][nkv][64][hd], rows in plain
// order, and one fp32 scale for each 16 positions of a page, kv head and K or V
// ([n_pages][layers][2][nkv][4]); a value is code * scale. Scales are powers of
// two, the smallest 2^e (e >= -126) with amax <= 448 * 2^e: e4m3 is a floating
// format, so a power of two costs no precision, and when a later position needs
// a larger scale the block's older codes go over to it exactly (but for those
// that become subnormal, which round once more).
#include "kv8_common.cuh"

namespace mmc {
namespace {

constexpr int kAppendThreads = 256;

// ---------------------------------------------------------------- append

// One CTA per window of `window` rows. A head's row is held by hd / 8 lanes, four
// elements of each half a lane, so that a lane has both ends of its rotations and
// loads and stores are 16, 8 (fp16 q) and 4 (codes) bytes wide. The q heads
// (RMSNorm, rotation, fp16) are dealt to the warps. Then, for each row that is the
// first of this call in its block of 16 positions, the CTA takes the whole block,
// two of its K and V heads at a time: the new rows stay in registers while their
// largest magnitudes go through shared memory, older codes go over to the new
// scale if it grew, and the new codes are written. With at most kStepRows rows a
// sequence (STEP) a window is one row and each K or V head one warp's, without
// barriers. A block has one owner, so no atomics on the cache and no order that
// could change the result.
//   Bound with many rows by the blocks' chains of loads, largest value and stores
// and by HBM (the raw projections, read once, are four times the bytes of all that
// is written): 11 prompts of 33 to 1401 rows (nq 32, nkv 8, hd 128) take 67 us, 4.2
// TB/s; 30 of 100 to 1000 with norms (nq 8, nkv 2, hd 96) 40 us; one of 200 or of 500
// (nq 32) 18 us, with fewer CTAs than SMs. Two heads at a time and four
// CTAs an SM: four heads leave registers for two CTAs (67 and 52 us), one head at a
// time spills at five (88 and 46), windows of 16 rows take 78 and 44. With few, by
// the chain of loads slot -> position -> page -> old scale, so the projections are
// loaded before it: 256 steps (nq 8, nkv 2, hd 96) 4.1 us, one 3.3 (with one CTA an
// SM 6.5, as 256 are two rounds then).
constexpr int kWindow = 8, kStepRows = 8;

template <int HD, bool STEP>
__global__ void __launch_bounds__(kAppendThreads, STEP ? 2 : 4) kv8_append_kernel(const Kv8AppendArgs a) {
  constexpr int window = STEP ? 1 : kWindow;
  constexpr int HALF = HD / 2, LPH = HD / 8;                                    // lanes of a head's row
  constexpr int GL = LPH <= 2 ? 2 : LPH <= 4 ? 4 : LPH <= 8 ? 8 : 16;           // lanes of a group
  constexpr int HPW = 32 / GL, BATCH = STEP ? 1 : 2;                                    // heads of a warp at once, and of a unit
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
    if (e < b && blockIdx.x == 0) set_error(c.err, kDevBadRows);  // (it has no rows to refuse)
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
      else if ((int64_t)pos0 + (last - first) > a.max_pos) e = kDevPositionLimit;
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

template <int HD>
cudaError_t append_hd(const Kv8AppendArgs& a, cudaStream_t s) {
  if (a.c.max_new <= kStepRows)
    kv8_append_kernel<HD, true><<<a.c.rows, kAppendThreads, 0, s>>>(a);
  else
    kv8_append_kernel<HD, false><<<(a.c.rows + kWindow - 1) / kWindow, kAppendThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

#define MMC_BY_HD(fn, ...)                                                                                          \
  (hd == 16 ? fn<16>(__VA_ARGS__) : hd == 32 ? fn<32>(__VA_ARGS__) : hd == 64 ? fn<64>(__VA_ARGS__)                 \
   : hd == 96 ? fn<96>(__VA_ARGS__) : hd == 128 ? fn<128>(__VA_ARGS__) : cudaErrorInvalidValue)

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, int hd, cudaStream_t s) { return MMC_BY_HD(append_hd, a, s); }

}  // namespace mmc
