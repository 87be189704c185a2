// Attention over the paged cache in 8 bits for steps and short runs of rows, the
// join of a sequence's parts, and the choice between this kernel and the one for
// long runs (kv8_prompts.cu). kv8.cu has the cache's layout.
#include "kv8_common.cuh"

#include <algorithm>

namespace mmc {
namespace {

constexpr int kAttnWarps = 4;  // warp w reads block w of each page
// m lies kHeadroom under the largest score when it is set, and is set again when a score exceeds it by more than kFollow
constexpr float kHeadroom = 7.f, kFollow = 15.f;

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
constexpr int kv8_ctas(int hd, int nt) { return nt == 1 ? (hd <= 96 ? 5 : 4) : nt == 2 || (nt == 3 && hd <= 64) ? 3 : 2; }

// One CTA: up to 8 NT rows (new position, q head of the group) of one sequence
// and kv head, over one part of `split_pages` pages. Each warp streams its own
// blocks of 16 positions (block w of every page) through a ring of its own, so
// the loop has no CTA barrier. On m16n8k16 the 16 positions are M and the rows
// are N: S^T = K Q^T and O^T += V^T P^T, so K and V are taken from e4m3 to fp16
// (exact) once for all rows, and a group of up to 8 q heads fills N.
//   Softmax: p = 2^(s - m), where m follows the largest score only when one
// exceeds it by more than 15, and then lies 7 below it: p stays below 2^15, within
// fp16, and most blocks need one vote and no reduction; the sums stay in each lane
// until the end. p goes to fp16 (2^-11 of each weight) for the products, the sums
// take the 32-bit weights.
//   V's scales are powers of two: with vref the largest so far, p * (scale /
// vref) loses nothing in fp16 down to scale = vref / 64 for weights from 2^-15 of
// the largest on, and O stays in units of vref. (With m at the largest score,
// thousands of weights of 2^-15 each lost up to 6 % in fp16's subnormals, 0.5 % of
// an output.) A block whose scale lies further below takes a second accumulator.
// The four warps' states are joined in shared memory in a fixed order; with
// several parts the joined states go to `part` and kv8_merge_kernel joins them,
// again in order.
//   What bounds it: instructions and their latency. 16 positions of hd 96 are 3 KB
// and some 250 instructions of a warp, 96 of them conversions and byte moves of the
// half-rate pipe. 64 sequences of 14000 to 32766 positions (nq 8, nkv 2): 111 to 123
// us by the GPU, 5.2 to 4.7 of 6.5 TB/s (hd 128: 133 us, 5.8 TB/s); the schedulers
// issue in 52 % of the cycles with 4.5 warps each, and wait for fixed latencies
// otherwise. 256 sequences of 16 to 2303: 34 us, as a CTA has 9 pages there and its
// start and join are 5 us; 32 x 3 to 5 rows: 20.5 us. Tried: two blocks a turn for more independent
// instructions (registers leave 12 warps instead of 20: 125 us), rings of four
// stages (119, but 256 sequences 40), 8-bit mma.sync with p and q in three parts
// (slower: it is emulated), the same on tcgen05 with positions on M (150: a tile of
// 128 positions waits for each of its copies, votes and products in turn), CTAs of
// a cluster joined in shared memory instead of the second kernel (the same), equal
// parts found on the device as for long runs (256 sequences: 47).
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
    const float2 sc = *reinterpret_cast<const float2*>(ring + st * C::STAGE + 2 * kKv8Block * C::PITCH);
    const float ks = sc.x * sl2, vs = sc.y;
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
      above |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] + kFollow || fmaxf(s[nt][1], s[nt][3]) > m[nt][1] + kFollow;
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
          mx = fmaxf(mx - kHeadroom, m[nt][r]);  // (the same in the row's eight lanes)
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
    // exponents: 1 .. 247; 255 where the block is lost (NaN). vref follows every larger scale, whatever the distance: what O
    // holds then loses bits only below 2^-126 of the new unit (2^-127 and on: all of it)
    const int ev = __float_as_uint(vs) >> 23 & 255;
    bool far = false;
    if (ev != eref) {
      if (ev > eref && ev != 255) {
        const float f = __uint_as_float(uint32_t(max(127 + eref - ev, 0)) << 23);
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
    auto values = [&](int kc, uint32_t (&a)[2][4]) {
      uint32_t r[4];
      ldsm_x4_t(vb + kc * 16, r[0], r[1], r[2], r[3]);
      // lane (g, t): columns 2 g, 2 g + 1 of positions 2 t, 2 t + 1 -> the pair of positions of each column; the even
      // columns are rows 0-7 of M, the odd ones rows 8-15
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t u0 = __byte_perm(r[2 * x], 0, 0x3120), u1 = __byte_perm(r[2 * x + 1], 0, 0x3120);
        a[x][0] = e4m3x2_half2(u0);
        a[x][1] = e4m3x2_half2(u0 >> 16);
        a[x][2] = e4m3x2_half2(u1);
        a[x][3] = e4m3x2_half2(u1 >> 16);
      }
    };
    if (!far) {  // (a loop of its own: with the seldom one in it, a step took 5 % longer)
#pragma unroll
      for (int kc = 0; kc < C::KC; kc += 2) {
        uint32_t a[2][4];
        values(kc, a);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (kc + x >= C::KC) break;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816(o[nt][kc + x], a[x][0], a[x][1], a[x][2], a[x][3], pb[nt][0], pb[nt][1]);
        }
      }
    } else {
      // vs / vref where it is not within P: 2^-7 and less, or NaN
      const float f = ev == 255 ? vs : exp2f(float(ev - eref));
#pragma unroll
      for (int kc = 0; kc < C::KC; kc += 2) {
        uint32_t a[2][4];
        values(kc, a);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (kc + x >= C::KC) break;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float d[4] = {};
            mma16816(d, a[x][0], a[x][1], a[x][2], a[x][3], pb[nt][0], pb[nt][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              // (a scale that is NaN is nothing to a row that sees none of the block)
              const bool sees = tok0 <= sq.pos0 + (fr0 + min(nt * 8 + 2 * t + (e & 1), n_fr - 1)) / rep;
              o[nt][kc + x][e] += sees ? f * d[e] : 0.f;
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
template <int HD, int ROWS, int WPR>
__global__ void __launch_bounds__(128) kv8_merge_kernel(const Kv8AttnArgs a) {
  constexpr int RPC = 4 / WPR, PER = (HD + 31) / 32, UN = 8;
  const Kv8Args& c = a.c;
  const int rep = c.nq / c.nkv, tile_rows = min(ROWS, c.max_new * rep);
  const int tiles = (c.max_new * rep + ROWS - 1) / ROWS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y, seq = blockIdx.z;
  const int fr = blockIdx.x * RPC + warp / WPR, sub = warp % WPR;  // (new position, q head) row, part of its parts
  __shared__ float s_val[WPR > 1 ? WPR : 1][HD], s_ml[WPR > 1 ? WPR : 1][2];
  const Kv8Seq sq = kv8_seq(c, a.max_ctx, seq, false);  // (the attention kernel writes none of this)
  // parts of this row's tile; a tile with one part has written its output
  const int last_row = min((fr / ROWS + 1) * ROWS, sq.n * rep) - 1;
  const int parts = (sq.pos0 + last_row / rep) / kPageTokens / a.split_pages + 1;
  const bool in = fr < sq.n * rep && sq.slot >= 0 && parts > 1;
  // Every warp waits, those without a row to join too: the attention kernel lets this one start before it has written its
  // rows, and what comes next on the stream waits for this grid only.
  pdl_wait();
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

template <int HD, int ROWS>
cudaError_t merge(const Kv8AttnArgs& a, cudaStream_t s) {
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
  return wpr == 4 ? cudaLaunchKernelEx(&cfg, kv8_merge_kernel<HD, ROWS, 4>, a)
                  : cudaLaunchKernelEx(&cfg, kv8_merge_kernel<HD, ROWS, 1>, a);
}
template <int HD, int NT>
cudaError_t attention_nt(const Kv8AttnArgs& a, cudaStream_t s) {
  kv8_attention_kernel<HD, NT>
      <<<dim3(a.tiles * a.splits, a.c.nkv, a.c.n_seqs), kAttnWarps * 32, Kv8Cfg<HD>::smem(8 * NT), s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess || a.splits == 1 ? e : merge<HD, 8 * NT>(a, s);
}
template <int HD>
cudaError_t attention_hd(const Kv8AttnArgs& a, cudaStream_t s) {
  return a.tile_rows == kKv8PromptRows ? launch_kv8_prompts(a, HD, s) : a.tile_rows == 8 ? attention_nt<HD, 1>(a, s)
         : a.tile_rows == 16 ? attention_nt<HD, 2>(a, s) : a.tile_rows == 24 ? attention_nt<HD, 3>(a, s) : attention_nt<HD, 4>(a, s);
}

template <int HD>
cudaError_t attr_hd() {
  const cudaError_t e1 = set_kernel_smem(kv8_attention_kernel<HD, 1>, Kv8Cfg<HD>::smem(8));
  const cudaError_t e2 = set_kernel_smem(kv8_attention_kernel<HD, 2>, Kv8Cfg<HD>::smem(16));
  const cudaError_t e3 = set_kernel_smem(kv8_attention_kernel<HD, 3>, Kv8Cfg<HD>::smem(24));
  const cudaError_t e4 = set_kernel_smem(kv8_attention_kernel<HD, 4>, Kv8Cfg<HD>::smem(32));
  return e1 != cudaSuccess ? e1 : e2 != cudaSuccess ? e2 : e3 != cudaSuccess ? e3 : e4;
}

}  // namespace

Kv8Plan kv8_plan(int n_seqs, int max_new, int nq, int nkv, int hd, int max_ctx, int sms) {
  const int64_t rows = (int64_t)max_new * (nq / nkv);
  const int64_t pages = ((int64_t)max_ctx + kPageTokens - 1) / kPageTokens;
  const int64_t heads = (int64_t)n_seqs * nkv;
  // Tiles of 8, 16, 24 or 32 rows, no more than the rows of a kv head fill, or the 128 of the kernel for long runs where there
  // is enough to do, in tiles of 32 rows x pages an SM: that one takes some 16 us to share its work out and join its parts.
  // Measured (smaller tiles / 128 rows, us), heads of 96: 4 sequences x 80 rows behind 4000 positions 21 / 30, 8 x 80 behind
  // 8000 44 / 31, 8 x 1200 behind 1000 89 / 44, 64 x 20 behind 2000 39 / 41, 256 x 20 105 / 96; heads of 128: 64 x 20
  // 62 / 52, 256 x 20 178 / 117; heads of 64: 256 x 20 85 / 91.
  const int64_t work = heads * ((rows + 31) / 32) * pages;
  const bool many = (rows > 32 ? work > 12 * (int64_t)sms
                               : rows > 16 && hd >= 96 && work > (hd == 96 ? 40 : 12) * (int64_t)sms) &&
                    heads * ((rows + kKv8PromptRows - 1) / kKv8PromptRows) < (int64_t(1) << 31);  // (its grid)
  const int tile_rows = many ? kKv8PromptRows : rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 24 ? 24 : 32;
  Kv8Plan p;
  p.tile_rows = tile_rows;
  p.tiles = int((rows + tile_rows - 1) / tile_rows);
  const int64_t items = heads * p.tiles;
  if (tile_rows == kKv8PromptRows) {
    // The kernel lengthens the parts as the call's lengths ask for; up to two and a half rounds of them, as sequences are
    // shorter than max_ctx. Parts of less than 4 pages cost more than they give.
    p.places = 2 * sms;
    int64_t splits = 1;
    if (items < p.places) splits = std::max<int64_t>(1, std::min((5 * p.places + 2 * items - 1) / (2 * items), pages / 4));
    p.split_pages = int((pages + splits - 1) / splits);
    p.splits = int((pages + p.split_pages - 1) / p.split_pages);
    if (p.splits > 1) p.part_floats = 4 + (size_t)items * p.splits * tile_rows * (hd + 2);
    return p;
  }
  const int64_t places = (int64_t)sms * kv8_ctas(hd, tile_rows / 8);  // CTAs on the GPU at once
  // one round of the places where that leaves parts of less than 8 pages, otherwise three, so that ragged lengths even
  // out, and four of long parts (heads of 128, 64 sequences of 14000 to 32766 positions: 142 us in three, 136 in four; 256
  // of 16 to 2303: 39.7 and 41.4)
  int64_t sp = (items * pages + places - 1) / places;
  if (sp > 8) sp = std::max<int64_t>(8, sp > 40 ? (sp + 3) / 4 : (sp + 2) / 3);
  sp = std::max<int64_t>(4, std::min(sp, pages));
  p.split_pages = int(sp);
  p.splits = int((pages + sp - 1) / sp);
  if (p.splits > 1) p.part_floats = (size_t)items * p.splits * std::min<int64_t>(tile_rows, rows) * (hd + 2);
  return p;
}

#define MMC_BY_HD(fn, ...)                                                                                          \
  (hd == 16 ? fn<16>(__VA_ARGS__) : hd == 32 ? fn<32>(__VA_ARGS__) : hd == 64 ? fn<64>(__VA_ARGS__)                 \
   : hd == 96 ? fn<96>(__VA_ARGS__) : hd == 128 ? fn<128>(__VA_ARGS__) : cudaErrorInvalidValue)

cudaError_t launch_kv8_attention(const Kv8AttnArgs& a, int hd, cudaStream_t s) {
  return MMC_BY_HD(attention_hd, a, s);
}
cudaError_t kv8_init_attributes() {
  for (int hd : {16, 32, 64, 96, 128}) {
    const cudaError_t e = MMC_BY_HD(attr_hd);
    if (e != cudaSuccess) return e;
  }
  return kv8_prompts_init_attributes();
}

}  // namespace mmc
