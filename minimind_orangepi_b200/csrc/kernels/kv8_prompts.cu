// Attention over the paged cache in 8 bits for long runs of rows: a sequence's
// new positions x the q heads of a kv head, 128 rows of them a CTA. kv8.cu has the
// cache's layout, kv8_attention.cu the kernel for fewer rows and the choice.
//
// For 128 rows the products are the work, so they go to tcgen05, in fp16 as q and p
// are (P rounds to 2^-11 of each weight; the sums take the weights as they were):
//   S [128 x 64] = Q K^T     O [128 x hd] += P V      a page of 64 positions a turn
// with rows as TMEM lanes, so that a thread has a row's scores and its softmax
// needs no exchange. The codes are taken to fp16 (exact) once for all 128 rows, and
// P stays in tensor memory, where its scores were.
//   Warps 0-3: softmax, warps 4-7: pages to fp16 tiles, warp 8: the matrix
// instructions, which compute the next page's scores before they wait for this
// page's P, warp 9: the pages' copies. Two CTAs share an SM, so one's
// softmax runs under the other's products. Every wait has a limit, after which the
// error word is set and the CTA drains and leaves.
//   Softmax: p = 2^(s - m), where m follows the largest score only when one
// exceeds it by more than 8; O is then scaled in TMEM.
//   What bounds it, measured on four prompts of 300 to 512 rows behind up to 4000
// positions (nq 8, nkv 2, hd 96): 46 us, where tiles of 32 rows on mma.sync took
// 111. A CTA takes 1.2 us a page, of which the softmax is 1.0 (64 exponentials a
// thread are 0.3 at the least; the rest is instruction latency, as two warps share
// a scheduler), some 8 us to find its unit and get its first page, 2.4 to write its
// part; the join takes 6. Tried: the scores in pieces of 16 columns, or held in
// registers from the maximum to the exponential (slower: trips to tensor memory,
// and spills), a part of the exponentials as polynomials (slower), packed fp32
// products and sums (the same), loads to registers instead of the page ring (48).
//   Scales: K's go to the scores in 32 bits. V's are powers of two: O is kept in
// units of 2^(eref - 7) where 2^eref is the largest scale so far, and a code goes
// to fp16 as code * 2^(ev - eref + 7): from 2^-9 * 2^-14 to 448 * 2^7, exact down to
// ev = eref - 21. A page whose blocks lie further apart is taken in several turns,
// each with a part of its blocks, and O changes its units in between, which is
// exact too. eref stays within 64 of the largest scale so far, so that O stays
// within 32 bits: at most 2^8 * 448 * 2^(64 + 7) a position, 2^40 positions. (So a
// block of less than 2^-85 of the largest scale so far counts as zeros.)
#include "kv8_common.cuh"
#include "tc_common.cuh"

#include <type_traits>

namespace mmc {
namespace {

constexpr int kRows = kKv8PromptRows;  // 128: M, and the softmax threads
constexpr int kThreads = 320;
constexpr int kListed = 1024;  // tiles of rows whose pages fit the shared memory of every head size
constexpr int kSpread = 21, kUnit = 7, kBelow = 64;  // kBelow: eref's distance from the largest scale so far, at most

template <int HD>
struct Prompts {
  static constexpr int PIECE = HD % 64 == 0 ? 64 : HD % 32 == 0 ? 32 : 16;  // columns of a piece: rows of one swizzle width
  static constexpr int ROWB = 2 * PIECE;
  static constexpr uint32_t SWZ = ROWB / 16 - 1;
  static constexpr uint64_t LAYOUT = ROWB == 128 ? 2 : ROWB == 64 ? 4 : 6;
  static constexpr int Q_BYTES = kRows * HD * 2, KV_BYTES = kPageTokens * HD * 2;
  static constexpr int OFF_KV = Q_BYTES;
  // fp16 tiles, and pages as they are in the cache: two CTAs an SM
  static constexpr int STAGES = HD <= 96 ? 3 : 2, RAW = HD <= 64 ? 4 : 1;
  static constexpr int SLAB = kPageTokens * HD, OFF_RAW = OFF_KV + STAGES * 2 * KV_BYTES;
  static constexpr int SMEM = 1024 + OFF_RAW + RAW * 2 * SLAB;  // the first kilobyte: barriers and notes
  static constexpr int O_COL = 2 * kPageTokens, TMEM = O_COL + HD <= 256 ? 256 : 512;
  // byte of column c, row r in a tile of `rows` rows: [piece][row][PIECE], swizzled
  static __device__ __forceinline__ uint32_t at(int rows, int r, int c) {
    uint32_t off = r * ROWB + c % PIECE * 2;
    off ^= ((off >> 7) & SWZ) << 4;
    return off + c / PIECE * (rows * ROWB);
  }
};

// What a turn is, beside its tiles.
struct Note {
  float ks[4];    // K's scales of the blocks that take part, times log2(e) / sqrt(hd): positive or NaN
  int tok0;       // first position
  uint32_t mask;  // blocks that take part; bit 4 + b: block b's V is lost
  int eref;       // units of O: 2^(eref - 127 - kUnit)
  int end;        // no turn: the end
};

__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo, uint32_t sbo, uint64_t layout) {
  return uint64_t((addr >> 4) & 0x3fff) | uint64_t((lbo >> 4) & 0x3fff) << 16 | uint64_t((sbo >> 4) & 0x3fff) << 32 |
         uint64_t(1) << 46 | layout << 61;
}
// 32 columns of this warp's lanes, in flight until the wait, which the values go through
__device__ __forceinline__ void tmem_fetch32(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr));
}
template <int COUNT>
__device__ __forceinline__ void tmem_arrived(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < COUNT; i += 8)
    asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]),
                      "+f"(v[i + 6]), "+f"(v[i + 7]));
}
// D[128 x N] (+)= A B with A in tensor memory: row = lane, two halves a column
__device__ __forceinline__ void umma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 codes to fp16, times `factor` (two halves)
template <bool SCALE>
__device__ __forceinline__ void widen(const uint4& codes, uint32_t factor, uint4 (&out)[2]) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[2 * i] = e4m3x2_half2(w[i]);
    h[2 * i + 1] = e4m3x2_half2(w[i] >> 16);
  }
  if (SCALE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = h2_mul(h[i], factor);
  }
  out[0] = make_uint4(h[0], h[1], h[2], h[3]);
  out[1] = make_uint4(h[4], h[5], h[6], h[7]);
}

// The pages that a tile of rows sees, 0 for one without rows.
__device__ __forceinline__ int tile_pages(const Kv8Seq& sq, int rep, int tile) {
  const int n_fr = min(kRows, sq.n * rep - tile * kRows);
  return sq.slot < 0 || n_fr <= 0 ? 0 : (sq.pos0 + (tile * kRows + n_fr - 1) / rep) / kPageTokens + 1;
}

// What a CTA does: a part of the pages of a sequence's tile of rows, for one kv head.
struct Unit {
  int seq, tile, h, part, split_pages;
};

__device__ __forceinline__ uint64_t block_sum(uint64_t x, uint64_t* place) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) place[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) x += place[w];
  return x;
}

// The call's lengths are known on the device only, so the CTAs share its work out
// here: of the units that there are, in order, CTA k takes the k-th, and those that
// are left without one are the last (empty ones in between would hold up what is
// behind them: the prompts case took 70 us). The pages of a part are the fewest of
// eight trials for which the units are no more than the CTAs that run at once: with
// N tiles and T pages of theirs, T / (places - N) always are. false: no unit.
__device__ bool find_unit(const Kv8AttnArgs& a, int tiles, int rep, uint8_t* smem, Unit& u) {
  const Kv8Args& c = a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint64_t* place = reinterpret_cast<uint64_t*>(smem);
  int* found = reinterpret_cast<int*>(smem + 128);
  int* pages = reinterpret_cast<int*>(smem + 1024);  // of tile i % tiles, from the last one, of sequence i / tiles
  const int n = c.n_seqs * tiles;
  uint64_t mine = 0;  // T, and N in the upper bits
  for (int i = tid; i < n; i += kThreads) {
    const int x = tile_pages(kv8_seq(c, a.max_ctx, i / tiles, false), rep, tiles - 1 - i % tiles);
    pages[i] = x;
    mine += x > 0 ? uint64_t(x) | uint64_t(1) << 40 : 0;
  }
  if (tid == 0) *found = -1;
  mine = block_sum(mine, place);
  int sp = 1 << 30;
  if (a.splits > 1) {
    const int64_t t = int64_t(mine & ((uint64_t(1) << 40) - 1)) * c.nkv, left = a.places - int64_t(mine >> 40) * c.nkv;
    const int low = int(t / a.places) + 1, high = int((t + left - 1) / left);  // (left > 0: tiles x kv heads < places)
    auto trial = [&](int j) { return max(a.split_pages, low + int(int64_t(high - low) * (j + 1) / 8)); };
    uint64_t units[2] = {};  // of four trials each; at most items x splits, a few thousand
    for (int i = tid; i < n; i += kThreads)
#pragma unroll
      for (int j = 0; j < 8; ++j) units[j / 4] += uint64_t((pages[i] + trial(j) - 1) / trial(j)) << (16 * (j % 4));
    units[0] = block_sum(units[0], place);
    units[1] = block_sum(units[1], place);
    sp = trial(7);
#pragma unroll
    for (int j = 6; j >= 0; --j)
      if (int64_t(units[j / 4] >> (16 * (j % 4)) & 0xffff) * c.nkv <= a.places) sp = trial(j);
    if (tid == 0 && blockIdx.x == 0) *reinterpret_cast<int*>(a.part) = sp;  // for the join
  }
  // the k-th unit: a run of the tiles a thread, the runs' sums in order
  const int k = blockIdx.x / c.nkv, per = (n + kThreads - 1) / kThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
  int sum = 0;
  for (int i = i0; i < i1; ++i) sum += (pages[i] + sp - 1) / sp;
  int before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  __syncthreads();
  if (lane == 31) place[warp] = before;
  __syncthreads();
  before -= sum;
  for (int w = 0; w < warp; ++w) before += int(place[w]);
  if (k >= before && k < before + sum)
    for (int i = i0; i < i1; ++i) {
      const int x = (pages[i] + sp - 1) / sp;
      if (k < before + x) {
        found[0] = i;
        found[1] = k - before;
        break;
      }
      before += x;
    }
  __syncthreads();
  u = {found[0] / tiles, tiles - 1 - found[0] % tiles, int(blockIdx.x % c.nkv), found[1], sp};
  const bool is = found[0] >= 0;
  __syncthreads();
  return is;
}

// Rows of unused sequences attend nothing, and are no unit; wrong ranges and slots
// are reported here. A sequence is CTA (sequence modulo CTAs)'s.
template <int HD>
__device__ void unused_rows(const Kv8AttnArgs& a) {
  for (int i = blockIdx.x; i < a.c.n_seqs; i += gridDim.x) {
    const Kv8Seq sq = kv8_seq(a.c, a.max_ctx, i, threadIdx.x == 0);
    if (sq.slot < 0)
      for (int64_t e = threadIdx.x; e < (int64_t)sq.n * a.c.nq * HD; e += kThreads)
        a.out[(size_t)sq.first * a.c.nq * HD + e] = __float2half_rn(0.f);
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 2) kv8_prompts_kernel(const Kv8AttnArgs a) {
  using C = Prompts<HD>;
  constexpr int kStages = C::STAGES, kRaw = C::RAW;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_raw);  // [kStages] the page's tiles and note
  uint64_t* empty = full + kStages;
  uint64_t* s_full = full + 2 * kStages;  // [2]
  uint64_t* p_ready = s_full + 2;
  uint64_t* pv_done = s_full + 3;  // [2], so that a wait needs the product three turns before to have ended, not the last
  uint64_t* drained = s_full + 5;
  uint64_t* raw_full = s_full + 6;  // [kRaw] a page has come
  uint64_t* raw_empty = raw_full + kRaw;
  float4* raw_scales = reinterpret_cast<float4*>(smem_raw + 512);  // [kRaw][K, V]
  int* raw_have = reinterpret_cast<int*>(smem_raw + 704);          // [kRaw]
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem_raw + 224);
  Note* notes = reinterpret_cast<Note*>(smem_raw + 256);  // [kStages]
  uint8_t* smem = smem_raw + 1024;
  const Kv8Args& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tiles = a.tiles, rep = c.nq / c.nkv;
  if (warp == 8) {  // first of all: an SM's second CTA starts when its first has given up the right to allocate
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)),
                 "r"(uint32_t(C::TMEM))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  auto leave = [&] {  // without work
    __syncwarp();
    if (warp == 8) tmem_dealloc<C::TMEM>(*s_tmem);
  };
  // Many more tiles than CTAs: each has its own, the last ones of a sequence, which see the most, first.
  Unit u{int(blockIdx.x / (c.nkv * tiles)), tiles - 1 - int(blockIdx.x / c.nkv % tiles), int(blockIdx.x % c.nkv), 0, 1 << 30};
  if (c.n_seqs * int64_t(tiles) <= kListed) {
    unused_rows<HD>(a);
    if (!find_unit(a, tiles, rep, smem_raw, u)) return leave();
  }
  const int seq = u.seq, tile = u.tile, h = u.h, split = u.part, split_pages = u.split_pages, fr0 = tile * kRows;
  const Kv8Seq sq = kv8_seq(c, a.max_ctx, seq, tid == 0);
  const int n_fr = min(kRows, sq.n * rep - fr0);  // this tile's rows
  if (n_fr <= 0) return leave();
  if (sq.slot < 0) {  // an unused sequence: its rows attend nothing
    for (int e = tid; e < n_fr * HD; e += kThreads) {
      const int fr = fr0 + e / HD;
      a.out[((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD + e % HD] = __float2half_rn(0.f);
    }
    return leave();
  }
  const int lim_lo = sq.pos0 + fr0 / rep, lim_hi = sq.pos0 + (fr0 + n_fr - 1) / rep;  // last positions seen
  const int end = sq.pos0 + sq.n;                                                     // positions written
  const int pages = lim_hi / kPageTokens + 1;
  const int p0 = split * split_pages, p1 = min(pages, p0 + split_pages);

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 4);
      mbar_init(empty + s, 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_full + 1, 1);
    for (int s = 0; s < kRaw; ++s) {
      mbar_init(raw_full + s, 1);
      mbar_init(raw_empty + s, 4);
    }
    mbar_init(p_ready, 4);
    mbar_init(pv_done, 1);
    mbar_init(pv_done + 1, 1);
    mbar_init(drained, 1);
    fence_mbar_init();
  }
  for (int i = tid; i < kRows * (HD / 8); i += kThreads) {
    const int r = i / (HD / 8), k = i % (HD / 8), fr = fr0 + r;
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (r < n_fr)
      x = *reinterpret_cast<const uint4*>(a.q + ((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD + 8 * k);
    *reinterpret_cast<uint4*>(smem + C::at(kRows, r, 8 * k)) = x;
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem, base = smem_u32(smem);
  pdl_launch_dependents();  // (the join's CTAs find room only where this kernel's leave some)
  bool ok = true;

  if (warp >= 4 && warp < 8) {
    // ================================================================ pages to fp16 tiles
    // A warp has a block of 16 positions, 16 codes a load. With heads of 64 and 128 its lanes lie along the rows, otherwise
    // two a row, so that neither the loads nor the stores meet in a bank (twice at most, stores of 128).
    constexpr bool ALONG = HD % 64 == 0;
    constexpr int PER = HD / 32 > 0 ? HD / 32 : 1;
    const int ct = tid - 128;
    const int row0 = ALONG ? ct / 32 * 16 + lane / (HD / 16) : HD == 16 ? ct & 63 : ct >> 1;
    const int col0 = ALONG ? lane % (HD / 16) * 16 : HD == 16 ? 0 : (ct & 1) * 16;
    constexpr int DROW = ALONG ? 512 / HD : 0, DCOL = ALONG ? 0 : 32;
    const bool mine = HD > 16 || ct < 64;
    const float sl2 = kLog2e / sqrtf(float(HD));
    int n = 0, eref = 0, largest = 0;  // turns so far; units, largest scale so far (0: no block yet)
    auto publish = [&](int s) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + s);
      ++n;
    };
    auto stage_free = [&]() {
      if (n >= kStages) ok = mbar_wait_bounded(empty + n % kStages, (n / kStages - 1) & 1, c.err);
      ok = __all_sync(0xffffffffu, ok);
      return ok;
    };
    const int my_b = row0 >> 4;
    for (int p = p0; p < p1 && ok; ++p) {
      const int tok0 = p * kPageTokens, rs = (p - p0) % kRaw;
      ok = mbar_wait_bounded(raw_full + rs, ((p - p0) / kRaw) & 1, c.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const bool have = raw_have[rs] != 0;
      const float4 ks4 = raw_scales[2 * rs], vs4 = raw_scales[2 * rs + 1];
      const uint8_t* raw = smem + C::OFF_RAW + rs * 2 * C::SLAB + row0 * HD + col0;
      uint4 kc[PER], vc[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        kc[i] = *reinterpret_cast<const uint4*>(raw + i * (DROW * HD + DCOL));
        vc[i] = *reinterpret_cast<const uint4*>(raw + C::SLAB + i * (DROW * HD + DCOL));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(raw_empty + rs);
      const float vs[4] = {vs4.x, vs4.y, vs4.z, vs4.w};
      const float my_vs = my_b == 0 ? vs[0] : my_b == 1 ? vs[1] : my_b == 2 ? vs[2] : vs[3];
      const int my_ev = __float_as_uint(my_vs) >> 23 & 255;
      uint32_t left = 0, lost = 0;  // blocks to come; those whose V scale is NaN
      int ev[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        ev[b] = __float_as_uint(vs[b]) >> 23 & 255;
        if (have && tok0 + 16 * b <= lim_hi) {
          left |= 1u << b;
          if (ev[b] == 255) lost |= 1u << b;
        }
      }
      while (left != 0) {
        if (!stage_free()) break;
        // the turn's units and blocks
        uint32_t take = left;
        const int top = max(max(ev[0], ev[1]), max(ev[2], ev[3])), low = min(min(ev[0], ev[1]), min(ev[2], ev[3]));
        if (left != 15u || top > eref || low < eref - kSpread) {  // (a lost block is above eref)
          int hi = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if ((left & ~lost) >> b & 1) hi = max(hi, ev[b]);
          largest = max(largest, hi);
          if (hi > eref || (hi != 0 && hi < eref - kSpread)) eref = max(hi, largest - kBelow);
          take = lost & left;
#pragma unroll
          for (int b = 0; b < 4; ++b)  // (all of them where eref stopped above hi: zeros)
            if ((left & ~lost) >> b & 1 && (ev[b] >= eref - kSpread || hi < eref - kSpread)) take |= 1u << b;
        }
        // 2^(ev - eref + kUnit) in fp16. Codes that take no part may be NaN, and codes that are no position's whatever was
        // there: 0 x NaN would spoil the sum
        const int e = my_ev - eref + kUnit;
        const bool zero = !((take & ~lost) >> my_b & 1) || e < kUnit - kSpread;
        const uint32_t factor = zero ? 0u : uint32_t(15 + e) * 0x04000400u;
        const int s = n % kStages;
        uint8_t* kt = smem + C::OFF_KV + s * 2 * C::KV_BYTES;
        uint8_t* vt = kt + C::KV_BYTES;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (!mine) break;
          const int row = row0 + i * DROW;
          const uint32_t off = C::at(kPageTokens, row, col0 + i * DCOL);
          uint4 w[2];
          widen<false>(kc[i], 0u, w);
          *reinterpret_cast<uint4*>(kt + off) = w[0];
          *reinterpret_cast<uint4*>(kt + (off ^ 16)) = w[1];
          widen<true>(zero || tok0 + row >= end ? make_uint4(0u, 0u, 0u, 0u) : vc[i], factor, w);
          *reinterpret_cast<uint4*>(vt + off) = w[0];
          *reinterpret_cast<uint4*>(vt + (off ^ 16)) = w[1];
        }
        if (ct == 0) {
          Note& note = notes[s];
          // (1 for a block that takes no part: where nothing has been written the scale may be anything, a sign included)
          note.ks[0] = take & 1u ? ks4.x * sl2 : 1.f;
          note.ks[1] = take & 2u ? ks4.y * sl2 : 1.f;
          note.ks[2] = take & 4u ? ks4.z * sl2 : 1.f;
          note.ks[3] = take & 8u ? ks4.w * sl2 : 1.f;
          note.tok0 = tok0;
          note.mask = take | (lost & take) << 4;
          note.eref = eref;
          note.end = 0;
        }
        left &= ~take;
        publish(s);
      }
    }
    if (ok && stage_free()) {
      if (ct == 0) notes[n % kStages].end = 1;
      publish(n % kStages);
    }
  } else if (warp == 9) {
    // ================================================================ copies
    const int* row_table = c.table + (size_t)sq.slot * c.max_pages;
    const size_t page_slabs = (size_t)c.layers * 2 * c.nkv, my_slab = (size_t)c.layer * 2 * c.nkv + h;  // K; V is nkv further
    int ids = 0, n = 0;  // the ids of 32 pages, one a lane; pages so far
    for (; n < p1 - p0; ++n) {
      if (n % 32 == 0) ids = p0 + n + lane < p1 ? row_table[p0 + n + lane] : -1;
      const int page = __shfl_sync(0xffffffffu, ids, n & 31), rs = n % kRaw;
      if (n >= kRaw) ok = mbar_wait_bounded(raw_empty + rs, (n / kRaw - 1) & 1, c.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        const bool have = unsigned(page) < unsigned(c.n_pages);
        raw_have[rs] = have;
        mbar_arrive_expect_tx(raw_full + rs, have ? 2 * C::SLAB + 32 : 0);
        if (have) {
          const size_t slab = page * page_slabs + my_slab;
          uint8_t* dst = smem + C::OFF_RAW + rs * 2 * C::SLAB;
          bulk_g2s(raw_scales + 2 * rs, c.scales + slab * kKv8BlocksPerPage, 16, raw_full + rs);
          bulk_g2s(raw_scales + 2 * rs + 1, c.scales + (slab + c.nkv) * kKv8BlocksPerPage, 16, raw_full + rs);
          bulk_g2s(dst, c.codes + slab * C::SLAB, C::SLAB, raw_full + rs);
          bulk_g2s(dst + C::SLAB, c.codes + (slab + c.nkv) * C::SLAB, C::SLAB, raw_full + rs);
        } else {
          set_error(c.err, kDevNoPage);
        }
      }
      __syncwarp();
    }
    if (lane == 0)  // no copy may be on its way when the CTA leaves
      for (int i = max(0, n - kRaw); i < n; ++i)
        if (!mbar_wait_bounded(raw_full + i % kRaw, (i / kRaw) & 1, c.err)) break;
    __syncwarp();
  } else if (warp == 8) {
    // ================================================================ matrix instructions
    if (lane == 0) {
      const uint32_t idesc_s = 1u << 4 | uint32_t(kPageTokens >> 3) << 17 | uint32_t(kRows >> 4) << 24;
      const uint32_t idesc_o = 1u << 4 | 1u << 16 | uint32_t(HD >> 3) << 17 | uint32_t(kRows >> 4) << 24;  // V: N-major
      auto scores = [&](int t) {  // false: the end, or a wait that ran out
        const int s = t % kStages;
        ok = mbar_wait_bounded(full + s, (t / kStages) & 1, c.err);
        if (!ok || notes[s].end) return false;
        tc_fence_after();
        const uint32_t kt = base + C::OFF_KV + s * 2 * C::KV_BYTES;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const int piece = 16 * k / C::PIECE, in = 16 * k % C::PIECE * 2;
          umma_f16(tmem + (t & 1) * kPageTokens, desc(base + piece * kRows * C::ROWB + in, 16, 8 * C::ROWB, C::LAYOUT),
                   desc(kt + piece * kPageTokens * C::ROWB + in, 16, 8 * C::ROWB, C::LAYOUT), idesc_s, k > 0);
        }
        umma_commit(s_full + (t & 1));
        return true;
      };
      bool more = scores(0);
      for (int t = 0; more; ++t) {
        more = scores(t + 1);
        if (!ok) break;
        ok = mbar_wait_bounded(p_ready, t & 1, c.err);
        if (!ok) break;
        tc_fence_after();
        const int s = t % kStages;
        const uint32_t vt = base + C::OFF_KV + s * 2 * C::KV_BYTES + C::KV_BYTES;
#pragma unroll
        for (int k = 0; k < kPageTokens / 16; ++k)
          umma_f16_ta(tmem + C::O_COL, tmem + (t & 1) * kPageTokens + k * 8,
                      desc(vt + k * 16 * C::ROWB, C::PIECE < HD ? kPageTokens * C::ROWB : 0, 8 * C::ROWB, C::LAYOUT), idesc_o,
                      t > 0 || k > 0);
        umma_commit(pv_done + (t & 1));
        umma_commit(empty + s);
      }
      umma_commit(drained);  // nothing may be running when the TMEM goes
      mbar_wait_bounded(drained, 0, c.err);
    }
    __syncwarp();
  } else {
    // ================================================================ softmax: thread = row
    const uint32_t lanes = uint32_t(warp * 32) << 16;
    const int fr = fr0 + min(tid, n_fr - 1);
    const int lim = sq.pos0 + fr / rep;  // the row's last position
    float m = kNoScore, l[4] = {0.f, 0.f, 0.f, 0.f};  // (four chains of sums)
    int eref = 0, t = 0;
    for (;; ++t) {
      const int s = t % kStages;
      ok = mbar_wait_bounded(full + s, (t / kStages) & 1, c.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const Note note = notes[s];
      if (note.end) break;
      ok = mbar_wait_bounded(s_full + (t & 1), (t >> 1) & 1, c.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_at = tmem + lanes + (t & 1) * kPageTokens;
      const bool edge = note.tok0 + kPageTokens - 1 > lim_lo || note.mask != 15u;
      const int seen = lim - note.tok0;
      // (a position that is not seen has no score, whatever its codes and scale are)
      auto none = [&](int i) { return i > seen || !(note.mask >> (i / 16) & 1); };
      float v[kPageTokens];
      tmem_fetch32(s_at, v);
      tmem_fetch32(s_at + 32, v + 32);
      tmem_arrived<kPageTokens>(v);
      if (edge) {
#pragma unroll
        for (int i = 0; i < kPageTokens; ++i) {
          if (none(i)) v[i] = -INFINITY;
          if (i % 16 == 0 && note.mask >> (4 + i / 16) & 1 && i <= seen) l[0] = __uint_as_float(0x7fc00000u);  // V is lost
        }
      }
      float mx = kNoScore;
#pragma unroll
      for (int j = 0; j < kPageTokens; j += 16) {
        float top[2] = {v[j], v[j + 1]};
#pragma unroll
        for (int k = 2; k < 16; ++k) top[k & 1] = fmaxf(top[k & 1], v[j + k]);
        mx = fmaxf(mx, fmaxf(top[0], top[1]) * note.ks[j / 16]);
      }
      if (__any_sync(0xffffffffu, mx > m + 8.f) || note.eref != eref) {
        const float m_new = fmaxf(m, mx);  // (NaN: m)
        const float f = ex2(m - m_new);
#pragma unroll
        for (int i = 0; i < 4; ++i) l[i] *= f;
        m = m_new;
        if (t > 0) {
          // (the scores of turn t were issued behind the product of turn t - 2: that one has ended)
          ok = mbar_wait_bounded(pv_done + ((t - 1) & 1), ((t - 1) >> 1) & 1, c.err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const int shift = eref - note.eref;  // -254 .. 64
          const float unit = f * ex2(float(max(shift, -126)));
          tc_fence_after();
#pragma unroll
          for (int d = 0; d < HD; d += 16) {
            float o[16];
            tmem_ld16(tmem + C::O_COL + lanes + d, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= unit;
            tmem_st16(tmem + C::O_COL + lanes + d, reinterpret_cast<const uint32_t*>(o));
          }
          tmem_st_wait();
        }
        eref = note.eref;
      }
      // P takes its scores' place in tensor memory
      auto emit = [&](auto masked) {  // (read again, as 64 values held on would not fit the registers)
#pragma unroll
        for (int j = 0; j < kPageTokens; j += 32) {
          float z[32];
          tmem_fetch32(s_at + j, z);
          tmem_arrived<32>(z);
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x = fmaf(z[i], note.ks[(j + i) / 16], -m), y = fmaf(z[i + 1], note.ks[(j + i) / 16], -m);
            if (masked.value) {  // (after the product: an infinity times a scale that is NaN)
              if (none(j + i)) x = -INFINITY;
              if (none(j + i + 1)) y = -INFINITY;
            }
            x = ex2(x);
            y = ex2(y);
            l[i & 3] += x;
            l[(i & 3) + 1] += y;
            w[i / 2] = pack_half2(x, y);
          }
          tmem_st16(s_at + j / 2, w);
        }
      };
      if (edge) emit(std::true_type{});
      else emit(std::false_type{});
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
    }
    // ---- the part's state, or the rows where the sequence has one part only
    if (ok && t > 0) {
      ok = mbar_wait_bounded(pv_done + ((t - 1) & 1), ((t - 1) >> 1) & 1, c.err);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    if (ok) {
      const float sum = (l[0] + l[1]) + (l[2] + l[3]);
      const float vref = eref > kUnit ? __uint_as_float(uint32_t(eref - kUnit) << 23)
                                      : __uint_as_float(1u << 23) * ex2(float(eref - kUnit - 1));
      const bool alone = pages <= split_pages;
      const float scale = alone ? (sum > 0.f || sum != sum ? vref / sum : 0.f) : vref;
      float* part = alone ? nullptr
                          : a.part + 4 + ((((size_t)seq * tiles + tile) * c.nkv + h) * a.splits + split) * kRows * (HD + 2);
      __half* out = a.out + ((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD;
#pragma unroll
      for (int d = 0; d < HD; d += 16) {
        float o[16];
        if (t > 0) {
          tmem_ld16(tmem + C::O_COL + lanes + d, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= scale;
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0.f;
        }
        if (tid >= n_fr) {
        } else if (alone) {
#pragma unroll
          for (int i = 0; i < 16; i += 8)
            *reinterpret_cast<uint4*>(out + d + i) = make_uint4(pack_half2(o[i], o[i + 1]), pack_half2(o[i + 2], o[i + 3]),
                                                                pack_half2(o[i + 4], o[i + 5]), pack_half2(o[i + 6], o[i + 7]));
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            part[(size_t)(d + i) * kRows + tid] = o[i];
        }
        __syncwarp();
      }
      if (!alone && tid < n_fr) {
        part[HD * kRows + tid] = m;
        part[(HD + 1) * kRows + tid] = sum;
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 8) tmem_dealloc<C::TMEM>(tmem);
}

// Joins the parts' states of a tile: a CTA takes 8 of its columns, a thread a row,
// as the parts lie there ([column][row], then m, then the sums), four groups of
// threads every fourth part each, in a fixed order. Bound by trips to L2.
constexpr int kMergeCols = 8, kMergeGroups = 4;
template <int HD>
__global__ void __launch_bounds__(kMergeGroups * kRows) kv8_prompts_merge_kernel(const Kv8AttnArgs a) {
  __shared__ float s_val[kMergeGroups][kMergeCols + 2][kRows];
  const Kv8Args& c = a.c;
  const int tid = threadIdx.x % kRows, group = threadIdx.x / kRows, tiles = a.tiles;
  const int tile = blockIdx.x / (HD / kMergeCols), d = blockIdx.x % (HD / kMergeCols) * kMergeCols;
  const int h = blockIdx.y, seq = blockIdx.z, rep = c.nq / c.nkv, fr0 = tile * kRows;
  const Kv8Seq sq = kv8_seq(c, a.max_ctx, seq, false);
  const int n_fr = min(kRows, sq.n * rep - fr0);
  pdl_wait();  // (ahead of every return: what comes next on the stream waits for this grid only)
  if (sq.slot < 0 || n_fr <= 0) return;
  const int split_pages = *reinterpret_cast<const int*>(a.part);
  const int parts = (tile_pages(sq, rep, tile) + split_pages - 1) / split_pages;
  if (parts == 1) return;
  constexpr size_t kState = size_t(kRows) * (HD + 2);
  const float* base = a.part + 4 + (((size_t)seq * tiles + tile) * c.nkv + h) * a.splits * kState + tid;
  float mx = kNoScore, sum = 0.f, val[kMergeCols] = {};
  if (tid < n_fr) {
#pragma unroll 8
    for (int s = group; s < parts; s += kMergeGroups) mx = fmaxf(mx, base[s * kState + HD * kRows]);
#pragma unroll 4
    for (int s = group; s < parts; s += kMergeGroups) {
      const float* p = base + s * kState;
      const float w = ex2(p[HD * kRows] - mx);
      sum += w * p[(HD + 1) * kRows];
#pragma unroll
      for (int i = 0; i < kMergeCols; ++i) val[i] += w * p[(d + i) * kRows];
    }
  }
#pragma unroll
  for (int i = 0; i < kMergeCols; ++i) s_val[group][i][tid] = val[i];
  s_val[group][kMergeCols][tid] = mx;
  s_val[group][kMergeCols + 1][tid] = sum;
  __syncthreads();
  if (group != 0 || tid >= n_fr) return;
#pragma unroll
  for (int g = 1; g < kMergeGroups; ++g) mx = fmaxf(mx, s_val[g][kMergeCols][tid]);
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMergeCols; ++i) val[i] = 0.f;
#pragma unroll
  for (int g = 0; g < kMergeGroups; ++g) {
    const float w = ex2(s_val[g][kMergeCols][tid] - mx);
    sum += w * s_val[g][kMergeCols + 1][tid];
#pragma unroll
    for (int i = 0; i < kMergeCols; ++i) val[i] += w * s_val[g][i][tid];
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const int fr = fr0 + tid;
  *reinterpret_cast<uint4*>(a.out + ((size_t)(sq.first + fr / rep) * c.nq + h * rep + fr % rep) * HD + d) =
      make_uint4(pack_half2(val[0] * inv, val[1] * inv), pack_half2(val[2] * inv, val[3] * inv),
                 pack_half2(val[4] * inv, val[5] * inv), pack_half2(val[6] * inv, val[7] * inv));
}

template <int HD>
cudaError_t prompts_hd(const Kv8AttnArgs& a, cudaStream_t s) {
  const int64_t items = (int64_t)a.tiles * a.c.nkv * a.c.n_seqs;
  kv8_prompts_kernel<HD><<<a.splits > 1 ? a.places : unsigned(items), kThreads, Prompts<HD>::SMEM, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || a.splits == 1) return e;
  cudaLaunchAttribute attr[1];  // its launch overlaps the end of the attention kernel
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.tiles * (HD / kMergeCols), a.c.nkv, a.c.n_seqs);
  cfg.blockDim = dim3(kMergeGroups * kRows);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv8_prompts_merge_kernel<HD>, a);
}

}  // namespace

cudaError_t launch_kv8_prompts(const Kv8AttnArgs& a, int hd, cudaStream_t s) {
  return hd == 16 ? prompts_hd<16>(a, s) : hd == 32 ? prompts_hd<32>(a, s)
         : hd == 64 ? prompts_hd<64>(a, s) : hd == 96 ? prompts_hd<96>(a, s)
         : hd == 128 ? prompts_hd<128>(a, s) : cudaErrorInvalidValue;
}
cudaError_t kv8_prompts_init_attributes() {
  for (const cudaError_t e :
       {set_kernel_smem(kv8_prompts_kernel<16>, Prompts<16>::SMEM), set_kernel_smem(kv8_prompts_kernel<32>, Prompts<32>::SMEM),
        set_kernel_smem(kv8_prompts_kernel<64>, Prompts<64>::SMEM), set_kernel_smem(kv8_prompts_kernel<96>, Prompts<96>::SMEM),
        set_kernel_smem(kv8_prompts_kernel<128>, Prompts<128>::SMEM)})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

}  // namespace mmc
