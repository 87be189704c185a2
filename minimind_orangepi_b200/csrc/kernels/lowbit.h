// Host-side launch interface of the low-bit operators: the 8-bit paged KV cache
// (kv8*.cu) and the 4-bit projections (w4.cu). Plain device pointers, launches on
// the caller's stream.
#pragma once

#include "kernels.h"

namespace mmc {

// Error codes of the low-bit operators' device error words, after DeviceError's.
enum LowBitError : int {
  kDevBadSlot = 16,       // slot outside [0, max_seqs) (negative: an unused row, no error)
  kDevBadRows = 17,       // a sequence's rows leave the batch, are more than max_new, or their range runs backwards
  kDevContextLimit = 18,  // positions past max_ctx or the block table's pages, or a negative position
  kDevSlotTwice = 19,     // two sequences of one append have the same slot
};

constexpr int kKv8Block = 16;  // positions that share one scale of a kv head
constexpr int kKv8BlocksPerPage = kPageTokens / kKv8Block;

// One call's view of the cache and the batch.
struct Kv8Args {
  // cache: codes [n_pages][layers][2 (K, V)][nkv][64][hd] e4m3, scales [n_pages][layers][2][nkv][4] fp32
  uint8_t* codes = nullptr;
  float* scales = nullptr;
  const int* table = nullptr;    // [max_seqs][max_pages]
  const int* seq_pos = nullptr;  // [max_seqs] positions before this call's rows
  int* err = nullptr;
  int n_pages = 0, layers = 0, layer = 0, nkv = 0, max_seqs = 0, max_pages = 0;
  // batch: sequence i owns rows [row_start[i], row_start[i + 1]) (null: row i)
  const int* slots = nullptr;
  const int* row_start = nullptr;
  int n_seqs = 0, rows = 0, max_new = 0, nq = 0;
};

struct Kv8AppendArgs {
  Kv8Args c;
  const float* qkv = nullptr;                           // [rows][(nq + 2 nkv) * hd]
  const float *q_norm = nullptr, *k_norm = nullptr;     // [hd] or both null
  const float *rope_cos = nullptr, *rope_sin = nullptr; // [max_pos][hd / 2]
  int max_pos = 0;
  float eps = 0.f;
  __half* q = nullptr;  // [rows][nq * hd]
};
cudaError_t launch_kv8_append(const Kv8AppendArgs& a, int hd, cudaStream_t s);

struct Kv8AttnArgs {
  Kv8Args c;
  const __half* q = nullptr;  // [rows][nq * hd]
  __half* out = nullptr;      // [rows][nq * hd]
  int max_ctx = 0;
  int split_pages = 1, splits = 1;  // pages of a part, parts of max_ctx positions
  int tile_rows = 8, tiles = 1;     // rows of a tile, tiles of a sequence
  int places = 0;                   // long runs: CTAs on the GPU at once
  float* part = nullptr;            // splits > 1: the plan's part_floats
};
// How a call is split over `sms` SMs.
struct Kv8Plan {
  int split_pages = 1, splits = 1, tile_rows = 8, tiles = 1, places = 0;
  size_t part_floats = 0;
};
Kv8Plan kv8_plan(int n_seqs, int max_new, int nq, int nkv, int hd, int max_ctx, int sms);
cudaError_t launch_kv8_attention(const Kv8AttnArgs& a, int hd, cudaStream_t s);
cudaError_t kv8_init_attributes();

struct W4Args {
  const uint8_t* codes = nullptr;   // [N][K / 2], column 2i in the low half of byte i
  const __half* scales = nullptr;   // [N][K / group]
  const uint8_t* zeros = nullptr;   // [N][K / group] or null (8)
  const __half* x = nullptr;        // [B][K]
  float* y = nullptr;               // [B][N]
  int B = 0, N = 0, K = 0, group = 0;
};
cudaError_t launch_w4_projection(const W4Args& a, int sms, cudaStream_t s);
cudaError_t w4_init_attributes();

}  // namespace mmc
