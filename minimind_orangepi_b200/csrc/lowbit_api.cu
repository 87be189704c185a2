// Entry points of the low-bit operators: append and attention over an 8-bit
// paged KV cache (kernels/kv8.cu, kv8_attention.cu, kv8_prompts.cu) and projections
// with 4-bit weights (kernels/w4.cu). Arguments that the host can see are checked here; what lies
// in device memory (slots, row ranges, positions, page ids) the kernels check
// before they use it and report in the cache's error word.
#include "../../include/minimind_cuda.h"
#include "kernels/lowbit.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

// Sets the thread-local text mmc_last_error() returns (defined in mmc_api.cu).
void mmc_set_last_error(const std::string& msg);

namespace {

struct Failure : std::runtime_error {
  int code;
  Failure(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

void require(bool ok, const char* msg) {
  if (!ok) throw Failure(MMC_ERR_INVALID, msg);
}
void ck(cudaError_t e, const char* what) {
  if (e != cudaSuccess) {
    cudaGetLastError();  // the caller's next CUDA call is not to find it
    throw Failure(MMC_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
}
// Runs f; nothing is thrown across the C boundary.
template <typename F>
int entry(F&& f) noexcept {
  try {
    f();
    return MMC_OK;
  } catch (const Failure& e) {
    try {
      mmc_set_last_error(e.what());
    } catch (...) {
    }
    return e.code;
  } catch (...) {
    try {
      mmc_set_last_error("unexpected exception");
    } catch (...) {
    }
    return MMC_ERR_CUDA;
  }
}

// The current device's SM count; kernel attributes are set once per device and thread.
int prepare_device() {
  static thread_local int done_dev = -1, sms = 0;
  int dev = 0;
  ck(cudaGetDevice(&dev), "device");
  if (done_dev != dev) {
    ck(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "device query");
    ck(mmc::kv8_init_attributes(), "attributes");
    ck(mmc::w4_init_attributes(), "attributes");
    done_dev = dev;
  }
  return sms;
}

// Refuses a pointer that the current device's kernels cannot read: host memory
// that is not mapped, or another device's.
void on_device(const void* p, const char* what) {
  cudaPointerAttributes at{};
  int dev = 0;
  ck(cudaGetDevice(&dev), "device");
  ck(cudaPointerGetAttributes(&at, p), what);
  if (at.type == cudaMemoryTypeManaged) return;
  require((at.type == cudaMemoryTypeDevice && at.device == dev) || (at.type == cudaMemoryTypeHost && at.devicePointer),
          what);
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

void check_batch(const mmc_kv8_cache* c, int32_t n_seqs, int32_t rows, int32_t max_new, int32_t nq) {
  require(c != nullptr, "null cache");
  require(c->n_pages >= 1 && c->layers >= 1 && c->nkv >= 1 && c->max_seqs >= 1 && c->max_pages >= 1,
          "cache sizes must be at least 1");
  require(c->hd == 16 || c->hd == 32 || c->hd == 64 || c->hd == 96 || c->hd == 128,
          "head_dim must be 16, 32, 64, 96 or 128");
  require(c->nkv <= 65535 && nq >= c->nkv && nq % c->nkv == 0 && nq <= 65535,
          "nq must be a multiple of nkv, at most 65535");
  require(n_seqs >= 1 && n_seqs <= 65535, "n_seqs must be in 1..65535");
  require(rows >= 1 && max_new >= 1 && max_new <= rows, "rows and max_new must be at least 1, max_new at most rows");
  require((int64_t)max_new * (nq / c->nkv) <= (int64_t(1) << 24), "max_new * (nq / nkv) is too large");
  const int64_t slabs = (int64_t)c->layers * 2 * c->nkv;  // of a page
  require(slabs < (int64_t(1) << 31) && c->n_pages * slabs < (int64_t(1) << 31), "n_pages * layers * 2 * nkv is too large");
}

mmc::Kv8Args make_args(const mmc_kv8_cache* c, int32_t layer, int32_t n_seqs, int32_t rows, int32_t max_new,
                       const int32_t* slots, const int32_t* row_start, int32_t nq) {
  require(layer >= 0 && layer < c->layers, "layer out of range");
  require(c->d_codes && c->d_scales && c->d_block_table && c->d_seq_pos && c->d_error && slots,
          "null cache, slots or error pointer");
  require(row_start != nullptr || (rows == n_seqs && max_new == 1),
          "without d_row_start each sequence has one row: rows == n_seqs, max_new == 1");
  require(aligned(c->d_codes, 16) && aligned(c->d_scales, 16), "d_codes and d_scales must be 16-byte aligned");
  mmc::Kv8Args k;
  k.codes = static_cast<uint8_t*>(c->d_codes);
  k.scales = c->d_scales;
  k.table = c->d_block_table;
  k.seq_pos = c->d_seq_pos;
  k.err = c->d_error;
  k.n_pages = c->n_pages;
  k.layers = c->layers;
  k.layer = layer;
  k.nkv = c->nkv;
  k.max_seqs = c->max_seqs;
  k.max_pages = c->max_pages;
  k.slots = slots;
  k.row_start = row_start;
  k.n_seqs = n_seqs;
  k.rows = rows;
  k.max_new = max_new;
  k.nq = nq;
  return k;
}

const char* error_text(int e) {
  switch (e) {
    case mmc::kDevWaitTimeout: return "a wait within the kernel ran out";
    case mmc::kDevNoPage: return "KV position not backed by a page of the pool";
    case mmc::kDevPositionLimit: return "position past the rotation tables (max_pos)";
    case mmc::kDevBadSlot: return "slot out of range";
    case mmc::kDevBadRows: return "a sequence's row range is not within the batch, or is longer than max_new";
    case mmc::kDevContextLimit: return "positions past max_ctx or the block table, or negative";
    case mmc::kDevSlotTwice: return "two sequences of one append have the same slot";
    default: return "unknown";
  }
}

}  // namespace

extern "C" {

int mmc_op_kv8_append(const mmc_kv8_cache* cache, int32_t layer, int32_t n_seqs, int32_t rows, int32_t max_new,
                      const int32_t* d_slots, const int32_t* d_row_start, int32_t nq, const float* d_qkv,
                      const float* d_q_norm, const float* d_k_norm, const float* d_rope_cos, const float* d_rope_sin,
                      int32_t max_pos, float eps, void* d_q_fp16, void* stream) {
  return entry([&] {
    check_batch(cache, n_seqs, rows, max_new, nq);
    mmc::Kv8AppendArgs a;
    a.c = make_args(cache, layer, n_seqs, rows, max_new, d_slots, d_row_start, nq);
    require(d_qkv && d_rope_cos && d_rope_sin && d_q_fp16, "null argument");
    require((d_q_norm == nullptr) == (d_k_norm == nullptr), "d_q_norm and d_k_norm go together");
    require(max_pos >= 1 && eps >= 0.f, "bad max_pos or eps");
    require(aligned(d_qkv, 16) && aligned(d_q_fp16, 16) && aligned(d_rope_cos, 16) && aligned(d_rope_sin, 16) &&
                aligned(d_q_norm, 16) && aligned(d_k_norm, 16),
            "d_qkv, norms, tables and d_q must be 16-byte aligned");
    on_device(cache->d_codes, "d_codes is not memory of the current device");
    on_device(d_qkv, "d_qkv is not memory of the current device");
    on_device(d_q_fp16, "d_q is not memory of the current device");
    prepare_device();
    a.qkv = d_qkv;
    a.q_norm = d_q_norm;
    a.k_norm = d_k_norm;
    a.rope_cos = d_rope_cos;
    a.rope_sin = d_rope_sin;
    a.max_pos = max_pos;
    a.eps = eps;
    a.q = static_cast<__half*>(d_q_fp16);
    ck(mmc::launch_kv8_append(a, cache->hd, static_cast<cudaStream_t>(stream)), "append launch");
  });
}

int mmc_op_kv8_attention_workspace_size(const mmc_kv8_cache* cache, int32_t n_seqs, int32_t rows, int32_t max_new,
                                        int32_t nq, int32_t max_ctx, size_t* bytes) {
  return entry([&] {
    check_batch(cache, n_seqs, rows, max_new, nq);
    require(bytes != nullptr, "null argument");
    require(max_ctx >= 1, "max_ctx must be at least 1");
    const mmc::Kv8Plan p = mmc::kv8_plan(n_seqs, max_new, nq, cache->nkv, cache->hd, max_ctx, prepare_device());
    *bytes = std::max<size_t>(16, p.part_floats * 4);
  });
}

int mmc_op_kv8_attention(const mmc_kv8_cache* cache, int32_t layer, int32_t n_seqs, int32_t rows, int32_t max_new,
                         const int32_t* d_slots, const int32_t* d_row_start, int32_t nq, const void* d_q_fp16,
                         int32_t max_ctx, void* d_out_fp16, void* d_workspace, size_t workspace_bytes, void* stream) {
  return entry([&] {
    check_batch(cache, n_seqs, rows, max_new, nq);
    mmc::Kv8AttnArgs a;
    a.c = make_args(cache, layer, n_seqs, rows, max_new, d_slots, d_row_start, nq);
    require(d_q_fp16 && d_out_fp16 && d_workspace, "null argument");
    require(max_ctx >= 1, "max_ctx must be at least 1");
    require(aligned(d_q_fp16, 16) && aligned(d_out_fp16, 16) && aligned(d_workspace, 16),
            "d_q, d_out and d_workspace must be 16-byte aligned");
    on_device(cache->d_codes, "d_codes is not memory of the current device");
    on_device(d_q_fp16, "d_q is not memory of the current device");
    on_device(d_out_fp16, "d_out is not memory of the current device");
    const mmc::Kv8Plan p = mmc::kv8_plan(n_seqs, max_new, nq, cache->nkv, cache->hd, max_ctx, prepare_device());
    require(workspace_bytes >= std::max<size_t>(16, p.part_floats * 4), "workspace too small");
    a.split_pages = p.split_pages;
    a.splits = p.splits;
    a.tile_rows = p.tile_rows;
    a.tiles = p.tiles;
    a.places = p.places;
    a.q = static_cast<const __half*>(d_q_fp16);
    a.out = static_cast<__half*>(d_out_fp16);
    a.max_ctx = max_ctx;
    a.part = static_cast<float*>(d_workspace);
    ck(mmc::launch_kv8_attention(a, cache->hd, static_cast<cudaStream_t>(stream)), "attention launch");
  });
}

int mmc_op_kv8_status(const mmc_kv8_cache* cache, void* stream) {
  return entry([&] {
    require(cache && cache->d_error, "null cache or error word");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int e = 0;
    ck(cudaMemcpyAsync(&e, cache->d_error, sizeof(int), cudaMemcpyDeviceToHost, s), "read error word");
    ck(cudaStreamSynchronize(s), "read error word");
    if (e != 0) {
      ck(cudaMemsetAsync(cache->d_error, 0, sizeof(int), s), "clear error word");
      ck(cudaStreamSynchronize(s), "clear error word");
      throw Failure(MMC_ERR_DEVICE, std::string("device error: ") + error_text(e) + " (code " + std::to_string(e) + ")");
    }
  });
}

int mmc_op_w4_projection(int32_t batch, int32_t n, int32_t k, int32_t group, const void* d_codes,
                         const void* d_scales_fp16, const void* d_zeros, const void* d_x_fp16, float* d_y,
                         void* stream) {
  return entry([&] {
    require(batch >= 1 && batch <= 65535 && n >= 1 && k >= 1, "batch (at most 65535), n and k must be at least 1");
    require(group == 32 || group == 64 || group == 128, "group must be 32, 64 or 128");
    require(k % group == 0, "k must be a multiple of group");
    require(n <= (1 << 30) && (int64_t)n * (k / group) < (int64_t(1) << 32), "n or n * (k / group) is too large");
    require(d_codes && d_scales_fp16 && d_x_fp16 && d_y, "null argument");
    require(aligned(d_codes, 16) && aligned(d_x_fp16, 16) && aligned(d_y, 16) && aligned(d_scales_fp16, 2),
            "d_codes, d_x and d_y must be 16-byte aligned");
    on_device(d_codes, "d_codes is not memory of the current device");
    on_device(d_x_fp16, "d_x is not memory of the current device");
    on_device(d_y, "d_y is not memory of the current device");
    const int sms = prepare_device();
    mmc::W4Args a;
    a.codes = static_cast<const uint8_t*>(d_codes);
    a.scales = static_cast<const __half*>(d_scales_fp16);
    a.zeros = static_cast<const uint8_t*>(d_zeros);
    a.x = static_cast<const __half*>(d_x_fp16);
    a.y = d_y;
    a.B = batch;
    a.N = n;
    a.K = k;
    a.group = group;
    ck(mmc::launch_w4_projection(a, sms, static_cast<cudaStream_t>(stream)), "projection launch");
  });
}

}  // extern "C"
