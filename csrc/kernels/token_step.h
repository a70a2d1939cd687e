// Launchers of the operators of one step of a served token model: rope.hip,
// kv_cache.hip, paged_attention.hip and lora.hip.
//
// Like the others (kernels.h) they are asynchronous on `stream`, allocate
// nothing and never synchronise.  Strides count elements; the last dimension of
// every tensor is contiguous.  They throw std::invalid_argument for what they do
// not take (a null pointer that is not called optional among it) and
// std::runtime_error for a launch that fails.
#pragma once

#include <hip/hip_runtime_api.h>
#include <hip/hip_vector_types.h>

#include <cstdint>

namespace sca::kern {

enum ElemType : int { kF32 = 0, kF16 = 1, kBF16 = 2, kE4M3 = 3, kI8 = 4 };

// n / d for n < 2^31 (the hardware divides no integers): with
// 2^(s-1) < d <= 2^s and mul = floor(2^32 (2^s - d) / d) + 1 the quotient is
// (high half of n * mul, + n) >> s (Granlund and Montgomery, 1994).
struct FastDiv {
  uint32_t d = 1, mul = 1, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((uint64_t(1) << shift) < d) ++shift;
    mul = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - d)) / d + 1);
  }
#ifdef __HIPCC__
  __device__ __forceinline__
#endif
  uint32_t div(uint32_t n) const { return (uint32_t((uint64_t(n) * mul) >> 32) + n) >> shift; }
};

// RMS norm of each head of q and k, then rotation of its first 2 * n_freq
// dimensions by pos * inv_freq, in one launch for both.
struct QkNormRopeArgs {
  const void* x[2] = {};        // q, k: [tokens, heads[i], dim]
  void* out[2] = {};            // may be x
  const void* weight[2] = {};   // [dim] or null (no learned weight)
  int heads[2] = {};
  int64_t x_token[2] = {}, x_head[2] = {}, out_token[2] = {}, out_head[2] = {};
  int64_t tokens = 0;
  int dim = 0;                  // even, <= 512
  int type = kBF16;             // of x and out: kF32, kF16 or kBF16
  int weight_f32 = 0;           // weights are fp32, not `type`
  const void* positions = nullptr;  // [tokens] int32 or int64
  int positions64 = 0;
  const void* inv_freq = nullptr;   // [n_freq] fp32 or fp64, radians per position
  int inv_freq64 = 0;
  int n_freq = 0;               // rotated pairs, <= dim / 2
  int interleaved = 0;          // pairs (2i, 2i + 1), else (i, i + n_freq)
  float eps = 1e-6f;
};
void qk_norm_rope(const QkNormRopeArgs& a, hipStream_t stream);

// Rows of k and v into a paged cache, or out of it.  An index of each pair is
// k's or v's.  A row whose slot is outside the cache is not written, and reads as zeros.
struct KvCacheArgs {
  void* x[2] = {};               // [rows, heads, dim]
  int64_t x_row[2] = {}, x_head[2] = {};
  int type = kBF16;              // of x: kF32, kF16 or kBF16
  void* cache[2] = {};           // [pages, page size, heads, dim]
  int64_t c_page[2] = {}, c_slot[2] = {}, c_head[2] = {};
  int cache_type = kBF16;
  float* scale[2] = {};          // [pages, page size, heads], of a kE4M3 or kI8 cache
  int64_t s_page[2] = {}, s_slot[2] = {}, s_head[2] = {};
  const void* slots = nullptr;   // [rows] int32 or int64
  int slots64 = 0;
  FastDiv page;                  // slots of a page
  int64_t slots_total = 0;       // pages * page size
  int64_t rows = 0;
  FastDiv heads;
  int dim = 0;                   // <= 512
};
void kv_cache_write(const KvCacheArgs& a, hipStream_t stream);
void kv_cache_read(const KvCacheArgs& a, hipStream_t stream);

// Attention of one new token for each request over a paged cache.  A token whose
// page is outside the cache is left out; a request that sees no token gets zeros
// and a logsumexp of -infinity.
struct PagedAttentionArgs {
  const void* q = nullptr;      // [batch, kv_heads * group, dim]
  int64_t q_batch = 0, q_head = 0;
  int type = kBF16;             // of q and out: kF16 or kBF16
  const void* cache[2] = {};    // k, v: [pages, page size, kv_heads, dim], of `type` or 8 bits
  int64_t c_page[2] = {}, c_slot[2] = {}, c_head[2] = {};
  int cache_type = kBF16;
  const float* cache_scale[2] = {};  // [pages, page size, kv_heads]
  int64_t s_page[2] = {}, s_slot[2] = {}, s_head[2] = {};
  const int32_t* table = nullptr;    // [batch, max_tokens / page size] pages
  int64_t table_row = 0;
  const int32_t* lengths = nullptr;  // [batch] tokens
  int pages = 0;
  FastDiv page;
  int max_tokens = 0;           // what a row of the table holds: longer lengths count as this
  int batch = 0, kv_heads = 0, group = 0, dim = 0;
  int window = 0;               // the last tokens that a request sees; 0: all
  float scale = 1.f;
  void* out = nullptr;          // [batch, kv_heads * group, dim], contiguous
  float* lse = nullptr;         // [batch, kv_heads * group] natural logsumexp of the scores, or null
  // filled in by paged_attention_plan()
  int q_heads = 0, row_blocks = 0, partial_rows = 0, grid = 0;
  float* partial_o = nullptr;   // [2 grid, partial_rows, padded dim]
  float* partial_ml = nullptr;  // [2 grid, partial_rows, 2]
};
// Checks the arguments, chooses the grid and returns the workspace in floats:
// partial_ml lies at its start, partial_o behind its 4 * grid * partial_rows floats.
int64_t paged_attention_plan(PagedAttentionArgs& a);
void paged_attention(const PagedAttentionArgs& a, hipStream_t stream);
int64_t paged_attention_workspace(int batch, int kv_heads, int group, int dim, bool eight_bit, int64_t max_tokens,
                                  int window);

// out = y + scale[a] * (x A[a]^T) B[a]^T for each row's adapter a.
struct LoraArgs {
  const void* x = nullptr;      // [rows, inner]
  const void* y = nullptr;      // [rows, outer]
  void* out = nullptr;          // [rows, outer], may be y
  int64_t x_row = 0, y_row = 0, out_row = 0;
  const void* A = nullptr;      // [adapters, rank, inner], contiguous
  const void* B = nullptr;      // [adapters, outer, rank], contiguous
  const void* ids = nullptr;    // [rows] int32 or int64; one that is no adapter leaves its row as y has it
  int ids64 = 0;
  const float* scales = nullptr;  // [adapters] or null
  int64_t rows = 0;
  int inner = 0, outer = 0, rank = 0, adapters = 0;
  int type = kBF16;             // of all but ids and scales: kF32, kF16 or kBF16
  float* h = nullptr;           // workspace of lora_workspace() floats
  // filled in by lora_add()
  int splits = 1, col_tiles = 1;
  int* grouped = nullptr;       // in the workspace: whether the rows lie in runs already
  int2* order = nullptr;        // else {row, adapter} sorted by adapter; null: never sorted
};
int64_t lora_workspace(int64_t rows, int inner, int rank, int adapters);
void lora_add(LoraArgs a, hipStream_t stream);

}  // namespace sca::kern
