// Host-side launchers of the operators around a paged cache held in 8 bits.
//
// Cache of one layer: kv[page][kv_head][K | V][16 tokens][head_dim] in E4M3 (the layout of kernels.h, a byte an element) and
// scales[page][kv_head][K | V] in f32. A scale is a power of two, the smallest 2^e with e >= -100 whose 448 * 2^e holds the
// largest finite magnitude put into the page: multiplying by it and by its reciprocal is exact, so a page whose scale grows
// loses nothing but what falls below the new scale's smallest step.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "util.cuh"

namespace omni {

constexpr int kPageTokens = 16;

// Lets a kernel have `bytes` of dynamic shared memory and clusters of sixteen, once a device.
template <auto kKernel>
inline cudaError_t allow_large(int bytes) {
  static std::atomic<bool> done[64];
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
  if (done[device].load(std::memory_order_acquire)) return cudaSuccess;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done[device].store(true, std::memory_order_release);
  return e;
}

// ---- page tables ------------------------------------------------------------------------------------------------------

enum TablesStatus : int32_t {
  kTablesBadLength = 1,
  kTablesNoPages = 2,
  kTablesRows = 4,
  kTablesPages = 8,
  kTablesFree = 16,
};
constexpr int kTablesMaxSeqs = 4096;             // five words a sequence in shared memory
constexpr int kPackedMaxSeqs = 16384;            // a block looks through all of them before its first waits run out
constexpr int64_t kTablesMaxEntries = 1ll << 26;  // tokens of so many pages still add up within 31 bits

struct TablesCall {
  const int32_t *lens, *add;
  int n;
  int32_t* table;  // [n][width]
  int width;
  int32_t* free_pages;
  int free_cap;
  const int32_t* free_count;
  int32_t *lens_out, *free_count_out;  // may be lens and free_count
  int32_t *indptr, *pages;
  int page_cap;
  int32_t *row_ptr, *pos, *slot, *seq;
  int row_cap;
  int32_t* status;
};
cudaError_t launch_kv_tables(const TablesCall& c, cudaStream_t s);

// ---- norm + rotary embedding --------------------------------------------------------------------------------------------

// out[r][head] = rotated(norm(x[r][head]) * gain) of the first hq + hk heads of every row with pos[r] >= 0; no gains: no norm.
// head_dim 64 or 128; 16-byte aligned rows; out may be x (with the same stride).
cudaError_t launch_qk_norm_rope(const bf16* x, int64_t ldx, const bf16* q_norm, const bf16* k_norm, const int32_t* pos, int rows,
                                int q_heads, int kv_heads, int head_dim, float eps, float theta, bf16* out, int64_t ldo,
                                cudaStream_t s);

// ---- cache ----------------------------------------------------------------------------------------------------------------

// K and V of every row with slot[r] >= 0 into its slot (page * 16 + token). Rows of one page are neighbours in ascending slots.
cudaError_t launch_kv8_append(const bf16* k, int64_t ldk, const bf16* v, int64_t ldv, const int32_t* slot, int rows, uint8_t* kv,
                              float* scales, int kv_pages, int kv_heads, int head_dim, uint32_t* err, cudaStream_t s);

// One query row each: row n against tokens 0..pos[n] of sequence seq[n] (n where seq is nullptr); pos[n] < 0: zeros.
struct Kv8Attend {
  const bf16* q;
  int64_t ldq;
  const uint8_t* kv;
  const float* scales;
  int kv_pages;
  const int32_t *pos, *seq, *indptr, *pages;
  int n_seqs, n_pages;  // indptr has n_seqs + 1 words, pages n_pages
  int rows, q_heads, kv_heads, head_dim;
  float scale;
  bf16* out;
  int64_t ldo;
};
// `pool`: where sums of rows in pieces are kept for the length of the call, in the stream's order.
cudaError_t launch_kv8_attend(const Kv8Attend& a, int sm_count, cudaMemPool_t pool, uint32_t* err, cudaStream_t s);

// ---- prompts ----------------------------------------------------------------------------------------------------------------

// Causal attention within each of n sequences, rows indptr[i] .. indptr[i + 1] of the packed q, k, v; other rows of out stay.
struct PackedAttend {
  const bf16* q;
  int64_t ldq;
  const bf16* k;
  int64_t ldk;
  const bf16* v;
  int64_t ldv;
  const int32_t* indptr;
  int n, rows, q_heads, kv_heads, head_dim;
  float scale;
  bf16* out;
  int64_t ldo;
};
cudaError_t launch_packed_attend(const PackedAttend& a, int sm_count, uint32_t* err, cudaStream_t s);

}  // namespace omni
