// Several requests at once over a key/value cache held in 4 bits: the cache's layout and what batch_api.cpp launches.
#pragma once
#include "layers.hpp"

constexpr int kPage = 64;   // positions of a page
constexpr int kGroup = 64;  // values that share a scale and an offset

inline bool page_dim(int dim) { return dim == 64 || dim == 128 || dim == 256; }
// A head's part of a page: keys [64][dim / 2], values [64][dim / 2], then the keys' parameters [dim / 64][scale, offset][64]
// in binary16 and the values'.  A key's row is four quarters, quarter k its values 64 g + 16 k .. + 15 of every group g; a value's row
// sixteen pieces, piece c its values 64 g + 4 c .. + 3: a lane of the matrix instructions takes a quarter or a piece, and what it takes
// of one group is whole words, which can be multiplied ahead of their scale (paged_attention.hip).
__host__ __device__ inline int64_t page_head_bytes(int dim) { return 72ll * dim; }
__host__ __device__ inline int key_nibble(int dim, int i) { return (i % 64 / 16) * (dim / 4) + 16 * (i / 64) + i % 16; }
__host__ __device__ inline int value_nibble(int dim, int i) { return (i % 64 / 4) * (dim / 16) + 4 * (i / 64) + i % 4; }
// offset in bytes of parameter `which` (0: scale, 1: offset) of group g of the keys (value 0) or the values (1) at a page's position
__host__ __device__ inline int page_parameter(int dim, int value, int g, int which, int position) {
  return 64 * dim + value * 4 * dim + ((g * 2 + which) * kPage + position) * 2;
}
// what a table's entry and a slot may be used for: the page, or -1 where nothing is held
__host__ __device__ inline int held_page(int entry, int n_pages) { return entry >= 0 && entry < n_pages ? entry : -1; }
__host__ __device__ inline int slot_page(int slot, int n_pages) { return slot >= 0 && slot / kPage < n_pages ? slot / kPage : -1; }

// Means of values as the activations' type has them: what is finite and beyond binary16 is its largest number (15 s + z may be, and the mean of
// values at its end under rounded weights).
__device__ __forceinline__ half_t held(float v, half_t) { return (half_t)(fabsf(v) < INFINITY ? __builtin_amdgcn_fmed3f(v, -65504.0f, 65504.0f) : v); }
__device__ __forceinline__ bf16_t held(float v, bf16_t) { return (bf16_t)v; }

inline bool launchable(int64_t blocks, int threads) { return blocks * threads < (1ll << 32); }  // HIP takes no more

int launch_page_plan(const awq_page_plan_args& a, hipStream_t st);
int launch_paged_append(const awq_paged_append_args& a, bool bf16, hipStream_t st);
int launch_paged_rows(const awq_paged_rows_args& a, bool bf16, hipStream_t st);
int64_t paged_workspace_bytes(int n_requests, int heads, int kv_heads, int dim, int max_pages);
int launch_paged_attention(const awq_paged_attention_args& a, bool bf16, hipStream_t st);
int launch_packed_attention(const awq_packed_attention_args& a, bool bf16, hipStream_t st);
int64_t sample_workspace_bytes(int64_t n_rows, int64_t vocab);
int launch_sample(const awq_sample_args& a, int dtype, hipStream_t st);
