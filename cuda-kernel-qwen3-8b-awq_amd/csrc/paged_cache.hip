// Rotary positions with the append to a cache in 4 bits, and its rows read back (batch.hpp).
#include "batch.hpp"
#include "lane_sums.hpp"

namespace {

template <typename T>
struct Eight {
  typedef T type __attribute__((ext_vector_type(8)));
};

__device__ __forceinline__ void narrow(float v, half_t& to) { to = to_half_rn(v); }
__device__ __forceinline__ void narrow(float v, bf16_t& to) { to = (bf16_t)v; }
// 64 bits to 16 in one rounding: by way of a binary32 number whose last bit says that something was cut off, which lies on the same side of
// every border of the 16-bit type
template <typename T>
__device__ __forceinline__ T rounded(double d) {
  float f = (float)d;
  if ((double)f != d) {
    uint32_t u = __float_as_uint(f);
    if (fabs((double)f) > fabs(d)) --u;
    f = __uint_as_float(u | 1u);
  }
  T to;
  narrow(f, to);
  return to;
}

// n s + z in one rounding: a multiply-add of binary16, or the sum of binary32 with the last bit as above (the product is exact, and the sum's
// rounding error is a number of binary32)
__device__ __forceinline__ half_t value_of(float n, half_t s, half_t z, half_t) { return __builtin_fmaf16((half_t)n, s, z); }
__device__ __forceinline__ bf16_t value_of(float n, half_t s, half_t z, bf16_t) {
  const float a = n * (float)s, b = (float)z;
  float f = a + b;
  const float rest = f - a, left = (a - (f - rest)) + (b - rest);
  if (left != 0.0f) {
    uint32_t u = __float_as_uint(f);
    if ((left < 0.0f) != (f < 0.0f)) --u;
    f = __uint_as_float(u | 1u);
  }
  return (bf16_t)f;
}

constexpr float kHalfMax = 65504.0f;

// A thread takes eight values of a head of a token, so that 64 values with one scale are eight lanes side by side and a head is within
// a wavefront.  Everything behind the load is in 64 bits, in which the turned values are exact: a value next to a border of the
// number format, and a quotient next to a half, then go where the formula sends them.
// 8,000 positions of 32 + 8 heads of 128, 64 of them turned, bfloat16: 56 us traced, 3.4 TB/s of what it reads and writes (190 MB), beside vector
// instructions for most of that time.  64 positions: 4 us, a launch.
template <typename T>
__global__ __launch_bounds__(256) void append_kernel(awq_paged_append_args a, int blocks) {
  typedef typename Eight<T>::type eight_t;
  const int64_t t = blockIdx.x / blocks;
  const int position = a.positions[t];
  const int slot = a.cache ? a.slots[t] : -1;
  const int dim = a.dim, shift = __builtin_ctz(dim) - 3;  // a head is a power of two
  const int unit = (int)(blockIdx.x - (uint32_t)t * blocks) * 256 + threadIdx.x;
  const int heads = a.q ? a.heads : 0, keys = a.k ? a.kv_heads : 0;
  int item = unit >> shift, at = (unit & ((1 << shift) - 1)) * 8;
  if (a.rot <= kGroup) {
    // all heads' first 64 values, then the next: a wavefront's lanes are turned together or not at all (half of heads of 128 turned: 55 us, head by head
    // 60; with more than 64 turned a pair may lie in two of these parts)
    const int items = heads + (a.cache ? 2 : 1) * keys, groups = dim / kGroup;
    item = unit >> 3;
    at = (unit & 7) * 8;
    for (int g = 1; g < groups; ++g)
      if (item >= items) item -= items, at += kGroup;
  }
  const bool is_q = item < heads, is_k = !is_q && item < heads + keys;
  const bool is_v = !is_q && !is_k && a.cache && item < heads + 2 * keys;
  const int head = is_q ? item : is_k ? item - heads : item - heads - keys;
  const T* src = is_q ? (const T*)a.q + t * a.ldq : is_k ? (const T*)a.k + t * a.ldk : (const T*)a.v + t * a.ldv;
  eight_t x;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (T)0.0f;
  if (is_q || is_k || is_v) x = *reinterpret_cast<const eight_t*>(src + (int64_t)head * dim + at);
  if (position < 0 || position >= a.max_pos) return;
  const int half = a.rot / 2;
  const bool turned = (is_q || is_k) && at < a.rot;
  if (a.interleaved) {
    if (turned) {
      typedef float f32x4_t __attribute__((ext_vector_type(4)));
      const f32x4_t c = *reinterpret_cast<const f32x4_t*>(a.cosines + (int64_t)position * half + at / 2);
      const f32x4_t s = *reinterpret_cast<const f32x4_t*>(a.sines + (int64_t)position * half + at / 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double u = (double)(float)x[2 * i], v = (double)(float)x[2 * i + 1], cd = (double)c[i], sd = (double)s[i];
        x[2 * i] = rounded<T>(u * cd - v * sd);
        x[2 * i + 1] = rounded<T>(u * sd + v * cd);
      }
    }
  } else if (a.rot && __builtin_amdgcn_ballot_w64(turned)) {
    // the other halves of the pairs are half / 8 lanes away; they are exchanged ahead of any store, so that q_out may be q
    const bool first = at < half;
    const int other = (int)(threadIdx.x & 63) + (turned ? (first ? half / 8 : -half / 8) : 0);
    typedef int i32x4_t __attribute__((ext_vector_type(4)));
    const i32x4_t mine = __builtin_bit_cast(i32x4_t, x);
    i32x4_t theirs;
#pragma unroll
    for (int i = 0; i < 4; ++i) theirs[i] = __shfl(mine[i], other, 64);
    const eight_t y = __builtin_bit_cast(eight_t, theirs);
    if (turned) {
      const float* const c = a.cosines + (int64_t)position * half + (first ? at : at - half);
      const float* const s = a.sines + (int64_t)position * half + (first ? at : at - half);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double u = (double)(float)x[i], v = (double)(float)y[i], cd = (double)c[i], sd = (double)s[i];
        x[i] = rounded<T>(first ? u * cd - v * sd : u * cd + v * sd);
      }
    }
  }
  if (is_q) *reinterpret_cast<eight_t*>((T*)a.q_out + t * a.ldq_out + (int64_t)head * dim + at) = x;
  if (is_k && a.k_out) *reinterpret_cast<eight_t*>((T*)a.k_out + t * a.ldk_out + (int64_t)head * dim + at) = x;
  const int page = slot_page(slot, a.n_pages);
  if (page < 0 || (!is_k && !is_v)) return;
  float least = INFINITY, largest = -INFINITY, bad = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = (float)x[i];
    if (!(fabsf(v) < INFINITY)) bad = 1.0f;
    least = fminf(least, v);
    largest = fmaxf(largest, v);
  }
  least = -lanes::maximum<8>(-least);
  largest = lanes::maximum<8>(largest);
  bad = lanes::maximum<8>(bad);
  half_t offset, scale;
  uint32_t word = 0;
  if (bad != 0.0f) {
    offset = scale = __builtin_bit_cast(half_t, (uint16_t)0x7e00);
  } else {
    offset = to_half_rn(fminf(fmaxf(least, -kHalfMax), kHalfMax)) + (half_t)0.0f;  // (one zero)
    scale = rounded<half_t>(fmin(((double)largest - (double)least) / 15.0, (double)kHalfMax));
    const double z = (double)(float)offset, s = (double)(float)scale;
    const float inverse = 1.0f / fmaxf((float)scale, 1e-10f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // (a guess that is off by one at most, put right by what is left of the exact difference)
      const double d = (double)(float)x[i] - z;
      float n = rintf(fminf(fmaxf((float)d * inverse, 0.0f), 15.0f));
      const double left = d - (double)n * s, half_step = 0.5 * s;
      const bool odd = ((int)n & 1) != 0;
      if (left > half_step || (left == half_step && odd)) n += 1.0f;
      else if (left < -half_step || (left == -half_step && odd)) n -= 1.0f;
      n = s > 0.0 ? fminf(fmaxf(n, 0.0f), 15.0f) : 0.0f;
      word |= (uint32_t)n << (4 * i);
    }
  }
  uint8_t* const base = (uint8_t*)a.cache + ((int64_t)page * a.kv_heads + head) * page_head_bytes(dim);
  const int p = slot % kPage, g = at / kGroup;
  if (is_k) {
    *reinterpret_cast<uint32_t*>(base + p * (dim / 2) + key_nibble(dim, at) / 2) = word;
  } else {
    uint8_t* const row = base + 32 * dim + p * (dim / 2);
    *reinterpret_cast<uint16_t*>(row + value_nibble(dim, at) / 2) = (uint16_t)word;
    *reinterpret_cast<uint16_t*>(row + value_nibble(dim, at + 4) / 2) = (uint16_t)(word >> 16);
  }
  if (at % kGroup == 0) {
    *reinterpret_cast<half_t*>(base + page_parameter(dim, is_v, g, 0, p)) = scale;
    *reinterpret_cast<half_t*>(base + page_parameter(dim, is_v, g, 1, p)) = offset;
  }
}

constexpr int kRowsStarts = 4096;

// A thread takes eight values of a row of keys or values; the request of a row is looked up among the starts.
// 8,000 rows of 8 heads of 128, bfloat16: 22 us traced, 17 in a row, for 42 MB; bound by its 350 instructions a thread, 100 of them for eight roundings that are one each
// (the requests' numbers in LDS for two trips to memory fewer: no gain).
template <typename T>
__global__ __launch_bounds__(256) void rows_kernel(awq_paged_rows_args a) {
  typedef typename Eight<T>::type eight_t;
  __shared__ int starts_of[kRowsStarts];
  const int n = a.n_requests;
  const bool here = n <= kRowsStarts;
  if (here)
    for (int i = threadIdx.x; i < n; i += 256) starts_of[i] = a.starts[i];
  __syncthreads();
  const int dim = a.dim, half = a.kv_heads * dim / 8, units = ((a.k != nullptr) + (a.v != nullptr)) * half;
  // (a 64-bit division takes longer than the rest of a row's eighth)
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, row = gridDim.x < 1u << 24 ? (int64_t)((uint32_t)unit / (uint32_t)units) : unit / units;
  if (row >= a.n_rows) return;
  const int in_row = (int)(unit - row * units);
  int lo = 0, hi = n;  // the last request that does not start behind the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((here ? starts_of[mid] : a.starts[mid]) <= row) lo = mid;
    else hi = mid;
  }
  const int start = here ? starts_of[lo] : a.starts[lo];
  if (row < start || row >= a.starts[lo + 1]) return;
  const int64_t p64 = (a.first ? max(a.first[lo], 0) : 0) + row - start;
  if (p64 >= min(a.lengths[lo], a.max_pages * kPage)) return;
  const bool value = a.k == nullptr || in_row >= half;
  const int p = (int)p64, in_heads = (in_row >= half ? in_row - half : in_row) * 8, at = in_heads & (dim - 1), head = in_heads >> __builtin_ctz(dim);
  const int page = held_page(a.table[(int64_t)lo * a.max_pages + p / kPage], a.n_pages);
  eight_t y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (T)0.0f;
  if (page >= 0) {
    const uint8_t* const base = (const uint8_t*)a.cache + ((int64_t)page * a.kv_heads + head) * page_head_bytes(dim);
    const int in_page = p % kPage, g = at / kGroup;
    uint32_t word;
    if (!value) {
      word = *reinterpret_cast<const uint32_t*>(base + in_page * (dim / 2) + key_nibble(dim, at) / 2);
    } else {
      const uint8_t* const r = base + 32 * dim + in_page * (dim / 2);
      word = *reinterpret_cast<const uint16_t*>(r + value_nibble(dim, at) / 2) |
             (uint32_t)*reinterpret_cast<const uint16_t*>(r + value_nibble(dim, at + 4) / 2) << 16;
    }
    const half_t s = *reinterpret_cast<const half_t*>(base + page_parameter(dim, value, g, 0, in_page));
    const half_t z = *reinterpret_cast<const half_t*>(base + page_parameter(dim, value, g, 1, in_page));
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = value_of((float)((word >> (4 * i)) & 15u), s, z, T());
    if constexpr (__is_same(T, half_t)) {
      const float furthest = fabsf(15.0f * (float)s + (float)z);  // (z is one of its numbers)
      if (furthest > kHalfMax && furthest < INFINITY) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (half_t)__builtin_amdgcn_fmed3f((float)y[i], -kHalfMax, kHalfMax);
      }
    }
  }
  T* const out = value ? (T*)a.v + row * a.ldv : (T*)a.k + row * a.ldk;
  *reinterpret_cast<eight_t*>(out + (int64_t)head * dim + at) = y;
}

}  // namespace

int launch_paged_append(const awq_paged_append_args& a, bool bf16, hipStream_t st) {
  const int items = (a.q ? a.heads : 0) + (a.k ? a.kv_heads : 0) + (a.k && a.cache ? a.kv_heads : 0);
  if (a.n_tokens == 0 || items == 0) return AWQ_OK;
  const int blocks = (items * (a.dim / 8) + 255) / 256;
  AWQ_REQUIRE(launchable(a.n_tokens * blocks, 256), "too many tokens and heads");
  const auto kernel = bf16 ? append_kernel<bf16_t> : append_kernel<half_t>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.n_tokens * blocks)), dim3(256), 0, st, a, blocks);
  AWQ_HIP_TRY(hipGetLastError());
  return AWQ_OK;
}

int launch_paged_rows(const awq_paged_rows_args& a, bool bf16, hipStream_t st) {
  if (a.n_rows == 0 || (!a.k && !a.v)) return AWQ_OK;
  const int64_t units = a.n_rows * ((a.k != nullptr) + (a.v != nullptr)) * (a.kv_heads * a.dim / 8);
  AWQ_REQUIRE(launchable((units + 255) / 256, 256), "too many rows and heads");
  const auto kernel = bf16 ? rows_kernel<bf16_t> : rows_kernel<half_t>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((units + 255) / 256)), dim3(256), 0, st, a);
  AWQ_HIP_TRY(hipGetLastError());
  return AWQ_OK;
}
