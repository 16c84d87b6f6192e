// Attention of one query a request over a cache in 4 bits (batch.hpp).
#include "batch.hpp"

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;     // of a workgroup, each with pages of its own
constexpr int kColumns = 16;  // query heads of one key/value head that share a pass over the pages

inline int columns_of(int group) { return std::min(group, kColumns); }
inline int streams_of(int heads, int kv_heads) { return kv_heads * ((heads / kv_heads + kColumns - 1) / kColumns); }
// wavefronts that share the pages of a stream (a key/value head and up to 16 of its query heads): as many as the chip holds with two
// pages each in LDS
inline int workers_of(int n_requests, int heads, int kv_heads, int dim, int max_pages) {
  const int64_t there = 256ll * (dim == 64 ? 16 : dim == 128 ? 8 : 4) / streams_of(heads, kv_heads);
  const int64_t most = (int64_t)n_requests * max_pages;
  return (int)std::max<int64_t>(kWaves, (std::min(there, most) + kWaves - 1) / kWaves * kWaves);
}

struct PagedArgs {
  awq_paged_attention_args a;
  int workers, streams, columns;
  float* sums;  // [streams][workers][2][columns][dim]
  float* ml;    // [streams][workers][2][columns][2]
};

template <int N>
__device__ __forceinline__ void wait_for_requests() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// sums and maxima over the four lanes with one lane % 16
__device__ __forceinline__ float over_quarters_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float over_quarters_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

__device__ __forceinline__ int pages_of(const awq_paged_attention_args& a, int r) {
  return (min(max(a.lengths[r], 0), a.max_pages * kPage) + kPage - 1) / kPage;
}

// Pages of the requests ahead of this lane's (64 runs of ceil(n / 64) requests, a lane each), and of all.
__device__ __forceinline__ int pages_ahead(const awq_paged_attention_args& a, int lane, int run, int& all) {
  int mine = 0;
  for (int r = lane * run; r < min((lane + 1) * run, a.n_requests); ++r) mine += pages_of(a, r);
  int sum = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(sum, off, 64);
    if (lane >= off) sum += v;
  }
  all = __builtin_amdgcn_readlane(sum, 63);
  return sum - mine;
}
__device__ __forceinline__ int first_page(int64_t worker, int all, int workers) { return (int)(worker * all / workers); }

// The pages of all requests in a row are cut evenly over `workers` wavefronts; a worker walks the requests that its run touches.  A page
// comes into LDS as it lies in memory but for the order of its 16-byte pieces, the next one while this one is worked on.  Operands of
// v_mfma_f32_16x16x32_f16, lane (m, kg) = (lane % 16, lane / 16), heads as columns:
//     S[key][head] = K q^T        sixteen keys; a lane takes quarter kg of key m's row
//     O[c][head] += V^T P         two of sixteen keys; a lane takes piece m of the rows of the keys 4 kg .. + 3 of both
// so that the weights a lane forms are the elements it supplies to the second product.  Nibbles go into the products as they are: as the last
// bits of a binary16 number they stand for n 2^-24, four bits up for 16 times that (the query's values there are divided by 16, and
// so are the sums of the values' pieces), so that a word of eight takes five instructions.  The scales are put on afterwards: on a key's
// sum over a group, s sum(q n) + z sum(q) in binary32, and on the weights, p s rounded to binary16 for the product, p z in binary32.
// Weights are relative to the largest of score + exponent of the page's largest value scale, so that p s is below 1 and as exact as
// binary16 can be whatever the values' size.
template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void paged_kernel(PagedArgs p) {
  constexpr int G = D / 64, PIECES = D / 32;  // groups; 16-byte pieces of a row
  constexpr int kBytes = 72 * D, kLoads = (kBytes / 16 + 63) / 64;
  typedef __attribute__((address_space(1))) const void* gptr_t;
  typedef __attribute__((address_space(3))) void* lptr_t;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves * 2 * kBytes];
  const awq_paged_attention_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, kg = lane >> 4;
  const int stream = blockIdx.x % p.streams, worker = blockIdx.x / p.streams * kWaves + wave;
  const int tiles = p.streams / a.kv_heads, kv_head = stream / tiles, group = a.heads / a.kv_heads;
  const int head0 = kv_head * group + stream % tiles * kColumns, columns = min(kColumns, group - stream % tiles * kColumns);
  uint8_t* const mine = lds + wave * 2 * kBytes;

  const int run = (a.n_requests + 63) / 64;
  int all;
  const int ahead = pages_ahead(a, lane, run, all);
  const int begin = first_page(worker, all, p.workers), end = first_page(worker + 1, all, p.workers);
  if (begin >= end) return;
  // the request of the first page: the last run of requests that does not start behind it, then one after the other
  const int at = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(ahead <= begin));
  int r = at * run, start = __builtin_amdgcn_readlane(ahead, at), n_pages = pages_of(a, r);
  while (start + n_pages <= begin) {
    start += n_pages;
    n_pages = pages_of(a, ++r);
  }

  // where the lane's 16 bytes of a request into LDS come from: a key's pieces rotated among its row's, so that those that lanes read together
  // lie in all banks; rows of values with those four apart side by side
  const auto piece_at = [&](int i) __attribute__((always_inline)) {
    const int x = 64 * i + lane;
    if (x < 64 * PIECES) {
      const int row = x / PIECES, part = x % PIECES;
      return row * PIECES + (part ^ ((row * PIECES / 16) & (PIECES - 1)));
    }
    if (x < 128 * PIECES) {
      const int slot = x / PIECES - 64, part = x % PIECES;
      return (64 + (slot & ~15) + (slot & 3) * 4 + ((slot & 15) >> 2)) * PIECES + part;
    }
    return x;
  };
  const auto request = [&](int page, int buffer) __attribute__((always_inline)) {
    const uint8_t* const src = (const uint8_t*)a.cache + ((int64_t)page * a.kv_heads + kv_head) * kBytes;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (64 * (i + 1) <= kBytes / 16 || lane < kBytes / 16 - 64 * i)
        __builtin_amdgcn_global_load_lds((gptr_t)(src + piece_at(i) * 16), (lptr_t)(mine + buffer * kBytes + i * 1024), 16, 0, 0);
  };

  for (int at_page = begin; at_page < end; ++r) {
    // one request: pages from .. to of it
    const int length = min(max(a.lengths[r], 0), a.max_pages * kPage);
    n_pages = (length + kPage - 1) / kPage;
    if (n_pages == 0) continue;
    const int from = at_page - start, to = min(n_pages, end - start);
    const int32_t* const table = a.table + (int64_t)r * a.max_pages;

    // the query: lane (m, kg) has values 64 g + 16 kg + 8 j .. + 7 of head m
    half8_t qop[2 * G];
    float q_sum[G], q_max = 0.0f;
    {
      float qv[2 * G][8];
      const T* const q = (const T*)a.q + (int64_t)r * a.ldq + (int64_t)(head0 + m) * D + 16 * kg;
      typedef T eight_t __attribute__((ext_vector_type(8)));
#pragma unroll
      for (int i = 0; i < 2 * G; ++i) {
        eight_t x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (T)0.0f;
        if (m < columns) x = *reinterpret_cast<const eight_t*>(q + 64 * (i / 2) + 8 * (i % 2));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          qv[i][e] = (float)x[e];
          q_max = fmaxf(q_max, fabsf(qv[i][e]));
        }
      }
      q_max = over_quarters_max(q_max);
      // a power of two brings the largest to 2^14: nothing is lost of what is within 2^-24 of it
      int e2 = 0;
      if (q_max > 0.0f && q_max < INFINITY) e2 = 15 - __builtin_amdgcn_frexp_expf(q_max);
      const float up = __builtin_amdgcn_ldexpf(1.0f, max(min(e2, 100), -100)), more = __builtin_amdgcn_ldexpf(1.0f, e2 - max(min(e2, 100), -100));
#pragma unroll
      for (int g = 0; g < G; ++g) {
        q_sum[g] = 0.0f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = qv[2 * g + j][e] * up * more;
            q_sum[g] += v[e];
          }
          qop[2 * g + j] = half8_t{(half_t)v[0], (half_t)v[4], (half_t)(v[1] * 0.0625f), (half_t)(v[5] * 0.0625f),
                                   (half_t)v[2], (half_t)v[6], (half_t)(v[3] * 0.0625f), (half_t)(v[7] * 0.0625f)};
        }
        q_sum[g] = over_quarters_sum(q_sum[g]);
      }
      q_max = __builtin_amdgcn_ldexpf(a.scale * 1.44269504088896340736f, -e2);
    }
    const float mul = q_max;

    f32x4_t o[G][4];
    float off[G], best = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      off[g] = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[g][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int entries = -1, entries_at = -64;
    const auto page_at = [&](int i) __attribute__((always_inline)) {
      if (i >= entries_at + 64) {
        entries_at = i;
        entries = i + lane < n_pages ? table[i + lane] : -1;
        // (waited for here: behind the branch the wait would be one for the pages on their way too, every time)
        asm volatile("" : "+v"(entries));
      }
      return held_page(__builtin_amdgcn_readlane(entries, i - entries_at), a.n_pages);
    };
    int page = page_at(from);
    if (page >= 0) request(page, 0);
    for (int i = from; i < to; ++i) {
      const int buffer = (i - from) & 1;
      const int next = i + 1 < to ? page_at(i + 1) : -1;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other buffer has been read
      if (next >= 0) {
        request(next, buffer ^ 1);
        wait_for_requests<kLoads>();
      } else {
        wait_for_requests<0>();
      }
      const int here = page;
      page = next;
      if (here < 0) continue;
      const uint8_t* const kb = mine + buffer * kBytes;
      const uint8_t* const vb = kb + 32 * D;
      const int left = length - i * kPage;  // positions of this page

      float score[4][4];
      float highest = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int row = 16 * t + m, turn = (row * PIECES / 16) & (PIECES - 1);
        uint32_t w[2 * G];
        if constexpr (G == 1) {
          const u32x2_t x = *reinterpret_cast<const u32x2_t*>(kb + row * 32 + (((kg >> 1) ^ turn) * 16) + (kg & 1) * 8);
          w[0] = x[0], w[1] = x[1];
        } else {
#pragma unroll
          for (int i4 = 0; i4 < G / 2; ++i4) {
            const u32x4_t x = *reinterpret_cast<const u32x4_t*>(kb + row * (D / 2) + ((kg * (G / 2) + i4) ^ turn) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * i4 + e] = x[e];
          }
        }
        f32x4_t s[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          s[g] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x = w[2 * g + j], y = x >> 8;
            const u32x4_t op = u32x4_t{x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
            s[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, op), qop[2 * g + j], s[g], 0, 0, 0);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) score[t][e] = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const half4_t sc = *reinterpret_cast<const half4_t*>(kb + page_parameter(D, 0, g, 0, 16 * t + 4 * kg));
          const half4_t zz = *reinterpret_cast<const half4_t*>(kb + page_parameter(D, 0, g, 1, 16 * t + 4 * kg));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            score[t][e] = __builtin_fmaf((float)sc[e], s[g][e] * 0x1p24f, __builtin_fmaf((float)zz[e], q_sum[g], score[t][e]));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          score[t][e] = 16 * t + 4 * kg + e < left ? score[t][e] * mul : -INFINITY;
          highest = fmaxf(highest, score[t][e]);
        }
      }
      half4_t vs[G][4], vz[G][4];
      float widest = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          vs[g][t] = *reinterpret_cast<const half4_t*>(kb + page_parameter(D, 1, g, 0, 16 * t + 4 * kg));
          vz[g][t] = *reinterpret_cast<const half4_t*>(kb + page_parameter(D, 1, g, 1, 16 * t + 4 * kg));
          if (left < kPage) {  // whatever lies behind the last position
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (16 * t + 4 * kg + e >= left) vs[g][t][e] = vz[g][t][e] = (half_t)0.0f;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) widest = fmaxf(widest, (float)vs[g][t][e]);
        }
      highest = over_quarters_max(highest);
      widest = over_quarters_max(widest);
      const float to_best = fmaxf(best, highest + (float)(widest > 0.0f ? __builtin_amdgcn_frexp_expf(widest) : -24));
      if (__builtin_amdgcn_ballot_w64(to_best > best)) {
        const float alpha = to_best > best ? __builtin_amdgcn_exp2f(best - to_best) : 1.0f;
        best = to_best;
        sum *= alpha;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          off[g] *= alpha;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[g][j] *= alpha;
        }
      }
      const float base = best == -INFINITY ? 0.0f : best;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        half8_t pop[G];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = 2 * u + (e >> 2);
          const float w = __builtin_amdgcn_exp2f(score[t][e & 3] - base);
          sum += w;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            pop[g][e] = (half_t)(w * (float)vs[g][t][e & 3]);
            off[g] = __builtin_fmaf(w, (float)vz[g][t][e & 3], off[g]);
          }
        }
        // rows of the keys 4 kg + e of both sixteens, this lane's piece of each
        uint32_t row[8][(G + 1) / 2];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint8_t* const v = vb + (32 * u + 16 * (e >> 2) + (e & 3) * 4 + kg) * (D / 2) + m * (D / 32);
          if constexpr (G == 1) row[e][0] = *reinterpret_cast<const uint16_t*>(v);
          else if constexpr (G == 2) row[e][0] = *reinterpret_cast<const uint32_t*>(v);
          else {
            const u32x2_t x = *reinterpret_cast<const u32x2_t*>(v);
            row[e][0] = x[0], row[e][1] = x[1];
          }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          uint32_t x[4], y[4];
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            x[i4] = __builtin_amdgcn_perm(row[2 * i4 + 1][g / 2], row[2 * i4][g / 2], g % 2 ? 0x07060302u : 0x05040100u);
            y[i4] = x[i4] >> 8;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t mask = j % 2 ? 0x00f000f0u : 0x000f000fu;
            u32x4_t op;
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) op[i4] = (j < 2 ? x[i4] : y[i4]) & mask;
            o[g][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, op), pop[g], o[g][j], 0, 0, 0);
          }
        }
      }
    }
    sum = over_quarters_sum(sum);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      off[g] = over_quarters_sum(off[g]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[g][j][e] = __builtin_fmaf(o[g][j][e], j % 2 ? 0x1p20f : 0x1p24f, off[g]);
    }
    // o[g][j][e]: value 64 g + 16 kg + 4 e + j of head m
    if (from == 0 && to == n_pages) {
      if (m < columns) {
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        T* const out = (T*)a.ctx + (int64_t)r * a.ldc + (int64_t)(head0 + m) * D + 16 * kg;
        typedef T four_t __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<four_t*>(out + 64 * g + 4 * e) =
                four_t{(T)(o[g][0][e] * inv), (T)(o[g][1][e] * inv), (T)(o[g][2][e] * inv), (T)(o[g][3][e] * inv)};
      }
    } else if (m < columns) {
      // (a worker has two such requests at most: the one that its run begins in and the one that it ends in)
      const int64_t slot = ((int64_t)stream * p.workers + worker) * 2 + (start < begin ? 0 : 1);
      float* const out = p.sums + (slot * p.columns + m) * D + 16 * kg;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<f32x4_t*>(out + 64 * g + 4 * e) = f32x4_t{o[g][0][e], o[g][1][e], o[g][2][e], o[g][3][e]};
      if (kg == 0) {
        p.ml[(slot * p.columns + m) * 2] = best;
        p.ml[(slot * p.columns + m) * 2 + 1] = sum;
      }
    }
    at_page = start + to;
    start += n_pages;
  }
}

constexpr int kJoin = 512;

// The parts of a request's sums, of one stream, whose workers lie side by side; requests without a position.
template <typename T>
__global__ __launch_bounds__(kJoin) void paged_join_kernel(PagedArgs p) {
  __shared__ int before_of[2];
  __shared__ float part[kJoin * 4];
  const awq_paged_attention_args& a = p.a;
  const int r = blockIdx.x / p.streams, stream = blockIdx.x % p.streams, tid = threadIdx.x, D = a.dim;
  const int tiles = p.streams / a.kv_heads, group = a.heads / a.kv_heads;
  const int head0 = stream / tiles * group + stream % tiles * kColumns, columns = min(kColumns, group - stream % tiles * kColumns);
  if (tid < 2) before_of[tid] = 0;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = tid; i < a.n_requests; i += kJoin) {
    const int n = pages_of(a, i);
    all += n;
    if (i < r) before += n;
  }
  if (all) atomicAdd(&before_of[0], all);
  if (before) atomicAdd(&before_of[1], before);
  const int n_pages = pages_of(a, r);
  __syncthreads();
  all = before_of[0];
  const int begin = before_of[1], end = begin + n_pages;
  T* const out = (T*)a.ctx + (int64_t)r * a.ldc + (int64_t)head0 * D;
  if (n_pages == 0) {
    for (int i = tid; i < columns * D; i += kJoin) out[i] = (T)0.0f;
    return;
  }
  // the worker of a page: the last whose first page is not behind it
  const auto worker_of = [&](int page) {
    int w = (int)((int64_t)page * p.workers / all);
    while (w + 1 < p.workers && first_page(w + 1, all, p.workers) <= page) ++w;
    while (first_page(w, all, p.workers) > page) --w;
    return w;
  };
  const int first = worker_of(begin), last = worker_of(end - 1);
  if (first == last) return;  // one worker had all of it
  const int64_t at = (int64_t)stream * p.workers;
  const auto slot_of = [&](int w) { return (at + w) * 2 + (w == first); };  // (it begins in the first and ran on in the others)
  const int quads = columns * D / 4, shares = max(1, kJoin / quads);
  for (int q0 = 0; q0 < quads; q0 += kJoin) {
    const int share = quads >= kJoin ? 0 : tid / quads, quad = quads >= kJoin ? q0 + tid : tid % quads;
    const bool mine = quad < quads && share < shares;
    const int head = min(quad * 4 / D, columns - 1);
    float best = -INFINITY, sum = 0.0f;
    f32x4_t o = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (mine) {
      for (int w = first; w <= last; ++w) {
        if (first_page(w, all, p.workers) == first_page(w + 1, all, p.workers)) continue;
        best = fmaxf(best, p.ml[(slot_of(w) * p.columns + head) * 2]);
      }
      const float base = best == -INFINITY ? 0.0f : best;
      for (int w = first + share; w <= last; w += shares) {
        if (first_page(w, all, p.workers) == first_page(w + 1, all, p.workers)) continue;
        const int64_t s = slot_of(w) * p.columns + head;
        const float f = __builtin_amdgcn_exp2f(p.ml[s * 2] - base);
        sum = __builtin_fmaf(f, p.ml[s * 2 + 1], sum);
        const f32x4_t v = *reinterpret_cast<const f32x4_t*>(p.sums + s * D + quad * 4 % D);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(f, v[e], o[e]);
      }
    }
    if (shares > 1) {
      __shared__ float sum_of[kJoin];
      *reinterpret_cast<f32x4_t*>(part + tid * 4) = o;
      sum_of[tid] = sum;
      __syncthreads();
      if (mine && share == 0)
        for (int s = 1; s < shares; ++s) {
          o = o + *reinterpret_cast<const f32x4_t*>(part + (s * quads + quad) * 4);
          sum += sum_of[s * quads + quad];
        }
    }
    if (mine && share == 0) {
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[quad * 4 + e] = (T)(o[e] * inv);
    }
  }
}

}  // namespace

int64_t paged_workspace_bytes(int n_requests, int heads, int kv_heads, int dim, int max_pages) {
  const int64_t parts = (int64_t)streams_of(heads, kv_heads) * workers_of(n_requests, heads, kv_heads, dim, max_pages) * 2 * columns_of(heads / kv_heads);
  return parts * (dim + 4) * 4;  // (a multiple of 16)
}

int launch_paged_attention(const awq_paged_attention_args& u, bool bf16, hipStream_t st) {
  if (u.n_requests == 0) return AWQ_OK;
  PagedArgs p;
  p.a = u;
  p.streams = streams_of(u.heads, u.kv_heads);
  p.workers = workers_of(u.n_requests, u.heads, u.kv_heads, u.dim, u.max_pages);
  p.columns = columns_of(u.heads / u.kv_heads);
  p.sums = (float*)u.workspace;
  p.ml = p.sums + (int64_t)p.streams * p.workers * 2 * p.columns * u.dim;
  const dim3 grid((unsigned)(p.workers / kWaves * p.streams)), block(64 * kWaves);
  const auto kernel = bf16 ? (u.dim == 64 ? paged_kernel<bf16_t, 64> : u.dim == 128 ? paged_kernel<bf16_t, 128> : paged_kernel<bf16_t, 256>)
                           : (u.dim == 64 ? paged_kernel<half_t, 64> : u.dim == 128 ? paged_kernel<half_t, 128> : paged_kernel<half_t, 256>);
  hipLaunchKernelGGL(kernel, grid, block, 0, st, p);
  AWQ_HIP_TRY(hipGetLastError());
  AWQ_REQUIRE((int64_t)u.n_requests * p.streams < (1ll << 31), "too many requests and heads");
  const dim3 join((unsigned)(u.n_requests * p.streams));
  hipLaunchKernelGGL(bf16 ? paged_join_kernel<bf16_t> : paged_join_kernel<half_t>, join, dim3(kJoin), 0, st, p);
  AWQ_HIP_TRY(hipGetLastError());
  return AWQ_OK;
}
