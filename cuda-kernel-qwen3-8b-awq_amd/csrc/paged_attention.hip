// Attention of one query a request over a cache in 4 bits (batch.hpp).
#include "batch.hpp"
#include "lane_sums.hpp"

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;     // of a workgroup, each with pages of its own
constexpr int kColumns = 16;  // query heads of one key/value head that share a pass over the pages
constexpr float kSlack = 8.0f, kNone = -1000.0f;  // kNone: r of a group without any products yet

// Wavefronts of a SIMD: as many as have all their numbers in registers.  Heads of 128, 64 requests of 8 key/value heads with 4 query heads each:
// 4 (some numbers in scratch memory) 49 us, 3 42, 2 44; 2 key/value heads with 16: 4 37 us, 2 20; heads of 256 with 16: 2 39 us, 1 25.
constexpr int resident(int dim, int columns) {
  return dim == 64 ? (columns > 8 ? 2 : 4) : dim == 128 ? (columns > 8 ? 2 : 3) : (columns > 8 ? 1 : 2);
}
inline int columns_of(int group) { return std::min(group, kColumns); }
inline int streams_of(int heads, int kv_heads) { return kv_heads * ((heads / kv_heads + kColumns - 1) / kColumns); }
// wavefronts that share the pages of a stream (a key/value head and up to 16 of its query heads): as many as the chip holds, each with a page in LDS
inline int workers_of(int n_requests, int heads, int kv_heads, int dim, int max_pages) {
  const int64_t there = 1024ll * resident(dim, heads / kv_heads) / streams_of(heads, kv_heads);
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

// over the lanes of one head: those 16 apart and, where FROM < 16, those FROM, 2 FROM .. apart too
template <int FROM, typename F>
__device__ __forceinline__ float over_head(float v, F f) {
  if constexpr (FROM <= 4) v = f(v, lanes::from<0x124>(v));  // rotated by 4 within 16 lanes, and by 8
  if constexpr (FROM <= 8) v = f(v, lanes::from<0x128>(v));
  return lanes::over_rows(v, f);
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
// pages of a worker: equal runs, the last ones may be without
__device__ __forceinline__ int run_of(int all, int workers) { return (all + workers - 1) / workers; }

// The pages of all requests in a row are cut evenly over `workers` wavefronts; a worker walks the requests that its run touches.  A page
// comes into LDS as it lies in memory but for the order of its 16-byte pieces, the next one's keys while this one's values are worked on and
// the other way round.  Operands of v_mfma_f32_16x16x32_f16, lane (m, kg) = (lane % 16, lane / 16), heads as columns:
//     S[key][head] = K q^T        sixteen keys; a lane takes quarter kg of key m's row
//     O[c][head] += V^T P         two of sixteen keys; a lane takes piece m of the rows of the keys 4 kg .. + 3 of both
// so that the weights a lane forms are the elements it supplies to the second product.  With COLUMNS heads below 16 the columns are the heads
// once for each of TP = 16 / COLUMNS sixteens of keys: a lane keeps the scores of its own sixteen (of every TP), supplies zeros to the
// second product for the others, and the columns of a head are added up at the end.  Softmax is then a quarter of the instructions at 4 heads.
// Nibbles go into the products as they are: as the last
// bits of a binary16 number they stand for n 2^-24, four bits up for 16 times that (the query's values there are divided by 16, and
// so are the sums of the values' pieces), so that a word of eight takes five instructions.  The scales are put on afterwards: on a key's
// sum over a group, s sum(q n) + z sum(q) in binary32, and on the weights, p s rounded to binary16 for the product, p z in binary32.
// Heads of 128, 32 over 8: 64 requests of 100 to 8,000 positions, bfloat16, 42 us, 4.2 TB/s of the cache; one of 40,960 positions, binary16, 17 us (its
// 640 pages leave a worker two); 12 requests of 5 to 300 positions, 16 heads of 64, 6 us (all traced).  Bound by memory and, at a few pages a worker, by the start.
// Weights are relative to the largest score, whose own is 1 then and its products p s exact.  A group's products are held relative to a power of two of
// its own, 2^r for a whole r, which moves once some are 2^kSlack above it: they are normal numbers of binary16 down to 2^-14 of the group's largest so
// far, whatever the scales of keys that weigh nothing and of other groups, and whatever their sign.
template <typename T, int D, int COLUMNS>
__global__ __launch_bounds__(64 * kWaves, resident(D, COLUMNS)) void paged_kernel(PagedArgs p) {
  constexpr int G = D / 64, PIECES = D / 32;  // groups; 16-byte pieces of a row
  constexpr int TP = 16 / COLUMNS, SETS = 4 / TP;
  constexpr int kBytes = 72 * D, kKeyLoads = D / 32 + (D + 127) / 128, kValueLoads = D / 32;
  typedef __attribute__((address_space(1))) const void* gptr_t;
  typedef __attribute__((address_space(3))) void* lptr_t;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves * kBytes];
  const awq_paged_attention_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, kg = lane >> 4;
  const int stream = blockIdx.x % p.streams, worker = blockIdx.x / p.streams * kWaves + wave;
  const int tiles = p.streams / a.kv_heads, kv_head = stream / tiles, group = a.heads / a.kv_heads;
  const int head0 = kv_head * group + stream % tiles * kColumns, columns = min(kColumns, group - stream % tiles * kColumns);
  const int column = m % COLUMNS, mine = m / COLUMNS;  // which sixteen of every TP
  // a page's keys, its parameters, its values
  uint8_t* const kb = lds + wave * kBytes;
  uint8_t* const pb = kb + 32 * D;
  uint8_t* const vb = pb + 8 * D;

  const int run = (a.n_requests + 63) / 64;
  int all;
  const int ahead = pages_ahead(a, lane, run, all);
  const int each = run_of(all, p.workers), begin = worker * each, end = min(begin + each, all);
  if (begin >= all) return;
  // pages of the four workers side by side, where all have some
  const int wg_begin = (worker - wave) * each, wg_end = wg_begin + 3 * each < all ? min(wg_begin + kWaves * each, all) : INT32_MAX;
  // the request of the first page: the last run of requests that does not start behind it, then one after the other
  const int at = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(ahead <= begin));
  int r = at * run, start = __builtin_amdgcn_readlane(ahead, at), n_pages = pages_of(a, r);
  while (start + n_pages <= begin) {
    start += n_pages;
    n_pages = pages_of(a, ++r);
  }

  // Where the lane's 16 bytes of a request into LDS come from: a key's pieces rotated among its row's, so that those that lanes read together
  // lie in all banks; rows of values with those four apart side by side.  A place of the wavefront and one of the lane, which is the same in every
  // request (of rows of 128 bytes a rotation by four pieces in every other).
  const uint32_t key_row = lane / PIECES, in_row = lane % PIECES;
  const uint32_t key_lane = (key_row * PIECES + (in_row ^ ((key_row * PIECES / 16) & (PIECES - 1)))) * 16;
  const uint32_t value_slot = lane / PIECES;
  const uint32_t value_lane = (((value_slot & ~15u) + (value_slot & 3) * 4 + ((value_slot & 15) >> 2)) * PIECES + in_row) * 16;
  const uint32_t parameter_lane = lane * 16;
  // (nothing of the compiler's may change the order of the requests: they are waited for by their number)
  const auto in_order = []() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto page_of = [&](int page) __attribute__((always_inline)) {
    return (const uint8_t*)a.cache + ((int64_t)__builtin_amdgcn_readfirstlane(page) * a.kv_heads + kv_head) * kBytes;
  };
  // (the wavefront's place stays in scalar registers, out of the compiler's hands: it would make 64-bit addresses of each lane's)
  const auto request = [&](const uint8_t* src, uint32_t of_lane, uint8_t* to) __attribute__((always_inline)) {
    uint64_t place = (uint64_t)src;
    asm volatile("" : "+s"(place));
    __builtin_amdgcn_global_load_lds((gptr_t)(place + of_lane), (lptr_t)to, 16, 0, 0);
  };
  const auto request_keys = [&](int page) __attribute__((always_inline)) {
    const uint8_t* const src = page_of(page);
    in_order();
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      request(src + i * 1024, D == 256 && i % 2 ? key_lane ^ 64u : key_lane, kb + i * 1024);
#pragma unroll
    for (int i = 0; i < (D + 127) / 128; ++i)
      if (D != 64 || lane < 32)
        request(src + 64 * D + i * 1024, parameter_lane, pb + i * 1024);
    in_order();
  };
  const auto request_values = [&](int page) __attribute__((always_inline)) {
    const uint8_t* const src = page_of(page);
    in_order();
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      request(src + 32 * D + (D == 256 ? (i / 2) * 2048 + (i % 2) * 256 : i * 1024), value_lane, vb + i * 1024);
    in_order();
  };

  for (int at_page = begin; at_page < end; ++r) {
    // one request: pages from .. to of it
    const int length = min(max(a.lengths[r], 0), a.max_pages * kPage);
    n_pages = (length + kPage - 1) / kPage;
    if (n_pages == 0) continue;
    const int from = at_page - start, to = min(n_pages, end - start);
    const int32_t* const table = a.table + (int64_t)r * a.max_pages;
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

    // the query: lane (m, kg) has values 64 g + 16 kg + 8 j .. + 7 of its head
    typedef T eight_t __attribute__((ext_vector_type(8)));
    eight_t qv[2 * G];
    {
      const T* const q = (const T*)a.q + (int64_t)r * a.ldq + (int64_t)(head0 + min(column, columns - 1)) * D + 16 * kg;
#pragma unroll
      for (int i = 0; i < 2 * G; ++i) qv[i] = *reinterpret_cast<const eight_t*>(q + 64 * (i / 2) + 8 * (i % 2));
    }
    int i = from;
    // (an entry that is no page is passed over)
    const auto next_page = [&]() __attribute__((always_inline)) {
      int page = -1;
      while (i < to && (page = page_at(i)) < 0) ++i;
      return page;
    };
    int here = next_page();
    if (here >= 0) {
      request_keys(here);
      request_values(here);
    }
    half8_t qop[2 * G];
    float q_sum[G], mul;
    {
      float q_max = 0.0f;
#pragma unroll
      for (int i = 0; i < 2 * G; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) q_max = fmaxf(q_max, fabsf((float)qv[i][e]));
      q_max = over_head<16>(q_max, lanes::Max());
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
            v[e] = (float)qv[2 * g + j][e] * up * more;
            q_sum[g] += v[e];
          }
          qop[2 * g + j] = half8_t{(half_t)v[0], (half_t)v[4], (half_t)(v[1] * 0.0625f), (half_t)(v[5] * 0.0625f),
                                   (half_t)v[2], (half_t)v[6], (half_t)(v[3] * 0.0625f), (half_t)(v[7] * 0.0625f)};
        }
        q_sum[g] = over_head<16>(q_sum[g], lanes::Add()) * 0x1p-24f;
      }
      mul = __builtin_amdgcn_ldexpf(a.scale * 1.44269504088896340736f, 24 - e2);
    }

    f32x4_t o[G][4];
    float off[G], r2[G], best = -INFINITY, sum = 0.0f;  // r2: the group's r
#pragma unroll
    for (int g = 0; g < G; ++g) {
      off[g] = 0.0f;
      r2[g] = kNone;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[g][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    while (here >= 0) {
      const int left = length - i * kPage;  // positions of this page
      ++i;
      const int next = next_page();
      // requests on their way: this page's keys and parameters, then its values
      wait_for_requests<kValueLoads>();
      f32x4_t s[SETS][G];
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
#pragma unroll
        for (int g = 0; g < G; ++g) {
          f32x4_t one = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x = w[2 * g + j], y = x >> 8;
            const u32x4_t op = u32x4_t{x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
            one = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, op), qop[2 * g + j], one, 0, 0, 0);
          }
          if (t % TP == 0) s[t / TP][g] = one;
          else
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t / TP][g][e] = mine == t % TP ? one[e] : s[t / TP][g][e];
        }
      }
      float score[SETS][4], highest = -INFINITY;
#pragma unroll
      for (int q = 0; q < SETS; ++q) {
        const int row = 16 * (q * TP + mine) + 4 * kg;  // of the lane's four keys
#pragma unroll
        for (int e = 0; e < 4; ++e) score[q][e] = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const half4_t sc = *reinterpret_cast<const half4_t*>(pb + ((g * 2) * kPage + row) * 2);
          const half4_t zz = *reinterpret_cast<const half4_t*>(pb + ((g * 2 + 1) * kPage + row) * 2);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            score[q][e] = __builtin_fmaf((float)sc[e], s[q][g][e], __builtin_fmaf((float)zz[e], q_sum[g], score[q][e]));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          score[q][e] = row + e < left ? score[q][e] * mul : -INFINITY;
          highest = fmaxf(highest, score[q][e]);
        }
      }
      half4_t vs[SETS][G], vz[SETS][G];
#pragma unroll
      for (int q = 0; q < SETS; ++q) {
        const int row = 16 * (q * TP + mine) + 4 * kg;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          vs[q][g] = *reinterpret_cast<const half4_t*>(pb + 4 * D + ((g * 2) * kPage + row) * 2);
          vz[q][g] = *reinterpret_cast<const half4_t*>(pb + 4 * D + ((g * 2 + 1) * kPage + row) * 2);
        }
        if (left < kPage) {  // whatever lies behind the last position
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (row + e >= left) vs[q][g][e] = vz[q][g][e] = (half_t)0.0f;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the keys and the parameters have been read
      if (next >= 0) request_keys(next);
      highest = over_head<COLUMNS>(highest, lanes::Max());
      const float to_best = fmaxf(best, highest);
      if (__builtin_amdgcn_ballot_w64(to_best > best)) {
        const float step = to_best > best ? to_best - best : 0.0f, alpha = __builtin_amdgcn_exp2f(-step);
        best = to_best;
        sum *= alpha;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          off[g] *= alpha;
          // (the group's largest so far are `step` less by now, and so is r as far as it stays whole)
          const float r = r2[g] - step;
          r2[g] = fmaxf(__builtin_ceilf(r), kNone);
          const float rest = __builtin_amdgcn_exp2f(r - r2[g]);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[g][j] *= rest;
        }
      }
      const float base = best == -INFINITY ? 0.0f : best;
      float w[SETS][4];
#pragma unroll
      for (int q = 0; q < SETS; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[q][e] = __builtin_amdgcn_exp2f(score[q][e] - base);
          sum += w[q][e];
        }
      u32x2_t weights[SETS][G];  // times the scales, four in binary16
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float widest = 0.0f;
#pragma unroll
        for (int q = 0; q < SETS; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            widest = fmaxf(widest, fabsf(w[q][e] * (float)vs[q][g][e]));
            off[g] = __builtin_fmaf(w[q][e], (float)vz[q][g][e], off[g]);
          }
        if (__builtin_amdgcn_ballot_w64(widest > __builtin_amdgcn_exp2f(r2[g] + kSlack))) {
          const float all = over_head<COLUMNS>(widest, lanes::Max()), to = all > 0.0f ? fmaxf((float)__builtin_amdgcn_frexp_expf(all), r2[g]) : r2[g];
          const float alpha = to > r2[g] ? __builtin_amdgcn_exp2f(r2[g] - to) : 1.0f;
          r2[g] = to;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[g][j] *= alpha;
        }
        const float up = __builtin_amdgcn_ldexpf(1.0f, (int)fminf(-r2[g], 126.0f));
#pragma unroll
        for (int q = 0; q < SETS; ++q) {
          half4_t ps;
#pragma unroll
          for (int e = 0; e < 4; ++e) ps[e] = (half_t)(w[q][e] * (float)vs[q][g][e] * up);
          weights[q][g] = __builtin_bit_cast(u32x2_t, ps);
        }
      }
      if (next >= 0) wait_for_requests<kKeyLoads>();
      else wait_for_requests<0>();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        half8_t pop[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          u32x4_t x;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = 2 * u + h;
            x[2 * h] = TP == 1 || mine == t % TP ? weights[t / TP][g][0] : 0u;
            x[2 * h + 1] = TP == 1 || mine == t % TP ? weights[t / TP][g][1] : 0u;
          }
          pop[g] = __builtin_bit_cast(half8_t, x);
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
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the values have been read
      if (next >= 0) request_values(next);
      here = next;
    }
    // the columns of a head together, its sums over all quarters of the keys
    const auto add_columns = [](float v) __attribute__((always_inline)) {
      if constexpr (COLUMNS <= 4) v += lanes::from<0x124>(v);
      if constexpr (COLUMNS <= 8) v += lanes::from<0x128>(v);
      return v;
    };
    sum = over_head<COLUMNS>(sum, lanes::Add());
#pragma unroll
    for (int g = 0; g < G; ++g) {
      off[g] = over_head<COLUMNS>(off[g], lanes::Add());
      const float size = __builtin_amdgcn_ldexpf(1.0f, (int)r2[g]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[g][j][e] = __builtin_fmaf(add_columns(o[g][j][e]) * size, j % 2 ? 0x1p20f : 0x1p24f, off[g]);
    }
    // o[g][j][e]: value 64 g + 16 kg + 4 e + j of the lane's head
    bool whole = from == 0 && to == n_pages, writes = m < columns;
    if (wg_begin >= start && wg_end <= start + n_pages) {
      // all four wavefronts have parts of this request and nothing else: together they are one
      float* const meet = reinterpret_cast<float*>(lds);  // [4][columns][D], then [4][columns][2]
      float* const meet_ml = meet + kWaves * COLUMNS * D;
      static_assert(kWaves * COLUMNS * (D + 2) * 4 <= kWaves * kBytes, "the sums take the place of the pages");
      __syncthreads();  // all pages have been read
      if (writes) {
        float* const out = meet + (wave * COLUMNS + m) * D + 16 * kg;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) *reinterpret_cast<f32x4_t*>(out + 64 * g + 4 * e) = f32x4_t{o[g][0][e], o[g][1][e], o[g][2][e], o[g][3][e]};
        if (kg == 0) meet_ml[(wave * COLUMNS + m) * 2] = best, meet_ml[(wave * COLUMNS + m) * 2 + 1] = sum;
      }
      __syncthreads();
      whole = wg_begin == start && wg_end == start + n_pages;
      const int64_t slot = ((int64_t)stream * p.workers + worker - wave) * 2 + (start < wg_begin ? 0 : 1);
      int tid = threadIdx.x;
      if constexpr (D == 256) asm volatile("" : "+v"(tid));  // (as below)
      for (int x = tid; x < columns * (D / 4); x += 64 * kWaves) {
        const int c = x / (D / 4), d = x % (D / 4) * 4;
        float top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, meet_ml[(w * COLUMNS + c) * 2]);
        const float base = top == -INFINITY ? 0.0f : top;
        f32x4_t y = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f(meet_ml[(w * COLUMNS + c) * 2] - base);
          const f32x4_t v = *reinterpret_cast<const f32x4_t*>(meet + (w * COLUMNS + c) * D + d);
          total = __builtin_fmaf(f, meet_ml[(w * COLUMNS + c) * 2 + 1], total);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(f, v[e], y[e]);
        }
        if (whole) {
          const float inv = total != 0.0f ? 1.0f / total : 0.0f;
          typedef T four_t __attribute__((ext_vector_type(4)));
          *reinterpret_cast<four_t*>((T*)a.ctx + (int64_t)r * a.ldc + (int64_t)(head0 + c) * D + d) =
              four_t{held(y[0] * inv, T()), held(y[1] * inv, T()), held(y[2] * inv, T()), held(y[3] * inv, T())};
        } else {
          *reinterpret_cast<f32x4_t*>(p.sums + (slot * p.columns + c) * D + d) = y;
          if (d == 0) p.ml[(slot * p.columns + c) * 2] = top, p.ml[(slot * p.columns + c) * 2 + 1] = total;
        }
      }
      return;
    }
    int quarter = kg, of_column = m;
    if constexpr (D == 256) asm volatile("" : "+v"(quarter), "+v"(of_column));  // (addresses are formed anew: one that waits through the pages would be a number too many)
    if (whole && writes) {
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      T* const out = (T*)a.ctx + (int64_t)r * a.ldc + (int64_t)(head0 + of_column) * D + 16 * quarter;
      typedef T four_t __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<four_t*>(out + 64 * g + 4 * e) =
              four_t{held(o[g][0][e] * inv, T()), held(o[g][1][e] * inv, T()), held(o[g][2][e] * inv, T()), held(o[g][3][e] * inv, T())};
    } else if (writes) {
      // (a worker has two such requests at most: the one that its run begins in and the one that it ends in)
      const int64_t slot = ((int64_t)stream * p.workers + worker) * 2 + (start < begin ? 0 : 1);
      float* const out = p.sums + (slot * p.columns + of_column) * D + 16 * quarter;
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

// The parts of a request's sums, of one stream, whose workers lie side by side: 4 `quads` values a workgroup, every 512 / quads-th part a
// thread; zeros for requests without a position.
template <typename T>
__global__ __launch_bounds__(kJoin) void paged_join_kernel(PagedArgs p, int chunks, int quads) {
  __shared__ int pages[2];
  __shared__ float best_of[kJoin], sum_of[kJoin];
  __shared__ f32x4_t o_of[kJoin];
  const awq_paged_attention_args& a = p.a;
  const int chunk = blockIdx.x % chunks, stream = blockIdx.x / chunks % p.streams, r = blockIdx.x / chunks / p.streams;
  const int tid = threadIdx.x, D = a.dim, shares = kJoin / quads;
  const int tiles = p.streams / a.kv_heads, group = a.heads / a.kv_heads;
  const int head0 = stream / tiles * group + stream % tiles * kColumns, columns = min(kColumns, group - stream % tiles * kColumns);
  const int value = (chunk * quads + tid % quads) * 4, share = tid / quads;  // of all columns' values
  if (tid < 2) pages[tid] = 0;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = tid; i < a.n_requests; i += kJoin) {
    const int n = pages_of(a, i);
    all += n;
    if (i < r) before += n;
  }
  if (all) atomicAdd(&pages[0], all);
  if (before) atomicAdd(&pages[1], before);
  const int n_pages = pages_of(a, r);
  __syncthreads();
  all = pages[0];
  const int begin = pages[1], end = begin + n_pages, each = run_of(all, p.workers);
  T* const out = (T*)a.ctx + (int64_t)r * a.ldc + (int64_t)head0 * D + value;
  typedef T four_t __attribute__((ext_vector_type(4)));
  if (n_pages == 0) {
    if (share == 0 && value < columns * D) *reinterpret_cast<four_t*>(out) = four_t{(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
    return;
  }
  const int first = begin / each, last = (end - 1) / each;
  // workgroups whose four workers have pages of this request alone have left one sum: workers from .. to
  int from = (first + kWaves - 1) / kWaves * kWaves, to = (last + 1) / kWaves * kWaves;
  if (from * each < begin) from += kWaves;
  if (to > from && min(to * each, all) > end) to -= kWaves;
  if (to < from) from = to = last + 1;
  if (first == last || (from == first && to == last + 1 && to - from == kWaves)) return;  // one worker or workgroup had all of it
  const int singles = from - first, wholes = (to - from) / kWaves, parts = singles + wholes + (last + 1 - to);
  const auto slot_of = [&](int i) {
    const int w = i < singles ? first + i : i < singles + wholes ? from + (i - singles) * kWaves : to + i - singles - wholes;
    return ((int64_t)stream * p.workers + w) * 2 + (w == first);  // (it begins in the first and ran on in the others)
  };
  const int head = min(value / D, columns - 1);
  f32x4_t o = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float best = -INFINITY, sum = 0.0f;
  const auto add = [&](float m, float l, f32x4_t v) __attribute__((always_inline)) {
    const float to = fmaxf(best, m), base = to == -INFINITY ? 0.0f : to;
    const float f = __builtin_amdgcn_exp2f(best - base), g = __builtin_amdgcn_exp2f(m - base);
    best = to;
    sum = __builtin_fmaf(g, l, sum * f);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(g, v[e], o[e] * f);
  };
#pragma unroll 4
  for (int i = share; i < parts; i += shares) {
    const int64_t s = slot_of(i) * p.columns + head;
    add(p.ml[s * 2], p.ml[s * 2 + 1], *reinterpret_cast<const f32x4_t*>(p.sums + s * D + value % D));
  }
  best_of[tid] = best;
  sum_of[tid] = sum;
  o_of[tid] = o;
  __syncthreads();
  if (share || value >= columns * D) return;
  for (int i = 1; i < min(shares, parts); ++i) add(best_of[i * quads + tid], sum_of[i * quads + tid], o_of[i * quads + tid]);
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  *reinterpret_cast<four_t*>(out) = four_t{held(o[0] * inv, T()), held(o[1] * inv, T()), held(o[2] * inv, T()), held(o[3] * inv, T())};
}

template <typename T, int D>
void launch_pages(const PagedArgs& p, dim3 grid, hipStream_t st) {
  if (p.columns <= 4) hipLaunchKernelGGL((paged_kernel<T, D, 4>), grid, dim3(64 * kWaves), 0, st, p);
  else if (p.columns <= 8) hipLaunchKernelGGL((paged_kernel<T, D, 8>), grid, dim3(64 * kWaves), 0, st, p);
  else hipLaunchKernelGGL((paged_kernel<T, D, 16>), grid, dim3(64 * kWaves), 0, st, p);
}

// wide pieces of a request's values where the workers are cut over many requests, few parts each; narrow ones, whose threads share the parts,
// where they are cut over few (one request of 40,960 positions 5.5 us with 32 pieces, 7.2 with 128; 64 requests 17.8 and 9.2; next to the border 5 requests
// of 8,000 with 32 pieces and 6 with 128 take 4.8 and 4.7)
int quads_of(const PagedArgs& p) { return p.workers / kWaves > 16ll * p.a.n_requests ? 32 : 128; }
int chunks_of(const PagedArgs& p) { return (p.columns * p.a.dim + 4 * quads_of(p) - 1) / (4 * quads_of(p)); }

template <typename T>
int launch(const PagedArgs& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.workers / kWaves * p.streams));
  if (p.a.dim == 64) launch_pages<T, 64>(p, grid, st);
  else if (p.a.dim == 128) launch_pages<T, 128>(p, grid, st);
  else launch_pages<T, 256>(p, grid, st);
  AWQ_HIP_TRY(hipGetLastError());
  const int quads = quads_of(p), chunks = chunks_of(p);
  hipLaunchKernelGGL(paged_join_kernel<T>, dim3((unsigned)(p.a.n_requests * p.streams * chunks)), dim3(kJoin), 0, st, p, chunks, quads);
  AWQ_HIP_TRY(hipGetLastError());
  return AWQ_OK;
}

}  // namespace

int64_t paged_workspace_bytes(int n_requests, int heads, int kv_heads, int dim, int max_pages) {
  const int64_t parts = (int64_t)streams_of(heads, kv_heads) * workers_of(n_requests, heads, kv_heads, dim, max_pages) * 2 * columns_of(heads / kv_heads);
  return parts * (dim + 4) * 4;  // (a multiple of 16)
}

int launch_paged_attention(const awq_paged_attention_args& u, bool bf16, hipStream_t st) {
  PagedArgs p;
  p.a = u;
  p.streams = streams_of(u.heads, u.kv_heads);
  p.workers = workers_of(u.n_requests, u.heads, u.kv_heads, u.dim, u.max_pages);
  p.columns = columns_of(u.heads / u.kv_heads);
  p.sums = (float*)u.workspace;
  p.ml = p.sums + (int64_t)p.streams * p.workers * 2 * p.columns * u.dim;
  AWQ_REQUIRE(launchable((int64_t)p.workers / kWaves * p.streams, 64 * kWaves) && launchable((int64_t)u.n_requests * p.streams * chunks_of(p), kJoin),
              "too many requests and heads");
  return bf16 ? launch<bf16_t>(p, st) : launch<half_t>(p, st);
}
