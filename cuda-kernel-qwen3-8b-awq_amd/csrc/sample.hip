// A token of each row of logits: temperature, top-k, top-p and min-p, from given uniform numbers (batch.hpp).
#include "batch.hpp"
#include "lane_sums.hpp"

namespace {

// Weights go into bins of a quarter of a nat, y = 4 l / T, bin floor(y); of a row or a part of it only the 256 bins from its largest logit's down
// are looked at: what lies further is below e^-63, and 64 bits of a sum would not show it.  Within a bin a weight is e^((y - bin - 1) / 4), between e^(-1/4) and 1, as a whole multiple of 2^-36, so that
// sums do not depend on their order; bins are joined in 64-bit floating point.  (Tokens with the largest logit are all in the first bin: their sums
// are exact, and uniform numbers such as 1/2 fall between two of them as they should.)
//   scan_kernel    parts of 8,192 logits: largest, sum of weights, and where a row is filtered a histogram, sums and counts by bin
//   choose_kernel  a workgroup a row: the bin in which the tokens kept end, the order within that bin alone, the part that the uniform
//                  number falls in, and the token in that part.
constexpr int kPart = 8192, kScan = 256, kChoose = 1024, kBins = 256, kChunk = 32, kHeld = 8192, kRanked = 512;
constexpr int kFixed = 36, kCountShift = 50;
constexpr double kFarthest = 0x1p50;  // of y: logits beyond 2^48 T count as that

struct Part {
  float largest;
  int32_t first;  // lowest id of the largest
  double sum;     // of the weights, relative to e^((bin + 1) / 4) of the largest's bin
};
struct SampleArgs {
  awq_sample_args a;
  int parts, chunks;
  Part* part;           // [rows][parts]
  uint64_t* histogram;  // [rows][parts][kBins]: count << 50 | sum, at bin mod 256
  float* chunk;         // [rows][chunks]: largest of 32 logits
};

struct Row {
  double per_t;  // 4 / T
  float top_p, min_p;
  int top_k;  // 0: not limited
  bool greedy, filtered;
};
__device__ __forceinline__ Row row_of(const awq_sample_args& a, int64_t row) {
  Row r;
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  r.greedy = !(t > 0.0f);
  r.per_t = 4.0 / (double)t;
  r.top_k = a.top_k ? a.top_k[row] : 0;
  if (r.top_k < 0 || r.top_k >= a.vocab) r.top_k = 0;
  r.top_p = a.top_p ? a.top_p[row] : 1.0f;
  if (!(r.top_p < 1.0f)) r.top_p = 1.0f;
  if (r.top_p <= 0.0f) r.top_k = 1, r.top_p = 1.0f;  // the first alone
  r.min_p = a.min_p ? a.min_p[row] : 0.0f;
  r.min_p = r.min_p > 0.0f ? fminf(r.min_p, 1.0f) : 0.0f;
  r.filtered = r.top_k > 0 || r.top_p < 1.0f || r.min_p > 0.0f;
  return r;
}

struct Binned {
  double bin, weight;  // weight relative to e^((bin + 1) / 4), a whole multiple of 2^-36
};
constexpr double kRound = 0x1.8p16;  // numbers of its size are 2^-36 apart
__device__ __forceinline__ double bin_of(double l, double per_t) { return floor(fmin(fmax(l * per_t, -kFarthest), kFarthest)); }
__device__ __forceinline__ Binned binned(float l, double per_t) {
  const double y = fmin(fmax((double)l * per_t, -kFarthest), kFarthest), b = floor(y);
  // e^(f - 1/8), f within 1/8 of 0: the series up to f^9 / 9!, the next term is below 3e-16
  const double f = (y - b) * 0.25 - 0.125;
  double e = 1.0 / 362880.0;
  e = fma(e, f, 1.0 / 40320.0);
  e = fma(e, f, 1.0 / 5040.0);
  e = fma(e, f, 1.0 / 720.0);
  e = fma(e, f, 1.0 / 120.0);
  e = fma(e, f, 1.0 / 24.0);
  e = fma(e, f, 1.0 / 6.0);
  e = fma(e, f, 0.5);
  e = fma(e, f, 1.0);
  e = fma(e, f, 1.0);
  return {b, fma(e, 0.88249690258459540286, kRound) - kRound};  // e^(-1/8)
}
__device__ __forceinline__ uint64_t fixed_of(double weight) { return (uint64_t)__double_as_longlong(weight + kRound) & ((1ull << 51) - 1); }
__device__ __forceinline__ int place_of(double bin) { return (int)((int64_t)bin & (kBins - 1)); }

__device__ __forceinline__ float logit(float v) { return v != v ? -INFINITY : v + 0.0f; }  // (-0 as 0)
// of a row with logits of +infinity those share the weight
__device__ __forceinline__ float finite(float v, bool infinite) { return infinite ? (v == INFINITY ? 0.0f : -INFINITY) : v; }

template <typename T, int N>
struct Some {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// kPart logits a workgroup, 32 a thread, in registers.
template <typename T>
__global__ __launch_bounds__(kScan) void scan_kernel(SampleArgs s) {
  constexpr int W = 16 / sizeof(T), L = kPart / kScan / W, LANES = kChunk / W;
  typedef typename Some<T, W>::type vec_t;
  __shared__ float largest_of[kScan / 64];
  __shared__ int first_of[kScan / 64];
  __shared__ double sum_of[kScan / 64];
  __shared__ unsigned long long bins[kScan / 64][kBins];
  __shared__ double table[kBins];
  const awq_sample_args& a = s.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / s.parts;
  const int part = blockIdx.x % s.parts;
  const Row r = row_of(a, row);
  const T* const x = (const T*)a.logits + row * a.ld;
  float v[L][W];
  float largest = -INFINITY;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int64_t at = (int64_t)part * kPart + (i * kScan + tid) * W;
    if (at + W <= a.vocab) {
      const vec_t u = *reinterpret_cast<const vec_t*>(x + at);
#pragma unroll
      for (int e = 0; e < W; ++e) v[i][e] = logit((float)u[e]);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) v[i][e] = at + e < a.vocab ? logit((float)x[at + e]) : -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < L; ++i) {
    float m = v[i][0];
#pragma unroll
    for (int e = 1; e < W; ++e) m = fmaxf(m, v[i][e]);
    largest = fmaxf(largest, m);
    if (r.filtered) {
      m = lanes::maximum<LANES>(m);
      const int64_t at = ((int64_t)part * kPart + (i * kScan + tid) * W) / kChunk;
      if (tid % LANES == 0 && at < s.chunks) s.chunk[row * s.chunks + at] = m;
    }
  }
  if (r.filtered && !r.greedy)
    for (int b = lane; b < kBins; b += 64) bins[wave][b] = 0;
  table[tid] = exp(-0.25 * tid);
  largest = lanes::maximum<64>(largest);
  if (lane == 0) largest_of[wave] = largest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kScan / 64; ++w) largest = fmaxf(largest, largest_of[w]);
  Part out{largest, 0, 0.0};
  if (r.greedy) {
    int first = INT32_MAX;
#pragma unroll
    for (int i = L - 1; i >= 0; --i)
#pragma unroll
      for (int e = W - 1; e >= 0; --e)
        if (v[i][e] == largest) first = part * kPart + (i * kScan + tid) * W + e;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) first = min(first, __shfl_xor(first, off, 64));
    if (lane == 0) first_of[wave] = first;
    __syncthreads();
    out.first = min(min(first_of[0], first_of[1]), min(first_of[2], first_of[3]));
  } else if (largest > -INFINITY) {
    const bool infinite = largest == INFINITY;
    const double top = bin_of(infinite ? 0.0 : (double)largest, r.per_t);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < L; ++i)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const Binned b = binned(finite(v[i][e], infinite), r.per_t);
        const double below = top - b.bin;
        if (below >= kBins || finite(v[i][e], infinite) == -INFINITY) continue;
        if (r.filtered) atomicAdd(&bins[wave][place_of(b.bin)], (1ull << kCountShift) | fixed_of(b.weight));
        else sum += b.weight * table[(int)below];
      }
    if (r.filtered) {
      __syncthreads();
      uint64_t* const to = s.histogram + ((int64_t)row * s.parts + part) * kBins;
      to[tid] = (bins[0][tid] + bins[1][tid]) + (bins[2][tid] + bins[3][tid]);
    } else {
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
      if (lane == 0) sum_of[wave] = sum;
      __syncthreads();
      out.sum = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
    }
  }
  if (tid == 0) s.part[row * s.parts + part] = out;
}

constexpr int kMostParts = 64;

// order of the tokens: falling logits, rising ids; larger numbers first
__device__ __forceinline__ uint64_t order_of(float l, uint32_t id) {
  const uint32_t u = __float_as_uint(l);
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~id;
}

template <typename T>
struct Choose {
  const SampleArgs& s;
  const Row& r;
  const T* x;
  const float* chunk;
  double top;      // the bin of the row's largest
  bool infinite;
  // shared memory
  uint64_t* held;        // [kHeld] order of the tokens of a bin
  uint64_t* digit;       // [256] sums
  uint32_t* digit_count; // [256]
  uint64_t* words;       // [4]
  uint32_t* count;

  __device__ __forceinline__ float at(int i) const { return finite(logit((float)x[i]), infinite); }
  // distance of a logit's bin from the row's first; 256: further or no weight
  __device__ __forceinline__ int below(const Binned& b, float l) const {
    const double d = top - b.bin;
    return l == -INFINITY || d >= kBins ? kBins : (int)d;
  }
  // every token of bin j: f(order, fixed weight); out of the row, by runs of 32 that can have one
  template <typename F>
  __device__ __forceinline__ void each_of_row(int j, F f) const {
    const int vocab = (int)s.a.vocab;
    for (int c = threadIdx.x / kChunk; c < s.chunks; c += kChoose / kChunk) {
      const float m = finite(chunk[c], infinite);
      if (m == -INFINITY || top - bin_of((double)m, r.per_t) > j) continue;
      const int i = c * kChunk + threadIdx.x % kChunk;
      if (i >= vocab) continue;
      const float l = at(i);
      const Binned b = binned(l, r.per_t);
      if (below(b, l) == j) f(order_of(l, i), fixed_of(b.weight));
    }
  }
  __device__ __forceinline__ float logit_of(uint64_t order) const {
    const uint32_t u = order >> 32;
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
  }
  template <typename F>
  __device__ __forceinline__ void each(int j, int n, F f) const {
    if (n <= kHeld) {
      for (int i = threadIdx.x; i < n; i += kChoose) f(held[i], fixed_of(binned(logit_of(held[i]), r.per_t).weight));
    } else {
      each_of_row(j, f);
    }
  }
  __device__ __forceinline__ void gather(int j, int n) const {
    if (n > kHeld) return;
    __syncthreads();
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
    each_of_row(j, [&](uint64_t order, uint64_t) {
      const uint32_t to = atomicAdd(count, 1u);
      if (to < (uint32_t)kHeld) held[to] = order;
    });
    __syncthreads();
  }
  // Of the n tokens of bin j the one with which the count (sum == false: `need` of them) or the sum of the fixed weights (the first at
  // which it reaches `reach`) is full.  words[0]: its order, 0 if there is none; words[1]: the sum up to it, itself included.
  __device__ __forceinline__ void last_kept(int j, int n, bool by_sum, uint32_t need, double reach) const {
    __syncthreads();
    if (threadIdx.x == 0) words[0] = words[1] = 0;
    __syncthreads();
    if (n <= kRanked) {
      if ((int)threadIdx.x < n) {
        const uint64_t mine = held[threadIdx.x], own = fixed_of(binned(logit_of(mine), r.per_t).weight);
        uint32_t ahead = 0;
        uint64_t sum = 0;
        for (int i = 0; i < n; ++i)
          if (held[i] > mine) ++ahead, sum += fixed_of(binned(logit_of(held[i]), r.per_t).weight);
        const bool last = by_sum ? (double)sum < reach && (double)(sum + own) >= reach : ahead + 1 == need;
        if (last) words[0] = mine, words[1] = sum + own;
      }
      __syncthreads();
      return;
    }
    uint64_t prefix = 0, sum = 0;
    uint32_t before = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
      __syncthreads();
      if (threadIdx.x < 256) digit[threadIdx.x] = 0, digit_count[threadIdx.x] = 0;
      __syncthreads();
      each(j, n, [&](uint64_t order, uint64_t weight) {
        if (shift < 56 && order >> (shift + 8) != prefix) return;
        const int d = (int)(order >> shift) & 255;
        atomicAdd((unsigned long long*)&digit[d], (unsigned long long)weight);
        atomicAdd(&digit_count[d], 1u);
      });
      __syncthreads();
      int d = 255;
      for (; d > 0; --d) {  // (the same in every thread)
        const bool full = by_sum ? (double)(sum + digit[d]) >= reach : before + digit_count[d] >= need;
        if (full && digit_count[d]) break;
        sum += digit[d];
        before += digit_count[d];
      }
      prefix = prefix << 8 | (uint64_t)d;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint64_t own = fixed_of(binned(logit_of(prefix), r.per_t).weight);
      words[0] = prefix;
      words[1] = sum + own;
    }
    __syncthreads();
  }
};

template <typename T>
__global__ __launch_bounds__(kChoose) void choose_kernel(SampleArgs s) {
  __shared__ uint64_t held[kHeld], digit[256], words[4], in_bin[kMostParts];
  __shared__ uint32_t digit_count[256], count;
  __shared__ double table[kBins], sums[kBins], part_sum[kMostParts], wave_sum[kChoose / 64];
  __shared__ uint32_t counts[kBins];
  __shared__ uint64_t fixed[kBins];
  __shared__ Part parts[kMostParts];
  __shared__ int pick, last;
  const awq_sample_args& a = s.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = s.parts;
  const int64_t row = blockIdx.x;
  const Row r = row_of(a, row);
  if (tid < S) parts[tid] = s.part[row * S + tid];
  if (tid < kBins) table[tid] = exp(-0.25 * tid);
  if (tid == 0) pick = INT32_MAX, last = 0;
  __syncthreads();
  float largest = -INFINITY;
  for (int i = 0; i < S; ++i) largest = fmaxf(largest, parts[i].largest);
  if (r.greedy || largest == -INFINITY) {
    if (tid == 0) {
      int id = 0;
      if (largest > -INFINITY)
        for (int i = 0; i < S; ++i)
          if (parts[i].largest == largest) {
            id = parts[i].first;
            break;
          }
      a.ids[row] = id;
    }
    return;
  }
  const bool infinite = largest == INFINITY;
  const double top = bin_of(infinite ? 0.0 : (double)largest, r.per_t);
  // how far the first bin of a part lies below the row's
  const auto behind = [&](int i) {
    const float m = finite(parts[i].largest, infinite);
    const double d = top - bin_of((double)m, r.per_t);
    return m == -INFINITY || d >= kBins ? kBins : (int)d;
  };
  const Choose<T> c{s, r, (const T*)a.logits + row * a.ld, s.chunk + row * s.chunks, top, infinite, held, digit, digit_count, words, &count};
  const uint64_t* const histogram = s.histogram + row * S * kBins;
  // weights, relative to e^((top + 1) / 4), of a part's bin
  const auto part_bin = [&](int i, int j) { return histogram[(int64_t)i * kBins + place_of(top - j)]; };
  constexpr uint64_t kSumMask = (1ull << kCountShift) - 1;
  constexpr double kUnit = 1.0 / (double)(1ll << kFixed);

  int end = kBins;          // bins below it are kept whole, those above it not at all
  uint64_t border = 0;      // of bin `end` the tokens that are not behind this in order
  bool at_least = false;    // and those of them that weigh at least min_p
  const double heaviest = infinite ? 0.0 : (double)largest * r.per_t * 0.25;
  const auto heavy = [&](float l) { return exp((double)l * r.per_t * 0.25 - heaviest) >= (double)r.min_p; };
  if (r.filtered) {
    if (tid < kBins) {
      uint64_t sum = 0;
      uint32_t n = 0;
      for (int i = 0; i < S; ++i)
        if (tid >= behind(i)) {
          const uint64_t h = part_bin(i, tid);
          sum += h & kSumMask;
          n += (uint32_t)(h >> kCountShift);
        }
      fixed[tid] = sum;
      counts[tid] = n;
    }
    __syncthreads();
    // every thread walks the bins; a row's tokens end in one of them
    double above = 0.0, all = 0.0;
    for (int j = 0; j < kBins; ++j) all += (double)fixed[j] * kUnit * table[j];
    if (r.top_k) {
      uint32_t n = 0;
      int j = 0;
      for (; j < kBins && n + counts[j] < (uint32_t)r.top_k; ++j) n += counts[j], above += (double)fixed[j] * kUnit * table[j];
      if (j < kBins) {
        end = j;
        c.gather(j, counts[j]);
        c.last_kept(j, counts[j], false, r.top_k - n, 0.0);
        border = words[0];
        all = above + (double)words[1] * kUnit * table[j];
      }
    }
    if (r.top_p < 1.0f) {
      const double target = (double)r.top_p * all;
      double sum = 0.0;
      int j = 0;
      for (; j < kBins && j < end; ++j) {
        const double with = sum + (double)fixed[j] * kUnit * table[j];
        if (with >= target) break;
        sum = with;
      }
      if (j < kBins && counts[j]) {
        if (j != end) c.gather(j, counts[j]);
        c.last_kept(j, counts[j], true, 0, (target - sum) / (kUnit * table[j]));
        // (nothing reaches it: a rounding away from the whole bin)
        if (j != end) border = words[0];
        else if (words[0] > border) border = words[0];
        end = j;
      }
    }
    if (r.min_p > 0.0f) {
      const double d = top - floor((heaviest + log((double)r.min_p)) * 4.0);
      const int j = d >= kBins ? kBins : max((int)d, 0);
      if (j < end) {
        end = j;
        border = 0;
        at_least = true;
        c.gather(j, counts[j]);
      } else if (j == end && j < kBins) {
        at_least = true;
      }
    }
    __syncthreads();
    if (tid < kMostParts) in_bin[tid] = 0;
    __syncthreads();
    if (end < kBins)
      c.each(end, counts[end], [&](uint64_t order, uint64_t weight) {
        if (order >= border && (!at_least || heavy(c.logit_of(order))))
          atomicAdd((unsigned long long*)&in_bin[(uint32_t)~(uint32_t)order / kPart], (unsigned long long)weight);
      });
    __syncthreads();
    for (int i = wave; i < S; i += kChoose / 64) {
      double sum = 0.0;
      const int from = behind(i);
      for (int j = lane; j < end; j += 64)
        if (j >= from) sum += (double)(part_bin(i, j) & kSumMask) * kUnit * table[j];
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
      if (lane == 0) part_sum[i] = end < kBins ? sum + (double)in_bin[i] * kUnit * table[end] : sum;
    }
  } else if (tid < S) {
    const int from = behind(tid);
    part_sum[tid] = from < kBins ? parts[tid].sum * table[from] : 0.0;
  }
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < S; ++i) total += part_sum[i];
  const double target = (double)fminf(fmaxf(a.uniform[row], 0.0f), 0x1.fffffep-1f) * total;
  double base = 0.0;
  int part = -1;
  for (int i = 0; i < S; ++i) {
    if (part_sum[i] <= 0.0) continue;
    if (part >= 0) base += part_sum[part];
    part = i;
    if (base + part_sum[i] > target) break;
  }
  // A uniform number this close to 0 asks for the first tokens, whose weights may be those that the sums do without: part after part.
  const bool least = target < total * 0x1p-60;
  if (least) base = 0.0, part = 0;
  for (;; ++part) {
    // eight logits of the part a thread, in order
    double mine[8], sum = 0.0;
    const int at = part * kPart + tid * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mine[e] = 0.0;
      if (at + e < a.vocab) {
        const float l = c.at(at + e);
        const Binned b = binned(l, r.per_t);
        const int j = c.below(b, l);
        if (j < end || (j == end && j < kBins && order_of(l, at + e) >= border && (!at_least || heavy(l)))) mine[e] = b.weight * table[j];
        if (least && j == kBins && end == kBins) mine[e] = exp((double)l * r.per_t * 0.25 - heaviest);
      }
      sum += mine[e];
    }
    double before = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double v = __shfl_up(before, off, 64);
      if (lane >= off) before += v;
    }
    if (lane == 63) wave_sum[wave] = before;
    __syncthreads();
    before = base + (before - sum);
    for (int w = 0; w < kChoose / 64; ++w) {
      if (w < wave) before += wave_sum[w];
      base += wave_sum[w];
    }
    int kept = -1;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (mine[e] > 0.0) {
        before += mine[e];
        kept = at + e;
        if (before > target) {
          atomicMin(&pick, at + e);
          break;
        }
      }
    }
    if (kept >= 0) atomicMax(&last, kept);
    __syncthreads();
    if (!least || pick != INT32_MAX || part + 1 == S) break;
    __syncthreads();  // everyone has seen that there is no pick yet
  }
  if (tid == 0) a.ids[row] = pick == INT32_MAX ? last : pick;  // (a rounding away from the end: the last one kept)
}

inline int parts_of(int64_t vocab) { return (int)((vocab + kPart - 1) / kPart); }
inline int chunks_of(int64_t vocab) { return (int)((vocab + kChunk - 1) / kChunk); }

template <typename T>
int launch(const SampleArgs& s, hipStream_t st) {
  hipLaunchKernelGGL(scan_kernel<T>, dim3((unsigned)(s.a.n_rows * s.parts)), dim3(kScan), 0, st, s);
  AWQ_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(choose_kernel<T>, dim3((unsigned)s.a.n_rows), dim3(kChoose), 0, st, s);
  AWQ_HIP_TRY(hipGetLastError());
  return AWQ_OK;
}

}  // namespace

int64_t sample_workspace_bytes(int64_t n_rows, int64_t vocab) {
  const int64_t parts = n_rows * parts_of(vocab);
  return parts * (int64_t)sizeof(Part) + parts * kBins * 8 + (n_rows * chunks_of(vocab) * 4 + 15) / 16 * 16;
}

int launch_sample(const awq_sample_args& a, int dtype, hipStream_t st) {
  if (a.n_rows == 0) return AWQ_OK;
  SampleArgs s;
  s.a = a;
  s.parts = parts_of(a.vocab);
  s.chunks = chunks_of(a.vocab);
  AWQ_REQUIRE(s.parts <= kMostParts && a.n_rows * s.parts < (1ll << 31), "too many logits");
  s.part = (Part*)a.workspace;
  s.histogram = (uint64_t*)(s.part + a.n_rows * s.parts);
  s.chunk = (float*)(s.histogram + a.n_rows * s.parts * kBins);
  if (dtype == AWQ_DTYPE_FLOAT32) return launch<float>(s, st);
  return dtype == AWQ_DTYPE_BFLOAT16 ? launch<bf16_t>(s, st) : launch<half_t>(s, st);
}
