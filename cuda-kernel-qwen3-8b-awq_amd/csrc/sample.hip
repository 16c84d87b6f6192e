// A token of each row of logits: temperature, top-k, top-p and min-p, from given uniform numbers (batch.hpp).
#include "batch.hpp"
#include "lane_sums.hpp"

namespace {

// Weights go into bins of an eighth of a nat, y = 8 l / T, bin floor(y); of a row or a part of it only the 512 bins from its largest logit's down
// are looked at: what lies further is below e^-63, and 64 bits of a sum would not show it.  Within a bin a weight is e^((y - bin - 1) / 8),
// between e^(-1/8) and 1, as a whole multiple of 2^-36, so that sums do not depend on their order; bins are joined in 64-bit floating point.
// (Tokens with the largest logit are all in the first bin: their sums are exact, and uniform numbers such as 1/2 fall between two of them as
// they should.)
// 151,936 logits a row, traced.  256 rows of binary32: scan 50 us filtered, 46 not, 29 greedy (33 us of a copy's rate; LDS additions and 64-bit arithmetic),
// choose 18 us for top-k 50, 44 to 64 for top-p (a bin of thousands, whose tokens are in most chunks: one compute unit reads the row again).  One row of binary16: 6 us,
// and 6 unfiltered, 15 top-k, 28 to 39 top-p: bound by steps one behind the other, of a trip to memory or a barrier each.
//   scan_kernel    parts of 8,192 logits: largest, sum of weights, and where a row is filtered a histogram, sums and counts by bin
//   choose_kernel  a workgroup a row: the bin in which the tokens kept end, the order within that bin alone, the part that the uniform
//                  number falls in, and the token in that part.
constexpr int kPart = 8192, kScan = 256, kChoose = 512, kBins = 512, kDigits = 256, kChunk = 32, kHeld = 8192, kFew = 128, kMostParts = 64;
constexpr int kMostChunks = kMostParts * kPart / kChunk, kCopies = 8;
constexpr int kFixed = 36, kCountShift = 50;
constexpr uint64_t kSumMask = (1ull << kCountShift) - 1;
constexpr double kUnit = 1.0 / (double)(1ll << kFixed);
constexpr double kRound = 0x1.8p16;  // numbers of its size are 2^-36 apart

struct Part {
  float largest;
  int32_t first;  // lowest id of the largest
  double sum;     // of the weights, relative to e^((bin + 1) / 8) of the largest's bin
};
struct SampleArgs {
  awq_sample_args a;
  int parts, chunks;
  Part* part;           // [rows][parts]
  uint64_t* histogram;  // [rows][parts][kBins]: count << 50 | sum, from the bin of the part's largest down
  float* chunk;         // [rows][chunks]: largest of 32 logits
};

// a value that all lanes have, in scalar registers: branches on it are the wavefront's, and it takes no lane's register through them
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(uniform(__float_as_uint(v))); }
__device__ __forceinline__ uint64_t uniform(uint64_t v) { return (uint64_t)uniform((uint32_t)(v >> 32)) << 32 | uniform((uint32_t)v); }
__device__ __forceinline__ double uniform(double v) { return __longlong_as_double((long long)uniform((uint64_t)__double_as_longlong(v))); }

__device__ __forceinline__ double last_lane(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

struct Row {
  double per_t;  // 8 / T
  float top_p, min_p;
  int top_k;  // 0: not limited
  bool greedy, filtered;
};
__device__ __forceinline__ Row row_of(const awq_sample_args& a, int64_t row) {
  Row r;
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  r.greedy = !(t > 0.0f);
  r.per_t = uniform(8.0 / (double)t);
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

__device__ __forceinline__ double bin_of(float l, const Row& r) { return floor((double)l * r.per_t); }
struct Binned {
  double bin, rounded;  // rounded: kRound + the weight relative to e^((bin + 1) / 8)
};
__device__ __forceinline__ Binned binned(float l, const Row& r) {
  // (of y beyond 2^53 x is 0, and different logits are too far from each other to meet)
  const double y = (double)l * r.per_t, b = floor(y), x = y - b;
  // e^((x - 1) / 8) for x from 0 to 1: the polynomial through its values at the six Chebyshev points, within 2.8e-12
  double e = 2.389384121670446e-07;
  e = fma(e, x, 8.96072434860192e-06);
  e = fma(e, x, 0.0002872797252023532);
  e = fma(e, x, 0.0068945050309035805);
  e = fma(e, x, 0.11031211299649428);
  e = fma(e, x, 0.8824969025821857);
  return {b, e + kRound};
}
// the weight as a multiple of 2^-36, and as a number
__device__ __forceinline__ uint64_t fixed_of(const Binned& b) { return (uint64_t)__double_as_longlong(b.rounded) & ((1ull << 51) - 1); }
__device__ __forceinline__ double weight_of(const Binned& b) { return b.rounded - kRound; }

__device__ __forceinline__ float logit(float v) { return v != v ? -INFINITY : v + 0.0f; }  // (-0 as 0)
// of a row with logits of +infinity those share the weight
__device__ __forceinline__ float finite(float v, bool infinite) { return infinite ? (v == INFINITY ? 0.0f : -INFINITY) : v; }

// order of logits as whole numbers
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(l);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// order of the tokens: falling logits, rising ids; larger numbers first
__device__ __forceinline__ uint64_t order_of(float l, uint32_t id) { return (uint64_t)key_of(l) << 32 | (uint32_t)~id; }

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
  // (copies by lane: lanes that meet in a bin wait for each other; a bin behind the last for what is further, which nobody reads)
  __shared__ unsigned long long bins[(kBins + 1) * kCopies];
  __shared__ double table[kBins + 1];
  const awq_sample_args& a = s.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / s.parts;
  const int part = blockIdx.x % s.parts;
  const T* const x = (const T*)a.logits + row * a.ld;
  float v[L][W];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int64_t at = (int64_t)part * kPart + (i * kScan + tid) * W;
    if (at + W <= a.vocab) {
      const vec_t u = *reinterpret_cast<const vec_t*>(x + at);
#pragma unroll
      for (int e = 0; e < W; ++e) v[i][e] = fmaxf((float)u[e], -INFINITY);  // (of NaN -infinity)
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) v[i][e] = at + e < a.vocab ? fmaxf((float)x[at + e], -INFINITY) : -INFINITY;
    }
  }
  const Row r = row_of(a, row);
  if (!r.greedy) {
    if (r.filtered) {
      for (int b = tid; b < kBins * kCopies; b += kScan) bins[b] = 0;
    } else {
      for (int b = tid; b < kBins; b += kScan) table[b] = exp(-0.125 * b);
      if (tid == 0) table[kBins] = 0.0;
    }
  }
  float largest = -INFINITY;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    float m = v[i][0];
#pragma unroll
    for (int e = 1; e < W; ++e) m = fmaxf(m, v[i][e]);
    largest = fmaxf(largest, m);
    if (r.filtered) {
      m = lanes::maximum<LANES>(m) + 0.0f;  // (-0 as 0)
      const int64_t at = ((int64_t)part * kPart + (i * kScan + tid) * W) / kChunk;
      if (tid % LANES == 0 && at < s.chunks) s.chunk[row * s.chunks + at] = m;
    }
  }
  largest = lanes::maximum<64>(largest) + 0.0f;
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
    if (infinite) {
#pragma unroll
      for (int i = 0; i < L; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e) v[i][e] = finite(v[i][e], true);
    }
    const double top = bin_of(finite(largest, infinite), r);
    // (a float as the number of a far bin is the largest of its kind)
    const auto place = [&](const Binned& b) __attribute__((always_inline)) { return min((uint32_t)__builtin_elementwise_min(top - b.bin, 4e9), (uint32_t)kBins); };
    double sum = 0.0;
    if (r.filtered) {
#pragma unroll
      for (int i = 0; i < L; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const Binned b = binned(v[i][e], r);
          atomicAdd(&bins[place(b) * kCopies + lane % kCopies], (1ull << kCountShift) | fixed_of(b));
        }
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const Binned b = binned(v[i][e], r);
          sum = fma(fmax(weight_of(b), 0.0), table[place(b)], sum);  // (of -infinity NaN)
        }
    }
    if (r.filtered) {
      __syncthreads();
      for (int b = tid; b < kBins; b += kScan) {
        unsigned long long all = 0;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) all += bins[b * kCopies + (c + tid) % kCopies];
        s.histogram[(row * s.parts + part) * kBins + b] = all;
      }
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

struct ChooseMemory {
  uint64_t held[kHeld];       // order of the tokens of a bin, where they are so few
  uint16_t list[kMostChunks]; // chunks that have some
  uint64_t few[kFew], few_weight[kFew];
  uint64_t digit[kDigits];
  uint32_t digit_count[kDigits];
  uint64_t word[2], in_bin[kMostParts];
  uint64_t fixed[kBins];
  uint32_t bin_count[kBins];
  double table[kBins], part_sum[kMostParts], wave_sum[kChoose / 64], until[kChoose];
  uint32_t wave_count[kChoose / 64];
  Part part[kMostParts];
  int behind[kMostParts];
  uint32_t held_count, list_count, few_count;
  int pick, last;
};

// The first of 64 N entries, N a lane, at which `full` holds of the sums up to it (itself included), and the sums ahead of it; 64 N: none.
// Every wavefront finds it for itself.
template <typename S>
struct Found {
  int at;
  S sum;
  uint32_t count;
};
template <int N, typename S, typename F>
__device__ __forceinline__ Found<S> first_full(const S (&sum)[N], const uint32_t (&count)[N], F full) {
  const int lane = threadIdx.x & 63;
  S mine = sum[0];
  uint32_t many = count[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mine += sum[i], many += count[i];
  S s = lanes::ahead<0x138, 0xf>(lanes::upto(mine));  // the sums ahead as they are formed, not as a difference
  uint32_t n = lanes::upto(many) - many;
  int at = N;
  S before = s;
  uint32_t before_count = n;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s += sum[i];
    n += count[i];
    if (at == N) {
      if (full(s, n)) at = i;
      else before = s, before_count = n;
    }
  }
  const unsigned long long any = __builtin_amdgcn_ballot_w64(at < N);
  if (any == 0) return {64 * N, (S)0, 0};
  const int from = __builtin_ctzll(any);
  return {uniform(N * from + __shfl(at, from, 64)), uniform(__shfl(before, from, 64)), uniform((uint32_t)__shfl((int)before_count, from, 64))};
}

template <typename T>
struct Choose {
  const SampleArgs& s;
  const Row& r;
  const T* x;
  const float* chunk;
  ChooseMemory& m;
  float largest;  // of the row
  double top;     // its bin
  bool infinite;

  __device__ __forceinline__ float of(T v) const { return finite(logit((float)v), infinite); }
  __device__ __forceinline__ float at(int i) const { return of(x[i]); }
  // distance of a logit's bin from the row's first; kBins: further or no weight
  __device__ __forceinline__ int below(const Binned& b, float l) const {
    const double d = top - b.bin;
    return l == -INFINITY || !(d < kBins) ? kBins : (int)d;
  }
  // the lowest order of a logit in bin j or ahead of it: among the 64 around the quotient, or else by 64 guesses at a time
  __device__ __forceinline__ uint32_t lowest_key(int j) const {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = key_of(-INFINITY), hi = uniform(key_of(largest));  // not in it, in it
    const auto in_bin = [&](uint32_t guess) __attribute__((always_inline)) { return guess >= hi || (guess > lo && top - bin_of(logit_of(guess), r) <= j); };
    const uint32_t around = uniform(key_of((float)((top - j) / r.per_t))) - 31;
    const unsigned long long near = __builtin_amdgcn_ballot_w64(in_bin(around + lane));
    if (near != 0 && !(near & 1)) return around + (uint32_t)__builtin_ctzll(near);
    for (int turn = 0; turn < 6 && hi - lo > 1; ++turn) {  // (2^32 in six turns)
      const uint32_t step = (hi - lo + 63) / 64;
      const unsigned long long in = __builtin_amdgcn_ballot_w64(in_bin(lo + step * (lane + 1)));
      const uint32_t first = __builtin_ctzll(in | 1ull << 63);  // (the last lane's guess is not below hi)
      hi = min(hi, lo + step * (first + 1));
      lo = lo + step * first;
    }
    return hi;
  }
  // the tokens of the orders a .. b - 1 into `held`, out of the row, by the chunks listed: 16 bytes of a chunk a thread and 64 logits at once.
  // First their ids, which a few lanes have at a time; then a logit a thread.
  __device__ __forceinline__ void hold(uint64_t a, uint64_t b) const {
    constexpr int W = 16 / sizeof(T), LANES = kChunk / W, AT_ONCE = kChoose / LANES, U = 64 / W;
    typedef typename Some<T, W>::type vec_t;
    const int vocab = (int)s.a.vocab, n = uniform((int)m.list_count), first = threadIdx.x / LANES, in_chunk = threadIdx.x % LANES * W;
    // (a and b are whole keys; of a row with +infinity the tokens that have it)
    const float least = infinite ? INFINITY : logit_of((uint32_t)(a >> 32)), most = infinite ? INFINITY : logit_of((uint32_t)(b >> 32) - 1);
    for (int c0 = 0; c0 < n; c0 += U * AT_ONCE) {
      vec_t v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c0 + u * AT_ONCE >= n) break;
        const int c = c0 + u * AT_ONCE + first, id = c < n ? m.list[c] * kChunk + in_chunk : vocab;
        if (id + W <= vocab) {
          v[u] = *reinterpret_cast<const vec_t*>(x + id);
        } else {
#pragma unroll
          for (int e = 0; e < W; ++e) v[u][e] = id + e < vocab ? x[id + e] : (T)-INFINITY;
        }
      }
      uint64_t in = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c0 + u * AT_ONCE >= n) break;
#pragma unroll
        for (int e = 0; e < W; ++e) in |= (uint64_t)((float)v[u][e] >= least && (float)v[u][e] <= most) << (u * W + e);
      }
      const uint32_t mine = __builtin_popcountll(in), upto = lanes::upto(mine);
      uint32_t to = 0;
      if ((threadIdx.x & 63) == 63 && upto) to = atomicAdd(&m.held_count, upto);
      to = (uint32_t)__builtin_amdgcn_readlane((int)to, 63) + upto - mine;
      for (; in; in &= in - 1, ++to) {
        const int bit = __builtin_ctzll(in);
        if (to < (uint32_t)kHeld) m.held[to] = (uint32_t)(m.list[c0 + bit / W * AT_ONCE + first] * kChunk + in_chunk + bit % W);
      }
    }
    __syncthreads();
    const int held = uniform(min((int)m.held_count, kHeld));
#pragma unroll 4
    for (int i = threadIdx.x; i < held; i += kChoose) {
      const int id = (int)m.held[i];
      m.held[i] = order_of(at(id), id);
    }
  }
  __device__ __forceinline__ uint64_t fixed_at(uint64_t order) const { return fixed_of(binned(logit_of((uint32_t)(order >> 32)), r)); }
  // every token of the orders a .. b - 1 of a bin of n; where they are not held a logit a thread (rows of some thousand equals)
  template <typename F>
  __device__ __forceinline__ void each(int n, uint64_t a, uint64_t b, F f) const {
    const int all = n <= kHeld ? n : uniform((int)m.list_count) * kChunk;
#pragma unroll 1
    for (int i = threadIdx.x; i < all; i += kChoose) {
      uint64_t order = 0;
      if (n <= kHeld) {
        order = m.held[i];
      } else {
        const int id = m.list[i / kChunk] * kChunk + i % kChunk;
        if (id < (int)s.a.vocab) order = order_of(at(id), id);
      }
      if (order >= a && order < b) f(order);
    }
  }
  // the chunks of bin j's n tokens (bin kBins: of those beyond the bins), and the tokens themselves where they are few; a, b: their orders
  __device__ __forceinline__ void gather(int j, int n, uint64_t& a, uint64_t& b) const {
    const uint32_t low = j < kBins ? lowest_key(j) : key_of(-INFINITY) + 1;
    a = (uint64_t)low << 32;
    b = (uint64_t)(j ? lowest_key(j - 1) : key_of(largest) + 1) << 32;
    __syncthreads();  // the last bin's readers are done
    if (threadIdx.x == 0) m.held_count = m.list_count = 0;
    __syncthreads();
    const int lane = threadIdx.x & 63;
    constexpr int U = 10;
    for (int c0 = 0; c0 < s.chunks; c0 += U * kChoose) {
      float largest_of[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * kChoose + threadIdx.x;
        largest_of[u] = c < s.chunks ? chunk[c] : -INFINITY;
      }
      uint32_t mine = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) mine += key_of(finite(largest_of[u], infinite)) >= low;
      const uint32_t upto = lanes::upto(mine);
      uint32_t to = 0;
      if (lane == 63 && upto) to = atomicAdd(&m.list_count, upto);
      to = (uint32_t)__builtin_amdgcn_readlane((int)to, 63) + upto - mine;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (key_of(finite(largest_of[u], infinite)) >= low) m.list[to++] = (uint16_t)(c0 + u * kChoose + threadIdx.x);
    }
    __syncthreads();
    if (n > kHeld) return;
    hold(a, b);
    __syncthreads();
  }
  // Of a bin's n tokens, of the orders a .. b - 1, the one with which the count (by_sum == false: `need` of them) or the sum of the weights (the first at
  // which it reaches `reach`) is full.  word[0]: its order, 0 if there is none; word[1]: the sum up to it, itself included.
  // By digits of the order until few are left, then each of those against all others.
  __device__ __forceinline__ void last_kept(int n, uint64_t a, uint64_t b, bool by_sum, uint32_t need, double reach) const {
    const int tid = threadIdx.x, lane = tid & 63, all = n;
    uint64_t ahead = 0;
    uint32_t ahead_count = 0;
    __syncthreads();
    if (tid == 0) m.word[0] = m.word[1] = 0;
    while (n > kFew) {
      const int shift = max(0, 56 - __builtin_clzll(b - a - 1));  // (b - a - 1) >> shift is below 256
      __syncthreads();
      if (tid < kDigits) m.digit[tid] = 0, m.digit_count[tid] = 0;
      __syncthreads();
      each(all, a, b, [&](uint64_t order) {
        const int d = (int)((order - a) >> shift);
        atomicAdd((unsigned long long*)&m.digit[d], (unsigned long long)fixed_at(order));
        atomicAdd(&m.digit_count[d], 1u);
      });
      __syncthreads();
      uint64_t sum[4];
      uint32_t count[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = m.digit[255 - 4 * lane - i], count[i] = m.digit_count[255 - 4 * lane - i];
      const Found<uint64_t> f = first_full(sum, count, [&](uint64_t su, uint32_t co) {
        return by_sum ? (double)(ahead + su) >= reach : ahead_count + co >= need;
      });
      if (f.at == kDigits) return;  // (a rounding away from all of them)
      const uint64_t d = 255 - f.at;
      ahead += f.sum;
      ahead_count += f.count;
      n = uniform((int)m.digit_count[d]);
      a += d << shift;
      if (b - a > 1ull << shift) b = a + (1ull << shift);
    }
    __syncthreads();
    if (tid == 0) m.few_count = 0;
    __syncthreads();
    each(all, a, b, [&](uint64_t order) {
      const uint32_t to = atomicAdd(&m.few_count, 1u);
      if (to < (uint32_t)kFew) {
        m.few[to] = order;
        m.few_weight[to] = fixed_at(order);
      }
    });
    __syncthreads();
    n = uniform(min((int)m.few_count, kFew));
    const int wide = n <= 8 ? 64 : kChoose >> (32 - __builtin_clz(n - 1));  // threads a token: 1 .. 64
    static_assert(kFew <= kChoose && 8 * 64 <= kChoose, "a thread a token at least");
    const int mine = tid / wide;
    const uint64_t order = mine < n ? m.few[mine] : ~0ull;
    uint64_t sum = 0;
    uint32_t count = 0;
#pragma unroll 4
    for (int i = tid % wide; i < n; i += wide) {
      const uint64_t weight = m.few_weight[i];
      const bool before = m.few[i] > order;
      count += before;
      sum += before ? weight : 0;
    }
    for (int off = wide / 2; off > 0; off >>= 1) {
      sum += __shfl_xor(sum, off, 64);
      count += __shfl_xor(count, off, 64);
    }
    if (mine < n && tid % wide == 0) {
      const uint64_t with = ahead + sum + m.few_weight[mine];
      if (by_sum ? (double)(ahead + sum) < reach && (double)with >= reach : ahead_count + count + 1 == need) m.word[0] = order, m.word[1] = with;
    }
    __syncthreads();
  }
};

// (512 threads: at 1,024 a thread has 128 registers, fewer than it needs)
template <typename T>
__global__ __launch_bounds__(kChoose) void choose_kernel(SampleArgs s) {
  __shared__ ChooseMemory m;
  const awq_sample_args& a = s.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = s.parts;
  const int64_t row = blockIdx.x;
  if (tid < S) m.part[tid] = s.part[row * S + tid];
  const Row r = row_of(a, row);
  static_assert(kBins == kChoose, "a thread a bin");
  if (!r.greedy) {
    m.table[tid] = exp(-0.125 * tid);
  }
  if (tid < kMostParts) m.in_bin[tid] = 0;
  if (tid == 0) m.pick = INT32_MAX, m.last = 0;
  const float uniform_number = a.uniform[row];
  __syncthreads();
  float largest = uniform(lanes::maximum<64>(lane < S ? m.part[lane].largest : -INFINITY));
  if (r.greedy || largest == -INFINITY) {
    if (tid == 0) {
      int id = 0;
      if (largest > -INFINITY)
        for (int i = 0; i < S; ++i)
          if (m.part[i].largest == largest) {
            id = m.part[i].first;
            break;
          }
      a.ids[row] = id;
    }
    return;
  }
  const bool infinite = largest == INFINITY;
  largest = finite(largest, infinite);
  const double top = uniform(bin_of(largest, r));
  const Choose<T> c{s, r, (const T*)a.logits + row * a.ld, s.chunk + row * s.chunks, m, largest, top, infinite};
  // how far the first bin of a part lies below the row's; its bin i is the row's behind + i
  if (tid < S) {
    const float l = finite(m.part[tid].largest, infinite);
    const double d = top - bin_of(l, r);
    m.behind[tid] = l == -INFINITY || !(d < kBins) ? kBins : (int)d;
  }
  __syncthreads();
  const uint64_t* const histogram = s.histogram + row * S * kBins;

  // A uniform number this close to 0 asks for the first tokens, whose weights may be those that the sums do without.
  const bool least = !(uniform_number >= 0x1p-60f);
  int end = kBins;          // bins below it are kept whole, those above it not at all
  uint64_t border = 0;      // of bin `end` the tokens that are not behind this in order (of those beyond the bins where it is kBins)
  float lightest = -INFINITY;  // no token behind this logit is kept
  bool at_least = false;    // and those of them that weigh at least min_p
  const double heaviest = uniform((double)largest * r.per_t * 0.125);
  const auto heavy = [&](float l) { return exp((double)l * r.per_t * 0.125 - heaviest) >= (double)r.min_p; };
  if (r.filtered) {
    {  // a bin of the row a thread
      uint64_t fixed = 0;
      uint32_t count = 0;
      constexpr int U = 20;
      for (int i0 = 0; i0 < S; i0 += U) {
        uint64_t h[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = min(i0 + u, S - 1), b = tid - m.behind[i];
          h[u] = i0 + u < S && b >= 0 ? histogram[i * kBins + b] : 0;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) fixed += h[u] & kSumMask, count += (uint32_t)(h[u] >> kCountShift);
      }
      m.fixed[tid] = fixed;
      m.bin_count[tid] = count;
      const double of_wave = lanes::upto((double)fixed * kUnit * m.table[tid]);
      count = lanes::upto(count);
      if (lane == 63) m.wave_sum[wave] = of_wave, m.wave_count[wave] = count;
    }
    __syncthreads();
    // the first bin at which `full` holds of the sums up to it: of 64 bins together, then of theirs; every wavefront for itself
    constexpr int N = kBins / 64;
    const double of_many = lane < N ? m.wave_sum[lane] : 0.0;
    const uint32_t count_of_many = lane < N ? m.wave_count[lane] : 0;
    const double many_upto = lanes::upto(of_many), many_ahead = lanes::ahead<0x138, 0xf>(many_upto);
    const uint32_t count_ahead = lanes::upto(count_of_many) - count_of_many;
    const auto first_bin = [&](auto full) __attribute__((always_inline)) {
      const unsigned long long any = __builtin_amdgcn_ballot_w64(lane < N && full(many_ahead + of_many, count_ahead + count_of_many));
      if (any == 0) return Found<double>{kBins, 0.0, 0};
      const int many = __builtin_ctzll(any), bin = 64 * many + lane;
      const double base = uniform(__shfl(many_ahead, many, 64));
      const uint32_t base_count = uniform((uint32_t)__shfl((int)count_ahead, many, 64)), count = m.bin_count[bin];
      const double upto = lanes::upto((double)m.fixed[bin] * kUnit * m.table[bin]), ahead = base + lanes::ahead<0x138, 0xf>(upto);
      const uint32_t count_upto = lanes::upto(count);
      // (the last of them has the sums that were looked at)
      const int from = __builtin_ctzll(__builtin_amdgcn_ballot_w64(full(base + upto, base_count + count_upto)) | 1ull << 63);
      return Found<double>{64 * many + from, uniform(__shfl(ahead, from, 64)), base_count + uniform((uint32_t)__shfl((int)(count_upto - count), from, 64))};
    };
    double all = last_lane(many_upto);
    const uint32_t in_bins = (uint32_t)__builtin_amdgcn_readlane((int)lanes::upto(count_of_many), 63);
    uint64_t from = 0, to = 0;  // the orders of bin `end`
    // top-k, top-p and min-p, each within what those ahead of it keep
#pragma unroll 1
    for (int filter = 0; filter < 3; ++filter) {
      int j;
      uint32_t need = 0;
      double reach = 0.0;
      if (filter < 2) {
        if (filter == 0 ? r.top_k == 0 : !(r.top_p < 1.0f)) continue;
        const double target = (double)r.top_p * all;
        Found<double> f = first_bin([&](double su, uint32_t n) { return filter ? su >= target : n >= (uint32_t)r.top_k; });
        // fewer tokens within the bins than top-k keeps: sums do without the others, their order matters if the first tokens are asked for
        if (f.at == kBins && (filter || !least)) continue;
        j = min(f.at, end);
        if (j < f.at) {  // (a rounding away from all that top-k keeps: the bin that it ends in)
          f.sum = 0.0;
          for (int i = 0; i < j; ++i) f.sum += (double)m.fixed[i] * kUnit * m.table[i];
          f.sum = uniform(f.sum);
        }
        need = r.top_k - (j < kBins ? f.count : in_bins);
        if (j < kBins) {
          reach = uniform((target - f.sum) / (kUnit * m.table[j]));
          if (filter == 0) all = f.sum;  // and what is kept of bin j
        }
      } else {
        if (!(r.min_p > 0.0f)) continue;
        const double d = top - floor((heaviest + log((double)r.min_p)) * 8.0);
        j = uniform(d >= kBins ? kBins : max((int)d, 0));
        if (j > end || j == kBins) continue;
        at_least = true;
        if (j == end) continue;
        border = 0;
      }
      const int n = j < kBins ? uniform((int)m.bin_count[j]) : kHeld + 1;  // (those beyond the bins are not held)
      if (j != end || j == kBins) c.gather(j, n, from, to);
      if (filter < 2) {
        c.last_kept(n, from, to, filter == 1, need, reach);
        const uint64_t last = uniform(m.word[0]);
        border = j == end && border > last ? border : last;
        if (j == kBins) continue;
        if (filter == 0) all = uniform(all + (double)m.word[1] * kUnit * m.table[j]);
      }
      end = j;
      lightest = logit_of((uint32_t)(from >> 32));
    }
    __syncthreads();
    if (end < kBins)
      c.each(uniform((int)m.bin_count[end]), from, to, [&](uint64_t order) {
        if (order >= border && (!at_least || heavy(logit_of((uint32_t)(order >> 32)))))
          atomicAdd((unsigned long long*)&m.in_bin[(uint32_t)~(uint32_t)order / kPart], (unsigned long long)c.fixed_at(order));
      });
    __syncthreads();
    constexpr int U = 4, WAVES = kChoose / 64;
    for (int i0 = wave; i0 < S; i0 += U * WAVES) {
      uint64_t h[U][2];  // of four parts the first 128 bins: mostly that is all
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int i = i0 + u * WAVES, b = 64 * v + lane;
          h[u][v] = i < S && b + m.behind[i] < end ? histogram[i * kBins + b] : 0;
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * WAVES;
        if (i >= S) break;
        const int behind = m.behind[i];
        double part = 0.0;
#pragma unroll
        for (int v = 0; v < 2; ++v) part += (double)(h[u][v] & kSumMask) * kUnit * m.table[min(64 * v + lane + behind, kBins - 1)];
        for (int b = 128 + lane; b + behind < end; b += 64) part += (double)(histogram[i * kBins + b] & kSumMask) * kUnit * m.table[b + behind];
        part = lanes::upto(part);
        if (lane == 63) m.part_sum[i] = end < kBins ? part + (double)m.in_bin[i] * kUnit * m.table[end] : part;
      }
    }
  } else if (tid < S) {
    m.part_sum[tid] = m.behind[tid] < kBins ? m.part[tid].sum * m.table[m.behind[tid]] : 0.0;
  }
  __syncthreads();
  const double of_part[1] = {lane < S ? m.part_sum[lane] : 0.0};
  const double total = last_lane(lanes::upto(of_part[0]));
  const double target = (double)fminf(fmaxf(uniform_number, 0.0f), 0x1.fffffep-1f) * total;
  const uint32_t nothing[1] = {0};
  static_assert(kMostParts == 64, "a part a lane");
  const Found<double> in_part = first_full(of_part, nothing, [&](double su, uint32_t) { return su > target; });
  double base = in_part.sum;
  int part = in_part.at < 64 ? in_part.at : 0;  // (a row has some weight, so one of its parts is it)
  if (least) base = 0.0, part = 0;  // part after part
  const auto weight_of_token = [&](T logit_of_it, int id) __attribute__((always_inline)) {
    const float l = c.of(logit_of_it);
    if (l < lightest) return 0.0;
    const Binned b = binned(l, r);
    const int j = c.below(b, l);
    if (j < end || (j == end && j < kBins && order_of(l, id) >= border && (!at_least || heavy(l)))) return weight_of(b) * m.table[j];
    const bool beyond = least && j == kBins && end == kBins && order_of(l, id) >= border && (!(r.min_p > 0.0f) || heavy(l));
    return beyond ? exp((double)l * r.per_t * 0.125 - heaviest) : 0.0;
  };
  constexpr int kEach = kPart / kChoose;
  for (;; ++part) {
    // sixteen logits of the part a thread, in order; then those of the thread that the number falls in, one a lane
    double sum = 0.0;
    const int at = part * kPart + tid * kEach;
    typedef typename Some<T, 16 / sizeof(T)>::type vec_t;
    constexpr int W = 16 / sizeof(T), L = kEach / W;
    vec_t v[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (at + (i + 1) * W <= a.vocab) {
        v[i] = *reinterpret_cast<const vec_t*>(c.x + at + i * W);
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) v[i][e] = at + i * W + e < a.vocab ? c.x[at + i * W + e] : (T)-INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < L; ++i)
#pragma unroll
      for (int e = 0; e < W; ++e) sum += weight_of_token(v[i][e], at + i * W + e);
    double before = lanes::upto(sum);
    if (lane == 63) m.wave_sum[wave] = before;
    __syncthreads();
    before += base;
#pragma unroll
    for (int w = 0; w < kChoose / 64; ++w) {
      if (w < wave) before += m.wave_sum[w];
      base += m.wave_sum[w];
    }
    const unsigned long long some = __builtin_amdgcn_ballot_w64(sum > 0.0), over = __builtin_amdgcn_ballot_w64(sum > 0.0 && before > target);
    if (lane == 0 && some) atomicMax(&m.last, tid + 63 - __builtin_clzll(some));  // (of the last part that is looked at)
    if (lane == 0 && over) atomicMin(&m.pick, tid + __builtin_ctzll(over));
    if (tid < kChoose) m.until[tid] = before - sum;
    __syncthreads();
    if (!least || m.pick != INT32_MAX || part + 1 == S) break;
    __syncthreads();  // everyone has seen that there is no pick yet
  }
  if (wave == 0) {
    const int thread = m.pick == INT32_MAX ? m.last : m.pick, id = part * kPart + thread * kEach + lane;
    const double w = lane < kEach && id < a.vocab ? weight_of_token(c.x[id], id) : 0.0;
    const double before = m.until[thread] + lanes::upto(w);
    const unsigned long long over = __builtin_amdgcn_ballot_w64(w > 0.0 && before > target), some = __builtin_amdgcn_ballot_w64(w > 0.0);
    // (a rounding away from the end: the last one kept)
    const int of_thread = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : 0;
    if (lane == 0) a.ids[row] = part * kPart + thread * kEach + of_thread;
  }
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
  AWQ_REQUIRE(s.parts <= kMostParts && launchable(a.n_rows * s.parts, kScan) && launchable(a.n_rows, kChoose), "too many logits");
  s.part = (Part*)a.workspace;
  s.histogram = (uint64_t*)(s.part + a.n_rows * s.parts);
  s.chunk = (float*)(s.histogram + a.n_rows * s.parts * kBins);
  if (dtype == AWQ_DTYPE_FLOAT32) return launch<float>(s, st);
  return dtype == AWQ_DTYPE_BFLOAT16 ? launch<bf16_t>(s, st) : launch<half_t>(s, st);
}
