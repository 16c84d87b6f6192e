// Attention of prompts of different lengths, one behind the other (batch.hpp).
#include "batch.hpp"
#include "lane_sums.hpp"
#include "tile_halves.hpp"

#include <type_traits>

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <typename T>
struct Vec {
  typedef T eight __attribute__((ext_vector_type(8)));
  typedef T four __attribute__((ext_vector_type(4)));
};
__device__ __forceinline__ f32x16_t product(Vec<half_t>::eight a, Vec<half_t>::eight b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t product(Vec<bf16_t>::eight a, Vec<bf16_t>::eight b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
constexpr int kQueries = 128;

// The tile of queries a workgroup takes: request r has ceil(queries / 128) of them.  Every wavefront looks its own up.  False: there are fewer tiles.
// Up to 64 requests, a lane each: tiles with the most keys first, by 128 keys; what runs last is short.  (13 prompts of 60 to 1,000 tokens, one request
// behind the other 50 us, so 47; 3 parts of long prompts, all long, 188 and 189; next to the border no gain, 32 prompts of 20 to 600 tokens 98 and 96,
// 64 of them 178 and 183.)  More requests: one behind the other, 64 at a time, the last tile of each first, which has
// the most keys; the search would read them all some ten times.
struct Tile {
  int q_begin, q_end, k_begin, k_end, first;  // first: of the tile's queries, from q_begin on
};
__device__ __forceinline__ int clamped(int64_t x, int64_t n) { return (int)(x < 0 ? 0 : x > n ? n : x); }
__device__ __forceinline__ bool find_tile(const awq_packed_attention_args& a, int tile, Tile& out) {
  const int lane = threadIdx.x & 63;
  const int* const starts = a.k_starts ? a.k_starts : a.q_starts;
  for (int r0 = 0; r0 < a.n_requests; r0 += 64) {
    const int r = r0 + lane;
    int b = 0, e = 0, kb = 0, ke = 0;
    if (r < a.n_requests) {
      b = clamped(a.q_starts[r], a.n_tokens), e = clamped(a.q_starts[r + 1], a.n_tokens);
      kb = clamped(starts[r], a.n_keys), ke = clamped(starts[r + 1], a.n_keys);
    }
    const int tiles = e > b ? (e - b + kQueries - 1) / kQueries : 0;
    const int sum = lanes::upto(tiles);
    const int all = __builtin_amdgcn_readlane(sum, 63);
    if (a.n_requests <= 64) {
      if (tile >= all) return false;
      // A request's tiles from the last on are at the levels top, top - 1, .. (all at top where all see all keys), those without keys at 0.
      const int nk = max(ke - kb, 0), top = (a.causal ? max(nk - (e - b - (tiles - 1) * kQueries), 0) : nk) / kQueries + 1;
      const auto from_level = [&](int level) __attribute__((always_inline)) {  // tiles at it or above
        return level <= 0 ? tiles : a.causal ? min(max(top - level + 1, 0), tiles) : level <= top ? tiles : 0;
      };
      const auto over_all = [](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(lanes::upto(v), 63); };
      // the level of the tile: the highest with more tiles from it on than are ahead of this one
      int lo = 0, hi = __builtin_amdgcn_readfirstlane((int)lanes::maximum<64>(tiles ? (float)top : 0.0f));  // (at most 2^24: exact)
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (over_all(from_level(mid)) > tile) lo = mid;
        else hi = mid - 1;
      }
      const int above = from_level(lo + 1), here = from_level(lo) - above, upto = lanes::upto(here), rest = tile - over_all(above);
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > rest) | 1ull << 63);
      const int behind = __builtin_amdgcn_readlane(above, at) + rest - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(here, at));
      out.q_begin = __builtin_amdgcn_readlane(b, at);
      out.q_end = __builtin_amdgcn_readlane(e, at);
      out.first = (__builtin_amdgcn_readlane(tiles, at) - 1 - behind) * kQueries;
      out.k_begin = __builtin_amdgcn_readlane(kb, at);
      out.k_end = __builtin_amdgcn_readlane(ke, at);
      return true;
    }
    if (tile < all) {
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > tile));
      const int behind = __builtin_amdgcn_readlane(sum, at) - 1 - tile;  // tiles of the request behind this one
      out.q_begin = __builtin_amdgcn_readlane(b, at);
      out.q_end = __builtin_amdgcn_readlane(e, at);
      // the last tile first: it has the most keys
      out.first = behind * kQueries;
      out.k_begin = __builtin_amdgcn_readlane(kb, at);
      out.k_end = __builtin_amdgcn_readlane(ke, at);
      return true;
    }
    tile -= all;
  }
  return false;
}

// bits 15 and 31 of the result: some of eight 16-bit numbers are infinite or NaN
template <typename T>
__device__ __forceinline__ uint32_t not_finite(u32x4_t v) {
  constexpr uint32_t to_bit = __is_same(T, half_t) ? 0x04000400u : 0x00800080u;
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= (v[i] & 0x7fff7fffu) + to_bit;
  return any;
}
// 0 in place of those that are
template <typename T>
__device__ __forceinline__ u32x4_t only_finite(u32x4_t v) {
  constexpr uint32_t e = __is_same(T, half_t) ? 0x7c00u : 0x7f80u;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] &= ((v[i] & e) == e ? 0xffff0000u : 0xffffffffu) & ((v[i] >> 16 & e) == e ? 0x0000ffffu : 0xffffffffu);
  return v;
}

// 128 queries of one head a workgroup, 32 a wavefront; 64 keys and values at a time come into LDS by themselves, the next ones while these are
// multiplied.  Queries are columns throughout, lane (n, kh) = (lane % 32, lane / 32):
//     S^T[key][query] = K Q^T,   O^T[c][query] += V^T P^T      v_mfma_f32_32x32x16
// so that a query's maximum, sum and rescaling stay in a lane and its partner, and the weights a lane forms are the elements it
// supplies to the second product (slice j: keys 16 j + 8 (e / 4) + 4 kh + e % 4; V^T by the transposing LDS read).  Scores, maxima and sums
// are binary32; a weight is rounded to the activations' type for the second product alone.
// A row's 16-byte pieces lie rotated in LDS so that the rows that lanes read together are in all banks.
// A step's scores are formed during the step ahead, each product of theirs beside a few of its weights, so that matrix and vector instructions of one
// wavefront run together; keys are therefore requested two steps ahead, values one.  (What is on its way is waited for ahead of a step's first
// transposing read, the compiler's doing, and ahead of the next barrier: a request runs beside the step's masks and maximum.)
// Heads of 128, 32 over 8: 13 prompts of 60 to 1,000 tokens, binary16, 42 us a call in a row, 46 traced; 3 parts of 500 to 1,100 tokens behind 3,500 each,
// bfloat16, 168 us, 0.79 PFLOP/s, and 205.  (The other figures here are traced ones of their time, against each other.)  Bound by the two kinds of instructions (each a third of the time) and by 800 workgroups on 512 places.  64 keys a step and two wavefronts a
// SIMD: 32 keys and three 57 and 236 us where these took 54 and 216; scores in their own step 53 and 206, formed a step ahead 50 and 188 (and 47 and 179 with the first values
// read ahead of them); heads of 64 with three wavefronts, some numbers in scratch memory, 74 us, with two 72.
// Where some query of the workgroup does not see all keys of a step, values that are not finite are kept out of the product, in which 0 times
// them is NaN, and are added for the queries that see them.
template <typename T, int D, int kStep, int WAVES>
__global__ __launch_bounds__(256, WAVES) void packed_kernel(awq_packed_attention_args a) {
  typedef typename Vec<T>::eight eight_t;
  typedef typename Vec<T>::four four_t;
  typedef __attribute__((address_space(1))) const void* gptr_t;
  typedef __attribute__((address_space(3))) void* lptr_t;
  constexpr int PIECES = D / 8, P = kStep * D / 2048;  // of a row; requests of a wavefront for a step's keys
  constexpr int kTile = kStep * D;
  __shared__ __attribute__((aligned(16))) T tiles[4 * kTile];  // keys, values, keys, values
  const int group = a.heads / a.kv_heads;
  const int g = blockIdx.x % a.kv_heads, h = g * group + blockIdx.x / a.kv_heads % group;
  Tile t;
  if (!find_tile(a, blockIdx.x / a.heads, t)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, kh = lane >> 5;
  const int nq = t.q_end - t.q_begin, nk = max(t.k_end - t.k_begin, 0);
  const auto seen_by = [&](int i) { return a.causal ? min(max(i + 1 + nk - nq, 0), nk) : nk; };
  const int qi = t.first + wave * 32 + n, qc = min(qi, nq - 1);
  const int seen = seen_by(qc);
  const int least = seen_by(min(t.first + wave * 32, nq - 1)), most = seen_by(min(t.first + wave * 32 + 31, nq - 1));
  const int end = seen_by(min(t.first + kQueries - 1, nq - 1));
  const T* const kg = (const T*)a.k + (int64_t)t.k_begin * a.ldk + (int64_t)g * D;
  const T* const vg = (const T*)a.v + (int64_t)t.k_begin * a.ldv + (int64_t)g * D;

  // rotations of a row's pieces (the same for the rows that one lane requests, 1024 / PIECES apart)
  const auto key_turn = [](int row) { return D == 64 ? (row >> 1) & 7 : D == 128 ? row & 15 : row & 7; };
  const auto value_turn = [](int row) { return D == 64 ? ((row >> 1) & 3) << 1 : (row & 7) << 1; };
  constexpr int kApart = 256 / PIECES;
  const int row = tid / PIECES, key_part = ((tid % PIECES) ^ key_turn(row)) * 16, value_part = ((tid % PIECES) ^ value_turn(row)) * 16;
  const int64_t key_row = a.ldk * 2, value_row = a.ldv * 2;  // bytes
  const uint32_t key_at = (uint32_t)row * (uint32_t)key_row + key_part, value_at = (uint32_t)row * (uint32_t)value_row + value_part;
  const auto request = [&](int k0, const T* from, int64_t row_bytes, uint32_t at, int part, T* tile) __attribute__((always_inline)) {
    const uint8_t* p = (const uint8_t*)from + k0 * row_bytes;
    T* const to = tile + wave * 512;
    if (k0 + kStep <= end) {
#pragma unroll
      for (int i = 0; i < P; ++i, p += kApart * row_bytes) __builtin_amdgcn_global_load_lds((gptr_t)(p + at), (lptr_t)(to + i * 2048), 16, 0, 0);
    } else {  // rows behind the last are masked, and are that one again
#pragma unroll 1
      for (int i = 0; i < P; ++i) {
        const uint32_t r = min(row + kApart * i, end - 1 - k0);
        __builtin_amdgcn_global_load_lds((gptr_t)(p + (r * (uint32_t)row_bytes + part)), (lptr_t)(to + i * 2048), 16, 0, 0);
      }
    }
  };
  const auto request_keys = [&](int k0, T* tile) __attribute__((always_inline)) { request(k0, kg, key_row, key_at, key_part, tile); };
  const auto request_values = [&](int k0, T* tile) __attribute__((always_inline)) { request(k0, vg, value_row, value_at, value_part, tile); };
  if (end > 0) {
    request_keys(0, tiles);
    request_values(0, tiles + kTile);
    if (end > kStep) request_keys(kStep, tiles + 2 * kTile);
  }
  eight_t qop[D / 16];
  {
    const T* const q = (const T*)a.q + (int64_t)(t.q_begin + qc) * a.ldq + (int64_t)h * D;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      qop[s] = *reinterpret_cast<const eight_t*>(q + 16 * s + 8 * kh);
      if (a.scale < 0.0f) {  // (the largest score is that of the largest product then)
        u32x4_t x = __builtin_bit_cast(u32x4_t, qop[s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] ^= 0x80008000u;
        qop[s] = __builtin_bit_cast(eight_t, x);
      }
    }
  }
  f32x16_t o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;  // (of this lane's keys alone)
  const float mul = fmaxf(fabsf(a.scale) * 1.44269504088896340736f, 0x1p-126f);  // (0 times -infinity would be NaN)

  // the scores of a step's keys; s[half][i]: key 32 half + 8 (i / 4) + 4 kh + i % 4
  const auto score = [&](const T* ks, f32x16_t (&s)[kStep / 32]) __attribute__((always_inline)) {
    int at = lane;
    if constexpr (D == 256) asm volatile("" : "+v"(at));  // addresses in LDS are formed anew each step: there are too many to keep
    const int n = at & 31, kh = at >> 5;
#pragma unroll
    for (int half = 0; half < kStep / 32; ++half)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[half][i] = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      if (D == 256 && d % 4 == 0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int half = 0; half < kStep / 32; ++half) {
        const int row = 32 * half + n;
        s[half] = product(*reinterpret_cast<const eight_t*>(ks + row * D + ((2 * d + kh) ^ key_turn(row)) * 8), qop[d], s[half]);
      }
    }
  };
  f32x16_t s[kStep / 32];
  // the step at k0, whose scores are there; `ks`: the next one's keys
  const auto step = [&](int k0, const T* ks, const T* vs) __attribute__((always_inline)) {
    int at = lane;
    if constexpr (D == 256) asm volatile("" : "+v"(at));
    const int L16 = at & 15, kh = at >> 5;
    // keys 16 j + 4 kh + L16 / 4 and 8 further, components 32 d + 16 ((lane / 16) % 2) + 4 (L16 % 4) .. + 3
    const auto values = [&](int j, int d) __attribute__((always_inline)) {
      const int row = 16 * j + 4 * kh + (L16 >> 2), piece = 4 * d + 2 * ((at >> 4) & 1) + ((L16 >> 1) & 1);
      const T* const lp = vs + row * D + (piece ^ value_turn(row)) * 8 + (L16 & 1) * 4;
      const T* const up = vs + (row + 8) * D + (piece ^ value_turn(row + 8)) * 8 + (L16 & 1) * 4;
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4_t __attribute__((address_space(3)))*)lp);
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4_t __attribute__((address_space(3)))*)up);
      const four_t l4 = __builtin_bit_cast(four_t, lo), u4 = __builtin_bit_cast(four_t, hi);
      return eight_t{l4[0], l4[1], l4[2], l4[3], u4[0], u4[1], u4[2], u4[3]};
    };
    if (k0 + kStep > least) {
      const int sees = seen - k0 - 4 * kh;
#pragma unroll
      for (int half = 0; half < kStep / 32; ++half)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[half][i] = 32 * half + 8 * (i >> 2) + (i & 3) < sees ? s[half][i] : -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int half = 0; half < kStep / 32; ++half)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[half][i]);
    const HalfPair best = half_pair(mx);
    mx = fmaxf(best.low, best.high);
    // (the scale goes into the exponent's multiply-add, whose product is exact where the maximum's is rounded: far from zero it is put on ahead)
    float scale = mul;
    if (__builtin_amdgcn_ballot_w64(fabsf(mx) * mul > 65536.0f && mx > -INFINITY)) {
      scale = 1.0f;
      mx *= mul;
#pragma unroll
      for (int half = 0; half < kStep / 32; ++half)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[half][i] *= mul;
    }
    move_maximum<true>(mx > -INFINITY ? mx * scale : -INFINITY, m_run, l_run, o);
    const float from = m_run == -INFINITY ? 0.0f : m_run;  // (no key seen yet: all weights are 0)
    eight_t pop[kStep / 16];
    const auto weights = [&](int first, int many) __attribute__((always_inline)) {  // of the lane's kStep / 2 scores
#pragma unroll
      for (int x = first; x < first + many; ++x) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x / 16][x % 16], scale, -from));
        l_run += p;
        pop[x / 8][x % 8] = (T)p;
      }
    };
    constexpr int HALVES = kStep / 32, ROUNDS = D / 16, EACH = kStep / 2 / ROUNDS;
    static_assert(ROUNDS * EACH == kStep / 2, "all weights");
    constexpr int PRODUCTS = kStep / 16 * (D / 32), AHEAD = 2;
    eight_t v[PRODUCTS];
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) v[x] = values(x / (D / 32), x % (D / 32));
    if (k0 + kStep < most) {  // a few weights behind each of the next scores' products, which take as long
      f32x16_t next[kStep / 32];
#pragma unroll
      for (int half = 0; half < kStep / 32; ++half)
#pragma unroll
        for (int i = 0; i < 16; ++i) next[half][i] = 0.0f;
      const auto key = [&](int d, int half) __attribute__((always_inline)) {
        const int row = 32 * half + (at & 31);
        return *reinterpret_cast<const eight_t*>(ks + row * D + ((2 * d + kh) ^ key_turn(row)) * 8);
      };
      eight_t ahead[HALVES];
#pragma unroll
      for (int half = 0; half < HALVES; ++half) ahead[half] = key(0, half);
#pragma unroll
      for (int d = 0; d < ROUNDS; ++d) {
        eight_t now[HALVES];
#pragma unroll
        for (int half = 0; half < HALVES; ++half) now[half] = ahead[half];
        if (d + 1 < ROUNDS)
#pragma unroll
          for (int half = 0; half < HALVES; ++half) ahead[half] = key(d + 1, half);
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          next[half] = product(now[half], qop[d], next[half]);
          weights(d * EACH + half * (EACH / HALVES), EACH / HALVES);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int half = 0; half < HALVES; ++half) s[half] = next[half];
    } else {
      weights(0, kStep / 2);
    }
#pragma unroll
    for (int x = 0; x < PRODUCTS; ++x) {
      if (x + AHEAD < PRODUCTS) v[x + AHEAD] = values((x + AHEAD) / (D / 32), (x + AHEAD) % (D / 32));
      o[x % (D / 32)] = product(v[x], pop[x / (D / 32)], o[x % (D / 32)]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const int unmasked = seen_by(min(t.first, nq - 1));  // keys that all queries of the workgroup see
  // A barrier does not wait for requests into LDS: every wavefront waits for its own ahead of it, also one without products in a step.
  const auto all_there = []() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  all_there();
  if (end > 0) score(tiles, s);
  T *here = tiles, *other = tiles + 2 * kTile;  // this step's keys and values, the next one's
  for (int k0 = 0; k0 < end; k0 += kStep) {
    all_there();  // the next keys and these values, and the last ones' readers are done
    bool strange = false;
    if (k0 + kStep > unmasked) {
      u32x4_t* const vs = reinterpret_cast<u32x4_t*>(here + kTile) + tid;
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < P; ++i) any |= not_finite<T>(vs[256 * i]);
      strange = __syncthreads_or(any & 0x80008000u) != 0;
      if (strange) {
#pragma unroll
        for (int i = 0; i < P; ++i) vs[256 * i] = only_finite<T>(vs[256 * i]);
        __syncthreads();
      }
    }
    if (k0 + 2 * kStep < end) request_keys(k0 + 2 * kStep, here);
    if (k0 + kStep < end) request_values(k0 + kStep, other + kTile);
    if (k0 < most) step(k0, other, here + kTile);
    if (strange) {
#pragma unroll 1
      for (int key = k0; key < min(k0 + kStep, most); ++key) {
        const T* const v = vg + (int64_t)key * a.ldv + 4 * kh;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float x = (float)v[32 * d + 8 * (c >> 2) + (c & 3)];
            o[d][c] += key < seen && !(fabsf(x) < INFINITY) ? x : 0.0f;
          }
        }
      }
    }
    T* const last = here;
    here = other;
    other = last;
  }
  if (qi >= nq) return;
  const HalfPair sums = half_pair(l_run);
  const float l = sums.low + sums.high, inv = l != 0.0f ? 1.0f / l : 0.0f;
  T* const out = (T*)a.ctx + (int64_t)(t.q_begin + qi) * a.ldc + (int64_t)h * D;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      four_t v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = held(o[d][4 * u + j] * inv, T());  // (rounded weights may lead a little beyond the largest value)
      *reinterpret_cast<four_t*>(out + 32 * d + 8 * u + 4 * kh) = v;
    }
}

template <typename T>
int launch(const awq_packed_attention_args& a, hipStream_t st) {
  const int64_t tiles = a.n_tokens / kQueries + std::min<int64_t>(a.n_requests, a.n_tokens);
  AWQ_REQUIRE(launchable(tiles * a.heads, 256), "too many queries and heads");
  const dim3 grid((unsigned)(tiles * a.heads));
  if (a.dim == 64) hipLaunchKernelGGL((packed_kernel<T, 64, 64, 2>), grid, dim3(256), 0, st, a);
  else if (a.dim == 128) hipLaunchKernelGGL((packed_kernel<T, 128, 64, 2>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((packed_kernel<T, 256, 64, 1>), grid, dim3(256), 0, st, a);
  AWQ_HIP_TRY(hipGetLastError());
  return AWQ_OK;
}

}  // namespace

int launch_packed_attention(const awq_packed_attention_args& a, bool bf16, hipStream_t st) {
  if (a.n_tokens == 0 || a.n_requests == 0) return AWQ_OK;
  return bf16 ? launch<bf16_t>(a, st) : launch<half_t>(a, st);
}
