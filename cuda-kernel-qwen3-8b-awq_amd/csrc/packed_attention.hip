// Attention of prompts of different lengths, one behind the other (batch.hpp).
#include "batch.hpp"
#include "tile_halves.hpp"

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
// any of eight 16-bit numbers infinite or NaN
template <typename T>
__device__ __forceinline__ bool not_finite(u32x4_t v) {
  constexpr uint32_t e = __is_same(T, half_t) ? 0x7c00u : 0x7f80u;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= (v[i] & e) == e || (v[i] >> 16 & e) == e;
  return any;
}

constexpr int kQueries = 128, kKeys = 32;

// The tile of queries a workgroup takes: request r has ceil(queries / 128) of them, tiles are numbered one request behind the other. Every
// wavefront looks its own up, 64 requests at a time.  False: there are fewer tiles.
struct Tile {
  int q_begin, q_end, k_begin, k_end, first;  // first: of the tile's queries, from q_begin on
};
__device__ __forceinline__ int clamped(int64_t x, int64_t n) { return (int)(x < 0 ? 0 : x > n ? n : x); }
__device__ __forceinline__ bool find_tile(const awq_packed_attention_args& a, int tile, Tile& out) {
  const int lane = threadIdx.x & 63;
  for (int r0 = 0; r0 < a.n_requests; r0 += 64) {
    const int r = r0 + lane;
    int b = 0, e = 0;
    if (r < a.n_requests) b = clamped(a.q_starts[r], a.n_tokens), e = clamped(a.q_starts[r + 1], a.n_tokens);
    const int tiles = e > b ? (e - b + kQueries - 1) / kQueries : 0;
    int sum = tiles;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(sum, off, 64);
      if (lane >= off) sum += v;
    }
    const int all = __builtin_amdgcn_readlane(sum, 63);
    if (tile < all) {
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > tile));
      const int behind = __builtin_amdgcn_readlane(sum, at) - 1 - tile;  // tiles of the request behind this one
      out.q_begin = __builtin_amdgcn_readlane(b, at);
      out.q_end = __builtin_amdgcn_readlane(e, at);
      // the last tile first: it has the most keys
      out.first = behind * kQueries;
      const int* const starts = a.k_starts ? a.k_starts : a.q_starts;
      out.k_begin = clamped(starts[r0 + at], a.n_keys);
      out.k_end = clamped(starts[r0 + at + 1], a.n_keys);
      return true;
    }
    tile -= all;
  }
  return false;
}

// 128 queries of one head a workgroup, 32 a wavefront; 64 keys and values at a time go through LDS.  Queries are columns throughout, lane
// (n, kh) = (lane % 32, lane / 32):
//     S^T[key][query] = K Q^T,   O^T[c][query] += V^T P^T      v_mfma_f32_32x32x16
// so that a query's maximum, sum and rescaling stay in a lane and its partner, and the weights a lane forms are the elements it
// supplies to the second product (slice j: keys 16 j + 8 (e / 4) + 4 kh + e % 4; V^T by the transposing LDS read).  Scores, maxima and sums
// are binary32; a weight is rounded to the activations' type for the second product, the sum of the weights is that of the rounded ones.
// Values that are not finite where some query of the tile does not see them are kept out of the product, in which 0 times them is NaN.
template <typename T, int D>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void packed_kernel(awq_packed_attention_args a) {
  typedef typename Vec<T>::eight eight_t;
  typedef typename Vec<T>::four four_t;
  constexpr int KS = D + 8, VS = D + 16, P = D / 32;  // strides in LDS; 16-byte pieces of 64 keys a thread
  __shared__ __attribute__((aligned(16))) T tiles[2 * kKeys * (KS + VS)];
  T *const ks = tiles, *const vs = tiles + 2 * kKeys * KS;
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
  const T* const q = (const T*)a.q + (int64_t)(t.q_begin + qc) * a.ldq + (int64_t)h * D;
  const T* const kg = (const T*)a.k + (int64_t)t.k_begin * a.ldk + (int64_t)g * D;
  const T* const vg = (const T*)a.v + (int64_t)t.k_begin * a.ldv + (int64_t)g * D;
  eight_t qop[D / 16];
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qop[s] = *reinterpret_cast<const eight_t*>(q + 16 * s + 8 * kh);
  f32x16_t o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;
  const float mul = a.scale * 1.44269504088896340736f;

  u32x4_t kr[P], vr[P];
  const auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int pc = tid + i * 256, key = k0 + pc / (D / 8), at = (pc % (D / 8)) * 8;
      kr[i] = vr[i] = u32x4_t{0, 0, 0, 0};
      if (key < end) {
        kr[i] = *reinterpret_cast<const u32x4_t*>(kg + (int64_t)key * a.ldk + at);
        vr[i] = *reinterpret_cast<const u32x4_t*>(vg + (int64_t)key * a.ldv + at);
      }
    }
  };
  const auto step = [&](int k0, int half, bool strange) __attribute__((always_inline)) {
    if (k0 >= most) return;
    const T* const klane = ks + (half * kKeys + n) * KS + 8 * kh;
    const int L16 = lane & 15;
    const T* const vlane = vs + (half * kKeys + 4 * kh + (L16 >> 2)) * VS + 16 * ((lane >> 4) & 1) + 4 * (L16 & 3);
    const auto values = [&](int j, int d) __attribute__((always_inline)) {
      const T* const vp = vlane + 16 * j * VS + d * 32;
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4_t __attribute__((address_space(3)))*)vp);
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4_t __attribute__((address_space(3)))*)(vp + 8 * VS));
      const four_t l4 = __builtin_bit_cast(four_t, lo), u4 = __builtin_bit_cast(four_t, hi);
      return eight_t{l4[0], l4[1], l4[2], l4[3], u4[0], u4[1], u4[2], u4[3]};
    };
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) s = product(*reinterpret_cast<const eight_t*>(klane + 16 * d), qop[d], s);
    // s[i]: key k0 + 8 (i / 4) + 4 kh + i % 4
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] *= mul;
    if (k0 + kKeys > least) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = k0 + 8 * (i >> 2) + 4 * kh + (i & 3) < seen ? s[i] : -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    const HalfPair best = half_pair(mx);
    move_maximum<false>(fmaxf(best.low, best.high), m_run, l_run, o);
    const float from = m_run == -INFINITY ? 0.0f : m_run;  // (no key seen yet: all weights are 0)
    float rs = 0.0f;
    eight_t pop[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const T p = (T)__builtin_amdgcn_exp2f(s[i] - from);
      rs += (float)p;
      pop[i >> 3][i & 7] = p;
    }
    const HalfPair sums = half_pair(rs);
    l_run += sums.low + sums.high;
    if (!strange) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int d = 0; d < D / 32; ++d) o[d] = product(values(j, d), pop[j], o[d]);
    } else {  // key by key, from memory
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const HalfPair p = half_pair((float)pop[i >> 3][i & 7]);
#pragma unroll
        for (int both = 0; both < 2; ++both) {
          const int key = k0 + 8 * (i >> 2) + 4 * both + (i & 3);
          if (key >= seen) continue;
          const T* const v = vg + (int64_t)key * a.ldv + 4 * kh;
          const float w = both ? p.high : p.low;
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int c = 0; c < 16; ++c) o[d][c] = __builtin_fmaf(w, (float)v[32 * d + 8 * (c >> 2) + (c & 3)], o[d][c]);
        }
      }
    }
  };
  const int unmasked = seen_by(min(t.first, nq - 1));  // keys that all queries of the tile see
  load(0);
  for (int k0 = 0; k0 < end; k0 += 2 * kKeys) {
    __syncthreads();  // the last tile's readers are done
    bool strange = false;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int pc = tid + i * 256, key = pc / (D / 8), at = (pc % (D / 8)) * 8;
      *reinterpret_cast<u32x4_t*>(ks + key * KS + at) = kr[i];
      *reinterpret_cast<u32x4_t*>(vs + key * VS + at) = vr[i];
      if (k0 + 2 * kKeys > unmasked) strange |= not_finite<T>(vr[i]);
    }
    strange = __syncthreads_or(strange) != 0;
    load(k0 + 2 * kKeys);
    step(k0, 0, strange);
    step(k0 + kKeys, 1, strange);
  }
  if (qi >= nq) return;
  const float inv = l_run != 0.0f ? 1.0f / l_run : 0.0f;
  T* const out = (T*)a.ctx + (int64_t)(t.q_begin + qi) * a.ldc + (int64_t)h * D;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      four_t v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (T)(o[d][4 * u + j] * inv);
      *reinterpret_cast<four_t*>(out + 32 * d + 8 * u + 4 * kh) = v;
    }
}

template <typename T>
int launch(const awq_packed_attention_args& a, hipStream_t st) {
  const int64_t tiles = a.n_tokens / kQueries + std::min<int64_t>(a.n_requests, a.n_tokens);
  AWQ_REQUIRE(tiles * a.heads < (1ll << 31), "too many queries and heads");
  const dim3 grid((unsigned)(tiles * a.heads));
  if (a.dim == 64) hipLaunchKernelGGL((packed_kernel<T, 64>), grid, dim3(256), 0, st, a);
  else if (a.dim == 128) hipLaunchKernelGGL((packed_kernel<T, 128>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((packed_kernel<T, 256>), grid, dim3(256), 0, st, a);
  AWQ_HIP_TRY(hipGetLastError());
  return AWQ_OK;
}

}  // namespace

int launch_packed_attention(const awq_packed_attention_args& a, bool bf16, hipStream_t st) {
  if (a.n_tokens == 0 || a.n_requests == 0) return AWQ_OK;
  return bf16 ? launch<bf16_t>(a, st) : launch<half_t>(a, st);
}
