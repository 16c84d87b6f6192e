// Pages and slots of a step's new positions from the requests' lengths (batch.hpp): integers, bound by their launches.
#include "batch.hpp"

namespace {

constexpr int kPlanThreads = 1024, kPlanTokens = 4096, kSlotThreads = 256, kSlotStarts = 4096;

struct Three {
  int a, b, c;
};

// sums of the lanes ahead of this one over the workgroup; `all`: over all lanes.  part [16][3]
__device__ __forceinline__ Three sums_ahead(Three v, int* part, Three& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Three s = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int a = __shfl_up(s.a, off, 64), b = __shfl_up(s.b, off, 64), c = __shfl_up(s.c, off, 64);
    if (lane >= off) s.a += a, s.b += b, s.c += c;
  }
  __syncthreads();  // the last call's readers of `part` are done
  if (lane == 63) part[3 * wave] = s.a, part[3 * wave + 1] = s.b, part[3 * wave + 2] = s.c;
  __syncthreads();
  Three ahead{s.a - v.a, s.b - v.b, s.c - v.c};
  all = Three{0, 0, 0};
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    const Three p{part[3 * w], part[3 * w + 1], part[3 * w + 2]};
    if (w < wave) ahead.a += p.a, ahead.b += p.b, ahead.c += p.c;
    all.a += p.a, all.b += p.b, all.c += p.c;
  }
  return ahead;
}

// the last of n ascending values that is not above x (the first is not)
template <typename P>
__device__ __forceinline__ int last_not_above(P v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void write_slot(const awq_page_plan_args& a, int64_t t, int request, int starts, int cached, int length) {
  const int p = cached + (int)t - starts;
  int slot = -1;
  if (p < length) {
    const int page = held_page(a.table[(int64_t)request * a.max_pages + p / kPage], a.n_pages);
    if (page >= 0) slot = page * kPage + p % kPage;
  }
  a.positions[t] = p;
  a.slots[t] = slot;
}

// One workgroup, 1,024 requests at a time: pages given back, then pages taken, each by a thread a page that looks its request up
// among the sums in LDS.  SLOTS: the new positions' slots too, where one workgroup has all requests in LDS and few
// positions a thread; slots_kernel otherwise.
// Bound by its trips to memory and barriers one behind the other, not by bytes: 200 answers, five of them ended, 9.8 us (traced).
template <bool SLOTS>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(awq_page_plan_args a) {
  __shared__ int part[48], sums[kPlanThreads], held_of[kPlanThreads], length_of[kPlanThreads], cached_of[kPlanThreads];
  const int tid = threadIdx.x, n = a.n_requests, capacity = a.max_pages * kPage;
  int available = min(max(*a.free_in, 0), a.n_pages);
  const auto cached_at = [&](int i) { return min(max(a.cached[i], 0), capacity); };
  const auto pages = [](int positions) { return (positions + kPage - 1) / kPage; };
  // (one tile of requests is read once)
  int cached = 0, fresh = 0;
  if (tid < n) cached = cached_at(tid), fresh = min(a.fresh[tid], capacity + 1);  // (more than capacity never fits)
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    if (i0) {
      cached = fresh = 0;
      if (i < n) cached = cached_at(i), fresh = a.fresh[i];
    }
    if (__syncthreads_or(i < n && fresh < 0 && cached > 0) == 0) continue;
    Three all;
    const int back = fresh < 0 ? pages(cached) : 0;
    const Three at = sums_ahead(Three{back, 0, 0}, part, all);
    sums[tid] = at.a;
    __syncthreads();
    for (int t0 = 0; t0 < all.a; t0 += kPlanThreads) {
      const int t = t0 + tid;
      int page = -1, to = available + tid, many = min(all.a - t0, kPlanThreads);
      if (t < all.a) {
        const int r = last_not_above(sums, kPlanThreads, t);  // (of requests that begin at one sum the last is the one with pages)
        page = held_page(a.table[(int64_t)(i0 + r) * a.max_pages + t - sums[r]], a.n_pages);
      }
      if (__syncthreads_or(t < all.a && page < 0)) {  // an entry that is no page is passed over
        Three pages_of_these;
        to = available + sums_ahead(Three{page >= 0 ? 1 : 0, 0, 0}, part, pages_of_these).a;
        many = pages_of_these.a;
      }
      if (page >= 0 && to < a.n_pages) a.free_pages[to] = page;
      available = min(available + many, a.n_pages);
    }
    __syncthreads();
  }
  int taken = 0, left = 0;
  Three base{0, 0, 0};  // pages needed, new positions, positions held by the requests ahead of this tile
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    if (n > kPlanThreads) {
      cached = fresh = 0;
      if (i < n) cached = cached_at(i), fresh = min(a.fresh[i], capacity + 1);
    }
    const bool fits = fresh <= capacity - cached;
    const int held = pages(cached), need = fresh > 0 && fits ? pages(cached + fresh) - held : 0, put = max(fresh, 0);
    Three all;
    const Three at = sums_ahead(Three{need, put, 0}, part, all);
    const bool served = i < n && fits && (need == 0 || base.a + at.a + need <= available);
    const int length = fresh < 0 ? 0 : served ? cached + fresh : cached;
    Three mine;
    const Three ahead = sums_ahead(Three{i < n ? length : 0, served && need ? need : 0, i < n && !served ? 1 : 0}, part, mine);
    if (i < n) {
      a.lengths[i] = length;
      a.starts[i] = base.b + at.b;
      if (a.key_starts) a.key_starts[i] = base.c + ahead.a;
      // (for slots_kernel: `lengths` may be `cached`)
      if (!SLOTS && put && base.b + at.b < a.max_tokens) a.positions[base.b + at.b] = cached;
    }
    sums[tid] = at.a;
    held_of[tid] = held;
    __syncthreads();
    // those served are the first of the tile that need pages, so that their pages lie side by side
    for (int t = tid; t < mine.b; t += kPlanThreads) {
      const int r = last_not_above(sums, kPlanThreads, t);
      a.table[(int64_t)(i0 + r) * a.max_pages + held_of[r] + t - sums[r]] = a.free_pages[available - 1 - (base.a + t)];
    }
    taken += mine.b;
    left += mine.c;
    base.a += all.a;
    base.b += all.b;
    base.c += mine.a;
    if constexpr (SLOTS) {
      __syncthreads();
      sums[tid] = base.b - all.b + at.b;
      length_of[tid] = length;
      cached_of[tid] = cached;
    }
  }
  if (tid == 0) {
    a.starts[n] = base.b;
    if (a.key_starts) a.key_starts[n] = base.c;
    *a.free_out = available - taken;
    if (a.left_out) *a.left_out = left;
  }
  if constexpr (SLOTS) {
    __syncthreads();  // the table's new entries are written
    for (int64_t t = tid; t < a.max_tokens; t += kPlanThreads) {
      if (t < base.b) {
        const int r = last_not_above(sums, n, (int)t);
        write_slot(a, t, r, sums[r], cached_of[r], length_of[r]);
      } else {
        a.positions[t] = 0;
        a.slots[t] = -1;
      }
    }
  }
}

// The first position of a request's new ones is there already, and is written again as it is.
__global__ __launch_bounds__(kSlotThreads) void slots_kernel(awq_page_plan_args a) {
  __shared__ int starts[kSlotStarts];
  const int n = a.n_requests;
  const bool here = n <= kSlotStarts;
  if (here)
    for (int i = threadIdx.x; i < n; i += kSlotThreads) starts[i] = a.starts[i];
  const int all = a.starts[n];
  __syncthreads();
  const int64_t t = (int64_t)blockIdx.x * kSlotThreads + threadIdx.x;
  if (t >= a.max_tokens) return;
  if (t >= all) {
    a.positions[t] = 0;
    a.slots[t] = -1;
    return;
  }
  const int r = here ? last_not_above(starts, n, (int)t) : last_not_above(a.starts, n, (int)t), start = here ? starts[r] : a.starts[r];
  write_slot(a, t, r, start, a.positions[start], a.lengths[r]);
}

}  // namespace

// One launch or two (traced, none ended): 200 requests with a position each 7.6 us in one, 6.6 + 2.5 in two; next to the border 1,000 requests with 4,000
// positions 10.9 and 8.0 + 4.1, 240 with 4,080 10.2 and 6.8 + 4.2; behind it 240 with 10,800 17.1 and 8.3 + 3.5.
int launch_page_plan(const awq_page_plan_args& a, hipStream_t st) {
  if (a.n_requests <= kPlanThreads && a.max_tokens <= kPlanTokens) {
    hipLaunchKernelGGL(plan_kernel<true>, dim3(1), dim3(kPlanThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL(plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, st, a);
    AWQ_HIP_TRY(hipGetLastError());
    if (a.max_tokens > 0)
      hipLaunchKernelGGL(slots_kernel, dim3((unsigned)((a.max_tokens + kSlotThreads - 1) / kSlotThreads)), dim3(kSlotThreads), 0, st, a);
  }
  AWQ_HIP_TRY(hipGetLastError());
  return AWQ_OK;
}
