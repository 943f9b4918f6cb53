// One serving step's bookkeeping on the GPU: pages for the requests that grow, the slot and position of every new token, packed
// offsets, lengths afterwards.  Integers only; a host that never learns the lengths can capture the step into a graph.
//
// Request r holds ceil(have / page) pages and needs ceil((have + new) / page).  The missing ones come off the free list in request
// order, so request r's start in the list is a prefix sum; a request whose row of the table or the list has no room is left as it
// was (the prefix sum goes on as if it had been served, so that the pages taken are always the list's first ones).  So is a request
// whose tokens would end behind the packed batch's rows: it, and every one behind it that brings any.  The sums stop at INT32_MAX,
// where they are behind any batch and any list: lengths may be anything.
//
// Latency-bound: a few bytes a token.  One launch: every CTA sums up all requests by itself (two prefix sums of b entries, from L2)
// and then writes its share of the tokens and of the table, a token a thread up to a CTA for every SM, so no CTA waits for another.
// 1024 requests with 33000 tokens: 6.35 us (with four tokens a thread and divisions of 64 bits 12.4), 0.27 of them for refusing what ends
// behind the batch; 8 requests 3.6.
#include <algorithm>

#include "common.cuh"

namespace fa {

constexpr int kPlanThreads = 256;

struct PlanRequest {
  int64_t have, add;
  int had, need;
  bool fits;
};
__device__ __forceinline__ PlanRequest plan_request(const fa_kvcache_plan_params& p, int have, int add) {
  PlanRequest q;
  q.have = have;
  q.add = max(add, 0);
  const int64_t after = q.have + q.add;
  q.fits = have >= 0 && add >= 0 && after <= (int64_t)p.cols * p.page_size;  // (which is within 32 bits)
  auto pages = [&](uint32_t n) { return n == 0 ? 0 : (int)((n - 1) / (uint32_t)p.page_size) + 1; };  // (32 bits: a division of 64 is a call)
  q.had = q.fits ? pages((uint32_t)have) : 0;
  q.need = q.fits ? pages((uint32_t)after) - q.had : 0;
  return q;
}
__device__ __forceinline__ PlanRequest plan_request(const fa_kvcache_plan_params& p, int r) { return plan_request(p, p.have[r], p.add[r]); }

// Sums of numbers that are not negative.
__device__ __forceinline__ int capped_sum(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7fffffffu); }
__device__ __forceinline__ int2 capped_sum(int2 a, int2 b) { return make_int2(capped_sum(a.x, b.x), capped_sum(a.y, b.y)); }

__global__ void __launch_bounds__(kPlanThreads) kvcache_plan_kernel(const __grid_constant__ fa_kvcache_plan_params p, int32_t* status) {
  extern __shared__ int2 s_pre[];  // per request: tokens and pages in front of it; [b]: of all
  __shared__ int2 s_warp[kPlanThreads / 32];
  __shared__ int s_pages;
  grid_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = ceil_div(p.b, kPlanThreads), r0 = min(p.b, tid * per), r1 = min(p.b, r0 + per);
  int2 sum = make_int2(0, 0);
  for (int rb = r0; rb < r1; rb += 4) {
    int have[4], add[4];  // (all on their way before the first is used)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = min(rb + k, r1 - 1);
      have[k] = p.have[r];
      add[k] = p.add[r];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (rb + k >= r1) break;
      const PlanRequest q = plan_request(p, have[k], add[k]);
      s_pre[rb + k] = sum;
      sum = capped_sum(sum, make_int2((int)q.add, q.need));
    }
  }
  int2 incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl.x, o), y = __shfl_up_sync(0xffffffffu, incl.y, o);
    if (lane >= o) incl = capped_sum(incl, make_int2(x, y));
  }
  if (lane == 31) s_warp[warp] = incl;
  if (tid == 0) s_pages = 0;
  __syncthreads();
  int2 base = make_int2(__shfl_up_sync(0xffffffffu, incl.x, 1), __shfl_up_sync(0xffffffffu, incl.y, 1));
  if (lane == 0) base = make_int2(0, 0);
  for (int w = 0; w < warp; ++w) base = capped_sum(base, s_warp[w]);
  for (int r = r0; r < r1; ++r) s_pre[r] = capped_sum(s_pre[r], base);
  if (tid == kPlanThreads - 1) s_pre[p.b] = capped_sum(base, sum);
  __syncthreads();

  int n_free = p.n_free;
  if (p.num_free) n_free = min(max(*p.num_free, 0), p.n_free);
  auto behind = [&](const PlanRequest& q, int r) { return s_pre[r + 1].x > (int)p.total && q.add > 0; };
  // (32 bits without a sign hold a sum of two numbers of 31)
  auto pages_left = [&](const PlanRequest& q, int r) { return q.need == 0 || (uint32_t)s_pre[r].y + (uint32_t)q.need <= (uint32_t)n_free; };
  auto granted = [&](const PlanRequest& q, int r) { return q.fits && pages_left(q, r) && !behind(q, r); };
  // requests: a warp each
  const int warps = gridDim.x * (kPlanThreads / 32), gw = blockIdx.x * (kPlanThreads / 32) + warp;
  for (int r = gw; r < p.b; r += warps) {
    const PlanRequest q = plan_request(p, r);
    const bool ok = granted(q, r);
    if (lane == 0) {
      p.after[r] = (int)(ok ? q.have + q.add : p.have[r]);
      p.cu_new[r] = min(s_pre[r].x, (int)p.total);
      if (q.have < 0 || p.add[r] < 0 || behind(q, r)) raise_bad_index(status);
    }
    if (ok)
      for (int i = lane; i < q.need; i += 32) p.table[(int64_t)r * p.table_stride + q.had + i] = p.free_pages[s_pre[r].y + i];
  }
  if (blockIdx.x == 0) {
    int most = 0;
    for (int r = tid; r < p.b; r += kPlanThreads) {
      const PlanRequest q = plan_request(p, r);
      if (q.need > 0 && granted(q, r)) most = max(most, s_pre[r].y + q.need);
    }
    atomicMax(&s_pages, most);
    __syncthreads();
    if (tid == 0) {
      *p.pages_taken = s_pages;
      p.cu_new[p.b] = min(s_pre[p.b].x, (int)p.total);
    }
  }
  // tokens
  const int last = s_pre[p.b].x;
  for (int64_t t = (int64_t)blockIdx.x * kPlanThreads + tid; t < p.total; t += (int64_t)gridDim.x * kPlanThreads) {
    int64_t slot = -1;
    int pos = 0;
    if (t < last) {
      int lo = 0, hi = p.b, end = last;  // the last request that starts at or in front of t (empty ones start where the next does), and its end
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1, at_mid = s_pre[mid].x;
        if (at_mid <= t) lo = mid;
        else hi = mid, end = at_mid;
      }
      const PlanRequest q = plan_request(p, lo);
      const int64_t at = q.have + (t - s_pre[lo].x);
      pos = (int)at;
      if (end <= (int)p.total && q.fits && pages_left(q, lo) && at >= 0 && at < q.have + q.add) {
        const int col = (int)((uint32_t)at / (uint32_t)p.page_size), in = (int)at - col * p.page_size;
        const int page = col < q.had ? p.table[(int64_t)lo * p.table_stride + col] : p.free_pages[s_pre[lo].y + col - q.had];
        slot = (int64_t)page * p.page_size + in;
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

cudaError_t launch_kvcache_plan(const fa_kvcache_plan_params& p, int num_sm, int32_t* status, cudaStream_t st) {
  int64_t grid = (p.total + kPlanThreads - 1) / kPlanThreads;
  grid = std::max<int64_t>(grid, ceil_div(p.b, kPlanThreads / 32));
  grid = std::min<int64_t>(std::max<int64_t>(grid, 1), num_sm);
  const size_t smem = (size_t)(p.b + 1) * sizeof(int2);
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kvcache_plan_kernel), (FA_B200_PLAN_MAX_REQUESTS + 1) * (int)sizeof(int2));
  if (e != cudaSuccess) return e;
  return launch_dependent(kvcache_plan_kernel, dim3((unsigned)grid), kPlanThreads, smem, st, p, status);
}

}  // namespace fa
