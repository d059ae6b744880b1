// Stable grouping of rows by id (expert, adapter): a counting sort whose bucket
// `groups` takes the ids outside [begin, begin + groups), so that order is a
// permutation with the rows in no group last.
#include <cuda_runtime.h>

#include "awqb200.h"
#include "awqb_common.h"

namespace awqb {
namespace {

constexpr int kMaxGroups = 1024;
constexpr int kChunk = 1024;  // ids per CTA of the multi-CTA sort
// Ids from which the multi-CTA sort is taken: one CTA's shared-memory atomics and
// match instructions are bound by its one SM. Measured, one / many CTAs in us for
// 128 groups: 4096 ids 7.9 / 13.3, 8192 12.8 / 14.3, 16384 22.2 / 15.0.
constexpr int64_t kMultiMin = 10240;

__device__ __forceinline__ int bucket_of(int id, int begin, int groups) {
  const int64_t g = (int64_t)id - begin;
  return g >= 0 && g < groups ? (int)g : groups;
}

// Exclusive prefix sum over the 1024 threads of the CTA; *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int* warp_tot, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) warp_tot[warp] = incl;
  __syncthreads();
  int t = warp_tot[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) t += u;
  }
  *total = __shfl_sync(0xffffffffu, t, 31);
  const int before = __shfl_sync(0xffffffffu, t, warp == 0 ? 0 : warp - 1);
  __syncthreads();
  return incl - v + (warp == 0 ? 0 : before);
}

// Writes the ids of [s0, s1) to their places in index order (one warp);
// pos[bucket] is the bucket's next place.
__device__ __forceinline__ void emit_slice(const int32_t* __restrict__ ids, int s0, int s1, int begin, int groups,
                                           int32_t* pos, int32_t* __restrict__ order) {
  const int lane = threadIdx.x & 31;
  const unsigned lt = (1u << lane) - 1u;
  for (int base = s0; base < s1; base += 32) {
    const int i = base + lane;
    const int b = i < s1 ? bucket_of(ids[i], begin, groups) : -1;
    const unsigned grp = __match_any_sync(0xffffffffu, b);
    if (b >= 0) order[pos[b] + __popc(grp & lt)] = i;
    __syncwarp();
    if (b >= 0 && (grp & lt) == 0) pos[b] += __popc(grp);
    __syncwarp();
  }
}

// One CTA: warp w counts, then emits, the contiguous slice w of the ids.
__global__ void __launch_bounds__(1024) group_small_kernel(const int32_t* __restrict__ ids, int n, int begin,
                                                           int groups, int32_t* __restrict__ order,
                                                           int32_t* __restrict__ offsets) {
  extern __shared__ int32_t cnt[];  // [32][groups + 1]
  __shared__ int warp_tot[32];
  const int B = groups + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = (n + 31) / 32;
  const int s0 = min(n, warp * slice), s1 = min(n, s0 + slice);
  for (int i = threadIdx.x; i < 32 * B; i += 1024) cnt[i] = 0;
  __syncthreads();
  for (int i = s0 + lane; i < s1; i += 32) atomicAdd(&cnt[warp * B + bucket_of(ids[i], begin, groups)], 1);
  __syncthreads();
  const int e = threadIdx.x;
  int tot = 0, total;
  if (e < groups)
    for (int w = 0; w < 32; ++w) tot += cnt[w * B + e];
  const int at = block_scan(tot, warp_tot, &total);
  if (e < groups) {
    offsets[e] = at;
    int run = at;
    for (int w = 0; w < 32; ++w) {
      const int c = cnt[w * B + e];
      cnt[w * B + e] = run;
      run += c;
    }
  }
  if (e == 1023) {  // the rows in no group
    offsets[groups] = total;
    int run = total;
    for (int w = 0; w < 32; ++w) {
      const int c = cnt[w * B + groups];
      cnt[w * B + groups] = run;
      run += c;
    }
  }
  __syncthreads();
  emit_slice(ids, s0, s1, begin, groups, cnt + warp * B, order);
}

__global__ void __launch_bounds__(256) group_hist_kernel(const int32_t* __restrict__ ids, int n, int begin, int groups,
                                                         int32_t* __restrict__ hist) {
  extern __shared__ int32_t h[];
  const int B = groups + 1;
  for (int b = threadIdx.x; b < B; b += 256) h[b] = 0;
  __syncthreads();
  const int i0 = blockIdx.x * kChunk;
  for (int i = i0 + threadIdx.x; i < min(n, i0 + kChunk); i += 256) atomicAdd(&h[bucket_of(ids[i], begin, groups)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < B; b += 256) hist[(int64_t)blockIdx.x * B + b] = h[b];
}

// One CTA of 1024: the chunks' counts become each chunk's first places.
__global__ void __launch_bounds__(1024) group_scan_kernel(int32_t* __restrict__ hist, int chunks, int groups,
                                                          int32_t* __restrict__ offsets) {
  __shared__ int warp_tot[32];
  const int B = groups + 1, e = threadIdx.x;
  int tot = 0, total;
  if (e < groups)
    for (int c = 0; c < chunks; ++c) tot += hist[(int64_t)c * B + e];
  const int at = block_scan(tot, warp_tot, &total);
  if (e < groups) offsets[e] = at;
  if (e == 1023) offsets[groups] = total;
  for (int b = e; b < B; b += 1024) {
    int run = b == groups ? total : at;
    for (int c = 0; c < chunks; ++c) {
      const int v = hist[(int64_t)c * B + b];
      hist[(int64_t)c * B + b] = run;
      run += v;
    }
  }
}

__global__ void __launch_bounds__(32) group_emit_kernel(const int32_t* __restrict__ ids, int n, int begin, int groups,
                                                        const int32_t* __restrict__ hist,
                                                        int32_t* __restrict__ order) {
  extern __shared__ int32_t pos[];
  const int B = groups + 1;
  for (int b = threadIdx.x; b < B; b += 32) pos[b] = hist[(int64_t)blockIdx.x * B + b];
  __syncwarp();
  const int s0 = blockIdx.x * kChunk;
  emit_slice(ids, s0, min(n, s0 + kChunk), begin, groups, pos, order);
}

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int64_t awqb_group_rows_workspace_bytes(int64_t n, int64_t groups) {
  return n < kMultiMin ? 0 : (n + kChunk - 1) / kChunk * (groups + 1) * 4;
}

extern "C" int awqb_group_rows(const int32_t* ids, int64_t n, int64_t begin, int64_t groups, int32_t* order,
                               int32_t* offsets, void* workspace, int64_t workspace_bytes, void* stream) {
  AWQB_REQUIRE(groups >= 1 && groups <= kMaxGroups, kInvalidArgument, "groups=%lld must be 1..%d", (long long)groups,
               kMaxGroups);
  AWQB_REQUIRE(n >= 0 && n < (1ll << 30), kInvalidArgument, "bad number of ids %lld", (long long)n);
  AWQB_REQUIRE(begin >= -(1ll << 31) && begin < (1ll << 31), kInvalidArgument, "bad first id %lld", (long long)begin);
  AWQB_REQUIRE(offsets != nullptr && (n == 0 || (ids != nullptr && order != nullptr)), kInvalidArgument,
               "null pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int B = (int)groups + 1;
  if (n < kMultiMin) {
    const int smem = 32 * B * 4;
    // (the most that any call wants: another thread's call may set it before this launch)
    if (smem > 48 * 1024 - 256)
      AWQB_CUDA(cudaFuncSetAttribute(group_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     32 * (kMaxGroups + 1) * 4));
    group_small_kernel<<<1, 1024, smem, st>>>(ids, (int)n, (int)begin, (int)groups, order, offsets);
    AWQB_LAUNCH_CHECK();
    return kOk;
  }
  const int64_t need = awqb_group_rows_workspace_bytes(n, groups);
  AWQB_REQUIRE(workspace != nullptr && workspace_bytes >= need, kInvalidArgument, "workspace too small: %lld < %lld bytes",
               (long long)workspace_bytes, (long long)need);
  const int chunks = (int)((n + kChunk - 1) / kChunk);
  int32_t* hist = static_cast<int32_t*>(workspace);
  group_hist_kernel<<<chunks, 256, B * 4, st>>>(ids, (int)n, (int)begin, (int)groups, hist);
  group_scan_kernel<<<1, 1024, 0, st>>>(hist, chunks, (int)groups, offsets);
  group_emit_kernel<<<chunks, 32, B * 4, st>>>(ids, (int)n, (int)begin, (int)groups, hist, order);
  AWQB_LAUNCH_CHECK();
  return kOk;
}
