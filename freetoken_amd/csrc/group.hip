// Routes grouped by expert (ftmoe_group_routes): the order of ftmoe_align with block
// size 1, without its padding, expert list and slot lookup, and beside it, for the
// int8 expert layer, the quantisation of the tokens, which needs nothing of it.
//
// A wave takes 64 routes at a time.  The lanes with the same expert are found by one
// ballot per bit of the expert id; a route's rank among them is a population
// count, and their first lane alone keeps the wave's count of that expert: no
// atomics, and the stable order.  Up to 2048 routes one workgroup does all of it in
// one launch; beyond, workgroups of 2048 routes count first, and in a second launch
// each adds up the counts before its own and places its routes.  That reads every
// count in every workgroup, which grows with the square of the routes: past
// kGroupCounts counts a launch between the two turns each expert's counts into
// their running sums.
//
// Bound by latency: 32 routes 3.5 us, 512 (with 64 tokens of 7168 quantised) 4.7 us,
// 32768 4.9 + 6.4 us, 65536 (with 8192 tokens of 2048, 50 MB) 12.6 + 8.7 us.
#include <algorithm>

#include "matmul.h"
#include "quant_int8.h"

namespace ftmoe {

namespace {

constexpr int kGroupWaves = 16;
constexpr int kGroupThreads = kGroupWaves * kWave;
constexpr int kGroupChunks = 2;  // 64-route chunks of a wave
constexpr int kGroupRoutes = kGroupThreads * kGroupChunks;
constexpr int kGroupQuantRows = 1 << 23;  // (four waves each: 2^31 threads, half of what a launch holds)

// Counts of all workgroups that each of them still adds up itself.  us in all, itself / with sums from a launch between:
// 65536 routes 128 experts 9.5 / 10.7, 1023 experts 21.0 / 14.6; 131072 routes 8 experts 7.5 / 9.7, 128 11.1 / 10.9, 1023
// 32.6 / 15.2; 1048576 routes 8 experts 12.1 / 12.8, 128 38.5 / 17.5, 1023 213 / 31.
constexpr int kGroupCounts = 8192;

int group_blocks(int numel) { return numel / kGroupRoutes + (numel % kGroupRoutes ? 1 : 0); }

// Whether the running sums come from a launch of their own, in one more row of counts.
bool group_sums(int blocks, int num_experts) { return static_cast<long long>(blocks) * (num_experts + 1) > kGroupCounts; }

struct GroupShared {
  uint16_t count[kGroupWaves][kCountMaxRows + 1];  // per wave and id, then the place of the wave's next route of it
  int scan[kGroupWaves];
  int sum[kCountMaxRows + 1], before[kCountMaxRows + 1];  // of every id: all routes, those of earlier workgroups
};

// Exclusive prefix of v over the workgroup's threads; the sum in *total.
__device__ __forceinline__ int group_scan(int v, GroupShared& s, int* total) {
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  int x = v;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int y = __shfl_up(x, off, kWave);
    if (lane >= off) x += y;
  }
  if (lane == kWave - 1) s.scan[wave] = x;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kGroupWaves; ++w) {
    const int c = s.scan[w];
    before += w < wave ? c : 0;
    sum += c;
  }
  *total = sum;
  return before + x - v;
}

// One workgroup's routes [first, first + kGroupRoutes).  hist: null, or [blocks][E + 1]
// counts of every workgroup (this one is `block`); summed: those of the workgroups before
// it instead, and behind them a row of all routes' counts.
__device__ __forceinline__ void group_block(const GroupArgs& a, int block, int blocks, const int32_t* hist,
                                            bool summed, GroupShared& s) {
  const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWave;
  const int ids = a.num_experts + 1;  // id num_experts has a place of its own behind the experts
  const int bits = 32 - __clz(a.num_experts);
  const int first = block * kGroupRoutes, here = min(a.numel - first, kGroupRoutes);
  const int per = (here + kGroupThreads - 1) / kGroupThreads;  // chunks of every wave
  for (int e = tid; e < ids; e += kGroupThreads) {
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) s.count[w][e] = 0;
    s.sum[e] = s.before[e] = 0;
  }
  int id[kGroupChunks], rank[kGroupChunks];
  unsigned long long same[kGroupChunks];
#pragma unroll
  for (int c = 0; c < kGroupChunks; ++c) {
    const int i = (wave * per + c) * kWave + lane;
    id[c] = c < per && i < here ? a.ids[first + i] : -1;
    if (id[c] < 0 || id[c] > a.num_experts) id[c] = -1;
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < kGroupChunks; ++c) {
    if (c >= per) break;
    same[c] = same_id(id[c], id[c] >= 0, bits);
    rank[c] = __popcll(same[c] & ((1ull << lane) - 1));
    if (id[c] >= 0 && rank[c] == 0) s.count[wave][id[c]] += static_cast<uint16_t>(__popcll(same[c]));
  }
  __syncthreads();
  if (hist && summed) {
    for (int e = tid; e < ids; e += kGroupThreads) {
      s.before[e] = hist[static_cast<size_t>(block) * ids + e];
      s.sum[e] = hist[static_cast<size_t>(blocks) * ids + e];
    }
    __syncthreads();
  } else if (hist) {  // (integer sums in LDS: the order does not matter)
    for (int i = tid; i < blocks * ids; i += kGroupThreads) {
      const int n = hist[i], b = i / ids, e = i - b * ids;
      if (!n) continue;
      atomicAdd(&s.sum[e], n);
      if (b < block) atomicAdd(&s.before[e], n);
    }
    __syncthreads();
  }
  // thread e: the places of id e before each wave, and the start of its group
  int sum = 0;
  if (tid < ids) {
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      const int n = s.count[w][tid];
      s.count[w][tid] = static_cast<uint16_t>(sum);
      sum += n;
    }
    if (hist) sum = s.sum[tid];
  }
  int total;
  const int start = group_scan(tid < ids ? sum : 0, s, &total);
  if (block == 0) {
    if (tid < ids) a.offsets[tid] = start;
    if (tid == 0) a.offsets[ids] = total;
  }
  if (tid < ids) s.before[tid] += start;
  __syncthreads();
#pragma unroll
  for (int c = 0; c < kGroupChunks; ++c) {
    if (c >= per) break;
    if (id[c] < 0) continue;
    const int at = s.count[wave][id[c]];
    a.order[s.before[id[c]] + at + rank[c]] = first + (wave * per + c) * kWave + lane;
    // (the wave's reads above are issued before this write)
    if (rank[c] == 0) s.count[wave][id[c]] = static_cast<uint16_t>(at + __popcll(same[c]));
  }
  for (long long i = static_cast<long long>(total) + block * kGroupThreads + tid; i < a.numel; i += blocks * kGroupThreads)
    a.order[i] = a.numel;
}

// The quantisation of rows by the workgroups behind the grouping ones.
template <int WPR>
__device__ __forceinline__ void quant_block(const GroupArgs& a, int block) {
  __shared__ uint32_t s_max[kGroupWaves];
  constexpr int kRowThreads = WPR * kWave;
  const int row = block * (kGroupThreads / kRowThreads) + threadIdx.x / kRowThreads;
  quant_row<WPR, 4>(a.x, row, row < a.x_rows, threadIdx.x % kRowThreads, a.K, a.q, a.scales, s_max);
}

// WPR: waves per quantised row, 0 without quantisation.
template <int WPR>
__global__ void __launch_bounds__(kGroupThreads) group_routes_kernel(GroupArgs a) {
  __shared__ GroupShared s;
  if constexpr (WPR > 0) {
    if (blockIdx.x > 0) return quant_block<WPR>(a, blockIdx.x - 1);
  }
  group_block(a, 0, 1, nullptr, false, s);
}

template <int WPR>
__global__ void __launch_bounds__(kGroupThreads) group_count_kernel(GroupArgs a, int blocks, int32_t* hist) {
  if constexpr (WPR > 0) {
    if (blockIdx.x >= blocks) return quant_block<WPR>(a, blockIdx.x - blocks);
  }
  __shared__ int bins[kCountMaxRows + 1];
  const int ids = a.num_experts + 1;
  for (int e = threadIdx.x; e < ids; e += kGroupThreads) bins[e] = 0;
  __syncthreads();
#pragma unroll
  for (int c = 0; c < kGroupChunks; ++c) {
    const long long i = static_cast<long long>(blockIdx.x) * kGroupRoutes + c * kGroupThreads + threadIdx.x;
    const int id = i < a.numel ? a.ids[i] : -1;
    if (id >= 0 && id < ids) atomicAdd(&bins[id], 1);  // (counts: the order does not matter)
  }
  __syncthreads();
  for (int e = threadIdx.x; e < ids; e += kGroupThreads) hist[static_cast<size_t>(blockIdx.x) * ids + e] = bins[e];
}

// Workgroup e: the counts of id e by workgroup become those of the workgroups before, all of them in row `blocks`.
__global__ void __launch_bounds__(kGroupThreads) group_sum_kernel(int ids, int blocks, int32_t* hist) {
  __shared__ GroupShared s;
  int before = 0;
  for (int b0 = 0; b0 < blocks; b0 += kGroupThreads) {  // (every thread takes part in the barriers)
    const int b = b0 + static_cast<int>(threadIdx.x);
    int32_t* const at = hist + static_cast<size_t>(b) * ids + blockIdx.x;
    int total;
    const int sum = group_scan(b < blocks ? *at : 0, s, &total);
    if (b < blocks) *at = before + sum;
    before += total;
    __syncthreads();  // (the scan's partial sums are read before they are written again)
  }
  if (threadIdx.x == 0) hist[static_cast<size_t>(blocks) * ids + blockIdx.x] = before;
}

__global__ void __launch_bounds__(kGroupThreads) group_place_kernel(GroupArgs a, int blocks, const int32_t* hist,
                                                                    bool summed) {
  __shared__ GroupShared s;
  group_block(a, blockIdx.x, blocks, hist, summed, s);
}

template <int WPR>
hipError_t launch_group(const GroupArgs& a, int32_t* hist, hipStream_t stream) {
  const int blocks = std::max(1, group_blocks(a.numel));
  const int quant = WPR ? (a.x_rows * WPR + kGroupWaves - 1) / kGroupWaves : 0;
  constexpr auto one = group_routes_kernel<WPR>;
  constexpr auto count = group_count_kernel<WPR>;
  if (blocks == 1) {
    hipLaunchKernelGGL(one, dim3(1 + quant), dim3(kGroupThreads), 0, stream, a);
  } else {
    hipLaunchKernelGGL(count, dim3(blocks + quant), dim3(kGroupThreads), 0, stream, a, blocks, hist);
    const bool summed = group_sums(blocks, a.num_experts);
    if (summed)
      hipLaunchKernelGGL(group_sum_kernel, dim3(a.num_experts + 1), dim3(kGroupThreads), 0, stream, a.num_experts + 1,
                         blocks, hist);
    hipLaunchKernelGGL(group_place_kernel, dim3(blocks), dim3(kGroupThreads), 0, stream, a, blocks,
                       static_cast<const int32_t*>(hist), summed);
  }
  return hipGetLastError();
}

}  // namespace

size_t group_hist_ints(int numel, int num_experts) {
  const int blocks = group_blocks(numel);
  return blocks > 1 ? (blocks + static_cast<size_t>(group_sums(blocks, num_experts))) * (num_experts + 1) : 0;
}

hipError_t launch_group_routes(const GroupArgs& a, int32_t* hist, hipStream_t stream) {
  if (!a.x) return launch_group<0>(a, hist, stream);
  if (a.x_rows <= kGroupQuantRows) {
    if (a.K <= 2048) return launch_group<1>(a, hist, stream);
    if (a.K <= 8192) return launch_group<4>(a, hist, stream);
  }
  // rows longer than a workgroup's registers, or too many for one launch: the quantisation in its own
  const hipError_t err = launch_act_quant_int8(a.x, a.x_rows, a.K, a.q, a.scales, stream);
  return err == hipSuccess ? launch_group<0>(a, hist, stream) : err;
}

}  // namespace ftmoe
