// Matrix products with one weight matrix per group of rows: dense int8 products
// (one group) and the products grouped by expert, bf16 or int8 (MatmulArgs).
//
// Weights are the MFMA A operand (rows = output features), rows of x the B
// operand (columns).  Both types take 64 bytes of a row per MFMA: 32 bf16 values
// (v_mfma_f32_16x16x32_bf16) or 64 int8 (v_mfma_i32_16x16x64_i8), a lane holding
// the 16 bytes of lane group l / 16.  A and B use the same placement of K, so the
// products pair up whatever the order inside the instruction.
#include <algorithm>

#include "kernels.h"

namespace ftmoe {

typedef int acc_i32 __attribute__((ext_vector_type(4)));

namespace {

template <bool INT8>
struct Acc {
  using type = f32x4;
};
template <>
struct Acc<true> {
  using type = acc_i32;
};

template <bool INT8>
__device__ __forceinline__ typename Acc<INT8>::type mma(u32x4 a, u32x4 b, typename Acc<INT8>::type c) {
  if constexpr (INT8)
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

// Rows [begin, end) of group e in the grouped order, cut to [0, rows] whatever
// the offsets hold.
__device__ __forceinline__ void group_range(const MatmulArgs& a, int e, int& begin, int& end) {
  if (!a.offsets) {
    begin = 0;
    end = a.rows;
    return;
  }
  begin = min(max(a.offsets[e], 0), a.rows);
  end = min(max(a.offsets[e + 1], begin), a.rows);
}

// The group of block b of the grid's blocks of `block` rows (one wave: a scan of
// the groups' block counts, 64 at a time); false past the last block.
__device__ __forceinline__ bool find_block(const MatmulArgs& a, int block, int b, int& e, int& begin, int& end) {
  const int lane = lane_id();
  int done = 0;
  for (int e0 = 0; e0 < a.E; e0 += kWave) {
    int lo = 0, hi = 0;
    if (e0 + lane < a.E) group_range(a, e0 + lane, lo, hi);
    const int nb = (hi - lo + block - 1) / block;
    int sum = nb;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int y = __shfl_up(sum, off, kWave);
      if (lane >= off) sum += y;
    }
    const unsigned long long past = __ballot(done + sum > b);
    if (past) {
      const int l = __ffsll(static_cast<long long>(past)) - 1;
      e = e0 + l;
      const int first = done + __shfl(sum - nb, l, kWave);
      begin = __shfl(lo, l, kWave) + (b - first) * block;
      end = min(__shfl(hi, l, kWave), begin + block);
      return true;
    }
    done += __shfl(sum, kWave - 1, kWave);
  }
  return false;
}

// One wave: 16 output features of 16 rows of one group.
template <bool INT8>
__global__ void __launch_bounds__(kWave) matmul_wave_kernel(MatmulArgs a) {
  using acc_t = typename Acc<INT8>::type;
  int e, begin, end;
  if (!find_block(a, 16, blockIdx.y, e, begin, end)) return;
  const int lane = lane_id(), r16 = lane & 15, g = lane >> 4;
  const int n_out = a.act < 0 ? a.N : a.N / 2;
  const int n0 = blockIdx.x * 16;
  const size_t kb = static_cast<size_t>(a.K) * (INT8 ? 1 : 2);
  // this lane's row of y
  int r = -1;
  if (begin + r16 < end) {
    r = a.order ? a.order[begin + r16] : begin + r16;
    if (r < 0 || r >= a.rows) r = -1;
  }
  const uint8_t* xr = a.x + static_cast<size_t>(r < 0 ? 0 : r / a.top_k) * kb;
  const uint8_t* we = a.w + static_cast<size_t>(e) * a.N * kb;
  const bool n_in = n0 + r16 < n_out;
  const uint8_t* wg = we + static_cast<size_t>(n_in ? n0 + r16 : 0) * kb;
  const uint8_t* wu = wg + static_cast<size_t>(n_out) * kb;
  acc_t acc_g = {}, acc_u = {};
  const u32x4 none = {0u, 0u, 0u, 0u};
  for (size_t at = 0; at < kb; at += 64) {
    const size_t c = at + 16 * g;
    const bool in = c < kb;
    const u32x4 xv = in && r >= 0 ? *reinterpret_cast<const u32x4*>(xr + c) : none;
    acc_g = mma<INT8>(in && n_in ? *reinterpret_cast<const u32x4*>(wg + c) : none, xv, acc_g);
    if (a.act >= 0) acc_u = mma<INT8>(in && n_in ? *reinterpret_cast<const u32x4*>(wu + c) : none, xv, acc_u);
  }
  if (r < 0) return;
  const float xs = INT8 ? a.xs[r / a.top_k] : 1.0f;
  const float rw = a.row_weight ? a.row_weight[r] : 1.0f;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int n = n0 + 4 * g + v;
    if (n >= n_out) break;
    float o = static_cast<float>(acc_g[v]);
    if constexpr (INT8) o *= a.ws[static_cast<size_t>(e) * a.N + n] * xs;
    if (a.act >= 0) {
      float u = static_cast<float>(acc_u[v]);
      if constexpr (INT8) u *= a.ws[static_cast<size_t>(e) * a.N + n_out + n] * xs;
      swiglu_clamp(a.limit, o, u);
      o = act_apply(a.act, o) * u;
    }
    o *= rw;
    const size_t at = static_cast<size_t>(r) * n_out + n;
    if (a.out_f32) static_cast<float*>(a.y)[at] = o;
    else static_cast<uint16_t*>(a.y)[at] = f32_to_bf16(o);
  }
}

// y[t] = bf16(sum of the routes' rows in route order + shared[t]), routes with
// ids outside [0, num_rows) skipped; H a multiple of 8.
__global__ void __launch_bounds__(256) combine_routes_kernel(const uint16_t* __restrict__ routes,
                                                             const int32_t* __restrict__ ids, int num_rows,
                                                             const float* __restrict__ shared, int M, int k, int H,
                                                             uint16_t* __restrict__ y) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int per = H / 8;
  if (i >= static_cast<long long>(M) * per) return;
  const int t = static_cast<int>(i / per), h = static_cast<int>(i % per) * 8;
  float acc[8] = {};
  for (int j = 0; j < k; ++j) {
    const int e = ids[static_cast<size_t>(t) * k + j];
    if (e < 0 || e >= num_rows) continue;
    const u32x4 v = *reinterpret_cast<const u32x4*>(routes + (static_cast<size_t>(t) * k + j) * H + h);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      acc[2 * w] += __uint_as_float(v[w] << 16);
      acc[2 * w + 1] += __uint_as_float(v[w] & 0xffff0000u);
    }
  }
  if (shared) {
#pragma unroll
    for (int w = 0; w < 8; ++w) acc[w] += shared[static_cast<size_t>(t) * H + h + w];
  }
  u32x4 o;
#pragma unroll
  for (int w = 0; w < 4; ++w) o[w] = pack_bf16x2(acc[2 * w], acc[2 * w + 1]);
  *reinterpret_cast<u32x4*>(y + static_cast<size_t>(t) * H + h) = o;
}

}  // namespace

hipError_t launch_matmul(const MatmulArgs& a, hipStream_t stream) {
  const int n_out = a.act < 0 ? a.N : a.N / 2;
  const int blocks = static_cast<int>(std::min<long long>(a.rows, a.rows / 16ll + a.E));
  const dim3 grid((n_out + 15) / 16, blocks);
  if (a.int8) hipLaunchKernelGGL(matmul_wave_kernel<true>, grid, dim3(kWave), 0, stream, a);
  else hipLaunchKernelGGL(matmul_wave_kernel<false>, grid, dim3(kWave), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_combine_routes(const uint16_t* routes, const int32_t* ids, int num_rows, const float* shared, int M,
                                 int k, int H, uint16_t* y, hipStream_t stream) {
  const long long n = static_cast<long long>(M) * (H / 8);
  hipLaunchKernelGGL(combine_routes_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, stream, routes,
                     ids, num_rows, shared, M, k, H, y);
  return hipGetLastError();
}

}  // namespace ftmoe
