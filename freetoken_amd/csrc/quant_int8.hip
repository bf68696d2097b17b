// Symmetric 8-bit quantisation, one scale per row (ftmoe_act_quant_int8).
//
// Bound by memory: x is read once and the codes written once.  Measured: 8192 rows of
// 7168 27.9 us (6.3 TB/s, most of it from the memory-side cache), 65536 of 768 26.5 us
// (5.7), one row of 7168 2.2 us.  Rows up to 2048 values take a wave, up to 8192 a
// workgroup of four: all of a row's loads are in flight together and its values
// stay in registers between the maximum and the codes.
#include <algorithm>

#include "quant_int8.h"

namespace ftmoe {

namespace {

constexpr int kQuantThreads = 256;

template <int WPR, int KEEP>
__global__ void __launch_bounds__(kQuantThreads) act_quant_int8_kernel(const uint16_t* __restrict__ x, int rows, int K,
                                                                       int8_t* __restrict__ q,
                                                                       float* __restrict__ scales) {
  constexpr int kRowThreads = WPR * kWave;
  __shared__ uint32_t s_max[kQuantThreads / kWave];
  const int row = blockIdx.x * (kQuantThreads / kRowThreads) + threadIdx.x / kRowThreads;
  quant_row<WPR, KEEP>(x, row, row < rows, threadIdx.x % kRowThreads, K, q, scales, s_max);
}

}  // namespace

hipError_t launch_act_quant_int8(const uint16_t* x, int rows, int K, int8_t* q, float* scales, hipStream_t stream) {
  constexpr int kMost = 1 << 23;  // rows of a launch, which holds below 2^32 threads
  for (long long first = 0; first < rows; first += kMost) {
    const int n = static_cast<int>(std::min<long long>(kMost, rows - first));
    const uint16_t* const xr = x + first * K;
    int8_t* const qr = q + first * K;
    float* const sr = scales + first;
    const dim3 block(kQuantThreads);
    if (K <= 2048)
      hipLaunchKernelGGL((act_quant_int8_kernel<1, 4>), dim3((n + 3) / 4), block, 0, stream, xr, n, K, qr, sr);
    else if (K <= 8192)
      hipLaunchKernelGGL((act_quant_int8_kernel<4, 4>), dim3(n), block, 0, stream, xr, n, K, qr, sr);
    else
      hipLaunchKernelGGL((act_quant_int8_kernel<4, 0>), dim3(n), block, 0, stream, xr, n, K, qr, sr);
  }
  return hipGetLastError();
}

}  // namespace ftmoe
