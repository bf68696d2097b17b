// Symmetric 8-bit quantisation, one scale per row: the row of a wave or of several,
// shared by the quantisation kernel (quant_int8.hip) and the grouping of an expert
// layer's routes (group.hip).
//
// With a = max |x| of a row: q = round(127 x / a), ties to even, scale a / 127.
// Ties are not rare (x = a/2 is 63.5), so the quotient has to be the correctly
// rounded one: t = 127 x is exact in float32 (8 by 7 bits), and with r = RN(1/a)
// and y = RN(t r) the corrected RN(y + r RN(t - y a)) is RN(t / a) (Markstein; the
// residual is exact in the FMA).  t / a has a 15-bit numerator and an 8-bit
// denominator, so RN(t / a) is a half exactly when t / a is, and otherwise on the
// same side of it: rounding it to an integer gives round(127 x / a).  Adding
// 1.5 2^23 does that rounding and leaves the code in the low byte.
//
// Magnitudes are compared as the integers of their bits, two bf16 at a time, where
// an infinity or a NaN is larger than every number.
#pragma once

#include "kernels.h"

namespace ftmoe {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t max_pair(uint32_t m, uint32_t v) {
  return __builtin_bit_cast(
      uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, v & 0x7fff7fffu)));
}

__device__ __forceinline__ uint32_t wave_max_pair(uint32_t m) {
  m = max_pair(m, dpp_u32<0xB1>(m));
  m = max_pair(m, dpp_u32<0x4E>(m));
  m = max_pair(m, dpp_u32<0x141>(m));
  m = max_pair(m, dpp_u32<0x140>(m));
  const auto lane = [&](int l) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(m), l)); };
  return max_pair(max_pair(lane(0), lane(16)), max_pair(lane(32), lane(48)));
}

struct RowScale {
  float a, r, mul;  // a and 127 scaled by the same power of two; r = RN(1/a)
};

// Rows far from 1 are scaled by 2^64 or 2^-64 first, which is exact for every
// value that does not quantise to 0, so that neither 127 x nor 1/a leaves the
// range of normal numbers.
__device__ __forceinline__ RowScale row_scale(float amax) {
  const float pre = amax > 0x1p60f ? 0x1p-64f : amax < 0x1p-60f ? 0x1p64f : 1.0f;
  RowScale s;
  s.a = amax * pre;
  s.r = __fdiv_rn(1.0f, s.a);
  s.mul = 127.0f * pre;
  return s;
}

// The code of x in the low byte.
__device__ __forceinline__ uint32_t code(float x, const RowScale& s) {
  const float t = x * s.mul;
  const float y = t * s.r;
  const float z = __builtin_fmaf(__builtin_fmaf(-y, s.a, t), s.r, y);
  return __float_as_uint(z + 0x1.8p23f);
}

__device__ __forceinline__ uint2 codes8(const u32x4& v, const RowScale& s) {
  uint32_t o[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t c0 = code(__uint_as_float(v[2 * h] << 16), s), c1 = code(__uint_as_float(v[2 * h] & 0xffff0000u), s);
    const uint32_t c2 = code(__uint_as_float(v[2 * h + 1] << 16), s);
    const uint32_t c3 = code(__uint_as_float(v[2 * h + 1] & 0xffff0000u), s);
    // low bytes of c0, c1 and of c2, c3, then the two halves
    const uint32_t lo = __builtin_amdgcn_perm(c1, c0, 0x0c0c0400u), hi = __builtin_amdgcn_perm(c3, c2, 0x0c0c0400u);
    o[h] = lo | (hi << 16);
  }
  return uint2{o[0], o[1]};
}

// Scale and codes of a row from the bits of its largest magnitudes (wave_max_pair).
struct RowCodes {
  float scale;
  bool live;  // the row has codes other than 0
  RowScale s;
  __device__ __forceinline__ uint2 codes(const u32x4& v) const { return live ? codes8(v, s) : uint2{0u, 0u}; }
};

__device__ __forceinline__ RowCodes row_codes(uint32_t pair) {
  const uint32_t bits = max(pair & 0xffffu, pair >> 16);
  const bool finite = bits < 0x7f80u;
  const float amax = __uint_as_float(bits << 16);
  RowCodes r;
  r.scale = finite ? __fdiv_rn(amax, 127.0f) : __uint_as_float(0x7fc00000u);
  r.live = finite && bits != 0;
  r.s = row_scale(r.live ? amax : 1.0f);
  return r;
}

// Quantises row `row` (live: it exists) with WPR waves, thread t of them; a thread
// holds up to KEEP 16-byte pieces of the row in registers (KEEP 0: any length, read
// twice, the second time from a cache).  s_max: a word per wave of the workgroup; with
// WPR > 1 every thread of the workgroup takes part in the barrier.
template <int WPR, int KEEP>
__device__ __forceinline__ void quant_row(const uint16_t* __restrict__ x, int row, bool live, int t, int K,
                                          int8_t* __restrict__ q, float* __restrict__ scales, uint32_t* s_max) {
  constexpr int kRowThreads = WPR * kWave;
  const int wave = threadIdx.x / kWave;
  const u32x4* xr = reinterpret_cast<const u32x4*>(x + static_cast<size_t>(row) * K);
  uint2* qr = reinterpret_cast<uint2*>(q + static_cast<size_t>(row) * K);
  const int n = live ? K / 8 : 0;
  u32x4 v[KEEP ? KEEP : 1];
  uint32_t m = 0;
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i) v[i] = t + i * kRowThreads < n ? xr[t + i * kRowThreads] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) m = max_pair(m, v[i][w]);
  } else {
    for (int p = t; p < n; p += kRowThreads) {
      const u32x4 u = xr[p];
#pragma unroll
      for (int w = 0; w < 4; ++w) m = max_pair(m, u[w]);
    }
  }
  m = wave_max_pair(m);
  if constexpr (WPR > 1) {
    if (lane_id() == 0) s_max[wave] = m;
    __syncthreads();
    const int first = wave / WPR * WPR;
#pragma unroll
    for (int w = 0; w < WPR; ++w) m = max_pair(m, s_max[first + w]);
  }
  const RowCodes r = row_codes(m);
  if (live && t == 0) scales[row] = r.scale;
  auto put = [&](int p, const u32x4& u) { qr[p] = r.codes(u); };
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (t + i * kRowThreads < n) put(t + i * kRowThreads, v[i]);
  } else {
    for (int p = t; p < n; p += kRowThreads) put(p, xr[p]);
  }
}

}  // namespace ftmoe
