// Pieces shared by the matrix products' kernels (matmul.hip, matmul_stream.hip, matmul_tile.hip) and the grouping of
// routes (group.hip).
#pragma once

#include "kernels.h"

namespace ftmoe {

typedef int acc_i32 __attribute__((ext_vector_type(4)));

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

// 32 x 32 outputs from 32 bytes of K: a lane holds the 16 bytes of half l / 32 of
// row l % 32, and results 8 (v / 4) + 4 (l / 32) + v % 4 (row of A), l % 32 (row of B).
typedef int acc32_i32 __attribute__((ext_vector_type(16)));
typedef float acc32_f32 __attribute__((ext_vector_type(16)));
template <bool INT8>
struct Acc32 {
  using type = acc32_f32;
};
template <>
struct Acc32<true> {
  using type = acc32_i32;
};

template <bool INT8>
__device__ __forceinline__ typename Acc32<INT8>::type mma32(u32x4 a, u32x4 b, typename Acc32<INT8>::type c) {
  if constexpr (INT8)
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

// An exact integer sum times its row's and its channel's scale, in an order that leaves the range of normal numbers
// only where the result does: a sum is 0 or at least 1 in magnitude, so the row's scale comes first where it is
// below 1 (the channel's may be large) and last where it is not (the channel's may be small).  One of the two parts
// is 1, so that there are two roundings; every form multiplies in this order.
struct RowFactor {
  float first, last;
};
__device__ __forceinline__ RowFactor row_factor(float scale) {
  return fabsf(scale) < 1.0f ? RowFactor{scale, 1.0f} : RowFactor{1.0f, scale};
}
__device__ __forceinline__ float scaled(float sum, const RowFactor& x, float ws) { return sum * x.first * ws * x.last; }

// swiglu_clamp that keeps a NaN (minima and maxima drop it): a row of NaN stays one.
__device__ __forceinline__ void clamp_numbers(float lim, float& g, float& u) {
  if (lim > 0.f) {
    g = g > lim ? lim : g;
    u = u > lim ? lim : u < -lim ? -lim : u;
  }
}

// Rows [begin, end) of group e in the grouped order, cut to [0, rows] whatever
// the offsets hold; group E is the extra one.
__device__ __forceinline__ void group_range(const MatmulArgs& a, int e, int& begin, int& end) {
  if (e == a.E) {
    begin = a.rows;
    end = a.rows + a.extra;
  } else if (!a.offsets) {
    begin = 0;
    end = a.rows;
  } else {
    begin = min(max(a.offsets[e], 0), a.rows);
    end = min(max(a.offsets[e + 1], begin), a.rows);
  }
}

// Lanes of the wave whose id equals this lane's (ids below 2^bits), among those with valid set.
__device__ __forceinline__ unsigned long long same_id(int id, bool valid, int bits) {
  unsigned long long m = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const unsigned long long set = __ballot((id >> b) & 1);
    m &= (id >> b) & 1 ? set : ~set;
  }
  return m;
}

__host__ __device__ inline int group_count(const MatmulArgs& a) { return a.E + (a.extra > 0 ? 1 : 0); }

// The streaming form, for few rows per group (matmul_stream.hip): a workgroup has
// 16 features x 16 rows with K split over its waves (split), 64 features x 16 rows,
// each wave with the whole of K (whole), or 32 features x 32 rows, split (wide; not
// where x is quantised on the way).
enum StreamShape { kStreamSplit, kStreamWhole, kStreamWide };
constexpr int kStreamQuantMaxK = 2048;
hipError_t launch_matmul_stream(const MatmulArgs& a, StreamShape shape, hipStream_t stream);

// The tiled form, for many rows per group (matmul_tile.hip): weight rows x rows of x
// of a workgroup; once: the weights are read about once, past the caches.
enum TileShape { kTile128x64, kTile256x128, kTile256x256 };
hipError_t launch_matmul_tile(const MatmulArgs& a, TileShape shape, bool once, hipStream_t stream);

}  // namespace ftmoe
