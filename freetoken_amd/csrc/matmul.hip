// Matrix products with one weight matrix per group of rows (MatmulArgs): dense
// int8 products (one group) and the products grouped by expert, bf16 or int8; and
// the sum of an expert layer's routes.  Here: the choice between the streaming form
// (matmul_stream.hip) and the tiled one (matmul_tile.hip).
//
// In both, weights are the MFMA A operand (rows = output features), rows of x the B
// operand (columns), and both types take 16 bytes of a row per lane: A and B use the same
// placement of K, so the products pair up whatever the order inside the instruction.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "matmul.h"

namespace ftmoe {

namespace {

constexpr int kCombineThreads = 64;  // (a decode step has few: spread over the CUs)

// Eight values of a route's row, past the caches: it is read once.
template <typename T>
__device__ __forceinline__ void load_row8(const T* p, u32x4 (&v)[sizeof(T) / 2]) {
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 2; ++i) v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + i);
}

template <typename T>
__device__ __forceinline__ void add_row8(float (&acc)[8], const u32x4 (&v)[sizeof(T) / 2]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4) acc[i] += __uint_as_float(v[i / 4][i % 4]);
    else acc[i] += __uint_as_float(i % 2 ? v[0][i / 2] & 0xffff0000u : v[0][i / 2] << 16);
  }
}

// y[t] = bf16(sum of the routes' rows in route order, then the shared row M k + t),
// routes with ids outside [0, num_rows) skipped; H a multiple of 8; rows of T, bf16 (uint16_t) or float32.
// The rows of eight routes are read before the first is added.  Bound by reading them: 8192 x 8
// rows of 2048 bf16 49 us (6.1 TB/s, part of it from the memory-side cache), float32 101 (5.7 TB/s).
template <typename T>
__global__ void __launch_bounds__(kCombineThreads) combine_routes_kernel(const T* __restrict__ routes,
                                                                         const int32_t* __restrict__ ids, int num_rows,
                                                                         int shared, int M, int k, int H,
                                                                         uint16_t* __restrict__ y) {
  const long long i = static_cast<long long>(blockIdx.x) * kCombineThreads + threadIdx.x;
  const int per = H / 8;
  if (i >= static_cast<long long>(M) * per) return;
  const int t = static_cast<int>(i / per), h = static_cast<int>(i % per) * 8;
  const int32_t* const tid = ids + static_cast<size_t>(t) * k;
  const T* const first = routes + static_cast<size_t>(t) * k * H + h;
  float acc[8] = {};
  for (int j0 = 0; j0 < k; j0 += 8) {
    u32x4 v[8][sizeof(T) / 2];
    bool in[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = j0 + j < k ? tid[j0 + j] : -1;
      in[j] = e >= 0 && e < num_rows;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (in[j]) load_row8(first + static_cast<size_t>(j0 + j) * H, v[j]);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (in[j]) add_row8<T>(acc, v[j]);
  }
  if (shared) {
    u32x4 v[sizeof(T) / 2];
    load_row8(routes + (static_cast<size_t>(M) * k + t) * H + h, v);
    add_row8<T>(acc, v);
  }
  u32x4 o;
#pragma unroll
  for (int w = 0; w < 4; ++w) o[w] = pack_bf16x2(acc[2 * w], acc[2 * w + 1]);
  *reinterpret_cast<u32x4*>(y + static_cast<size_t>(t) * H + h) = o;
}

}  // namespace

// Forms and tiles are chosen from the sizes known on the host: the rows per group
// are R / E on average.  Measured (us, int8 unless said; streams split / whole /
// wide | tiles of 128 x 64 / 256 x 128):
//   one group, N 4096, K 7168: 1 row 7.1 / - / 9.9 | 22 / 38, 16 rows 8.4 / - / 10.6 | 22, 48 rows 19 / - / 12.6 | 22;
//   N 7168, K 2048: 16 rows 6.5 / - / 5.7 | 10, 64 rows - / - / 9 | 10.5, 128 rows - / - / 15 | 10.7 / 16;
//   128 experts, N 1536 (gate and up), K 2048: 8 rows 9.1 / 10.1 / 9.9 | 14, 64 rows 39 / 30 / 35 | 36, 256 rows 76 /
//   58 / 69 | 62, 512 rows 82 / 61 / 73 | 64; N 2048, K 768: 64 rows 30 / 17 / 25 | 20, 512 rows 70 / 35 / 52 | 38;
//   64 experts, N 7168, K 2048, 512 rows 209 / 150 / 158 | 147;
//   rows of 4 KB and more: bf16 N 1536, K 2048, 64 rows over 128 experts 56 / 68 / 58 | 70; N 4096, K 7168, 9 rows
//   over 65 43 / 56 / 47 | 57, 300 over 64 270 / 268 / 268 | 273.
namespace {

enum class Form { kTiles, kSplit, kWhole, kWide };

Form form_of(const MatmulArgs& a) {
  const long long n_out = a.act < 0 ? a.N : a.N / 2, rows = a.rows, E = a.E;
  const long long tiles = (n_out + 15) / 16;  // of 16 features
  if (tiles > 1 << 24) return Form::kTiles;   // a launch holds below 2^32 threads, 256 for 16 to 64 features when streaming
  if (E == 1) return rows <= 16 && tiles <= 384 ? Form::kSplit : rows <= 64 ? Form::kWide : Form::kTiles;
  if (rows > 4 * E) return rows <= 16 * E && tiles * E <= 1536 ? Form::kWide : Form::kTiles;
  // K is split where there are too few workgroups without it, or rows long enough for four streams
  const long long row_bytes = static_cast<long long>(a.K) * (a.int8 ? 1 : 2);
  return row_bytes >= 4096 || tiles * std::min(rows, E) <= 512 ? Form::kSplit : Form::kWhole;
}

}  // namespace

bool launch_matmul_quantises(const MatmulArgs& a) {
  const Form form = form_of(a);
  // Saves a launch each, but every workgroup quantises its group's rows anew.  An expert layer (us, neither product /
  // the down product / both): 8 routes over 16 experts (H 1024, I 512) 17.9 / 17.2 / 14.6; over 128 (H 2048, I 768)
  // 8 routes 22.8 / 21.2 / 18.1, 32 routes - / 39.7 / 36.8, 64 routes 55.2 / 60.7, 512 routes 106 / 121.
  return a.int8 && a.K <= kStreamQuantMaxK && a.rows <= 32 &&
         (form == Form::kSplit || form == Form::kWhole);
}

hipError_t launch_matmul(const MatmulArgs& a, hipStream_t stream) {
  switch (form_of(a)) {
    case Form::kSplit: return launch_matmul_stream(a, kStreamSplit, stream);
    case Form::kWhole: return launch_matmul_stream(a, kStreamWhole, stream);
    case Form::kWide: return launch_matmul_stream(a, kStreamWide, stream);
    default: break;
  }
  const long long n_out = a.act < 0 ? a.N : a.N / 2, rows = a.rows;
  // Tiles: the time of a shape goes by its rounds over the workgroups that fit the
  // chip at once (the mean of the whole rounds and the fraction) times what a round
  // of it takes, from the rates that large calls reach (dense 8192 x 4096 x 7168: 2360, 2140 and
  // 1430 T/s).  Up to 32 rows per group the smallest tiles, whose weights pass
  // the caches (1000 rows over 64 experts, N 7168, K 2048: 162, cached 176; 4000 rows 264 / 221);
  // tiles of 128 rows read past the caches up to 64 (4000 rows 191 / 200, 8000 291 / 240).
  if (rows <= 32ll * a.E && a.E > 1) return launch_matmul_tile(a, kTile128x64, true, stream);
  struct Shape {
    TileShape shape;
    int feats, rows, slots;
    double round;
  };
  constexpr Shape kShapes[] = {
      {kTile128x64, 128, 64, 512, 11.5}, {kTile256x128, 256, 128, 256, 15.3}, {kTile256x256, 256, 256, 256, 28.3}};
  const Shape* best = nullptr;
  double least = 0;
  for (const Shape& s : kShapes) {
    const int feats = a.act < 0 ? s.feats : s.feats / 2;
    // blocks of rows: a group's last one is half full on average
    const double blocks = a.E == 1 ? static_cast<double>((rows + s.rows - 1) / s.rows)
                                   : std::max<double>(std::min<long long>(rows, a.E),
                                                      static_cast<double>(rows) / s.rows + 0.5 * a.E);
    const double rounds = blocks * static_cast<double>((n_out + feats - 1) / feats) / s.slots;
    const double t = 0.5 * (rounds + std::ceil(rounds)) * s.round;
    if (!best || t < least) {
      best = &s;
      least = t;
    }
  }
  return launch_matmul_tile(a, best->shape, best->shape == kTile256x128 && a.E > 1 && rows <= 64ll * a.E, stream);
}

hipError_t launch_combine_routes(const void* routes, bool f32, const int32_t* ids, int num_rows, bool shared, int M,
                                 int k, int H, uint16_t* y, hipStream_t stream) {
  const long long n = static_cast<long long>(M) * (H / 8);
  const dim3 grid(static_cast<unsigned>((n + kCombineThreads - 1) / kCombineThreads)), block(kCombineThreads);
  if (f32)
    hipLaunchKernelGGL(combine_routes_kernel<float>, grid, block, 0, stream, static_cast<const float*>(routes), ids,
                       num_rows, static_cast<int>(shared), M, k, H, y);
  else
    hipLaunchKernelGGL(combine_routes_kernel<uint16_t>, grid, block, 0, stream, static_cast<const uint16_t*>(routes),
                       ids, num_rows, static_cast<int>(shared), M, k, H, y);
  return hipGetLastError();
}

}  // namespace ftmoe
