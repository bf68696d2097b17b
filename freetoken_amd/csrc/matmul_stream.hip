// Streaming form of the matrix products of MatmulArgs, for few rows per group:
// the time is that of reading the weights once.
//
// A workgroup has 4 waves, a wave 16 RT weight rows x 16 CT rows of x of one group.
// KS waves share the same weight rows and split K between them, adding their sums
// through LDS in a fixed order; groups of KS waves have weight rows of their own.  Each
// wave copies its weight lines global -> LDS by LDS-DMA into a ring of its own (no
// barrier in the K loop): an instruction covers 8 whole 128-byte lines, where a
// register load in the operand layout covers half lines.  x comes straight to registers.
// Three stages of 2 KB a wave (4 with gate and up rows), two of them on their way while the third is multiplied: where
// there are enough workgroups six (three) of them share a CU, with 144 KB of LDS and 96 KB of weights on their way.
// Where there are not (one row, N 4096: one a CU) it is 16 KB, and latency bounds the call.  Measured: 512 rows over
// 128 experts, N 1536 (gate and up), K 2048, 61 us (6.6 TB/s of weights), 8 rows 9.1 us (2.8 TB/s: latency of one short
// pass).
//
// QX: x is bf16.  The workgroup quantises its rows (quant_int8.h, the codes that
// act_quant_int8 gives) into LDS while its first weights are on their way, which saves
// a step of one or a few tokens the launch between an expert's two products, and
// with the rows' experts found from their ids in every workgroup (ten ballots) also the
// launch before the first.
#include <algorithm>

#include "kernels.h"
#include "lds_ring.h"
#include "matmul.h"
#include "quant_int8.h"

namespace ftmoe {

namespace {

constexpr int kTile = 16 * 128;  // bytes of 16 weight rows of one K step

// The group and rows of block b of the grid's blocks of `block` rows: a scan of the
// groups' block counts, 64 at a time; false past the last block.
__device__ __forceinline__ bool find_block(const MatmulArgs& a, int block, int b, int& e, int& begin, int& end) {
  if (!a.offsets) {
    e = 0;
    begin = b * block;
    end = min(begin + block, a.rows);
    return begin < a.rows;
  }
  const int lane = lane_id();
  int done = 0;
  const int groups = group_count(a);
  for (int e0 = 0; e0 < groups; e0 += kWave) {
    int lo = 0, hi = 0;
    if (e0 + lane < groups) group_range(a, e0 + lane, lo, hi);
    const int nb = (hi - lo + block - 1) / block;
    int sum = nb;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int y = __shfl_up(sum, off, kWave);
      if (lane >= off) sum += y;
    }
    const unsigned long long past = __ballot(done + sum > b);
    if (past) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<long long>(past)) - 1);
      e = e0 + l;
      const int first = done + __builtin_amdgcn_readlane(sum - nb, l);
      begin = __builtin_amdgcn_readlane(lo, l) + (b - first) * block;
      end = min(__builtin_amdgcn_readlane(hi, l), begin + block);
      return true;
    }
    done += __builtin_amdgcn_readlane(sum, kWave - 1);
  }
  return false;
}

// The same from the rows' ids (at most 64, one per lane): blocks of 16 rows, the groups
// in the order of their first rows, and the row of this lane's column or -1.
__device__ __forceinline__ bool find_rows(const MatmulArgs& a, int b, int& e, int& row) {
  const int lane = lane_id(), r16 = lane & 15;
  const int id = lane < a.rows ? a.ids[lane] : -1;
  const bool valid = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.E);
  const unsigned long long same = same_id(id, valid, 32 - __builtin_clz(a.E));
  const int rank = __popcll(same & ((1ull << lane) - 1));
  const int nb = valid && rank == 0 ? (__popcll(same) + 15) / 16 : 0;
  int sum = nb;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int y = __shfl_up(sum, off, kWave);
    if (lane >= off) sum += y;
  }
  const unsigned long long past = __ballot(sum > b);
  if (!past) {
    e = a.E;
    const int i = a.rows + 16 * (b - __builtin_amdgcn_readlane(sum, kWave - 1)) + r16;
    row = i < a.rows + a.extra ? i : -1;
    return __ballot(row >= 0) != 0;
  }
  const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<long long>(past)) - 1);
  e = __builtin_amdgcn_readlane(id, l);
  const int j = b - __builtin_amdgcn_readlane(sum - nb, l);
  const bool mine = id == e && rank / 16 == j;
  const int count = __popcll(__ballot(mine));
  // lane numbers to the lanes of their columns, the others' to one that is not read
  const int at = __builtin_amdgcn_ds_permute((mine ? rank % 16 : kWave - 1) * 4, lane);
  const int r = __shfl(at, r16, kWave);
  row = r16 < count ? r : -1;
  return true;
}

template <bool INT8, bool GATE, bool QX, int RT, int CT, int S, int KS, int W>
__global__ void __launch_bounds__(W* kWave) matmul_stream_kernel(MatmulArgs a) {
  using acc_t = typename Acc<INT8>::type;
  constexpr int kStage = RT * kTile, kRing = S * kStage;
  constexpr int kGroups = W / KS;  // waves that own rows of their own
  constexpr int kRed = KS > 1 ? W * RT * CT * kWave * 16 : 0;
  constexpr int kPerStep = 2 * RT + (QX ? 0 : 2 * CT);  // vector memory instructions of a step
  // The quantised rows, chunk c (16 bytes) of row k at c ^ k % 16; their scales, where the rings were (two
  // workgroups of gate and up rows just fit a CU).
  constexpr int kXRow = kStreamQuantMaxK, kXRows = QX ? 16 * CT * kXRow : 0;
  constexpr int kScales = QX ? 16 * CT * 4 : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[std::max(W * kRing, kRed + kScales) + kXRows];
  uint8_t* const xq = lds + std::max(W * kRing, kRed + kScales);
  float* const s_xs = reinterpret_cast<float*>(lds + kRed);
  const int lane = lane_id(), r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int e, begin = 0, end = 0, listed = -1;
  const bool by_id = QX && a.ids;
  if (by_id ? !find_rows(a, blockIdx.y, e, listed) : !find_block(a, 16 * CT, blockIdx.y, e, begin, end)) return;
  const int n_out = GATE ? a.N / 2 : a.N;
  constexpr int NJ = GATE ? RT / 2 : RT;
  const int wk = wave % KS;
  const int n0 = (blockIdx.x * kGroups + wave / KS) * 16 * NJ;
  const uint32_t rb = static_cast<uint32_t>(a.K) * (INT8 ? 1 : 2);

  const bool extra = e == a.E;
  const uint8_t* const w = extra ? a.extra_w : a.w + static_cast<size_t>(e) * a.N * rb;
  const float* const ws = extra ? a.extra_ws : a.ws + static_cast<size_t>(e) * a.N;
  const float limit = extra ? a.extra_limit : a.limit;
  auto x_row = [&](int r) -> uint32_t { return r < a.rows ? r / a.top_k : r - a.rows + a.extra_x; };

  // rows of y and of x in this lane's columns
  int route[CT];
  uint32_t xvoff[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int i = begin + 16 * c + r16;
    int r = listed;
    if (!by_id && i < end) {
      r = a.order && !extra ? a.order[i] : i;
      if (static_cast<uint32_t>(r) >= static_cast<uint32_t>(a.rows + a.extra)) r = -1;
    }
    route[c] = r;
    xvoff[c] = r < 0 ? kOutOfRange : x_row(r) * rb + 16 * g;
  }
  // weights: lane l of copy h of a tile takes chunk (l % 8) ^ (l / 8) of row 8h + l / 8
  const int q = (lane & 7) ^ (lane >> 3);
  const uint8_t* wexp = w + static_cast<size_t>(n0) * rb;
  const __amdgpu_buffer_rsrc_t rw =
      make_rsrc(wexp, static_cast<uint32_t>(max(GATE ? a.N - n0 : min(a.N - n0, 16 * RT), 0)) * rb);
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(a.x, static_cast<uint32_t>(a.x_rows) * rb);
  uint32_t wvoff[RT][2];
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      wvoff[j][h] = static_cast<uint32_t>((j < NJ ? 16 * j : n_out + 16 * (j - NJ)) + 8 * h + (lane >> 3)) * rb + 16 * q;
  const int nst = static_cast<int>((rb + 127) / 128);
  const int lo = wk * nst / KS, hi = (wk + 1) * nst / KS, n = hi - lo;
  // the last step's chunks past the rows' end
  const uint32_t tail = static_cast<uint32_t>(nst - 1) * 128;
  const uint32_t wdead = tail + 16 * q >= rb ? kOutOfRange : 0u;
  const uint32_t xdead[2] = {tail + 16 * g >= rb ? kOutOfRange : 0u, tail + 64 + 16 * g >= rb ? kOutOfRange : 0u};

  uint8_t* const ring = lds + wave * kRing;
  u32x4 xf[S][CT][2];
  // QX: row k of the workgroup's columns belongs to wave k % W, lane l holding its pieces l, l + 64, ...
  constexpr int kMine = QX ? 16 * CT / W : 1, kPieces = QX ? kStreamQuantMaxK / 8 / kWave : 1;
  u32x4 raw[kMine][kPieces];
  int mine[kMine];
  float scale[kMine];
  if constexpr (QX) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int k = m * W + wave, c = m * W / 16;  // (W divides 16: a constant column tile)
      mine[m] = __builtin_amdgcn_readlane(route[c], k & 15);
      const u32x4* row = reinterpret_cast<const u32x4*>(a.x + static_cast<size_t>(x_row(max(mine[m], 0))) * rb * 2);
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const int at = lane + p * kWave;
        raw[m][p] = mine[m] >= 0 && at < a.K / 8 ? row[at] : u32x4{0u, 0u, 0u, 0u};
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  auto issue = [&](int s, int slot) {  // step s of this wave; past its end: the same instructions, reading zeros
    const uint32_t off = s < n ? 0u : kOutOfRange;
    const bool last = lo + s == nst - 1;
    const uint32_t so = static_cast<uint32_t>(lo + s) * 128;
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        lds_buf16_nt(rw, ring + slot * kStage + j * kTile + h * 1024, wvoff[j][h] | off | (last ? wdead : 0u), so);
    if constexpr (!QX)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int p = 0; p < 2; ++p) xf[slot][c][p] = buf_x4(rx, (xvoff[c] | off | (last ? xdead[p] : 0u)) + 64 * p, so);
  };
  acc_t acc[RT][CT];
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[j][c] = acc_t{};
  auto compute = [&](int slot, int s) {
    if constexpr (QX) {  // (steps past the end, and past K in the last one, meet zero weights)
      const uint8_t* const at = xq + r16 * kXRow;
      const int chunk = min(lo + s, nst - 1) * 8 + g;
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          xf[slot][c][p] = *reinterpret_cast<const u32x4*>(at + c * 16 * kXRow + 16 * ((chunk + 4 * p) ^ r16));
    }
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      const uint8_t* row = ring + slot * kStage + j * kTile + r16 * 128;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(row + (((4 * p + g) ^ (r16 & 7)) << 4));
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[j][c] = mma<INT8>(w, xf[slot][c][p], acc[j][c]);
      }
    }
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    issue(s, s);
    __builtin_amdgcn_sched_barrier(0);
  }
  if constexpr (QX) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      scale[m] = 0.f;
      if (mine[m] < 0) continue;
      const int k = m * W + wave;
      uint32_t top = 0;
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
#pragma unroll
        for (int w4 = 0; w4 < 4; ++w4) top = max_pair(top, raw[m][p][w4]);
      const RowCodes rc = row_codes(wave_max_pair(top));
      scale[m] = rc.scale;
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
        if (lane + p * kWave < a.K / 8)
          *reinterpret_cast<uint2*>(xq + k * kXRow + 16 * ((lane + p * kWave) / 2 ^ (k & 15)) + 8 * (lane & 1)) =
              rc.codes(raw[m][p]);
    }
    wait_lgkm0();
    bare_barrier();
  }
  for (int i = 0; i < n; i += S) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      // (steps past the end compute on zeros: the sums stay, and every wait counts whole steps)
      issue(i + s + S - 1, (s + S - 1) % S);
      wait_vm<(S - 1) * kPerStep>();
      __builtin_amdgcn_sched_barrier(0);
      compute(s, i + s);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // ---- the waves' sums through LDS; of the KS waves of the same rows, wave w finishes the tiles t with t % KS == w
  acc_t* const red = reinterpret_cast<acc_t*>(lds);
  const int w0 = wave - wk;
  if constexpr (KS > 1 || QX) {
    wait_vm<0>();
    __syncthreads();
    if constexpr (KS > 1)
#pragma unroll
      for (int j = 0; j < RT; ++j)
#pragma unroll
        for (int c = 0; c < CT; ++c) red[((wave * RT + j) * CT + c) * kWave + lane] = acc[j][c];
    if constexpr (QX)
#pragma unroll
      for (int m = 0; m < kMine; ++m)
        if (lane == 0) s_xs[m * W + wave] = scale[m];
    __syncthreads();
  }
  auto sum = [&](int j, int c) {
    if constexpr (KS == 1) return acc[j][c];
    acc_t s = red[((w0 * RT + j) * CT + c) * kWave + lane];
#pragma unroll
    for (int w = 1; w < KS; ++w) s += red[(((w0 + w) * RT + j) * CT + c) * kWave + lane];
    return s;
  };
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int r = route[c];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if ((j * CT + c) % KS != wk) continue;
      const int nn = n0 + 16 * j + 4 * g;
      if (r < 0 || nn >= n_out) continue;
      const acc_t sg = sum(j, c);
      const acc_t su = GATE ? sum(NJ + j, c) : sg;
      const float xs = QX ? s_xs[16 * c + r16] : INT8 ? a.xs[x_row(r)] : 1.0f;
      const float wt = a.row_weight && r < a.rows ? a.row_weight[r] : 1.0f;
      const RowFactor rf = row_factor(xs);
      float o[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int f = min(nn + v, n_out - 1);
        float y = static_cast<float>(sg[v]);
        if (INT8) y = scaled(y, rf, ws[f]);
        if constexpr (GATE) {
          float u = static_cast<float>(su[v]);
          if (INT8) u = scaled(u, rf, ws[n_out + f]);
          clamp_numbers(limit, y, u);
          y = act_apply(a.act, y) * u;
        }
        o[v] = y * wt;
      }
      const size_t at = static_cast<size_t>(r) * n_out + nn;
      if (n_out % 4 == 0) {
        if (a.out_f32) *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + at) = f32x4{o[0], o[1], o[2], o[3]};
        else
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + at) =
              uint2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          if (nn + v >= n_out) break;
          if (a.out_f32) static_cast<float*>(a.y)[at + v] = o[v];
          else static_cast<uint16_t*>(a.y)[at + v] = f32_to_bf16(o[v]);
        }
      }
    }
  }
}

template <bool INT8, bool GATE, bool QX, int RT, int CT, int S, int KS, int W>
hipError_t launch_one(const MatmulArgs& a, hipStream_t stream) {
  constexpr auto kernel = matmul_stream_kernel<INT8, GATE, QX, RT, CT, S, KS, W>;
  const int n_out = GATE ? a.N / 2 : a.N, feats = 16 * (GATE ? RT / 2 : RT) * (W / KS);
  const long long blocks =
      std::min<long long>(a.rows, a.rows / (16 * CT) + a.E) + (a.extra + 16 * CT - 1) / (16 * CT);
  hipLaunchKernelGGL(kernel, dim3((n_out + feats - 1) / feats, static_cast<unsigned>(blocks)),
                     dim3(W * kWave), 0, stream, a);
  return hipGetLastError();
}

// NJ: 16-feature tiles of a wave (with gate and up rows, twice as many weight tiles)
template <int NJ, int CT, int S, int KS, int W>
hipError_t launch_stream(const MatmulArgs& a, hipStream_t stream) {
  if (a.int8)
    return a.act < 0 ? launch_one<true, false, false, NJ, CT, S, KS, W>(a, stream)
                     : launch_one<true, true, false, 2 * NJ, CT, S, KS, W>(a, stream);
  return a.act < 0 ? launch_one<false, false, false, NJ, CT, S, KS, W>(a, stream)
                   : launch_one<false, true, false, 2 * NJ, CT, S, KS, W>(a, stream);
}

}  // namespace

hipError_t launch_matmul_stream(const MatmulArgs& a, StreamShape shape, hipStream_t stream) {
  if (a.quantise && a.act < 0)
    return shape == kStreamWhole ? launch_one<true, false, true, 1, 1, 3, 1, 4>(a, stream)
                                 : launch_one<true, false, true, 1, 1, 3, 4, 4>(a, stream);
  if (a.quantise)
    return shape == kStreamWhole ? launch_one<true, true, true, 2, 1, 3, 1, 4>(a, stream)
                                 : launch_one<true, true, true, 2, 1, 3, 4, 4>(a, stream);
  switch (shape) {
    case kStreamSplit: return launch_stream<1, 1, 3, 4, 4>(a, stream);
    case kStreamWhole: return launch_stream<1, 1, 3, 1, 4>(a, stream);
    default: return launch_stream<2, 2, 2, 4, 4>(a, stream);
  }
}

}  // namespace ftmoe
