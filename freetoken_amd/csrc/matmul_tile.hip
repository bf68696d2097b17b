// Tiled form of the matrix products of MatmulArgs, for many rows per group.
//
// A workgroup of WR x WC waves computes ROWS = 32 RT WR weight rows x COLS =
// 32 CT WC rows of x of one group, a wave RT x CT MFMA tiles of 32 x 32.  A K step is one
// 128-byte line of every row (128 int8 or 64 bf16 values), copied global -> LDS by
// the LDS-DMA form of the buffer loads into a ring of S stages: the copies of the
// next S - 1 steps are in flight while a step computes, and the ring runs on from
// tile to tile (the workgroups are persistent, one walk over the tiles each).
//
// int8 sums stay int32 to the end (exact), bf16 ones float32; a result is the sum
// times its channel's and its row's scale (and weight), rounded to bf16 once; the
// factors are multiplied as in the streaming form (matmul.h: scaled).
//
// Two waves per SIMD and 32 x 32 MFMAs: one wave with 16 x 16 ones issues 2930 int8
// T/s at most, two 4000, one with 32 x 32 ones 4100 (8192 x 4096 x 7168: 227 us with 4
// waves of 16 x 16, 204 with 8 of 32 x 32 = 2360 T/s).  Tiles of 256 x 256 hold two
// stages, 256 x 128 three; 128 x 64 leave room for a second workgroup on the CU, which
// multiplies while the first one stores.
//
// What bounds it: 65536 rows over 128 experts, N 2048, K 768 (256 x 128) take 173 us.  Timed by
// parts when they took 201 (before bf16 results passed the caches): the MFMAs and LDS reads alone 93,
// the copies alone 103 (66 where every tile reads the same lines: they wait for lines that miss L2, two
// steps ahead fill the LDS), and the results overlap with neither.  Float32 results go out in pieces
// of 32 bytes: inside an expert layer 270 to 292 us, bf16 ones 200 to 234.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "lds_ring.h"
#include "matmul.h"

namespace ftmoe {

namespace {

// Chunk c (16 bytes) of line l lies at c ^ swz(l): free of bank conflicts for reads
// of one chunk of 32 lines (2% of the LDS cycles; with the line's low three bits, or
// swz_pair, 49%: rocprofv3 SQ_LDS_BANK_CONFLICT over SQ_LDS_IDX_ACTIVE).
__device__ __forceinline__ int swz(int line) { return (line >> 1) & 7; }

struct MTile {
  int e, begin, end, ntile;  // group, its rows [begin, end) of this tile in the grouped order, weight tile
};

template <int ROWS, int COLS, int WAVES, int S>
struct TileLds {
  static constexpr int kA = ROWS * 128, kB = COLS * 128, kStage = kA + kB;
  static constexpr int kACopies = ROWS / 8 / WAVES, kBCopies = COLS / 8 / WAVES;  // 1 KB copies per wave and step
  static constexpr int kPerStep = kACopies + kBCopies;
  static constexpr int kRing = S * kStage;
  // per tile parity: the tile's rows of y, their scales and weights, and the channel scales
  static constexpr int kSide = (3 * COLS + ROWS) * 4;
  static constexpr int kFixed = kRing + 2 * kSide;
  static int bytes(int groups) { return kFixed + 2 * (groups + 1) * static_cast<int>(sizeof(int)); }
};

template <bool INT8, bool GATE, int WR, int WC, int RT, int CT, int S, bool NT>
__global__ void __launch_bounds__(kWave* WR* WC) matmul_tile_kernel(MatmulArgs a) {
  using acc_t = typename Acc32<INT8>::type;
  constexpr int ROWS = 32 * RT * WR, COLS = 32 * CT * WC;
  using L = TileLds<ROWS, COLS, WR * WC, S>;
  constexpr int D = S - 1;  // prefetch distance in K steps
  constexpr int kChunk = 2048 / COLS;  // M blocks that sweep the N tiles together
  extern __shared__ __attribute__((aligned(16))) uint8_t t_lds[];
  const int E = a.E, G = group_count(a);
  int* const s_blk = reinterpret_cast<int*>(t_lds + L::kFixed);  // [G + 1] first block of every group
  int* const s_beg = s_blk + G + 1;                              // [E + 1] first row of every group, the last one's end
  const auto s_route = [&](int b) { return reinterpret_cast<int*>(t_lds + L::kRing + b * L::kSide); };
  const auto s_xs = [&](int b) { return reinterpret_cast<float*>(t_lds + L::kRing + b * L::kSide) + COLS; };
  const auto s_rw = [&](int b) { return reinterpret_cast<float*>(t_lds + L::kRing + b * L::kSide) + 2 * COLS; };
  const auto s_ws = [&](int b) { return reinterpret_cast<float*>(t_lds + L::kRing + b * L::kSide) + 3 * COLS; };

  const int tid = threadIdx.x, lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wr = wave / WC, wc = wave % WC;
  const int r32 = lane & 31, half = lane >> 5;
  const int n_out = GATE ? a.N / 2 : a.N;
  constexpr int kOutRows = GATE ? ROWS / 2 : ROWS;  // output features of a tile
  const int ntiles = (n_out + kOutRows - 1) / kOutRows;
  const uint32_t rb = static_cast<uint32_t>(a.K) * (INT8 ? 1 : 2);  // bytes of a row
  const int nkb = static_cast<int>((rb + 127) / 128);

  // ---- blocks of every group
  if (wave == 0) {
    int done = 0;
    for (int e0 = 0; e0 <= G; e0 += kWave) {
      int lo = 0, hi = 0;
      if (e0 + lane < G) group_range(a, e0 + lane, lo, hi);
      const int nb = (hi - lo + COLS - 1) / COLS;
      int sum = nb;
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) {
        const int y = __shfl_up(sum, off, kWave);
        if (lane >= off) sum += y;
      }
      if (e0 + lane <= G) s_blk[e0 + lane] = done + sum - nb;
      if (e0 + lane < E) s_beg[e0 + lane] = lo;
      done += __shfl(sum, kWave - 1, kWave);
    }
    if (lane == 0) s_beg[E] = a.offsets ? min(max(a.offsets[E], 0), a.rows) : a.rows;
  }
  __syncthreads();

  const auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const int total = uniform(s_blk[G]) * ntiles;
  auto map_tile = [&](int b, MTile& t) -> bool {
    if (b >= total) return false;
    const int wg = xcd_major(b, total);
    int owner = 0;
    if (G > 1) {  // the largest group whose first tile is <= wg
      owner = -1;
      const int l = fresh_lane();
      for (int e0 = 0; e0 < G; e0 += kWave)
        owner += __popcll(__ballot(e0 + l < G && s_blk[min(e0 + l, G)] * ntiles <= wg));
      owner = uniform(owner);
    }
    const int b0 = uniform(s_blk[owner]), nb = uniform(s_blk[owner + 1]) - b0;
    const MNTile mn = chunked<kChunk>(wg - b0 * ntiles, nb, ntiles);
    const bool extra = owner == E;
    const int beg = extra ? a.rows : uniform(s_beg[owner]);
    const int end = extra ? a.rows + a.extra : max(beg, uniform(s_beg[min(owner, E - 1) + 1]));
    t.e = owner;
    t.begin = beg + mn.m * COLS;
    t.end = min(end, t.begin + COLS);
    t.ntile = mn.ntile;
    return true;
  };

  // weight row of tile row R, relative to the tile's first
  auto trow_rel = [&](int R) -> int {
    const int q = R / (32 * RT), j = R / 32 % RT;
    if (GATE) return (j < RT / 2 ? 0 : n_out) + 16 * RT * q + 32 * (j % (RT / 2)) + (R & 31);
    return R;
  };

  // ---- sources of the copies.  A copy fills 8 lines; a lane's chunk of a line goes by the copy's parity.
  const int q16[2] = {16 * ((lane & 7) ^ swz(lane >> 3)), 16 * ((lane & 7) ^ swz(8 + (lane >> 3)))};
  uint32_t last_dead[2];  // the last step's chunks past the rows' end
  uint32_t avoff[L::kACopies], xvoff[L::kBCopies];
#pragma unroll
  for (int p = 0; p < 2; ++p) last_dead[p] = static_cast<uint32_t>(nkb - 1) * 128 + q16[p] >= rb ? kOutOfRange : 0u;
#pragma unroll
  for (int c = 0; c < L::kACopies; ++c)
    avoff[c] = static_cast<uint32_t>(trow_rel(8 * (wave * L::kACopies + c) + (lane >> 3))) * rb + q16[c & 1];
  const __amdgpu_buffer_rsrc_t rsrc_x = make_rsrc(a.x, static_cast<uint32_t>(a.x_rows) * rb);
  const __amdgpu_buffer_rsrc_t rsrc_xs = make_rsrc(a.xs, static_cast<uint32_t>(a.x_rows) * 4);
  uint64_t wbase = 0;
  uint32_t wrange = 0;
  auto n0_of = [&](const MTile& t) { return t.ntile * kOutRows; };
  const uint32_t magic = a.top_k == 1 ? 0u : static_cast<uint32_t>(((uint64_t{1} << 32) + a.top_k - 1) / a.top_k);
  auto x_row = [&](int r) -> uint32_t {
    uint32_t q = static_cast<uint32_t>(r);
    if (r >= a.rows) {
      q += a.extra_x - a.rows;
    } else if (magic) {
      q = __umulhi(q, magic);
      // the rounded-up reciprocal gives at most one too many
      q -= q * static_cast<uint32_t>(a.top_k) > static_cast<uint32_t>(r) ? 1u : 0u;
    }
    return q;
  };
  // row of y in column col of tile t, or -1
  auto route_of = [&](const MTile& t, int b, int col) -> int {
    const int r = s_route(b)[col];
    return t.begin + col < t.end && static_cast<uint32_t>(r) < static_cast<uint32_t>(a.rows + a.extra) ? r : -1;
  };
  auto fetch_routes = [&](const MTile& t, int b) {  // wave w: columns [64 w, 64 w + 64)
    if (64 * wave >= COLS) return;
    const int ln = fresh_lane();
    if (a.order && t.e != E)
      lds_buf4(make_rsrc(a.order + t.begin, static_cast<uint32_t>(t.end - t.begin) * 4),
               reinterpret_cast<uint8_t*>(s_route(b) + 64 * wave), (64 * wave + ln) * 4, 0);
    else
      s_route(b)[64 * wave + ln] = t.begin + 64 * wave + ln;
  };
  auto setup = [&](const MTile& t, int b) {
    const int n0 = n0_of(t);
    const bool extra = t.e == E;
    const uint64_t first = (extra ? 0 : static_cast<uint64_t>(t.e) * static_cast<uint32_t>(a.N)) + static_cast<uint32_t>(n0);
    wbase = uniform_u64(reinterpret_cast<uint64_t>(extra ? a.extra_w : a.w) + first * rb);
    wrange = uniform(static_cast<int>(static_cast<uint32_t>(GATE ? a.N - n0 : min(a.N - n0, ROWS)) * rb));
    const int ln = fresh_lane();
#pragma unroll
    for (int c = 0; c < L::kBCopies; ++c) {
      const int r = route_of(t, b, 8 * (wave * L::kBCopies + c) + (ln >> 3));
      xvoff[c] = r < 0 ? kOutOfRange : x_row(r) * rb + 16 * ((ln & 7) ^ swz(8 * (c & 1) + (ln >> 3)));
    }
    if (64 * wave < COLS) {
      const int r = route_of(t, b, 64 * wave + ln);
      if (INT8)
        lds_buf4(rsrc_xs, reinterpret_cast<uint8_t*>(s_xs(b) + 64 * wave), r < 0 ? kOutOfRange : x_row(r) * 4, 0);
      if (a.row_weight)  // (rows < 2^31: 64-bit addresses through the descriptor's base would not reach past 2 GiB)
        s_rw(b)[64 * wave + ln] = r < 0 ? 0.f : r < a.rows ? a.row_weight[r] : 1.0f;
    }
    if (INT8 && 64 * wave < ROWS) {
      const uint64_t ws = uniform_u64(reinterpret_cast<uint64_t>(extra ? a.extra_ws : a.ws) + first * 4);
      // (N below 2^27 with gate and up rows: check_product)
      lds_buf4(make_rsrc(reinterpret_cast<const void*>(ws), uniform((GATE ? a.N - n0 : min(a.N - n0, ROWS)) * 4)),
               reinterpret_cast<uint8_t*>(s_ws(b) + 64 * wave), static_cast<uint32_t>(trow_rel(64 * wave + ln)) * 4, 0);
    }
  };

  auto issue_piece = [&](int q, int kb, int stg) {
    uint8_t* st = t_lds + stg * L::kStage;
    const uint32_t dead = kb == nkb - 1 ? last_dead[(q < L::kACopies ? q : q - L::kACopies) & 1] : 0u;
    if (q < L::kACopies) {
      const auto copy = NT ? lds_buf16_nt : lds_buf16;
      copy(make_rsrc(reinterpret_cast<const void*>(wbase), wrange), st + (wave * L::kACopies + q) * 1024,
           avoff[q] | dead, static_cast<uint32_t>(kb) * 128);
    } else {
      const int c = q - L::kACopies;
      lds_buf16(rsrc_x, st + L::kA + (wave * L::kBCopies + c) * 1024, xvoff[c] | dead, static_cast<uint32_t>(kb) * 128);
    }
  };
  auto issue = [&](int kb, int stg) {
#pragma unroll
    for (int q = 0; q < L::kPerStep; ++q) issue_piece(q, kb, stg);
  };

  acc_t acc[RT][CT];

  // One K step from stage stg; with ikb >= 0 the copies of step ikb into stage
  // istg are issued between the column tiles.
  constexpr int kSpread = S == 2 ? 2 : 4;  // of the step's four parts
  constexpr int kPer = (L::kPerStep + kSpread - 1) / kSpread;
  auto compute = [&](int stg, int ikb, int istg) {
    const uint8_t* st = t_lds + stg * L::kStage;
    const uint8_t* const ws = st + (32 * RT * wr + r32) * 128;
    const uint8_t* const xs = st + L::kA + (32 * CT * wc + r32) * 128;
    u32x4 wf[2][RT], xf[2][CT];
    auto read = [&](int s) {  // 32 bytes of K: chunks 2s and 2s + 1
      const int at = ((2 * s + half) ^ swz(r32)) * 16;
#pragma unroll
      for (int i = 0; i < CT; ++i) xf[s & 1][i] = *reinterpret_cast<const u32x4*>(xs + at + 4096 * i);
#pragma unroll
      for (int j = 0; j < RT; ++j) wf[s & 1][j] = *reinterpret_cast<const u32x4*>(ws + at + 4096 * j);
    };
    read(0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s + 1 < 4) read(s + 1);
      __builtin_amdgcn_sched_barrier(0);
      if (ikb >= 0) {
#pragma unroll
        for (int q = kPer * s; q < kPer * s + kPer; ++q)
          if (q < L::kPerStep) issue_piece(q, ikb, istg);
      }
#pragma unroll
      for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[j][i] = mma32<INT8>(wf[s & 1][j], xf[s & 1][i], acc[j][i]);
    }
  };

  // ---- epilogue: a lane holds features 32j + 8q + 4 half + [0, 4) of column
  // 32i + r32 of its wave.  bf16 results are staged in LDS (stg, which no copy
  // targets before the next tile's K loop; every wave in its own part) and stored
  // as 16-byte pieces of contiguous rows.
  // plain: the results are bf16, an activation silu without a limit (chosen once a tile, not once a value: an expert
  // layer of 65536 rows, gate and up of N 1536, K 2048, 692 us in all, else 727).
  auto epilogue = [&](const MTile& t, int b, uint8_t* stg, auto plain) {
    const bool out_f32 = !plain.value && a.out_f32;
    constexpr int NJ = GATE ? RT / 2 : RT;
    constexpr int RB = 64 * NJ;          // bytes of a row of y that a wave holds
    constexpr int NC = 4 * NJ;           // 16-byte chunks of it
    constexpr int kRowsPer = kWave / NC; // rows of y per store instruction
    const int nw = n0_of(t) + 32 * NJ * wr;  // the wave's first output feature
    uint8_t* const mine = stg + wave * (32 * RB);
    static_assert(WR * WC * 32 * RB <= L::kStage, "the staging areas fit a stage");
    const bool whole = n_out % 8 == 0;
    const float limit = t.e == E ? a.extra_limit : a.limit;
    f32x4 ws[RT][4];  // read once for all columns
    if (INT8) {
      const float* const wsp = s_ws(b) + 32 * RT * wr + 4 * half;
#pragma unroll
      for (int j = 0; j < RT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) ws[j][q] = *reinterpret_cast<const f32x4*>(wsp + 32 * j + 8 * q);
    }
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      const int col = 32 * CT * wc + 32 * i + r32;
      const float xs = INT8 ? s_xs(b)[col] : 1.0f;
      const float rw = a.row_weight ? s_rw(b)[col] : 1.0f;
      const RowFactor rf = row_factor(xs);
      const int r = out_f32 ? route_of(t, b, col) : 0;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float o[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float y = static_cast<float>(acc[j][i][4 * q + v]);
            if (INT8) y = scaled(y, rf, ws[j][q][v]);
            if constexpr (GATE) {
              float u = static_cast<float>(acc[RT / 2 + j][i][4 * q + v]);
              if (INT8) u = scaled(u, rf, ws[RT / 2 + j][q][v]);
              if constexpr (plain.value) {
                y = act_apply(ACT_SILU, y) * u;
              } else {
                clamp_numbers(limit, y, u);
                y = act_apply(a.act, y) * u;
              }
            }
            o[v] = y * rw;
          }
          if (!out_f32) {
            const int chunk = (4 * j + q) ^ (r32 & (NC - 1));
            *reinterpret_cast<uint2*>(mine + r32 * RB + chunk * 16 + half * 8) =
                uint2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
          } else if (r >= 0) {
            const int n = nw + 32 * j + 8 * q + 4 * half;
            float* const dst = static_cast<float*>(a.y) + static_cast<size_t>(r) * n_out + n;
            if (whole && n < n_out) {
              *reinterpret_cast<f32x4*>(dst) = f32x4{o[0], o[1], o[2], o[3]};
            } else {
#pragma unroll
              for (int v = 0; v < 4; ++v)
                if (n + v < n_out) dst[v] = o[v];
            }
          }
        }
      if (out_f32) continue;
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
      for (int kk = 0; kk < 32 / kRowsPer; ++kk) {
        const int c = kRowsPer * kk + lane / NC, chunk = lane % NC;
        const u32x4 v = *reinterpret_cast<const u32x4*>(mine + c * RB + ((chunk ^ (c & (NC - 1))) * 16));
        const int row = route_of(t, b, 32 * CT * wc + 32 * i + c);
        const int n = nw + 8 * chunk;
        if (row < 0 || n >= n_out) continue;
        uint16_t* const dst = static_cast<uint16_t*>(a.y) + static_cast<size_t>(row) * n_out + n;
        if (whole && !GATE) {  // written once, past the caches (65536 rows, N 2048, K 768: 190, cached 211)
          __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(dst));
        } else if (whole) {    // (the activations are read again at once)
          *reinterpret_cast<u32x4*>(dst) = v;
        } else {
#pragma unroll
          for (int w = 0; w < 8; ++w)
            if (n + w < n_out) dst[w] = static_cast<uint16_t>(v[w / 2] >> (16 * (w & 1)));
        }
      }
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    }
  };

  // ---- persistent loop (as prefill_qgemm_kernel): the last D steps of a tile
  // issue the next tile's first D, which land while the epilogue runs
  int v = blockIdx.x;
  MTile cur;
  if (!map_tile(v, cur)) return;
  fetch_routes(cur, 0);
  wait_vm<0>();
  __syncthreads();
  setup(cur, 0);
  int buf = 0, g0 = 0;
  bool ahead = false;
  for (;;) {
    if (!ahead) {
#pragma unroll
      for (int d = 0; d < D; ++d)
        if (d < nkb) issue(d, ring<S>(g0 + d));
    }
    MTile nxt;
    const bool has_next = map_tile(v + static_cast<int>(gridDim.x), nxt);
    const bool cross = has_next && nkb > D;
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        acc[j][i] = acc_t{};
        pin(acc[j][i]);
      }
    // step 0 (and all before it) has landed once at most the D - 1 later steps' copies are outstanding
    if (nkb >= D) wait_vm<(D - 1) * L::kPerStep>();
    else wait_vm<0>();
    wait_lgkm0();
    bare_barrier();
    if (has_next) fetch_routes(nxt, buf ^ 1);
    int kb = 0;
    for (; kb < nkb - D; ++kb) {
      compute(ring<S>(g0 + kb), kb + D, ring<S>(g0 + kb + D));
      wait_vm<(D - 1) * L::kPerStep>();
      wait_lgkm0();
      bare_barrier();
    }
    // the next tile's rows were copied before step D's copies: from nkb = 2D on the waits above covered them
    if (has_next && nkb < 2 * D) {
      wait_vm<0>();
      wait_lgkm0();
      bare_barrier();
    }
    if (cross) setup(nxt, buf ^ 1);
    for (; kb < nkb; ++kb) {
      compute(ring<S>(g0 + kb), cross ? kb + D - nkb : -1, ring<S>(g0 + kb + D));
      if (kb + 1 < nkb) {
        if (cross) wait_vm<(D - 1) * L::kPerStep>();
        else wait_vm<0>();
      }
      wait_lgkm0();
      bare_barrier();
    }
    uint8_t* const stg = t_lds + ring<S>(g0 + nkb + D) * L::kStage;
    const float limit = cur.e == E ? a.extra_limit : a.limit;
    if (!a.out_f32 && (!GATE || (a.act == ACT_SILU && !(limit > 0.f)))) epilogue(cur, buf, stg, std::true_type{});
    else epilogue(cur, buf, stg, std::false_type{});
    if (!has_next) break;
    ahead = cross;
    cur = nxt;
    buf ^= 1;
    g0 += nkb;
    v += static_cast<int>(gridDim.x);
    if (!ahead) setup(cur, buf);
  }
}

template <bool INT8, bool GATE, int WR, int WC, int RT, int CT, int S, bool NT>
hipError_t launch_tile(const MatmulArgs& a, hipStream_t stream) {
  constexpr int ROWS = 32 * RT * WR, COLS = 32 * CT * WC;
  constexpr auto kernel = matmul_tile_kernel<INT8, GATE, WR, WC, RT, CT, S, NT>;
  using L = TileLds<ROWS, COLS, WR * WC, S>;
  const int lds = L::bytes(group_count(a));
  // once on every device
  int dev = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err != hipSuccess) return err;
  static std::atomic<uint64_t> ready{0};  // (two threads at once set the same attribute twice)
  if (dev > 63 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
    err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                              160 * 1024);
    if (err != hipSuccess) return err;
    if (dev <= 63) ready.fetch_or(uint64_t{1} << dev, std::memory_order_release);
  }
  const int n_out = GATE ? a.N / 2 : a.N, out_rows = GATE ? ROWS / 2 : ROWS;
  const long long blocks =
      std::min<long long>(a.rows, static_cast<long long>(a.rows) / COLS + a.E) + (a.extra + COLS - 1) / COLS;
  const long long tiles = blocks * ((n_out + out_rows - 1) / out_rows);
  const int per_cu = std::max(1, 160 * 1024 / lds);
  const int wgs = static_cast<int>(std::min<long long>(tiles, 256ll * per_cu));
  hipLaunchKernelGGL(kernel, dim3(wgs), dim3(kWave * WR * WC), lds, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_matmul_tile(const MatmulArgs& a, TileShape shape, bool once, hipStream_t stream) {
#define FTMOE_TILE(...)                                                                          \
  return a.int8 ? (a.act < 0 ? launch_tile<true, false, __VA_ARGS__>(a, stream)                  \
                             : launch_tile<true, true, __VA_ARGS__>(a, stream))                  \
                : (a.act < 0 ? launch_tile<false, false, __VA_ARGS__>(a, stream)                 \
                             : launch_tile<false, true, __VA_ARGS__>(a, stream))
  switch (shape) {
    case kTile256x256: FTMOE_TILE(4, 2, 2, 4, 2, false);
    case kTile256x128:
      if (once) FTMOE_TILE(4, 2, 2, 2, 3, true);
      FTMOE_TILE(4, 2, 2, 2, 3, false);
    default:
      if (once) FTMOE_TILE(2, 2, 2, 1, 3, true);
      FTMOE_TILE(2, 2, 2, 1, 3, false);
  }
#undef FTMOE_TILE
}

}  // namespace ftmoe
