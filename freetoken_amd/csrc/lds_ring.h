// Pieces of the GEMMs whose operands come through a ring of LDS stages by direct
// global -> LDS copies (prefill.hip, matmul_stream.hip, matmul_tile.hip): explicit waits and barriers, the
// copies, the LDS swizzle and the tiles' order.
#pragma once

#include "ftmoe_common.h"

namespace ftmoe {

constexpr int kXcds = 8;

// Position of workgroup b of n in an order that gives every XCD (workgroup b runs
// on XCD b % 8) a contiguous range.
__device__ __forceinline__ int xcd_major(int b, int n) {
  const int per = n / kXcds, rem = n % kXcds;
  const int x = b % kXcds, i = b / kXcds;
  return x * per + min(x, rem) + i;
}

struct MNTile {
  int m, ntile;
};

// (M block, N tile) of position `local` in a group of nb M blocks x ntiles:
// chunks of kQChunk M blocks, each chunk sweeping all N tiles.
// (Returned by value, and from one call per mapping: results written through
// references from two calls lived in scratch memory, whose loads wait for the
// copies in flight.)
template <int kQChunk>
__device__ __forceinline__ MNTile chunked(int local, int nb, int ntiles) {
  const int full = nb / kQChunk, rem = nb - full * kQChunk;
  const int span = kQChunk * ntiles;
  const bool whole = local < full * span;
  const int c = whole ? local / span : full;
  const int w = local - c * span, in = whole ? kQChunk : rem;
  const int ntile = w / in;
  return {c * kQChunk + (w - ntile * in), ntile};
}

// Lane index as an asm result: the compiler can neither hoist nor merge it,
// so per-tile set-up code recomputes its lane-derived values instead of keeping
// them live (or spilled) across the K loop.
__device__ __forceinline__ int fresh_lane() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}

// s_barrier without the memory fence of __syncthreads (which would wait for
// every copy in flight); the clobber keeps the compiler from moving LDS
// accesses across it.
__device__ __forceinline__ void bare_barrier() { asm volatile("s_barrier" ::: "memory"); }

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ void wait_lgkm0() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// LDS-DMA copies through a buffer descriptor: each lane's 16 (4) bytes at lane
// offset voff plus the wave-uniform soff land at dst + lane * 16 (4), dst
// wave-uniform; a lane offset at or past the descriptor's range reads zeros
// without memory traffic.
__device__ __forceinline__ void lds_buf16(__amdgpu_buffer_rsrc_t r, uint8_t* dst, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, soff, 0, 0);
}
// (nontemporal: for weights that are read once)
__device__ __forceinline__ void lds_buf16_nt(__amdgpu_buffer_rsrc_t r, uint8_t* dst, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, soff, 0, 2);
}
__device__ __forceinline__ void lds_buf4(__amdgpu_buffer_rsrc_t r, uint8_t* dst, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 4, voff, soff, 0, 0);
}

// 128-byte lines read as chunk pairs (2g, 2g + 1): chunk c of line l at c ^ swz_pair(l)
// is free of bank conflicts (measured; prefill.hip).
__device__ __forceinline__ int swz_pair(int line) { return ((line & 3) << 1) | ((line >> 2) & 1); }

// Position of a running count in a ring of N.  (Unsigned: the signed remainders
// were a dozen more scalar operations at the head of every step, before its
// first LDS read; FP8 calls gained 0.3-0.8%.)
template <int N>
__device__ __forceinline__ int ring(int i) {
  return static_cast<int>(static_cast<unsigned>(i) % N);
}

// Empty asm that keeps the value's update at this point of the instruction
// stream (no code is emitted).
template <typename T>
__device__ __forceinline__ void pin(T& v) {
  asm volatile("" : "+v"(v));
}

__device__ __forceinline__ uint64_t uniform_u64(uint64_t v) { return readlane_u64(v, 0); }

}  // namespace ftmoe
