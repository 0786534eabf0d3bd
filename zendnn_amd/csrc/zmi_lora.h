// What the kernels of k_lora.hip and k_lora_expand.hip share.
#pragma once
#include "zmi_device.h"
#include "zmi_launch.h"

#define LORA_WAVES 4
#define LORA_SMALL_T 64     // rows up to which wavefronts plan for themselves

// How a call goes out (k_lora.hip: lora_shape)
struct LoraShape {
  bool small;
  bool dma;            // rows of x and A and their addresses are 16-byte multiples
  int rt;              // 16-row groups of a shrink tile
  int nt;              // rank tiles of a shrink unit
  int ny;              // units over the rank tiles
  int ks;              // small: K slices
  int grid;            // planned: shrink workgroups
  int64_t tiles;       // tiles there can be
  int64_t groups;      // 16-row groups there can be
  int kt;              // 32-rank blocks an expand wavefront holds
  int nj;              // its column tiles of 16
  int64_t col_blocks;
  int64_t runs;        // planned: expand workgroups down the rows
  int terms;
};

hipError_t lora_launch_expand(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream);

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 16 / 8 bytes at any 2-byte aligned address (global memory takes unaligned vector accesses on this device)
__device__ __forceinline__ u32x4 load16(const void *p) { u32x4 v; __builtin_memcpy(&v, p, 16); return v; }
__device__ __forceinline__ void store16(void *p, u32x4 v) { __builtin_memcpy(p, &v, 16); }

// the first n (< 8) of eight 16-bit elements, zeros behind them
__device__ __forceinline__ u32x4 load16_head(const uint16_t *p, int n) {
  u32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) v[i / 2] |= (uint32_t)p[i] << (16 * (i % 2));
  return v;
}

__device__ __forceinline__ int lora_rank(const ZmiLora &p, int slot) {
  if (!p.ranks) return p.rank;
  const int r = p.ranks[slot];
  return r < 0 ? 0 : r > p.rank ? p.rank : r;
}

struct Tile {
  int slot;   // n_slots: rows without an adapter
  int n;      // rows of the tile
  int group;  // planned: number of its first 16-row group
  int row;    // unplanned: lane l's row is that of position l % 16
};

// Tile `want` of up to 64 rows: slots in the order of their first rows, 16 rows each.
__device__ __forceinline__ bool lora_find_tile(const ZmiLora &p, int want, Tile &t) {
  const int lane = threadIdx.x % 64;
  int id = -1;
  if (lane < p.T) {
    id = p.slot_ids[lane];
    if ((unsigned)id >= (unsigned)p.n_slots) id = p.n_slots;
  }
  uint64_t left = __ballot(lane < p.T);
  int seen = 0;
  while (left) {
    const int slot = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t m = __ballot(id == slot);
    const int c = __popcll(m), tiles = (c + 15) / 16;
    if (want < seen + tiles) {
      const int sub = want - seen;
      const int pos = __popcll(m & ((1ull << lane) - 1));
      const bool in = id == slot && pos / 16 == sub;
      // (lanes outside push to the upper lanes, which nobody reads)
      const int got = __builtin_amdgcn_ds_permute(4 * (in ? pos % 16 : 63), lane);
      t.slot = slot;
      t.n = c - 16 * sub < 16 ? c - 16 * sub : 16;
      t.group = 0;
      t.row = __shfl(got, lane % 16, 64);
      return true;
    }
    seen += tiles;
    left &= ~m;
  }
  return false;
}

template <bool F16>
__device__ __forceinline__ f32x4 mma_x(u32x4 a, u32x4 b, f32x4 c) {
  if (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// v as TERMS bf16 terms, largest first; what is left of a value that is not finite is zero
template <int TERMS, int N>
__device__ __forceinline__ void split(const float (&v)[N], __bf16 (&t)[TERMS][N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float rest = v[i];
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
      t[k][i] = (__bf16)rest;
      const float hi = (float)t[k][i];
      rest = __builtin_fabsf(hi) < __builtin_inff() ? rest - hi : 0.0f;
    }
  }
}

template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// (LDS reads of the step before are over when a wavefront arrives: what follows may write where it read)
__device__ __forceinline__ void group_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace
