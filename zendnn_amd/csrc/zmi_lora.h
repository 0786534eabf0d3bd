// What the kernels of k_lora.hip and k_lora_expand.hip share.
#pragma once
#include "zmi_device.h"
#include "zmi_launch.h"

#define LORA_WAVES 4
#define LORA_TERMS 3   // bf16 terms that h is held in: 24 bits, all that f32 has
// Rows up to which wavefronts plan for themselves: any slots, or few slots and ranks (a round of the search per distinct slot,
// and a tile's 16 rows read all of their slot's A and B)
#define LORA_SMALL_T 128
#define LORA_SMALL_MOST 512
#define LORA_SMALL_SLOTS 16
#define LORA_SMALL_RANKS 64

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
};

hipError_t lora_launch_expand(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream);

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 16 bytes at any 2-byte aligned address (global memory takes unaligned vector accesses on this device)
__device__ __forceinline__ u32x4 load16(const void *p) { u32x4 v; __builtin_memcpy(&v, p, 16); return v; }

// the first n (1 .. 7) of eight 16-bit elements, zeros behind them: four, two and one, as n has them
__device__ __forceinline__ u32x4 load16_head(const uint16_t *p, int n) {
  uint32_t four[2] = {0, 0}, two = 0, one = 0;
  if (n & 4) __builtin_memcpy(four, p, 8);
  if (n & 2) __builtin_memcpy(&two, p + (n & 4), 4);
  if (n & 1) one = p[n & 6];
  const uint32_t lo = n & 2 ? two : one, hi = n & 2 ? one : 0;
  return n & 4 ? u32x4{four[0], four[1], lo, hi} : u32x4{lo, hi, 0, 0};
}

__device__ __forceinline__ int lora_rank(const ZmiLora &p, int slot) {
  if (!p.ranks) return p.rank;
  const int r = p.ranks[slot];
  return r < 0 ? 0 : r > p.rank ? p.rank : r;
}

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int lora_dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
// sum over the lanes up to this one
__device__ __forceinline__ int lora_running_sum(int v) {
  v += lora_dpp<0x111>(v);        // row_shr 1, 2, 4, 8: inside rows of 16
  v += lora_dpp<0x112>(v);
  v += lora_dpp<0x114>(v);
  v += lora_dpp<0x118>(v);
  v += lora_dpp<0x142, 0xa>(v);   // row_bcast 15 into rows 1 and 3
  v += lora_dpp<0x143, 0xc>(v);   // row_bcast 31 into rows 2 and 3
  return v;
}

struct Tile {
  int slot;   // n_slots: rows without an adapter
  int n;      // rows of the tile
  int group;  // planned: number of its first 16-row group
  int row;    // unplanned: lane l's row is that of position l % 16
};

// The tile of rows `sub` * 16 .. +15 among the c rows of a slot, whose lanes (row 64 h + lane) are m[h].
template <int H>
__device__ __forceinline__ void lora_tile_rows(const uint64_t (&m)[H], int c, int slot, int sub, Tile &t) {
  const int lane = threadIdx.x % 64;
  int got = 0, before = 0;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int pos = before + __popcll(m[h] & ((1ull << lane) - 1));
    const bool in = ((m[h] >> lane) & 1) && pos / 16 == sub;
    // (lanes outside push to the upper lanes, which nobody reads; a lane that nothing is pushed to gets 0)
    const int row = __builtin_amdgcn_ds_permute(4 * (in ? pos % 16 : 16 + lane % 48), in ? lane + 64 * h + 1 : 0);
    got = row > got ? row : got;
    before += __popcll(m[h]);
  }
  t.slot = slot;
  t.n = c - 16 * sub < 16 ? c - 16 * sub : 16;
  t.group = 0;
  t.row = __shfl(got, lane % 16, 64) - 1;
}

// Tile `want` of up to 64 H rows: slots in the order of their first rows, 16 rows each; a round per distinct id.
template <int H>
__device__ __forceinline__ bool lora_find_tile_few_slots(const ZmiLora &p, int want, Tile &t) {
  const int lane = threadIdx.x % 64, parts = (p.T + 63) / 64;
  int id[H];
#pragma unroll
  for (int h = 0; h < H; ++h) id[h] = h < parts ? p.slot_ids[lane + 64 * h < p.T ? lane + 64 * h : p.T - 1] : 0;
  uint64_t left[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    if ((unsigned)id[h] >= (unsigned)p.n_slots) id[h] = p.n_slots;
    left[h] = __ballot(lane + 64 * h < p.T);
  }
  int seen = 0;
  for (;;) {
    int slot = -1;
#pragma unroll
    for (int h = H - 1; h >= 0; --h)
      if (left[h]) slot = __builtin_amdgcn_readlane(id[h], __builtin_ctzll(left[h]));
    if (slot < 0) return false;
    uint64_t m[H];
    int c = 0;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      m[h] = h < parts ? __ballot(id[h] == slot) & left[h] : 0;
      c += __popcll(m[h]);
    }
    const int tiles = (c + 15) / 16;
    if (want < seen + tiles) {
      lora_tile_rows<H>(m, c, slot, want - seen, t);
      return true;
    }
    seen += tiles;
#pragma unroll
    for (int h = 0; h < H; ++h) left[h] &= ~m[h];
  }
}

// The same of up to 128 rows, without the rounds: every lane finds the rows that share its slot bit by bit, the first of
// them counts their tiles, and a running sum over the lanes says whose tile it is.
__device__ __forceinline__ bool lora_find_tile_few_rows(const ZmiLora &p, int want, Tile &t) {
  const int lane = threadIdx.x % 64;
  const uint64_t below = (1ull << lane) - 1;
  int id[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) id[h] = p.slot_ids[lane + 64 * h < p.T ? lane + 64 * h : p.T - 1];
  uint64_t m[2][2];   // [this lane's row of half h][rows of half g that share its slot]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if ((unsigned)id[h] >= (unsigned)p.n_slots) id[h] = p.n_slots;
#pragma unroll
    for (int g = 0; g < 2; ++g) m[h][g] = __ballot(lane + 64 * g < p.T);
  }
  const int bits = 32 - __builtin_clz(p.n_slots);
  for (int b = 0; b < bits; ++b) {
    const uint64_t one[2] = {__ballot((id[0] >> b) & 1), __ballot((id[1] >> b) & 1)};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < 2; ++g) m[h][g] &= (id[h] >> b) & 1 ? one[g] : ~one[g];
  }
  int c[2], tiles[2], end[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    c[h] = __popcll(m[h][0]) + __popcll(m[h][1]);
    const bool first = lane + 64 * h < p.T && !(m[h][h] & below) && (h == 0 || !m[h][0]);
    tiles[h] = first ? (c[h] + 15) / 16 : 0;
    end[h] = lora_running_sum(tiles[h]);
  }
  end[1] += __builtin_amdgcn_readlane(end[0], 63);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint64_t hit = __ballot(want < end[h] && want >= end[h] - tiles[h]);
    if (!hit) continue;
    const int at = __builtin_ctzll(hit);
    uint64_t mine[2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
      mine[g] = (uint32_t)__builtin_amdgcn_readlane((int)m[h][g], at) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(m[h][g] >> 32), at) << 32;
    lora_tile_rows<2>(mine, __builtin_amdgcn_readlane(c[h], at), __builtin_amdgcn_readlane(id[h], at),
                      want - __builtin_amdgcn_readlane(end[h] - tiles[h], at), t);
    return true;
  }
  return false;
}

__device__ __forceinline__ bool lora_find_tile(const ZmiLora &p, int want, Tile &t) {
  if (p.T > 128) return lora_find_tile_few_slots<LORA_SMALL_MOST / 64>(p, want, t);
  return p.n_slots <= LORA_SMALL_SLOTS ? lora_find_tile_few_slots<2>(p, want, t) : lora_find_tile_few_rows(p, want, t);
}

template <bool F16>
__device__ __forceinline__ f32x4 mma_x(u32x4 a, u32x4 b, f32x4 c) {
  if (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// v as TERMS bf16 terms, largest first.  A finite value's terms are finite (bf16's largest stands for what would round beyond
// it, the next term holds the rest); what is left of a value that is not finite is zero.
template <int TERMS, int N>
__device__ __forceinline__ void split(const float (&v)[N], __bf16 (&t)[TERMS][N]) {
  const float most = 0x1.fep127f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float rest = v[i];
    const bool finite = __builtin_fabsf(rest) < __builtin_inff();
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
      t[k][i] = (__bf16)(k == 0 && finite ? __builtin_amdgcn_fmed3f(rest, -most, most) : rest);
      rest = finite ? rest - (float)t[k][i] : 0.0f;
    }
  }
}

template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// (LDS reads of the step before are over when a wavefront arrives: what follows may write where it read)
__device__ __forceinline__ void group_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace
