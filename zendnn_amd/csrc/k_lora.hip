// Low-rank adapters of many requests beside a shared projection (gfx950); see zmi_lowoha.h.
//
//   h[t][s, r] = sum_k x[t][k] A[a][s rank + r][k],  dst[t][n] = base[t][n] + scales[a] sum_r h[t][s, r] B_s[a][n][r]
//
// with a = slot_ids[t].  Per byte that has to move (x, dst, base, the used slots' A and B) there are at most `rank`
// multiply-adds, so HBM bounds every size, and latency the small ones.  Rows of one slot are gathered into tiles of
// 16 RT rows, so that a tile reads its slot's A and B once and both products run on the 16 x 16 x 32 MFMA:
//
//   plan    (more than 64 rows) one workgroup sorts the rows by slot and lists the tiles; up to 64 rows every
//           wavefront finds its tile by itself from a ballot per distinct id, and there is no such launch;
//   shrink  h of a tile, K through an LDS ring.  K is cut into slices where the tiles alone do not fill the device;
//   expand  dst.  A wavefront keeps 32 .. 128 columns' B in registers and goes down the rows of its slot.
//
// The MFMA takes 16-bit operands: x, A exactly as they are; h, which is f32, as a sum of bf16 terms (2 terms hold 16
// bits, for f32 destinations 3 hold 24), and f16 B, which the range of h does not allow to meet in f16, as two bf16 terms
// that hold it exactly.  All products are accumulated in f32.
#include "zmi_device.h"
#include "zmi_launch.h"

#include <type_traits>

#define LORA_WAVES 4
#define LORA_SMALL_T 64     // rows up to which wavefronts plan for themselves

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
  int first;  // planned: position of its first row in the sorted order
  int row;    // unplanned: lane l's row is that of position l % 16
  int group;  // planned: number of its first 16-row group in h
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
      t.first = 0;
      t.row = __shfl(got, lane % 16, 64);
      return true;
    }
    seen += tiles;
    left &= ~m;
  }
  return false;
}

__device__ __forceinline__ bool lora_planned_tile(const int32_t *table, int count, int want, Tile &t) {
  if (want >= count) return false;
  const int *e = table + 4 * (int64_t)want;
  t.slot = __builtin_amdgcn_readfirstlane(e[0]);
  t.first = __builtin_amdgcn_readfirstlane(e[1]);
  t.n = __builtin_amdgcn_readfirstlane(e[2]);
  t.group = __builtin_amdgcn_readfirstlane(e[3]);
  t.row = 0;
  return true;
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

extern __shared__ __attribute__((aligned(16))) char lora_smem[];

}  // namespace

// ---------------------------------------------------------------------------------------------------------------
// plan: rows sorted by slot (the order within a slot does not matter: rows are computed independently of each other),
// the shrink launch's tiles of `tile` rows and the expand launch's, of `wide` times as many.
// ---------------------------------------------------------------------------------------------------------------
#define LORA_PLAN_KEEP 8   // ids a thread keeps between the passes

__global__ __launch_bounds__(1024) void zmi_lora_plan_kernel(ZmiLora p, ZmiLoraPlan w, int tile, int wide) {
  __shared__ int count[ZMI_LORA_MAX_SLOTS + 1];
  __shared__ int wave_sums[3][16];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, n = p.n_slots + 1;
  auto slot_of = [&](int t) {
    if (t >= p.T) return -1;
    const int id = p.slot_ids[t];
    return (unsigned)id < (unsigned)p.n_slots ? id : p.n_slots;
  };
  int id[LORA_PLAN_KEEP], pos[LORA_PLAN_KEEP];
#pragma unroll
  for (int i = 0; i < LORA_PLAN_KEEP; ++i) id[i] = slot_of(i * 1024 + tid);
  for (int i = tid; i < n; i += 1024) count[i] = 0;
  for (int i = tid; i < w.n_arrivals; i += 1024) w.arrivals[i] = 0;
  __syncthreads();
  // a row's place among its slot's rows: rows of a wavefront that share a slot take their places with one atomic (the
  // first few distinct slots; neighbouring rows mostly belong to one request)
  auto place = [&](int mine) {
    int at = 0;
    bool open = mine >= 0;
    for (int k = 0; k < 4; ++k) {
      const uint64_t left = __ballot(open);
      if (!left) return at;
      const int first = __builtin_ctzll(left), slot = __builtin_amdgcn_readlane(mine, first);
      const uint64_t same = __ballot(open && mine == slot);
      int base = 0;
      if (lane == first) base = atomicAdd(&count[slot], (int)__popcll(same));
      base = __builtin_amdgcn_readlane(base, first);
      if (open && mine == slot) { at = base + __popcll(same & ((1ull << lane) - 1)); open = false; }
    }
    if (open) at = atomicAdd(&count[mine], 1);
    return at;
  };
#pragma unroll
  for (int i = 0; i < LORA_PLAN_KEEP; ++i)
    if (i * 1024 < p.T) pos[i] = place(id[i]);
  for (int t0 = LORA_PLAN_KEEP * 1024; t0 < p.T; t0 += 1024) {
    const int at = place(slot_of(t0 + tid));
    if (t0 + tid < p.T) w.place[t0 + tid] = at;
  }
  __syncthreads();
  // thread i owns slots [i per, (i + 1) per)
  const int per = (n + 1023) / 1024;
  int sums[3] = {0, 0, 0};   // rows, tiles, wide tiles
  for (int i = tid * per; i < (tid + 1) * per && i < n; ++i) {
    const int c = count[i];
    sums[0] += c;
    sums[1] += (c + tile - 1) / tile;
    sums[2] += (c + tile * wide - 1) / (tile * wide);
  }
  int start[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    int v = sums[k];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(v, d, 64);
      if (lane >= d) v += o;
    }
    if (lane == 63) wave_sums[k][wave] = v;
    start[k] = v - sums[k];
  }
  __syncthreads();
  for (int i = 0; i < wave; ++i)
#pragma unroll
    for (int k = 0; k < 3; ++k) start[k] += wave_sums[k][i];
  if (tid == 1023) {
    w.header[0] = start[1] + sums[1];
    w.header[1] = start[2] + sums[2];
  }
  for (int i = tid * per; i < (tid + 1) * per && i < n; ++i) {
    const int c = count[i], tile0 = start[1];
    for (int j = 0; j < c; j += tile)
      *(int4 *)(w.tiles + 4 * (int64_t)start[1]++) = make_int4(i, start[0] + j, c - j < tile ? c - j : tile, (tile0 + j / tile) * (tile / 16));
    for (int j = 0; j < c; j += tile * wide)
      *(int4 *)(w.wide + 4 * (int64_t)start[2]++) = make_int4(i, start[0] + j, c - j < tile * wide ? c - j : tile * wide, (tile0 + j / tile) * (tile / 16));
    count[i] = start[0];
    start[0] += c;
  }
  __syncthreads();
  // (each thread reads back the places that it wrote itself)
  for (int t = LORA_PLAN_KEEP * 1024 + tid; t < p.T; t += 1024) w.order[count[slot_of(t)] + w.place[t]] = t;
#pragma unroll
  for (int i = 0; i < LORA_PLAN_KEEP; ++i)
    if (id[i] >= 0) w.order[count[id[i]] + pos[i]] = i * 1024 + tid;
}

// ---------------------------------------------------------------------------------------------------------------
// shrink: workgroup (x: tile, y: NT rank tiles of 16, z: K slice).  MFMA rows are ranks, columns the tile's rows: lane
// l holds ranks (l / 16) * 4 .. +3 of row l % 16.  Rank tiles are numbered over the live ones of all slices (an adapter
// of a smaller rank has fewer); ranks and rows beyond the last one repeat it and are dropped.
//
// K goes through an LDS ring of D stages of KS elements: x rows and A rows alike are moved in units of 8 rows x 128
// bytes, one 16-byte piece a lane.  (MFMA operands read from global memory directly put 16 rows under 16 neighbouring
// lanes: every 16 bytes a cache line of its own, and the compute unit's address path, not HBM, sets the pace: 148 us for
// 8192 rows of K = 14336 at rank 128 against 62 us through LDS.)  Piece c of row r stands at slot c ^ (r % 8), which
// spreads the operand reads over the banks.  With rows, strides and addresses of 16-byte multiples the units are moved
// by global -> LDS loads (DMA), D - 1 stages ahead; otherwise through registers, one stage ahead.
// The four wavefronts share a stage as WR x WN x WK over row groups, rank tiles and 64-element blocks of K.
// ---------------------------------------------------------------------------------------------------------------
template <bool F16, int RT, int NT, int KS, int WR, int WN, int D, bool DMA, bool SMALL>
__global__ __launch_bounds__(LORA_WAVES * 64, 2) void zmi_lora_shrink_kernel(ZmiLora p, ZmiLoraPlan w) {
  constexpr int WK = LORA_WAVES / (WR * WN), RW = RT / WR, NW = NT / WN;
  constexpr int BLOCKS = KS / 64;                       // 64-element blocks of a stage
  constexpr int UNITS = (RT + NT) * 2 * BLOCKS;         // 1 KiB each, [block][8 rows]
  constexpr int OPS = (UNITS + LORA_WAVES - 1) / LORA_WAVES;
  constexpr int STAGE = UNITS * 1024;
  static_assert(BLOCKS % WK == 0 && (D - 2) * OPS < 64, "blocks split over wavefronts; the wait counter");
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), g = lane / 16, c16 = lane % 16;
  Tile t;
  if (!(SMALL ? lora_find_tile(p, blockIdx.x, t) : lora_planned_tile(w.tiles, w.header[0], blockIdx.x, t))) return;
  if (t.slot == p.n_slots) return;
  const int rank = lora_rank(p, t.slot), lt = (rank + 15) / 16, live = lt * p.n_slices;
  const int q0 = blockIdx.y * NT;
  if (q0 >= live) return;
  // this lane's pieces of a stage
  const uint16_t *from[OPS];
  uint32_t into[OPS];
#pragma unroll
  for (int i = 0; i < OPS; ++i) {
    int u = wave + i * LORA_WAVES;
    if (u >= UNITS) u = UNITS - 1;                      // (the last unit again: the same bytes to the same place)
    const int block = u / ((RT + NT) * 2), r = u % ((RT + NT) * 2) * 8 + lane / 8, piece = lane % 8 ^ (lane / 8);
    into[i] = u * 1024;
    if (r < RT * 16) {
      const int at = r < t.n ? r : 0;
      const int row = SMALL ? __shfl(t.row, at, 64) : w.order[t.first + at];
      from[i] = (const uint16_t *)p.x + row * p.ldx;
    } else {
      const int q = q0 + (r - RT * 16) / 16 < live ? q0 + (r - RT * 16) / 16 : live - 1, s = q / lt;
      const int k = (q - s * lt) * 16 + r % 16;
      from[i] = (const uint16_t *)p.a + t.slot * p.a_slot + (s * p.rank + (k < rank ? k : rank - 1)) * p.a_ld;
    }
    from[i] += block * 64 + piece * 8;
  }
  const int stages = (p.K + KS - 1) / KS, full = p.K / KS;
  const int s0 = (int)((int64_t)stages * blockIdx.z / gridDim.z), s1 = (int)((int64_t)stages * (blockIdx.z + 1) / gridDim.z);
  f32x4 acc[RW][NW];
#pragma unroll
  for (int i = 0; i < RW; ++i)
#pragma unroll
    for (int j = 0; j < NW; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  const int wr = wave % WR, wn = wave / WR % WN, wk = wave / (WR * WN);
  // where this lane's operands stand in a stage: row c16 of 16, slot of piece h * 4 + g
  const uint32_t at0 = wk * ((RT + NT) * 2048) + c16 / 8 * 1024 + c16 % 8 * 128 + ((uint32_t)g ^ (c16 & 3)) * 16;
  const uint32_t side = (c16 & 4) * 16;                 // (the slot's upper bit: h ^ bit 2 of the row)
  auto compute = [&](const char *stage) {
#pragma unroll
    for (int b = 0; b < BLOCKS / WK; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const char *at = stage + b * WK * ((RT + NT) * 2048) + at0 + ((h * 64) ^ side);
        u32x4 x[RW], a[NW];
#pragma unroll
        for (int i = 0; i < RW; ++i) x[i] = *(const u32x4 *)(at + (wr * RW + i) * 2048);
#pragma unroll
        for (int j = 0; j < NW; ++j) a[j] = *(const u32x4 *)(at + (RT + wn * NW + j) * 2048);
#pragma unroll
        for (int j = 0; j < NW; ++j)
#pragma unroll
          for (int i = 0; i < RW; ++i) acc[i][j] = mma_x<F16>(a[j], x[i], acc[i][j]);
      }
  };
  // stage s through registers (the only way where K ends inside it, or without the alignment)
  u32x4 reg[OPS];
  auto fetch = [&](int s) {
    const int64_t k = (int64_t)s * KS;
    if (s < full) {
#pragma unroll
      for (int i = 0; i < OPS; ++i) reg[i] = load16(from[i] + k);
    } else {
#pragma unroll
      for (int i = 0; i < OPS; ++i) {
        const int u = wave + i * LORA_WAVES < UNITS ? wave + i * LORA_WAVES : UNITS - 1;
        const int n = p.K - (int)k - u / ((RT + NT) * 2) * 64 - (lane % 8 ^ (lane / 8)) * 8;
        reg[i] = n >= 8 ? load16(from[i] + k) : load16_head(from[i] + k, n);
      }
    }
  };
  auto put = [&](int slot) {
#pragma unroll
    for (int i = 0; i < OPS; ++i) *(u32x4 *)(lora_smem + slot * STAGE + into[i] + lane * 16) = reg[i];
  };
  if (DMA) {
    const int n = (s1 < full ? s1 : full) - s0;
    auto issue = [&](int i, int slot) {
#pragma unroll
      for (int k = 0; k < OPS; ++k) {
        const uint16_t *src = from[k] + (int64_t)(s0 + i) * KS;
        asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(slot * STAGE + into[k]), "v"(src) : "memory", "m0");
      }
    };
    for (int i = 0; i < D - 1; ++i)
      if (i < n) issue(i, i);
    int slot = 0, next = D - 1;
    for (int i = 0; i < n; ++i) {
      if (i + D - 2 < n) wait_loads<(D - 2) * OPS>();
      else wait_loads<0>();
      group_barrier();
      if (i + D - 1 < n) issue(i + D - 1, next);
      compute(lora_smem + slot * STAGE);
      slot = slot + 1 == D ? 0 : slot + 1;
      next = next + 1 == D ? 0 : next + 1;
    }
    if (s1 > full) {
      fetch(full);
      group_barrier();
      put(0);
      group_barrier();
      compute(lora_smem);
    }
  } else {
    fetch(s0);
    for (int s = s0; s < s1; ++s) {
      put((s - s0) & 1);
      group_barrier();
      if (s + 1 < s1) fetch(s + 1);
      compute(lora_smem + ((s - s0) & 1) * STAGE);
    }
  }
  const int kt = (p.rank + 31) / 32;
  // one finished fragment (row group i, rank tile q) as the expand launch's MFMA operands: blocks of 32 ranks, in each
  // block lane (r / 8 % 4) * 16 + row holds ranks r .. r + 7
  auto finish = [&](int i, int q, f32x4 v) {
    const int s = q / lt, r = (q - s * lt) * 16 + g * 4;
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = r + e < rank ? v[e] : 0.0f;
    auto put = [&](auto terms) {
      constexpr int TERMS = decltype(terms)::value;
      __bf16 h[TERMS][4];
      split<TERMS>(f, h);
      char *to = (char *)w.h + ((((int64_t)(t.group + i) * p.n_slices + s) * kt + r / 32) * TERMS) * 1024 +
                 (r / 8 % 4 * 16 + c16) * 16 + r % 8 * 2;
#pragma unroll
      for (int k = 0; k < TERMS; ++k) {
        *(bf16x4 *)(to + k * 1024) = bf16x4{h[k][0], h[k][1], h[k][2], h[k][3]};
        // (a block whose upper half no rank tile fills)
        if (q - s * lt == lt - 1 && lt % 2) *(u32x2 *)(to + k * 1024 + 512) = u32x2{0, 0};
      }
    };
    if (p.dt_dst == ZMI_DT_F32) put(std::integral_constant<int, 3>());
    else put(std::integral_constant<int, 2>());
  };
  // where the sums of K slice z stand: [tile][rank tile][row group][lane]
  auto partial = [&](int z, int i, int q) {
    const int64_t at = (((int64_t)z * gridDim.x + blockIdx.x) * (p.n_slices * ((p.rank + 15) / 16)) + q) * RT + i;
    return w.partial + (at * 64 + lane) * 4;
  };
  if (WK > 1) {   // the wavefronts' shares of K meet in LDS; the first of each set goes on
    f32x4 *red = (f32x4 *)lora_smem + lane;
    group_barrier();
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
      for (int j = 0; j < NW; ++j) red[(wave * RW * NW + i * NW + j) * 64] = acc[i][j];
    group_barrier();
    if (wk == 0) {
#pragma unroll
      for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < NW; ++j)
#pragma unroll
          for (int k = 1; k < WK; ++k) acc[i][j] += red[((wave + k * WR * WN) * RW * NW + i * NW + j) * 64];
    }
  }
  const bool split_k = !SMALL && gridDim.z > 1;
  if (wk == 0) {
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        const int rg = wr * RW + i, q = q0 + wn * NW + j;
        if (q >= live || rg * 16 >= t.n) continue;
        const f32x4 v = acc[i][j];
        if (SMALL) {
          *(f32x4 *)partial(blockIdx.z, rg, q) = v;
        } else if (!split_k) {
          finish(rg, q, v);
        } else {
          // (written through to device scope, so that the slice that arrives last can read it: see below)
          uint64_t *to = (uint64_t *)partial(blockIdx.z, rg, q);
          __hip_atomic_store(to, __builtin_bit_cast(uint64_t, u32x2{__float_as_uint(v[0]), __float_as_uint(v[1])}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __hip_atomic_store(to + 1, __builtin_bit_cast(uint64_t, u32x2{__float_as_uint(v[2]), __float_as_uint(v[3])}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
  }
  if (!split_k) return;
  // The slice that arrives last at the tile's word adds all slices' sums, in slice order, and leaves the operands.
  wait_loads<0>();   // (stores count as well)
  group_barrier();
  int *is_last = (int *)lora_smem;
  if (threadIdx.x == 0)
    *is_last = __hip_atomic_fetch_add(w.arrivals + blockIdx.y * gridDim.x + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.z - 1;
  __syncthreads();
  if (!*is_last) return;
  for (int f = wave; f < RT * NT; f += LORA_WAVES) {
    const int i = f % RT, q = q0 + f / RT;
    if (q >= live || i * 16 >= t.n) continue;
    f32x4 v = {0, 0, 0, 0};
    for (unsigned z = 0; z < gridDim.z; ++z) {
      const uint64_t *src = (const uint64_t *)partial(z, i, q);
      const u32x2 a = __builtin_bit_cast(u32x2, __hip_atomic_load(src, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      const u32x2 b = __builtin_bit_cast(u32x2, __hip_atomic_load(src + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      v += f32x4{__uint_as_float(a[0]), __uint_as_float(a[1]), __uint_as_float(b[0]), __uint_as_float(b[1])};
    }
    finish(i, q, v);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// expand: workgroup (x: columns of a slice, y: tile), 16 NJ columns a wavefront.  MFMA rows are the tile's rows, MFMA
// columns columns of dst: of column tile j lane l holds column n0 + l % 16 * NJ + j of rows (l / 16) * 4 .. +3, so that
// a lane's NJ columns lie together and 16 lanes take 32 NJ contiguous bytes of a row.  B stays in registers for all of the
// tile's 16-row groups.
// ---------------------------------------------------------------------------------------------------------------
template <bool F16, int NJ, int KT, int TERMS, bool D32, bool SMALL>
__global__ __launch_bounds__(LORA_WAVES * 64, KT * NJ * (F16 ? 2 : 1) > 16 ? 2 : 3) void zmi_lora_expand_kernel(ZmiLora p, ZmiLoraPlan w, int slices) {
  constexpr int ES = D32 ? 4 : 2;            // bytes of a dst element
  constexpr int BYTES = NJ * ES, WORDS = BYTES / 4;   // a lane's run of a row
  constexpr int COLS = LORA_WAVES * 16 * NJ;
  typedef uint32_t run_t __attribute__((ext_vector_type(WORDS)));
  const int lane = threadIdx.x % 64, g = lane / 16, c16 = lane % 16;
  Tile t;
  if (!(SMALL ? lora_find_tile(p, blockIdx.y, t) : lora_planned_tile(w.wide, w.header[1], blockIdx.y, t))) return;
  int s = 0, blk = blockIdx.x, col0 = 0;
  while (blk >= (p.N[s] + COLS - 1) / COLS) {
    blk -= (p.N[s] + COLS - 1) / COLS;
    col0 += p.N[s++];
  }
  const int N = p.N[s], n0 = blk * COLS + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 16 * NJ;
  if (n0 >= N) return;
  const bool none = t.slot == p.n_slots;
  if (none && p.base == p.dst) return;
  const int n = n0 + c16 * NJ, cols = N - n < NJ ? N - n : NJ;   // this lane's columns (none where cols <= 0)
  int rank = 0, kts = 0;
  float scale = 0.0f;
  u32x4 b[KT][NJ][F16 ? 2 : 1];
  if (!none) {
    rank = lora_rank(p, t.slot);
    kts = (rank + 31) / 32;
    scale = p.scales ? p.scales[t.slot] : 1.0f;
#pragma unroll
    for (int c = 0; c < KT; ++c)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int at = n + j < N ? n + j : N - 1, left = rank - c * 32 - g * 8;   // ranks that this lane's eight elements may read
        const uint16_t *br = (const uint16_t *)p.b[s] + t.slot * p.b_slot[s] + at * p.b_ld[s] + c * 32 + g * 8;
        u32x4 v = left >= 8 ? load16(br) : load16_head(br, left);
        if (F16) {
          float f[8];
          const f16x8 half = __builtin_bit_cast(f16x8, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = (float)half[e];
          __bf16 q[2][8];
          split<2>(f, q);
#pragma unroll
          for (int k = 0; k < 2; ++k) b[c][j][F16 ? k : 0] = __builtin_bit_cast(u32x4, bf16x8{q[k][0], q[k][1], q[k][2], q[k][3], q[k][4], q[k][5], q[k][6], q[k][7]});
        } else {
          b[c][j][0] = v;
        }
      }
  }
  for (int g0 = 0; g0 < t.n; g0 += 16) {
    // ---- rows and base ----
    int64_t row[4];
    run_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = g0 + g * 4 + i;
      row[i] = at >= t.n || cols <= 0 ? -1 : SMALL ? 0 : w.order[t.first + at];
      if (SMALL) { const int r = __shfl(t.row, g * 4 + i, 64); if (row[i] >= 0) row[i] = r; }
#pragma unroll
      for (int k = 0; k < WORDS; ++k) y[i][k] = 0;
    }
    if (p.base) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (row[i] < 0) continue;
        const char *at = (const char *)p.base + (row[i] * p.ld_base + col0 + n) * ES;
        if (cols == NJ) {
          __builtin_memcpy(&y[i], at, BYTES);
        } else {
#pragma unroll
          for (int e = 0; e < NJ; ++e) {
            if (e >= cols) continue;
            if (D32) y[i][e % WORDS] = ((const uint32_t *)at)[e];
            else y[i][e / 2] |= (uint32_t)((const uint16_t *)at)[e] << (16 * (e % 2));
          }
        }
      }
    }
    f32x4 acc[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < KT; ++c) {
      if (c >= kts) break;
      u32x4 h[TERMS];
      if (SMALL) {
        // the K slices' sums as the shrink launch left them: ranks (r % 16 / 4) * 16 + row, four to a lane
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const int r = c * 32 + g * 8, lt = (rank + 15) / 16, left = rank - r;
        if (left > 0 && c16 < t.n) {
          for (int z = 0; z < slices; ++z) {
            const int64_t at = ((int64_t)z * gridDim.y + blockIdx.y) * (p.n_slices * ((p.rank + 15) / 16)) + s * lt + r / 16;
            const f32x4 *src = (const f32x4 *)w.partial + at * 64 + r % 16 / 4 * 16 + c16;
            const f32x4 lo = src[0], hi = src[16];
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[e] += lo[e]; v[4 + e] += hi[e]; }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e >= left) v[e] = 0.0f;
        }
        __bf16 q[TERMS][8];
        split<TERMS>(v, q);
#pragma unroll
        for (int k = 0; k < TERMS; ++k) h[k] = __builtin_bit_cast(u32x4, bf16x8{q[k][0], q[k][1], q[k][2], q[k][3], q[k][4], q[k][5], q[k][6], q[k][7]});
      } else {
#pragma unroll
        for (int k = 0; k < TERMS; ++k)
          h[k] = ((const u32x4 *)w.h)[((((int64_t)(t.group + g0 / 16) * p.n_slices + s) * ((p.rank + 31) / 32) + c) * TERMS + k) * 64 + lane];
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#pragma unroll
        for (int k = 0; k < TERMS; ++k) acc[j] = mma_x<false>(h[k], b[c][j][0], acc[j]);
        // (the product of the last terms is beyond the precision kept)
#pragma unroll
        for (int k = 0; F16 && k + 1 < TERMS; ++k) acc[j] = mma_x<false>(h[k], b[c][j][F16 ? 1 : 0], acc[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (row[i] < 0) continue;
      run_t out;
      if (none) {
        out = y[i];
      } else if (D32) {
#pragma unroll
        for (int e = 0; e < NJ; ++e) out[e % WORDS] = __float_as_uint(__builtin_fmaf(scale, acc[e][i], __uint_as_float(y[i][e % WORDS])));
      } else {
#pragma unroll
        for (int e = 0; e < WORDS; ++e) {
          const uint32_t old = y[i][e];
          const float d0 = acc[2 * e % NJ][i], d1 = acc[(2 * e + 1) % NJ][i];
          if (p.dt_dst == ZMI_DT_BF16) {
            out[e] = zmi_pack_bf16(__builtin_fmaf(scale, d0, zmi_bf16_to_f32((uint16_t)old)),
                                   __builtin_fmaf(scale, d1, zmi_bf16_to_f32((uint16_t)(old >> 16))));
          } else {
            const _Float16 lo = (_Float16)__builtin_fmaf(scale, d0, zmi_f16_to_f32((uint16_t)old));
            const _Float16 hi = (_Float16)__builtin_fmaf(scale, d1, zmi_f16_to_f32((uint16_t)(old >> 16)));
            out[e] = (uint32_t)__builtin_bit_cast(uint16_t, lo) | (uint32_t)__builtin_bit_cast(uint16_t, hi) << 16;
          }
        }
      }
      char *at = (char *)p.dst + (row[i] * p.ld_dst + col0 + n) * ES;
      if (cols == NJ) {
        __builtin_memcpy(at, &out, BYTES);
      } else {
#pragma unroll
        for (int e = 0; e < NJ; ++e) {
          if (e >= cols) continue;
          if (D32) ((uint32_t *)at)[e] = out[e % WORDS];
          else ((uint16_t *)at)[e] = (uint16_t)(out[e / 2] >> (16 * (e % 2)));
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
namespace {

struct Shape {
  bool small;
  bool dma;          // rows of x and A and their addresses are 16-byte multiples
  int rt;            // 16-row groups of a tile
  int nt;            // rank tiles of a shrink workgroup
  int ny;            // shrink workgroups over the rank tiles
  int ks;            // K slices
  int64_t tiles;     // tiles there can be
  int kt;            // 32-rank blocks an expand wavefront holds
  int nj;            // its column tiles
  int wide;          // tiles of an expand workgroup
  int64_t wide_tiles;
  int64_t col_blocks;
  int terms;
};

// elements of K in a stage of the shrink launch: a stage is 10 .. 24 KiB whatever the tile's shape
constexpr int lora_ks(int rt, int nt) { return rt + nt <= 3 ? (rt + nt == 2 ? 256 : rt == 1 ? 256 : 128) : rt == 1 && nt == 4 ? 128 : rt == 2 && nt == 2 ? 128 : 64; }

Shape lora_shape(const ZmiLora &p) {
  Shape s;
  s.small = p.T <= LORA_SMALL_T;
  const int64_t ids = p.T < p.n_slots + 1 ? p.T : p.n_slots + 1;
  const int64_t avg = p.T / ids;
  s.rt = s.small || avg < 20 ? 1 : avg < 48 ? 2 : 4;
  s.tiles = ids + (p.T - ids) / (16 * s.rt);
  const int qt = p.n_slices * ((p.rank + 15) / 16);
  s.nt = qt >= 8 ? 8 : qt > 2 ? 4 : qt;
  s.ny = (qt + s.nt - 1) / s.nt;
  const int stages = (p.K + lora_ks(s.rt, s.nt) - 1) / lora_ks(s.rt, s.nt);
  int64_t want = 512 / (s.tiles * s.ny), most = stages / 4;
  s.ks = (int)(want < most ? want : most);
  if (s.ks > 16) s.ks = 16;
  if (s.ks < 1) s.ks = 1;
  s.terms = p.dt_dst == ZMI_DT_F32 ? 3 : 2;
  s.dma = p.ldx % 8 == 0 && p.a_ld % 8 == 0 && p.a_slot % 8 == 0 && (uintptr_t)p.x % 16 == 0 && (uintptr_t)p.a % 16 == 0;
  s.kt = p.rank <= 32 ? 1 : p.rank <= 64 ? 2 : p.rank <= 128 ? 4 : 8;
  s.nj = s.small || s.terms == 3 || s.kt == 8 || p.dt_x == ZMI_DT_F16 ? (s.kt == 8 && p.dt_x == ZMI_DT_F16 ? 2 : 4) : 8;
  s.col_blocks = 0;
  const int cols = LORA_WAVES * 16 * s.nj;
  for (int i = 0; i < p.n_slices; ++i) s.col_blocks += (p.N[i] + cols - 1) / cols;
  s.wide = s.col_blocks * s.tiles >= 4 * 512 ? 4 : s.col_blocks * s.tiles >= 2 * 512 ? 2 : 1;
  s.wide_tiles = ids + (p.T - ids) / (16 * s.rt * s.wide);
  return s;
}

size_t pad256(size_t n) { return (n + 255) / 256 * 256; }

// the parts of the workspace; base null: only the size is wanted
size_t lora_layout(const ZmiLora &p, const Shape &s, char *base, ZmiLoraPlan *w) {
  size_t at = 0;
  auto take = [&](size_t n) { char *q = base + at; at += pad256(n); return q; };
  const size_t qt = (size_t)p.n_slices * ((p.rank + 15) / 16);
  ZmiLoraPlan l = {};
  if (!s.small) {
    l.header = (int32_t *)take(16);
    l.tiles = (int32_t *)take((size_t)s.tiles * 16);
    l.wide = (int32_t *)take((size_t)s.wide_tiles * 16);
    l.order = (int32_t *)take((size_t)p.T * 4);
    l.place = (int32_t *)take(p.T > LORA_PLAN_KEEP * 1024 ? (size_t)p.T * 4 : 0);
    l.n_arrivals = (int32_t)(s.tiles * s.ny);
    l.arrivals = (uint32_t *)take((size_t)l.n_arrivals * 4);
    l.h = take((size_t)s.tiles * s.rt * p.n_slices * ((p.rank + 31) / 32) * s.terms * 1024);
  }
  if (s.small || s.ks > 1) l.partial = (float *)take((size_t)s.ks * s.tiles * qt * s.rt * 1024);
  if (w) *w = l;
  return at;
}

template <bool F16, int RT, int NT, int WR, int WN, bool SMALL>
hipError_t launch_shrink_as(const ZmiLora &p, const ZmiLoraPlan &w, const Shape &s, hipStream_t stream) {
  constexpr int KS = lora_ks(RT, NT), STAGE = (RT + NT) * 32 * KS, D = STAGE <= 18432 ? 4 : 3;
  static_assert(LORA_WAVES / (WR * WN) * WR * WN == LORA_WAVES && D * STAGE <= 80 * 1024, "two workgroups a compute unit");
  const dim3 grid((unsigned)s.tiles, (unsigned)s.ny, (unsigned)s.ks), block(LORA_WAVES * 64);
  if (s.dma) {
    const auto kernel = zmi_lora_shrink_kernel<F16, RT, NT, KS, WR, WN, D, true, SMALL>;
    const hipError_t e = zmi_func_smem_once((const void *)kernel, D * STAGE);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, grid, block, D * STAGE, stream, p, w);
  } else {
    const auto kernel = zmi_lora_shrink_kernel<F16, RT, NT, KS, WR, WN, D, false, SMALL>;
    hipLaunchKernelGGL(kernel, grid, block, 2 * STAGE, stream, p, w);
  }
  return hipGetLastError();
}

template <bool F16, int RT, bool SMALL>
hipError_t launch_shrink(const ZmiLora &p, const ZmiLoraPlan &w, const Shape &s, hipStream_t stream) {
  constexpr int R2 = RT >= 2 ? 2 : 1;
  if (s.nt == 1) return launch_shrink_as<F16, RT, 1, RT, 1, SMALL>(p, w, s, stream);
  if (s.nt == 2) return launch_shrink_as<F16, RT, 2, RT, RT == 2 ? 2 : 1, SMALL>(p, w, s, stream);
  if (s.nt == 4) return launch_shrink_as<F16, RT, 4, R2, 4 / R2, SMALL>(p, w, s, stream);
  return launch_shrink_as<F16, RT, 8, R2, 4 / R2, SMALL>(p, w, s, stream);
}

template <bool F16, bool SMALL, int NJ, int KT, bool D32>
hipError_t launch_expand_as(const ZmiLora &p, const ZmiLoraPlan &w, const Shape &s, hipStream_t stream) {
  const dim3 grid((unsigned)s.col_blocks, (unsigned)(SMALL ? s.tiles : s.wide_tiles)), block(LORA_WAVES * 64);
  hipLaunchKernelGGL((zmi_lora_expand_kernel<F16, NJ, KT, D32 ? 3 : 2, D32, SMALL>), grid, block, 0, stream, p, w, s.ks);
  return hipGetLastError();
}

template <bool F16, bool SMALL, int KT>
hipError_t launch_expand_kt(const ZmiLora &p, const ZmiLoraPlan &w, const Shape &s, hipStream_t stream) {
  constexpr int FEW = KT == 8 && F16 ? 2 : 4, NJ = SMALL || F16 || KT == 8 ? FEW : 8;
  if (s.terms == 3) return launch_expand_as<F16, SMALL, FEW, KT, true>(p, w, s, stream);
  return launch_expand_as<F16, SMALL, NJ, KT, false>(p, w, s, stream);
}

template <bool F16, bool SMALL>
hipError_t launch_expand(const ZmiLora &p, const ZmiLoraPlan &w, const Shape &s, hipStream_t stream) {
  return s.kt == 1 ? launch_expand_kt<F16, SMALL, 1>(p, w, s, stream) : s.kt == 2 ? launch_expand_kt<F16, SMALL, 2>(p, w, s, stream)
       : s.kt == 4 ? launch_expand_kt<F16, SMALL, 4>(p, w, s, stream) : launch_expand_kt<F16, SMALL, 8>(p, w, s, stream);
}

template <bool F16>
hipError_t launch_both(const ZmiLora &p, const ZmiLoraPlan &w, const Shape &s, hipStream_t stream) {
  const hipError_t e = s.small ? launch_shrink<F16, 1, true>(p, w, s, stream) : s.rt == 1 ? launch_shrink<F16, 1, false>(p, w, s, stream)
                     : s.rt == 2 ? launch_shrink<F16, 2, false>(p, w, s, stream) : launch_shrink<F16, 4, false>(p, w, s, stream);
  if (e != hipSuccess) return e;
  return s.small ? launch_expand<F16, true>(p, w, s, stream) : launch_expand<F16, false>(p, w, s, stream);
}

}  // namespace

size_t zmi_lora_workspace_bytes(const ZmiLora &p) { return p.T > 0 ? lora_layout(p, lora_shape(p), nullptr, nullptr) : 0; }

hipError_t zmi_launch_lora(const ZmiLora &p, hipStream_t stream, const char **name) {
  if (p.T <= 0) return hipSuccess;
  if (!p.workspace || p.n_slots > ZMI_LORA_MAX_SLOTS || p.n_slices > 4) return hipErrorInvalidValue;
  const Shape s = lora_shape(p);
  if (s.tiles > 65535 || s.ny > 65535) return hipErrorInvalidValue;
  ZmiLoraPlan w;
  lora_layout(p, s, (char *)p.workspace, &w);
  if (!s.small) hipLaunchKernelGGL(zmi_lora_plan_kernel, dim3(1), dim3(1024), 0, stream, p, w, 16 * s.rt, s.wide);
  *name = s.small ? "lora_small" : "lora_planned";
  return p.dt_x == ZMI_DT_F16 ? launch_both<true>(p, w, s, stream) : launch_both<false>(p, w, s, stream);
}
