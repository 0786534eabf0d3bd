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
//   shrink  h of a tile.  Wavefronts split K, not the tile: operands go straight from memory to registers, each
//           wavefront has its own loads in flight and no barrier in its loop; partial sums meet in LDS, and across
//           the workgroups of one tile (K in slices, where the tiles alone do not fill the device) in memory;
//   expand  dst.  A wavefront takes 64 columns of a tile's rows and reads h as MFMA operands.
//
// The MFMA takes 16-bit operands: x, A exactly as they are; h, which is f32, as a sum of bf16 terms (2 terms hold 16
// bits, for f32 destinations 3 hold 24), and f16 B, which the range of h does not allow to meet in f16, as two bf16 terms
// that hold it exactly.  All products are accumulated in f32.
#include "zmi_device.h"
#include "zmi_launch.h"

#include <type_traits>

#define LORA_WAVES 4
#define LORA_SMALL_T 64     // rows up to which wavefronts plan for themselves
#define LORA_COLS 256       // columns of an expand workgroup

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

__device__ __forceinline__ bool lora_planned_tile(const ZmiLoraPlan &w, int want, Tile &t) {
  if (want >= w.header[0]) return false;
  const int *e = w.tiles + 4 * (int64_t)want;
  t.slot = __builtin_amdgcn_readfirstlane(e[0]);
  t.first = __builtin_amdgcn_readfirstlane(e[1]);
  t.n = __builtin_amdgcn_readfirstlane(e[2]);
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

}  // namespace

// ---------------------------------------------------------------------------------------------------------------
// plan: rows sorted by slot (the order within a slot does not matter: rows are computed independently of each other),
// tiles of at most `tile` rows.
// ---------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(1024) void zmi_lora_plan_kernel(ZmiLora p, ZmiLoraPlan w, int tile) {
  __shared__ int cursor[ZMI_LORA_MAX_SLOTS + 1];
  __shared__ int wave_rows[16], wave_tiles[16];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, n = p.n_slots + 1;
  for (int i = tid; i < n; i += 1024) cursor[i] = 0;
  for (int i = tid; i < w.n_arrivals; i += 1024) w.arrivals[i] = 0;
  __syncthreads();
  auto slot_of = [&](int t) {
    const int id = p.slot_ids[t];
    return (unsigned)id < (unsigned)p.n_slots ? id : p.n_slots;
  };
  for (int t = tid; t < p.T; t += 1024) atomicAdd(&cursor[slot_of(t)], 1);
  __syncthreads();
  // thread i owns slots [i per, (i + 1) per)
  const int per = (n + 1023) / 1024;
  int rows = 0, tiles = 0;
  for (int i = tid * per; i < (tid + 1) * per && i < n; ++i) {
    rows += cursor[i];
    tiles += (cursor[i] + tile - 1) / tile;
  }
  int r = rows, q = tiles;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int a = __shfl_up(r, d, 64), b = __shfl_up(q, d, 64);
    if (lane >= d) { r += a; q += b; }
  }
  if (lane == 63) { wave_rows[wave] = r; wave_tiles[wave] = q; }
  __syncthreads();
  int row0 = r - rows, tile0 = q - tiles;
  for (int i = 0; i < wave; ++i) { row0 += wave_rows[i]; tile0 += wave_tiles[i]; }
  if (tid == 1023) w.header[0] = tile0 + tiles;
  for (int i = tid * per; i < (tid + 1) * per && i < n; ++i) {
    const int c = cursor[i];
    for (int j = 0; j < c; j += tile) {
      int *e = w.tiles + 4 * (int64_t)tile0++;
      e[0] = i;
      e[1] = row0 + j;
      e[2] = c - j < tile ? c - j : tile;
    }
    cursor[i] = row0;
    row0 += c;
  }
  __syncthreads();
  for (int t = tid; t < p.T; t += 1024) w.order[atomicAdd(&cursor[slot_of(t)], 1)] = t;
}

// ---------------------------------------------------------------------------------------------------------------
// shrink: workgroup (x: tile, y: NT rank tiles of 16, z: K slice).  MFMA rows are ranks, columns the tile's rows: lane
// l holds ranks (l / 16) * 4 .. +3 of row l % 16.  Rank tiles are numbered over the live ones of all slices (an adapter
// of a smaller rank has fewer); ranks and rows beyond the last one repeat it and are dropped.
// ---------------------------------------------------------------------------------------------------------------
template <bool F16, int RT, int NT, int DEPTH, bool SMALL>
__global__ __launch_bounds__(LORA_WAVES * 64, RT * NT < 32 ? 2 : 1) void zmi_lora_shrink_kernel(ZmiLora p, ZmiLoraPlan w) {
  constexpr int FRAGS = RT * NT;
  constexpr int PART = FRAGS < 8 ? FRAGS : 8;   // fragments summed over the wavefronts at a time
  __shared__ f32x4 red[LORA_WAVES][PART][64];
  __shared__ int is_last;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), g = lane / 16, c16 = lane % 16;
  Tile t;
  if (!(SMALL ? lora_find_tile(p, blockIdx.x, t) : lora_planned_tile(w, blockIdx.x, t))) return;
  if (t.slot == p.n_slots) return;
  const int rank = lora_rank(p, t.slot), lt = (rank + 15) / 16, live = lt * p.n_slices;
  const int q0 = blockIdx.y * NT;
  if (q0 >= live) return;
  const uint16_t *xr[RT], *ar[NT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int at = i * 16 + c16 < t.n ? i * 16 + c16 : 0;
    const int row = SMALL ? __shfl(t.row, at, 64) : w.order[t.first + at];
    xr[i] = (const uint16_t *)p.x + row * p.ldx + g * 16;
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int q = q0 + i < live ? q0 + i : live - 1, s = q / lt;
    const int r = (q - s * lt) * 16 + c16;
    ar[i] = (const uint16_t *)p.a + t.slot * p.a_slot + (s * p.rank + (r < rank ? r : rank - 1)) * p.a_ld + g * 16;
  }
  // K in groups of DEPTH steps of 32 elements: lane group g takes elements g * 16 + 0 .. 7 of a 64-element chunk in its
  // first step and + 8 .. 15 in its second, so that two steps read whole 128-byte lines
  constexpr int GROUP = 32 * DEPTH;
  const int groups = (p.K + GROUP - 1) / GROUP;
  const int parts = gridDim.z * LORA_WAVES, part = blockIdx.z * LORA_WAVES + wave;
  const int g0 = (int)((int64_t)groups * part / parts), g1 = (int)((int64_t)groups * (part + 1) / parts);
  const int whole = g1 * GROUP <= p.K ? g1 : g1 - 1;
  f32x4 acc[RT][NT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  u32x4 xf[DEPTH][RT], af[DEPTH][NT];
  auto load = [&](u32x4 (&x)[RT], u32x4 (&a)[NT], int64_t k) {
#pragma unroll
    for (int j = 0; j < RT; ++j) x[j] = load16(xr[j] + k);
#pragma unroll
    for (int j = 0; j < NT; ++j) a[j] = load16(ar[j] + k);
  };
  auto mma = [&](const u32x4 (&x)[RT], const u32x4 (&a)[NT]) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[i][j] = mma_x<F16>(a[j], x[i], acc[i][j]);
  };
  if (g0 < whole) {   // DEPTH steps are in flight
    int64_t k = (int64_t)g0 * GROUP;
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(xf[d], af[d], k + d / 2 * 64 + d % 2 * 8);
#pragma unroll 1
    for (int i = g0 + 1; i < whole; ++i) {
      k += GROUP;
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        mma(xf[d], af[d]);
        load(xf[d], af[d], k + d / 2 * 64 + d % 2 * 8);
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) mma(xf[d], af[d]);
  }
  if (whole < g1) {   // the last group when it is not whole
    const int k0 = whole * GROUP;
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int k = k0 + d / 2 * 64 + d % 2 * 8;
#pragma unroll
      for (int j = 0; j < RT; ++j) xf[d][j] = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < NT; ++j) af[d][j] = u32x4{0, 0, 0, 0};
      if (k + g * 16 + 8 <= p.K) load(xf[d], af[d], k);
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) mma(xf[d], af[d]);
    if (p.K % 8) {   // (the first lane group takes what is left)
      const int n = g == 0 ? p.K % 8 : 0, k = p.K - p.K % 8;
#pragma unroll
      for (int j = 0; j < RT; ++j) xf[0][j] = load16_head(xr[j] + k, n);
#pragma unroll
      for (int j = 0; j < NT; ++j) af[0][j] = load16_head(ar[j] + k, n);
      mma(xf[0], af[0]);
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
      char *to = (char *)w.h + (((((int64_t)blockIdx.x * RT + i) * p.n_slices + s) * kt + r / 32) * TERMS) * 1024 +
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
#pragma unroll
  for (int f0 = 0; f0 < FRAGS; f0 += PART) {
    if (f0) __syncthreads();
#pragma unroll
    for (int f = 0; f < PART; ++f) red[wave][f][lane] = acc[(f0 + f) % RT][(f0 + f) / RT];
    __syncthreads();
    for (int f = wave; f < PART; f += LORA_WAVES) {
      const int i = (f0 + f) % RT, q = q0 + (f0 + f) / RT;
      if (q >= live || i * 16 >= t.n) continue;
      const f32x4 v = red[0][f][lane] + red[1][f][lane] + red[2][f][lane] + red[3][f][lane];
      if (SMALL) {
        *(f32x4 *)partial(blockIdx.z, i, q) = v;
      } else if (gridDim.z == 1) {
        finish(i, q, v);
      } else {
        // (written through to device scope, so that the slice that arrives last can read it: see below)
        uint64_t *to = (uint64_t *)partial(blockIdx.z, i, q);
        __hip_atomic_store(to, __builtin_bit_cast(uint64_t, u32x2{__float_as_uint(v[0]), __float_as_uint(v[1])}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(to + 1, __builtin_bit_cast(uint64_t, u32x2{__float_as_uint(v[2]), __float_as_uint(v[3])}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (SMALL || gridDim.z == 1) return;
  // The slice that arrives last at the tile's word adds all slices' sums, in slice order, and leaves the operands.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    is_last = __hip_atomic_fetch_add(w.arrivals + blockIdx.y * gridDim.x + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.z - 1;
  __syncthreads();
  if (!is_last) return;
  for (int f = wave; f < FRAGS; f += LORA_WAVES) {
    const int i = f % RT, q = q0 + f / RT;
    if (q >= live || i * 16 >= t.n) continue;
    f32x4 v = {0, 0, 0, 0};
    for (unsigned z = 0; z < gridDim.z; ++z) {
      const uint64_t *from = (const uint64_t *)partial(z, i, q);
      const u32x2 a = __builtin_bit_cast(u32x2, __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      const u32x2 b = __builtin_bit_cast(u32x2, __hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      v += f32x4{__uint_as_float(a[0]), __uint_as_float(a[1]), __uint_as_float(b[0]), __uint_as_float(b[1])};
    }
    finish(i, q, v);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// expand: workgroup (x: 256 columns of a slice, y: tile), 64 columns a wavefront.  MFMA rows are columns of dst, MFMA
// columns the tile's rows: of 16-column tile j lane l holds n0 + (j / 2) * 32 + (l / 16) * 8 + j % 2 * 4 .. +3 of row l % 16,
// so that a lane's columns are two runs of eight and every access to base and dst takes 64 contiguous bytes of a row.
// ---------------------------------------------------------------------------------------------------------------
template <bool F16, int RT, int TERMS, bool D32, bool SMALL>
__global__ __launch_bounds__(LORA_WAVES * 64) void zmi_lora_expand_kernel(ZmiLora p, ZmiLoraPlan w, int slices) {
  constexpr int ES = D32 ? 4 : 2;          // bytes of a dst element
  constexpr int W = D32 ? 2 : 1;           // 16-byte words of a run of eight
  const int lane = threadIdx.x % 64, g = lane / 16, c16 = lane % 16;
  Tile t;
  if (!(SMALL ? lora_find_tile(p, blockIdx.y, t) : lora_planned_tile(w, blockIdx.y, t))) return;
  int s = 0, blk = blockIdx.x, col0 = 0;
  while (blk >= (p.N[s] + LORA_COLS - 1) / LORA_COLS) {
    blk -= (p.N[s] + LORA_COLS - 1) / LORA_COLS;
    col0 += p.N[s++];
  }
  const int N = p.N[s], n0 = blk * LORA_COLS + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 64;
  if (n0 >= N) return;
  const bool none = t.slot == p.n_slots;
  if (none && p.base == p.dst) return;
  int64_t row[RT];
  bool have[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    have[i] = i * 16 + c16 < t.n;
    const int at = have[i] ? i * 16 + c16 : 0;
    row[i] = SMALL ? __shfl(t.row, at, 64) : w.order[t.first + at];
  }
  // ---- base ----
  u32x4 y[RT][2][W];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = n0 + h * 32 + g * 8;
#pragma unroll
      for (int k = 0; k < W; ++k) y[i][h][k] = u32x4{0, 0, 0, 0};
      if (!p.base || !have[i] || n >= N) continue;
      const char *at = (const char *)p.base + (row[i] * p.ld_base + col0 + n) * ES;
      if (n + 8 <= N) {
#pragma unroll
        for (int k = 0; k < W; ++k) y[i][h][k] = load16(at + 16 * k);
      } else if (D32) {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (n + e < N) y[i][h][e / 4][e % 4] = ((const uint32_t *)at)[e];
      } else {
        y[i][h][0] = load16_head((const uint16_t *)at, N - n);
      }
    }
  f32x4 acc[RT][4];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  float scale = 0.0f;
  if (!none) {
    const int rank = lora_rank(p, t.slot), kts = (rank + 31) / 32, kt = (p.rank + 31) / 32;
    scale = p.scales ? p.scales[t.slot] : 1.0f;
    const uint16_t *br[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + (j >> 1) * 32 + c16 / 4 * 8 + (j & 1) * 4 + c16 % 4;
      br[j] = (const uint16_t *)p.b[s] + t.slot * p.b_slot[s] + (n < N ? n : N - 1) * p.b_ld[s] + g * 8;
    }
    for (int c = 0; c < kts; ++c) {
      const int left = rank - c * 32 - g * 8;   // ranks that this lane's eight elements may read
      u32x4 b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = left >= 8 ? load16(br[j] + c * 32) : load16_head(br[j] + c * 32, left);
      u32x4 hf[RT][TERMS];
      if (SMALL) {
        // the K slices' sums as the shrink launch left them: ranks (r % 16 / 4) * 16 + row, four to a lane
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const int r = c * 32 + g * 8, lt = (rank + 15) / 16;
        if (left > 0) {
          for (int z = 0; z < slices; ++z) {
            const int64_t at = ((int64_t)z * gridDim.y + blockIdx.y) * (p.n_slices * ((p.rank + 15) / 16)) + s * lt + r / 16;
            const f32x4 *from = (const f32x4 *)w.partial + at * 64 + r % 16 / 4 * 16 + c16;
            const f32x4 lo = from[0], hi = from[16];
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[e] += lo[e]; v[4 + e] += hi[e]; }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e >= left) v[e] = 0.0f;
        }
        __bf16 h[TERMS][8];
        split<TERMS>(v, h);
#pragma unroll
        for (int k = 0; k < TERMS; ++k) hf[0][k] = __builtin_bit_cast(u32x4, bf16x8{h[k][0], h[k][1], h[k][2], h[k][3], h[k][4], h[k][5], h[k][6], h[k][7]});
      } else {
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int k = 0; k < TERMS; ++k)
            hf[i][k] = ((const u32x4 *)w.h)[(((((int64_t)blockIdx.y * RT + i) * p.n_slices + s) * kt + c) * TERMS + k) * 64 + lane];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (F16) {
          float v[8];
          const f16x8 half = __builtin_bit_cast(f16x8, b[j]);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (float)half[e];
          __bf16 q[2][8];
          split<2>(v, q);
          const u32x4 hi = __builtin_bit_cast(u32x4, bf16x8{q[0][0], q[0][1], q[0][2], q[0][3], q[0][4], q[0][5], q[0][6], q[0][7]});
          const u32x4 lo = __builtin_bit_cast(u32x4, bf16x8{q[1][0], q[1][1], q[1][2], q[1][3], q[1][4], q[1][5], q[1][6], q[1][7]});
#pragma unroll
          for (int i = 0; i < RT; ++i) {
#pragma unroll
            for (int k = 0; k < TERMS; ++k) acc[i][j] = mma_x<false>(hi, hf[i][k], acc[i][j]);
            // (the product of the last terms is beyond the precision kept)
#pragma unroll
            for (int k = 0; k + 1 < TERMS; ++k) acc[i][j] = mma_x<false>(lo, hf[i][k], acc[i][j]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int k = 0; k < TERMS; ++k) acc[i][j] = mma_x<false>(b[j], hf[i][k], acc[i][j]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = n0 + h * 32 + g * 8;
      if (!have[i] || n >= N) continue;
      u32x4 out[W];
      if (none) {
#pragma unroll
        for (int k = 0; k < W; ++k) out[k] = y[i][h][k];
      } else if (D32) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          out[e / 4][e % 4] = __float_as_uint(__builtin_fmaf(scale, acc[i][2 * h + e / 4][e % 4], __uint_as_float(y[i][h][e / 4][e % 4])));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t old = y[i][h][0][e];
          const float d0 = acc[i][2 * h + e / 2][e % 2 * 2], d1 = acc[i][2 * h + e / 2][e % 2 * 2 + 1];
          if (p.dt_dst == ZMI_DT_BF16) {
            out[0][e] = zmi_pack_bf16(__builtin_fmaf(scale, d0, zmi_bf16_to_f32((uint16_t)old)),
                                      __builtin_fmaf(scale, d1, zmi_bf16_to_f32((uint16_t)(old >> 16))));
          } else {
            const _Float16 a = (_Float16)__builtin_fmaf(scale, d0, zmi_f16_to_f32((uint16_t)old));
            const _Float16 b = (_Float16)__builtin_fmaf(scale, d1, zmi_f16_to_f32((uint16_t)(old >> 16)));
            out[0][e] = (uint32_t)__builtin_bit_cast(uint16_t, a) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
          }
        }
      }
      char *at = (char *)p.dst + (row[i] * p.ld_dst + col0 + n) * ES;
      if (n + 8 <= N) {
#pragma unroll
        for (int k = 0; k < W; ++k) store16(at + 16 * k, out[k]);
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e) {
          if (n + e >= N) continue;
          if (D32) ((uint32_t *)at)[e] = out[e / 4][e % 4];
          else ((uint16_t *)at)[e] = (uint16_t)(out[0][e / 2] >> (16 * (e % 2)));
        }
      }
    }
}

// ---------------------------------------------------------------------------------------------------------------
namespace {

struct Shape {
  bool small;
  int rt;            // 16-row groups of a tile
  int nt;            // rank tiles of a shrink workgroup
  int ny;            // shrink workgroups over the rank tiles
  int ks;            // K slices
  int64_t tiles;     // tiles there can be
  int terms;
};

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
  int64_t want = 512 / (s.tiles * s.ny), most = (p.K + 255) / 256 / LORA_WAVES;
  s.ks = (int)(want < most ? want : most);
  if (s.ks > 16) s.ks = 16;
  if (s.ks < 1) s.ks = 1;
  s.terms = p.dt_dst == ZMI_DT_F32 ? 3 : 2;
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
    l.order = (int32_t *)take((size_t)p.T * 4);
    l.n_arrivals = (int32_t)(s.tiles * s.ny);
    l.arrivals = (uint32_t *)take((size_t)l.n_arrivals * 4);
    l.h = take((size_t)s.tiles * s.rt * p.n_slices * ((p.rank + 31) / 32) * s.terms * 1024);
  }
  if (s.small || s.ks > 1) l.partial = (float *)take((size_t)s.ks * s.tiles * qt * s.rt * 1024);
  if (w) *w = l;
  return at;
}

template <bool F16, int RT, bool SMALL>
void launch_shrink(const ZmiLora &p, const ZmiLoraPlan &w, const Shape &s, hipStream_t stream) {
  const dim3 grid((unsigned)s.tiles, (unsigned)s.ny, (unsigned)s.ks), block(LORA_WAVES * 64);
  constexpr int D1 = RT == 4 ? 4 : 8, D4 = RT == 4 ? 2 : 4;
  if (s.nt == 1) hipLaunchKernelGGL((zmi_lora_shrink_kernel<F16, RT, 1, D1, SMALL>), grid, block, 0, stream, p, w);
  else if (s.nt == 2) hipLaunchKernelGGL((zmi_lora_shrink_kernel<F16, RT, 2, 4, SMALL>), grid, block, 0, stream, p, w);
  else if (s.nt == 4) hipLaunchKernelGGL((zmi_lora_shrink_kernel<F16, RT, 4, D4, SMALL>), grid, block, 0, stream, p, w);
  else hipLaunchKernelGGL((zmi_lora_shrink_kernel<F16, RT, 8, 2, SMALL>), grid, block, 0, stream, p, w);
}

template <bool F16, int RT, bool SMALL>
void launch_expand(const ZmiLora &p, const ZmiLoraPlan &w, const Shape &s, hipStream_t stream) {
  int64_t blocks = 0;
  for (int i = 0; i < p.n_slices; ++i) blocks += (p.N[i] + LORA_COLS - 1) / LORA_COLS;
  const dim3 grid((unsigned)blocks, (unsigned)s.tiles), block(LORA_WAVES * 64);
  if (p.dt_dst == ZMI_DT_F32) hipLaunchKernelGGL((zmi_lora_expand_kernel<F16, RT, 3, true, SMALL>), grid, block, 0, stream, p, w, s.ks);
  else hipLaunchKernelGGL((zmi_lora_expand_kernel<F16, RT, 2, false, SMALL>), grid, block, 0, stream, p, w, s.ks);
}

template <bool F16>
void launch_both(const ZmiLora &p, const ZmiLoraPlan &w, const Shape &s, hipStream_t stream) {
  if (s.small) {
    launch_shrink<F16, 1, true>(p, w, s, stream);
    launch_expand<F16, 1, true>(p, w, s, stream);
  } else if (s.rt == 1) {
    launch_shrink<F16, 1, false>(p, w, s, stream);
    launch_expand<F16, 1, false>(p, w, s, stream);
  } else if (s.rt == 2) {
    launch_shrink<F16, 2, false>(p, w, s, stream);
    launch_expand<F16, 2, false>(p, w, s, stream);
  } else {
    launch_shrink<F16, 4, false>(p, w, s, stream);
    launch_expand<F16, 4, false>(p, w, s, stream);
  }
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
  if (!s.small) hipLaunchKernelGGL(zmi_lora_plan_kernel, dim3(1), dim3(1024), 0, stream, p, w, 16 * s.rt);
  if (p.dt_x == ZMI_DT_F16) launch_both<true>(p, w, s, stream);
  else launch_both<false>(p, w, s, stream);
  *name = s.small ? "lora_small" : "lora_planned";
  return hipGetLastError();
}
