// The second product of the low-rank adapters (k_lora.hip): dst[t][n] = base[t][n] + scales[a] sum_r h[t][s, r] B_s[a][n][r].
//
// MFMA rows are 16 rows of the batch that share a slot, MFMA columns columns of dst: of column tile j lane l holds column
// n0 + l % 16 * NJ + j of rows (l / 16) * 4 .. +3, so that a lane's NJ columns lie together and 16 lanes take whole lines
// of a row.  (With the operands the other way round 16 neighbouring lanes stand in 16 rows, and the address path of the
// compute unit takes four times as long over every access.)
//
// HBM bounds it: base and dst once, B and h from L2.  Planned calls run down the 16-row groups of the batch with B in
// registers, reloaded where the slot changes; each workgroup takes an equal share of the groups, h of the next group goes
// to LDS and its base to registers while one is computed, and a group's stores go out behind the next group's loads.
#include <type_traits>

#include "zmi_lora.h"

namespace {

template <int NJ, int DST>   // DST: ZMI_DT_*
struct Out {
  static constexpr int ES = DST == ZMI_DT_F32 ? 4 : 2, BYTES = NJ * ES, WORDS = BYTES / 4;
  static constexpr int TERMS = DST == ZMI_DT_F32 ? 3 : 2;
  static constexpr int COLS = LORA_WAVES * 16 * NJ;   // of a workgroup
  typedef uint32_t run_t __attribute__((ext_vector_type(WORDS)));   // a lane's columns of a row

  // cols < NJ: only that many (edge: some lane of the wavefront has fewer)
  static __device__ __forceinline__ run_t load(const char *at, int cols, bool edge) {
    run_t y;
    if (!edge) {
      __builtin_memcpy(&y, at, BYTES);
    } else {
#pragma unroll
      for (int k = 0; k < WORDS; ++k) y[k] = 0;
#pragma unroll
      for (int e = 0; e < NJ; ++e) {
        if (e >= cols) continue;
        if (ES == 4) y[e % WORDS] = ((const uint32_t *)at)[e];
        else y[e / 2 % WORDS] |= (uint32_t)((const uint16_t *)at)[e] << (16 * (e % 2));
      }
    }
    return y;
  }
  static __device__ __forceinline__ void store(char *at, run_t y, int cols, bool edge) {
    if (!edge) {
      __builtin_memcpy(at, &y, BYTES);
    } else {
#pragma unroll
      for (int e = 0; e < NJ; ++e) {
        if (e >= cols) continue;
        if (ES == 4) ((uint32_t *)at)[e] = y[e % WORDS];
        else ((uint16_t *)at)[e] = (uint16_t)(y[e / 2 % WORDS] >> (16 * (e % 2)));
      }
    }
  }
  // base + scale * delta of row i of the lane's four, rounded once
  static __device__ __forceinline__ run_t sum(run_t y, const f32x4 (&acc)[NJ], int i, float scale) {
    run_t out;
#pragma unroll
    for (int e = 0; e < WORDS; ++e) {
      if (DST == ZMI_DT_F32) {
        out[e] = __float_as_uint(__builtin_fmaf(scale, acc[e % NJ][i], __uint_as_float(y[e])));
      } else {
        const float d0 = acc[2 * e % NJ][i], d1 = acc[(2 * e + 1) % NJ][i];
        if (DST == ZMI_DT_BF16) {
          out[e] = zmi_pack_bf16(__builtin_fmaf(scale, d0, zmi_bf16_to_f32((uint16_t)y[e])),
                                 __builtin_fmaf(scale, d1, zmi_bf16_to_f32((uint16_t)(y[e] >> 16))));
        } else {
          const _Float16 lo = (_Float16)__builtin_fmaf(scale, d0, zmi_f16_to_f32((uint16_t)y[e]));
          const _Float16 hi = (_Float16)__builtin_fmaf(scale, d1, zmi_f16_to_f32((uint16_t)(y[e] >> 16)));
          out[e] = (uint32_t)__builtin_bit_cast(uint16_t, lo) | (uint32_t)__builtin_bit_cast(uint16_t, hi) << 16;
        }
      }
    }
    return out;
  }
};

__device__ __forceinline__ u32x4 pack8(const __bf16 (&v)[8]) {
  return __builtin_bit_cast(u32x4, bf16x8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]});
}

// B of a lane's NJ columns from column n on, as MFMA operands: ranks c * 32 + g * 8 .. +7, zeros from `rank` on
template <bool F16, int NJ, int KT>
__device__ __forceinline__ void load_b(const ZmiLora &p, int s, int slot, int rank, int n, u32x4 (&b)[KT][NJ][F16 ? 2 : 1]) {
  const int g = threadIdx.x % 64 / 16;
  u32x4 v[KT][NJ];
#pragma unroll
  for (int c = 0; c < KT; ++c)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int at = n + j < p.N[s] ? n + j : p.N[s] - 1, left = rank - c * 32 - g * 8;
      const uint16_t *br = (const uint16_t *)p.b[s] + slot * p.b_slot[s] + at * p.b_ld[s] + c * 32 + g * 8;
      v[c][j] = left >= 8 ? load16(br) : load16_head(br, left);
    }
#pragma unroll
  for (int c = 0; c < KT; ++c)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (F16) {
        float f[8];
        const f16x8 half = __builtin_bit_cast(f16x8, v[c][j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)half[e];
        __bf16 q[2][8];
        split<2>(f, q);
        b[c][j][0] = pack8(q[0]);
        b[c][j][F16 ? 1 : 0] = pack8(q[1]);
      } else {
        b[c][j][0] = v[c][j];
      }
    }
}

// acc += h (term k of `terms`) times B
template <bool F16, int NJ>
__device__ __forceinline__ void mma_h(f32x4 (&acc)[NJ], u32x4 h, const u32x4 (&b)[NJ][F16 ? 2 : 1], bool last) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = mma_x<false>(h, b[j][0], acc[j]);
  // (the product of the last terms is beyond the precision kept)
  if (F16 && !last)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] = mma_x<false>(h, b[j][F16 ? 1 : 0], acc[j]);
}

}  // namespace

// Planned: workgroup (x: columns of a slice, y: share of the 16-row groups).
template <bool F16, int NJ, int KT, int DST>
__global__ __launch_bounds__(LORA_WAVES * 64, 2) void zmi_lora_expand_kernel(ZmiLora p, ZmiLoraPlan w) {
  typedef Out<NJ, DST> O;
  constexpr int TERMS = O::TERMS;
  __shared__ __attribute__((aligned(16))) char ring[2][KT * TERMS * 1024];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), g = lane / 16, c16 = lane % 16;
  // (in place the rows without an adapter, which come last, are left alone)
  const int64_t groups = __builtin_amdgcn_readfirstlane(w.header[p.base == p.dst ? 1 : 2]);
  const int a = (int)(groups * blockIdx.y / gridDim.y), z = (int)(groups * (blockIdx.y + 1) / gridDim.y);
  if (a >= z) return;
  int s = 0, blk = blockIdx.x, col0 = 0;
  while (blk >= (p.N[s] + O::COLS - 1) / O::COLS) {
    blk -= (p.N[s] + O::COLS - 1) / O::COLS;
    col0 += p.N[s++];
  }
  const int n0 = blk * O::COLS + wave * 16 * NJ, n = n0 + c16 * NJ, cols = p.N[s] - n;
  const bool here = n0 < p.N[s], edge = n0 + 16 * NJ > p.N[s];   // (a wavefront without columns still moves its part of h)
  const int kt = (p.rank + 31) / 32;

  auto rows_of = [&](int i) { return *(const int4 *)(w.order + (int64_t)i * 16 + g * 4); };
  auto send_h = [&](int i) {   // 1 KiB operand blocks, as many as the group's adapter has
    const int units = (w.group_slot[2 * i + 1] + 31) / 32 * TERMS;
    const uint32_t into = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)(char *)ring[i & 1]);
    const char *from = (const char *)w.h + ((int64_t)i * p.n_slices + s) * kt * TERMS * 1024 + lane * 16;
    for (int u = wave; u < units; u += LORA_WAVES)
      asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off"
                   ::"s"(into + u * 1024), "v"(from + u * 1024) : "memory", "m0");
  };
  auto load_base = [&](typename O::run_t (&y)[4], int4 rows) {
    const int row[4] = {rows.x, rows.y, rows.z, rows.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p.base) y[i] = O::load((const char *)p.base + ((int64_t)(row[i] < 0 ? 0 : row[i]) * p.ld_base + col0 + n) * O::ES, cols, edge);
      else
#pragma unroll
        for (int k = 0; k < O::WORDS; ++k) y[i][k] = 0;
    }
  };
  auto store = [&](const typename O::run_t (&y)[4], int4 rows) {
    const int row[4] = {rows.x, rows.y, rows.z, rows.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (row[i] >= 0) O::store((char *)p.dst + ((int64_t)row[i] * p.ld_dst + col0 + n) * O::ES, y[i], cols, edge);
  };

  u32x4 b[KT][NJ][F16 ? 2 : 1];
  typename O::run_t y[4], y_next[4], out[4];
  int4 rows = rows_of(a), rows_next = rows_of(a + 1 < z ? a + 1 : a), rows_out = rows;
  int slot = -1, kts = 0;
  float scale = 0.0f;
  send_h(a);
  if (here) load_base(y, rows);
  for (int i = a; i < z; ++i) {
    __builtin_amdgcn_s_waitcnt(0x0f70);   // all that was asked for one group ago
    group_barrier();
    const int4 rows_after = rows_of(i + 2 < z ? i + 2 : z - 1);
    if (i + 1 < z) {
      if (here) load_base(y_next, rows_next);
      send_h(i + 1);
    }
    if (here) {
      if (i > a) store(out, rows_out);
      const int now = __builtin_amdgcn_readfirstlane(w.group_slot[2 * i]);
      if (now != slot) {
        slot = now;
        const int rank = __builtin_amdgcn_readfirstlane(w.group_slot[2 * i + 1]);
        kts = (rank + 31) / 32;
        if (kts) {
          scale = p.scales ? p.scales[slot] : 1.0f;
          load_b<F16, NJ, KT>(p, s, slot, rank, n, b);
        }
      }
      if (kts) {
        f32x4 acc[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < KT; ++c) {
          if (c >= kts) break;
#pragma unroll
          for (int k = 0; k < TERMS; ++k) mma_h<F16, NJ>(acc, *(const u32x4 *)(ring[i & 1] + (c * TERMS + k) * 1024 + lane * 16), b[c], k + 1 == TERMS);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) out[r] = O::sum(y[r], acc, r, scale);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) out[r] = y[r];
      }
    }
    rows_out = rows;
    rows = rows_next;
    rows_next = rows_after;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = y_next[r];
  }
  if (here) store(out, rows_out);
}

// Up to 64 rows: workgroup (x: columns of a slice, y: tile of up to 16 rows); h comes as the K slices' sums.
template <bool F16, int NJ, int KT, int DST>
__global__ __launch_bounds__(LORA_WAVES * 64, 2) void zmi_lora_expand_small_kernel(ZmiLora p, ZmiLoraPlan w, int slices) {
  typedef Out<NJ, DST> O;
  constexpr int TERMS = O::TERMS;
  const int lane = threadIdx.x % 64, g = lane / 16, c16 = lane % 16;
  Tile t;
  if (!lora_find_tile(p, blockIdx.y, t)) return;
  int s = 0, blk = blockIdx.x, col0 = 0;
  while (blk >= (p.N[s] + O::COLS - 1) / O::COLS) {
    blk -= (p.N[s] + O::COLS - 1) / O::COLS;
    col0 += p.N[s++];
  }
  const int n0 = blk * O::COLS + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 16 * NJ;
  if (n0 >= p.N[s]) return;
  const bool none = t.slot == p.n_slots, edge = n0 + 16 * NJ > p.N[s];
  if (none && p.base == p.dst) return;
  const int n = n0 + c16 * NJ, cols = p.N[s] - n;
  int64_t row[4];
  typename O::run_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = g * 4 + i;
    row[i] = __shfl(t.row, at < t.n ? at : 0, 64);
    if (p.base) y[i] = O::load((const char *)p.base + (row[i] * p.ld_base + col0 + n) * O::ES, cols, edge);
    else
#pragma unroll
      for (int k = 0; k < O::WORDS; ++k) y[i][k] = 0;
  }
  if (!none) {
    const int rank = lora_rank(p, t.slot), kts = (rank + 31) / 32, lt = (rank + 15) / 16, qt = p.n_slices * ((p.rank + 15) / 16);
    const float scale = p.scales ? p.scales[t.slot] : 1.0f;
    u32x4 b[KT][NJ][F16 ? 2 : 1];
    load_b<F16, NJ, KT>(p, s, t.slot, rank, n, b);
    f32x4 acc[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < KT; ++c) {
      if (c >= kts) break;
      // ranks (r % 16 / 4) * 16 + row, four to a lane
      float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      const int r = c * 32 + g * 8, left = rank - r;
      if (left > 0 && c16 < t.n) {
        for (int k = 0; k < slices; ++k) {
          const int64_t at = ((int64_t)k * gridDim.y + blockIdx.y) * qt + s * lt + r / 16;
          const f32x4 *src = (const f32x4 *)w.partial + at * 64 + r % 16 / 4 * 16 + c16;
          const f32x4 lo = src[0], hi = src[16];
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
      for (int k = 0; k < TERMS; ++k) mma_h<F16, NJ>(acc, pack8(h[k]), b[c], k + 1 == TERMS);
    }
    if (kts) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = O::sum(y[i], acc, i, scale);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (g * 4 + i < t.n) O::store((char *)p.dst + (row[i] * p.ld_dst + col0 + n) * O::ES, y[i], cols, edge);
}

namespace {

template <bool F16, int KT, int DST>
void launch_as(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream) {
  constexpr int FEW = KT == 8 ? 2 : 4, NJ = F16 || KT == 8 || DST == ZMI_DT_F32 ? FEW : 8;
  const dim3 block(LORA_WAVES * 64);
  if (s.small) hipLaunchKernelGGL((zmi_lora_expand_small_kernel<F16, FEW, KT, DST>), dim3((unsigned)s.col_blocks, (unsigned)s.tiles), block, 0, stream, p, w, s.ks);
  else hipLaunchKernelGGL((zmi_lora_expand_kernel<F16, NJ, KT, DST>), dim3((unsigned)s.col_blocks, (unsigned)s.runs), block, 0, stream, p, w);
}

template <bool F16, int KT>
void launch_dst(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream) {
  if (p.dt_dst == ZMI_DT_F32) launch_as<F16, KT, ZMI_DT_F32>(p, w, s, stream);
  else if (p.dt_dst == ZMI_DT_BF16) launch_as<F16, KT, ZMI_DT_BF16>(p, w, s, stream);
  else launch_as<F16, KT, ZMI_DT_F16>(p, w, s, stream);
}

template <bool F16>
void launch_kt(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream) {
  if (s.kt == 1) launch_dst<F16, 1>(p, w, s, stream);
  else if (s.kt == 2) launch_dst<F16, 2>(p, w, s, stream);
  else if (s.kt == 4) launch_dst<F16, 4>(p, w, s, stream);
  else launch_dst<F16, 8>(p, w, s, stream);
}

}  // namespace

hipError_t lora_launch_expand(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream) {
  if (p.dt_x == ZMI_DT_F16) launch_kt<true>(p, w, s, stream);
  else launch_kt<false>(p, w, s, stream);
  return hipGetLastError();
}
