// The second product of the low-rank adapters (k_lora.hip): dst[t][n] = base[t][n] + scales[a] sum_r h[t][s, r] B_s[a][n][r].
//
// MFMA rows are 16 rows of the batch that share a slot, MFMA columns columns of dst: of column tile j lane l holds column
// n0 + l % 16 * NJ + j of rows (l / 16) * 4 .. +3, so that a lane's NJ columns lie together and 16 lanes take whole lines
// of a row.  (With the operands the other way round 16 neighbouring lanes stand in 16 rows, and the address path of the
// compute unit takes four times as long over every access.)
//
// HBM bounds it: base and dst once, B and h from L2 (2048 rows, 2 x 14336 columns, rank 32: 235 MB of base and dst in 51 us,
// 4.6 TB/s where a large copy reaches 4.9; 8192 rows, 4096 columns, rank 128: 43 us, of which three terms of h instead of two
// are 2 to 3).  Planned calls run down the 16-row groups of the batch with B in
// registers, reloaded where the slot changes; each workgroup takes an equal share of the groups, h of the next group goes
// to LDS and its base to registers while one is computed, and a group's stores go out behind the next group's loads.
#include <type_traits>

#include "zmi_lora.h"

namespace {

template <int NJ, int DST>   // DST: ZMI_DT_*
struct Out {
  static constexpr int ES = DST == ZMI_DT_F32 ? 4 : 2, BYTES = NJ * ES, WORDS = BYTES / 4;
  static constexpr int COLS = LORA_WAVES * 16 * NJ;   // of a workgroup
  typedef uint32_t run_t __attribute__((ext_vector_type(WORDS)));   // a lane's columns of a row

  // EDGE: only `cols` of them are there (of some lanes of the wavefront), none where that is not positive; with eight columns
  // a lane all or none are (the host sees to it)
  template <bool EDGE>
  static __device__ __forceinline__ run_t load(const char *at, int cols) {
    run_t y;
    if (!EDGE) {
      __builtin_memcpy(&y, at, BYTES);
    } else if (NJ == 8) {
#pragma unroll
      for (int k = 0; k < WORDS; ++k) y[k] = 0;
      if (cols > 0) __builtin_memcpy(&y, at, BYTES);
    } else {
      // (the slice's last column in the place of those behind it: no branches, all loads in flight)
      uint32_t v[NJ];
#pragma unroll
      for (int e = 0; e < NJ; ++e) {
        const int i = e < cols ? e : cols - 1;
        v[e] = ES == 4 ? ((const uint32_t *)at)[i] : ((const uint16_t *)at)[i];
      }
#pragma unroll
      for (int k = 0; k < WORDS; ++k) y[k] = ES == 4 ? v[k % NJ] : v[2 * k % NJ] | v[(2 * k + 1) % NJ] << 16;
    }
    return y;
  }
  template <bool EDGE>
  static __device__ __forceinline__ void store(char *at, run_t y, int cols) {
    if (!EDGE || NJ == 8) {
      if (!EDGE || cols > 0) __builtin_memcpy(at, &y, BYTES);
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

// this lane's number, made where it is used (kept over the whole run of a full wavefront it is a register spilled, and reading
// it back waits for all loads ahead)
__device__ __forceinline__ int lane_here() {
  uint32_t all = ~0u;
  asm volatile("" : "+s"(all));
  return __builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0));
}

__device__ __forceinline__ u32x4 pack8(const __bf16 (&v)[8]) {
  return __builtin_bit_cast(u32x4, bf16x8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]});
}

// B of a lane's NJ columns from column n on, as MFMA operands: ranks c * 32 + g * 8 .. +7, zeros from `rank` on
template <bool F16, int NJ, int KT>
__device__ __forceinline__ void load_b(const ZmiLora &p, int s, int slot, int rank, int n, u32x4 (&b)[KT][NJ][F16 ? 2 : 1]) {
  const int g = threadIdx.x % 64 / 16;
  u32x4 v[KT][NJ];
  const uint16_t *from[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) from[j] = (const uint16_t *)p.b[s] + slot * p.b_slot[s] + (n + j < p.N[s] ? n + j : p.N[s] - 1) * p.b_ld[s] + g * 8;
  // (zeros first, then one masked load each: a second writer of the same registers would have to wait for the first)
#pragma unroll
  for (int c = 0; c < KT; ++c) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) v[c][j] = u32x4{0, 0, 0, 0};
    if (rank - c * 32 - g * 8 >= 8) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) v[c][j] = load16(from[j] + c * 32);
    }
  }
  if (rank % 8) {
#pragma unroll
    for (int c = 0; c < KT; ++c) {
      const int left = rank - c * 32 - g * 8;
      if (left > 0 && left < 8) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) v[c][j] = load16_head(from[j] + c * 32, left);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < KT; ++c)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (F16) {   // (every f16 value is the sum of its two terms)
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

// acc += a term of h times B
template <bool F16, int NJ>
__device__ __forceinline__ void mma_h(f32x4 (&acc)[NJ], u32x4 h, const u32x4 (&b)[NJ][F16 ? 2 : 1], bool last) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = mma_x<false>(h, b[j][0], acc[j]);
  // (the last terms' product is at most 2^-25 of the whole one, less than a rounding of the sum)
  if (F16 && !last)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] = mma_x<false>(h, b[j][F16 ? 1 : 0], acc[j]);
}

// An infinite h or B meets zeros and opposite signs among the other operand's terms, which the definition does not know: where
// the terms' products leave NaN, the sum over the ranks is made again from h and B themselves.  h_of(i, r): h of rank r of
// row i of the lane's four.  Not a fast path: rows of NaN, as a padded batch may hold, are let be; a row or column with an
// infinity takes a load for every rank of each of its elements (8192 rows of K=14336, 4096 columns, rank 128: 132 us, with
// NaN in every row 140, an infinity in one row of 16 236, in one column of B 583).
template <bool F16, int NJ, class H>
__device__ __forceinline__ void redo_nan(const ZmiLora &p, int s, int slot, int rank, int n, f32x4 (&acc)[NJ], H h_of) {
  f32x4 top = acc[0];   // (IEEE 754's maximum: NaN where either is)
#pragma unroll
  for (int j = 1; j < NJ; ++j) top = __builtin_elementwise_maximum(top, acc[j]);
  const float any = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top[0], top[1]), __builtin_elementwise_maximum(top[2], top[3]));
  if (__builtin_expect(any == any, 1)) return;
  bool done[4];   // (a NaN in h stays)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float h = h_of(i, 0);
    done[i] = h != h;
  }
  asm volatile("" : "+v"(n));   // (no address of this is made ahead, in registers that the rows in front would lack)
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const uint16_t *b = (const uint16_t *)p.b[s] + slot * p.b_slot[s] + (n + j < p.N[s] ? n + j : p.N[s] - 1) * p.b_ld[s];
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // (one at a time: what is live here adds to what the rows in front keep in registers)
      if (done[i] || acc[j][i] == acc[j][i]) continue;
      float sum = 0.0f;
#pragma unroll 1
      for (int r = 0; r < rank && sum == sum; ++r) sum = __builtin_fmaf(h_of(i, r), F16 ? zmi_f16_to_f32(b[r]) : zmi_bf16_to_f32(b[r]), sum);
      acc[j][i] = sum;
    }
  }
}

}  // namespace

// Planned: workgroup (x: columns of a slice, y: share of the 16-row groups).
template <bool F16, int NJ, int KT, int DST>
__global__ __launch_bounds__(LORA_WAVES * 64, 2) void zmi_lora_expand_kernel(ZmiLora p, ZmiLoraPlan w) {
  typedef Out<NJ, DST> O;
  __shared__ __attribute__((aligned(16))) char ring[2][KT * LORA_TERMS * 1024];
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
    const int units = (w.group_slot[2 * i + 1] + 31) / 32 * LORA_TERMS;
    const uint32_t into = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)(char *)ring[i & 1]);
    const char *from = (const char *)w.h + ((int64_t)i * p.n_slices + s) * kt * LORA_TERMS * 1024 + lane * 16;
    for (int u = wave; u < units; u += LORA_WAVES)
      asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off"
                   ::"s"(into + u * 1024), "v"(from + u * 1024) : "memory", "m0");
  };
  auto run = [&](auto edge_of) {
    constexpr bool EDGE = decltype(edge_of)::value;
    auto load_base = [&](typename O::run_t (&y)[4], int4 rows) {
      const int row[4] = {rows.x, rows.y, rows.z, rows.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (p.base) y[i] = O::template load<EDGE>((const char *)p.base + ((int64_t)(row[i] < 0 ? 0 : row[i]) * p.ld_base + col0 + n) * O::ES, cols);
        else
#pragma unroll
          for (int k = 0; k < O::WORDS; ++k) y[i][k] = 0;
      }
    };
    auto store = [&](const typename O::run_t (&y)[4], int4 rows) {
      const int row[4] = {rows.x, rows.y, rows.z, rows.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row[i] >= 0) O::template store<EDGE>((char *)p.dst + ((int64_t)row[i] * p.ld_dst + col0 + n) * O::ES, y[i], cols);
    };

    u32x4 b[KT][NJ][F16 ? 2 : 1];
    typename O::run_t y[4], y_next[4], out[4];
    int4 rows = rows_of(a), rows_next = rows_of(a + 1 < z ? a + 1 : a), rows_out = rows;
    int slot = -1, rank = 0, kts = 0;
    float scale = 0.0f;
    auto take_slot = [&](int i) {
      const int now = __builtin_amdgcn_readfirstlane(w.group_slot[2 * i]);
      if (now == slot) return;
      slot = now;
      rank = __builtin_amdgcn_readfirstlane(w.group_slot[2 * i + 1]);
      kts = (rank + 31) / 32;
      if (!kts) return;
      scale = p.scales ? p.scales[slot] : 1.0f;
      load_b<F16, NJ, KT>(p, s, slot, rank, n, b);
      __builtin_amdgcn_s_waitcnt(0x0f70);   // (waited for here, B holds up no group of the same slot until the loads ahead are back)
    };
    send_h(a);
    if (here) {
      load_base(y, rows);
      take_slot(a);
    }
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
        take_slot(i);
        if (kts) {
          const char *const h_at = ring[i & 1] + lane_here() * 16;
          f32x4 acc[NJ];
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < KT; ++c) {
            if (c >= kts) break;
#pragma unroll
            for (int k = 0; k < LORA_TERMS; ++k) mma_h<F16, NJ>(acc, *(const u32x4 *)(h_at + (c * LORA_TERMS + k) * 1024), b[c], k + 1 == LORA_TERMS);
          }
          redo_nan<F16, NJ>(p, s, slot, rank, n, acc, [&](int q, int r) {
            const char *at = ring[i & 1] + r / 32 * LORA_TERMS * 1024 + (r / 8 % 4 * 16 + g * 4 + q) * 16 + r % 8 * 2;
            float h = 0.0f;
#pragma unroll
            for (int k = LORA_TERMS - 1; k >= 0; --k) h += zmi_bf16_to_f32(*(const uint16_t *)(at + k * 1024));
            return h;
          });
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
  };
  if (edge) run(std::true_type());   // (the barriers of either are the same ones)
  else run(std::false_type());
}

// Calls without a plan launch: workgroup (x: columns of a slice, y: tile of up to 16 rows); h comes as the K slices' sums.
// Latency bounds it, the chain from the tile's entry over B and the sums to dst: 4.9 us for one row of 4096 columns at rank
// 16, 10.4 us for 48 rows of 6144 columns at rank 64, whose B alone is 16 MB.
template <bool F16, int NJ, int KT, int DST>
__global__ __launch_bounds__(LORA_WAVES * 64, 2) void zmi_lora_expand_small_kernel(ZmiLora p, ZmiLoraPlan w, int slices) {
  typedef Out<NJ, DST> O;
  const int lane = threadIdx.x % 64, g = lane / 16, c16 = lane % 16;
  // the tile as the shrink launch found it
  const int32_t *entry = w.tiles + blockIdx.y * 20;
  const int4 e = *(const int4 *)entry, rows = *(const int4 *)(entry + 4 + g * 4);
  const int slot = __builtin_amdgcn_readfirstlane(e.x), count = __builtin_amdgcn_readfirstlane(e.y), rank = __builtin_amdgcn_readfirstlane(e.z);
  if (!count) return;
  int s = 0, blk = blockIdx.x, col0 = 0;
  while (blk >= (p.N[s] + O::COLS - 1) / O::COLS) {
    blk -= (p.N[s] + O::COLS - 1) / O::COLS;
    col0 += p.N[s++];
  }
  const int n0 = blk * O::COLS + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 16 * NJ;
  if (n0 >= p.N[s]) return;
  const bool none = slot == p.n_slots, edge = n0 + 16 * NJ > p.N[s];
  if (none && p.base == p.dst) return;
  const int n = n0 + c16 * NJ, cols = p.N[s] - n;
  const int row[4] = {rows.x, rows.y, rows.z, rows.w};
  auto run = [&](auto edge_of) {
    constexpr bool EDGE = decltype(edge_of)::value;
    typename O::run_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p.base) y[i] = O::template load<EDGE>((const char *)p.base + ((int64_t)(row[i] < 0 ? 0 : row[i]) * p.ld_base + col0 + n) * O::ES, cols);
      else
#pragma unroll
        for (int k = 0; k < O::WORDS; ++k) y[i][k] = 0;
    }
    if (!none) {
      const int kts = (rank + 31) / 32, lt = (rank + 15) / 16, qt = p.n_slices * ((p.rank + 15) / 16);
      const float scale = p.scales ? p.scales[slot] : 1.0f;
      u32x4 b[KT][NJ][F16 ? 2 : 1];
      load_b<F16, NJ, KT>(p, s, slot, rank, n, b);
      f32x4 acc[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < KT; ++c) {
        if (c >= kts) break;
        // ranks (r % 16 / 4) * 16 + row, four to a lane
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const int r = c * 32 + g * 8, left = rank - r;
        if (left > 0 && c16 < count) {
          const f32x4 *src = (const f32x4 *)w.partial + ((int64_t)blockIdx.y * qt + s * lt + r / 16) * 64 + r % 16 / 4 * 16 + c16;
          const int64_t step = (int64_t)gridDim.y * qt * 64;
          for (int k0 = 0; k0 < slices; k0 += 4) {   // (four slices' sums in flight)
            f32x4 part[4][2];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const f32x4 *at = src + (k0 + k < slices ? k0 + k : k0) * step;
              part[k][0] = at[0];
              part[k][1] = at[16];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                v[e] += k0 + k < slices ? part[k][0][e] : 0.0f;
                v[4 + e] += k0 + k < slices ? part[k][1][e] : 0.0f;
              }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e >= left) v[e] = 0.0f;
        }
        __bf16 h[LORA_TERMS][8];
        split<LORA_TERMS>(v, h);
#pragma unroll
        for (int k = 0; k < LORA_TERMS; ++k) mma_h<F16, NJ>(acc, pack8(h[k]), b[c], k + 1 == LORA_TERMS);
      }
      redo_nan<F16, NJ>(p, s, slot, rank, n, acc, [&](int i, int r) {
        if (g * 4 + i >= count) return 0.0f;
        const float *src = w.partial + (((int64_t)blockIdx.y * qt + s * lt + r / 16) * 64 + r % 16 / 4 * 16 + g * 4 + i) * 4 + r % 4;
        float h = 0.0f;
        for (int k = 0; k < slices; ++k) h += src[(int64_t)k * gridDim.y * qt * 256];
        return h;
      });
      if (kts) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = O::sum(y[i], acc, i, scale);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (row[i] >= 0) O::template store<EDGE>((char *)p.dst + ((int64_t)row[i] * p.ld_dst + col0 + n) * O::ES, y[i], cols);
  };
  if (edge) run(std::true_type());
  else run(std::false_type());
}

namespace {

template <bool F16, int KT, int DST>
void launch_as(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream) {
  constexpr int FEW = KT == 8 ? 2 : 4;
  const dim3 block(LORA_WAVES * 64);
  if (s.small) {
    hipLaunchKernelGGL((zmi_lora_expand_small_kernel<F16, FEW, KT, DST>), dim3((unsigned)s.col_blocks, (unsigned)s.tiles), block, 0, stream, p, w, s.ks);
    return;
  }
  const dim3 grid((unsigned)s.col_blocks, (unsigned)s.runs);
  if constexpr (KT <= (F16 ? 1 : 4) && DST != ZMI_DT_F32) {
    if (s.nj == 8) {
      hipLaunchKernelGGL((zmi_lora_expand_kernel<F16, 8, KT, DST>), grid, block, 0, stream, p, w);
      return;
    }
  }
  hipLaunchKernelGGL((zmi_lora_expand_kernel<F16, FEW, KT, DST>), grid, block, 0, stream, p, w);
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
