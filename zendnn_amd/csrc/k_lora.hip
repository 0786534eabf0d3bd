// Low-rank adapters of many requests beside a shared projection (gfx950); see zmi_lowoha.h.
//
//   h[t][s, r] = sum_k x[t][k] A[a][s rank + r][k],  dst[t][n] = base[t][n] + scales[a] sum_r h[t][s, r] B_s[a][n][r]
//
// with a = slot_ids[t].  Per byte that has to move (x, dst, base, the used slots' A and B) there are at most `rank`
// multiply-adds, so HBM bounds every size, and latency the small ones.  Rows of one slot are gathered into tiles of
// 16 RT rows, so that a tile reads its slot's A and B once and both products run on the 16 x 16 x 32 MFMA:
//
//   plan    (many rows) one workgroup sorts the rows by slot and lists the tiles; with few rows every
//           wavefront finds its tile by itself from a ballot per distinct id, and there is no such launch;
//   shrink  h of a tile, K through an LDS ring.  K is cut into slices where the tiles alone do not fill the device;
//   expand  dst.  A wavefront keeps 32 .. 128 columns' B in registers and goes down the rows of its slot.
//
// The MFMA takes 16-bit operands: x, A exactly as they are; h, which is f32, as a sum of three bf16 terms, which hold all of
// its 24 bits (down to bf16's least value, 2^-133), and f16 B, which the range of h does not allow to meet in f16, as two bf16
// terms that hold it exactly.  All products are accumulated in f32.
#include "zmi_lora.h"

#define LORA_RUN 4   // least stages of a shrink workgroup's run

namespace {

extern __shared__ __attribute__((aligned(16))) char lora_smem[];

}  // namespace

// ---------------------------------------------------------------------------------------------------------------
// plan: the rows of each slot, in the batch's order (so that a call repeats its bits), in groups of 16, -1 in the last one's
// empty places, and the shrink launch's tiles of up to `tile` rows; rows without an adapter come last.
//
// `waves` wavefronts of the one workgroup walk a contiguous share of the batch each, 64 rows at a time, and count per slot
// in their own row of LDS; a row's place is its slot's count plus the number of lower lanes with the same slot.  Latency bounds
// it: 5.8 us for 2048 rows of 8 slots, 11 for 8192; rows beyond those that stay in registers cost a memory latency for every 64
// of a wavefront, 39 us for 32768 (of 2048 slots, which leave LDS for fewer wavefronts' counts: 21, 59 and 208).
// ---------------------------------------------------------------------------------------------------------------
#define LORA_PLAN_KEEP 8   // rows a lane keeps between the passes

__global__ __launch_bounds__(1024) void zmi_lora_plan_kernel(ZmiLora p, ZmiLoraPlan w, int tile, int waves) {
  __shared__ int wave_sums[2][16];
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = p.n_slots + 1;
  int4 *of = (int4 *)lora_smem;                // [n]
  int *count = (int *)(lora_smem + n * 16);   // [waves][n]
  const int share = (p.T + waves * 64 - 1) / (waves * 64) * 64;   // rows of a wavefront
  const int t0 = wave < waves ? wave * share : p.T, t1 = t0 + share < p.T ? t0 + share : p.T;
  auto slot_of = [&](int t, int raw) { return t >= t1 ? -1 : (unsigned)raw < (unsigned)p.n_slots ? raw : p.n_slots; };
  int id[LORA_PLAN_KEEP], pos[LORA_PLAN_KEEP];
#pragma unroll
  for (int i = 0; i < LORA_PLAN_KEEP; ++i) {   // (all loads in flight: no branch in front of them)
    const int t = t0 + i * 64 + lane;
    id[i] = p.slot_ids[t < p.T ? t : p.T - 1];
  }
  for (int i = tid; i < waves * n; i += 1024) count[i] = 0;
  for (int i = tid; i < w.n_arrivals; i += 1024) w.arrivals[i] = 0;
  __syncthreads();
  constexpr int MOST = (ZMI_LORA_MAX_SLOTS + 1 + 1023) / 1024;   // slots of a thread
  int total[MOST], rank[MOST];
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    const int i = tid * ((n + 1023) / 1024) + k;
    rank[k] = k < (n + 1023) / 1024 && i < p.n_slots ? lora_rank(p, i) : 0;
  }
#pragma unroll
  for (int i = 0; i < LORA_PLAN_KEEP; ++i) id[i] = slot_of(t0 + i * 64 + lane, id[i]);
  const int bits = 32 - __builtin_clz(n);
  int *mine = count + (wave < waves ? wave : 0) * n;
  auto place = [&](int slot) {
    uint64_t same = __ballot(slot >= 0);
    for (int b = 0; b < bits; ++b) {
      const uint64_t one = __ballot((slot >> b) & 1);
      same &= (slot >> b) & 1 ? one : ~one;
    }
    int at = 0;
    if (slot >= 0) {
      at = mine[slot] + __popcll(same & ((1ull << lane) - 1));
      // (LDS serves a wavefront in order: everybody has read before the last lane of each slot writes)
      if (same >> lane == 1) mine[slot] = at + 1;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (other lanes' writes are read by the next 64 rows)
    return at;
  };
#pragma unroll
  for (int i = 0; i < LORA_PLAN_KEEP; ++i)
    if (t0 + i * 64 < t1) pos[i] = place(id[i]);
  for (int t = t0 + LORA_PLAN_KEEP * 64; t < t1; t += 64) {
    const int at = place(slot_of(t + lane, p.slot_ids[t + lane < p.T ? t + lane : p.T - 1]));
    if (t + lane < t1) w.place[t + lane] = at;
  }
  __syncthreads();
  // thread i owns slots [i per, (i + 1) per)
  const int per = (n + 1023) / 1024;
  int sums[2] = {0, 0};   // 16-row groups, tiles
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    const int i = tid * per + k;
    total[k] = 0;
    if (k >= per || i >= n) continue;
    int c = 0, own[16];   // its rows; a wavefront's count becomes the number of rows before its own
#pragma unroll
    for (int v = 0; v < 16; ++v) own[v] = v < waves ? count[v * n + i] : 0;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      if (v < waves) count[v * n + i] = c;
      c += own[v];
    }
    total[k] = c;
    sums[0] += (c + 15) / 16;
    sums[1] += (c + tile - 1) / tile;
  }
  int start[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int v = lora_running_sum(sums[k]);
    if (lane == 63) wave_sums[k][wave] = v;
    start[k] = v - sums[k];
  }
  if (n > 64) {   // (else the first wavefront has all slots)
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) start[k] += i < wave ? wave_sums[k][i] : 0;
  }
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    const int i = tid * per + k;
    if (k >= per || i >= n) continue;
    of[i] = make_int4(start[0], start[1], total[k], rank[k]);
    start[0] += (total[k] + 15) / 16;
    if (i == p.n_slots) {   // (the rows without an adapter)
      w.header[0] = start[1];
      w.header[1] = start[0] - (total[k] + 15) / 16;
      w.header[2] = start[0];
    }
    start[1] += (total[k] + tile - 1) / tile;
  }
  __syncthreads();
  // every row to its place; the first of a group or tile writes its entry, a slot's last row the empty places behind it
  auto put = [&](int t, int slot, int at) {
    const int4 o = of[slot];   // first group, first tile, rows, rank
    const int q = mine[slot] + at;
    w.order[(int64_t)o.x * 16 + q] = t;
    if (q % 16 == 0) *(int2 *)(w.group_slot + 2 * (int64_t)(o.x + q / 16)) = make_int2(slot, o.w);
    if (q % tile == 0 && slot < p.n_slots) *(int4 *)(w.tiles + 4 * (int64_t)(o.y + q / tile)) = make_int4(slot, o.x + q / 16, o.z - q < tile ? o.z - q : tile, o.w);
    if (q == o.z - 1)
      for (int j = q + 1; j % 16; ++j) w.order[(int64_t)o.x * 16 + j] = -1;
  };
  // (each lane reads back the places that it wrote itself)
  for (int t = t0 + LORA_PLAN_KEEP * 64 + lane; t < t1; t += 64) put(t, slot_of(t, p.slot_ids[t]), w.place[t]);
#pragma unroll
  for (int i = 0; i < LORA_PLAN_KEEP; ++i)
    if (id[i] >= 0) put(t0 + i * 64 + lane, id[i], pos[i]);
}

// ---------------------------------------------------------------------------------------------------------------
// shrink: h of a tile's rows by NT rank tiles of 16, over a run of K.  MFMA rows are ranks, columns the tile's rows: lane
// l holds ranks (l / 16) * 4 .. +3 of row l % 16.  Rank tiles are numbered over the live ones of all slices (an adapter
// of a smaller rank has fewer); ranks and rows beyond the last one repeat it and are dropped.
//
// K goes through an LDS ring of D stages of KS elements: x rows and A rows alike are moved in units of 8 rows x 128
// bytes, one 16-byte piece a lane.  (MFMA operands read from global memory directly put 16 rows under 16 neighbouring
// lanes: every 16 bytes an access of its own, and the compute unit's address path, not HBM, sets the pace: 148 us for
// 8192 rows of K = 14336 at rank 128 against 78 us through LDS.)  Piece c of row r stands at slot c ^ (r % 8), which
// spreads the operand reads over the banks.  With rows, strides and addresses of 16-byte multiples the units are moved
// by global -> LDS loads (DMA), D - 1 stages ahead; otherwise through registers, one stage ahead.
// The four wavefronts share a stage as WR x WN x WK over row groups, rank tiles and 64-element blocks of K.
//
// What bounds it: the cache lines a compute unit can have outstanding.  In the 78 us above 4.3 M lines of 128 bytes (206 MB
// of x, 346 MB of A read again by every tile; 71 % of the accesses that L2 counts are misses) are read with a latency of 806 clocks
// on average, which is some 70 lines in flight in a compute unit (at 2.4 GHz); without its arithmetic the launch takes the
// same 78 us, with all loads but the first stages' left out 54.  2048 rows of K = 4096, two slices of rank 32: 13 us for
// 16 MB of x and A.
// ---------------------------------------------------------------------------------------------------------------
template <bool F16, int RT, int NT, int KS, int WR, int WN, int D, bool DMA, bool SMALL>
__global__ __launch_bounds__(LORA_WAVES * 64, 2) void zmi_lora_shrink_kernel(ZmiLora p, ZmiLoraPlan w, int ny) {
  constexpr int WK = LORA_WAVES / (WR * WN), RW = RT / WR, NW = NT / WN;
  constexpr int BLOCKS = KS / 64;                       // 64-element blocks of a stage
  constexpr int UNITS = (RT + NT) * 2 * BLOCKS;         // 1 KiB each, [block][8 rows]
  constexpr int OPS = (UNITS + LORA_WAVES - 1) / LORA_WAVES;
  constexpr int STAGE = UNITS * 1024;
  static_assert(BLOCKS % WK == 0 && (D - 2) * OPS < 64, "blocks split over wavefronts; the wait counter");
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), g = lane / 16, c16 = lane % 16;
  const int stages = (p.K + KS - 1) / KS, full = p.K / KS, qt = p.n_slices * ((p.rank + 15) / 16);
  // Planned: the units (tile, group of rank tiles) x stages are cut into as many equal runs as there are workgroups, so that
  // every compute unit has the same to move; a unit's pieces meet below.  Workgroups go to the eight XCDs in turn, and each
  // XCD takes a contiguous eighth of the runs, so that a slot's A is read into few L2s.
  const int me = SMALL ? 0 : blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
  const int all = SMALL ? 0 : __builtin_amdgcn_readfirstlane(w.header[0]) * ny * stages;   // (below 2^31: zmi_api_lora.hip)
  const int run = all > 0 ? (all - 1) / (int)gridDim.x + 1 : 1;
  const int begin = me * run < all ? me * run : all, end = begin + run < all ? begin + run : all;
  int unit = SMALL ? 0 : begin / stages;
  do {
    if (!SMALL && unit * stages >= end) return;
    Tile t;
    int q0, s0, s1;
    if (SMALL) {
      const bool found = lora_find_tile(p, blockIdx.x, t);
      if (blockIdx.y == 0 && blockIdx.z == 0 && wave == 0) {   // the expand launch's entry: {slot, rows, rank, -}, 16 rows
        int32_t *e = w.tiles + blockIdx.x * 20;
        if (lane == 0) *(int4 *)e = found ? make_int4(t.slot, t.n, t.slot < p.n_slots ? lora_rank(p, t.slot) : 0, 0) : make_int4(0, 0, 0, 0);
        if (found && lane < 16) e[4 + lane] = lane < t.n ? t.row : -1;
      }
      if (!found || t.slot == p.n_slots) return;
      q0 = blockIdx.y * NT;
      s0 = (int)((int64_t)stages * blockIdx.z / gridDim.z);
      s1 = (int)((int64_t)stages * (blockIdx.z + 1) / gridDim.z);
    } else {
      const int *e = w.tiles + unit / ny * 4;
      t.slot = __builtin_amdgcn_readfirstlane(e[0]);
      t.group = __builtin_amdgcn_readfirstlane(e[1]);
      t.n = __builtin_amdgcn_readfirstlane(e[2]);
      q0 = unit % ny * NT;
      s0 = begin > unit * stages ? begin - unit * stages : 0;
      s1 = end < (unit + 1) * stages ? end - unit * stages : stages;
    }
    const int rank = SMALL ? lora_rank(p, t.slot) : __builtin_amdgcn_readfirstlane(w.tiles[unit / ny * 4 + 3]), lt = (rank + 15) / 16, live = lt * p.n_slices;
    if (q0 >= live) {
      if (SMALL) return;
      ++unit;
      continue;
    }
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
        const int row = SMALL ? __shfl(t.row, at, 64) : w.order[(int64_t)t.group * 16 + at];
        from[i] = (const uint16_t *)p.x + row * p.ldx;
      } else {
        const int q = q0 + (r - RT * 16) / 16 < live ? q0 + (r - RT * 16) / 16 : live - 1, s = q / lt;
        const int k = (q - s * lt) * 16 + r % 16;
        from[i] = (const uint16_t *)p.a + t.slot * p.a_slot + (s * p.rank + (k < rank ? k : rank - 1)) * p.a_ld;
      }
      from[i] += block * 64 + piece * 8;
    }
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
    auto left = [&](int i, int k) {   // elements of K from this lane's piece on
      const int u = wave + i * LORA_WAVES < UNITS ? wave + i * LORA_WAVES : UNITS - 1;
      return p.K - k - u / ((RT + NT) * 2) * 64 - (lane % 8 ^ (lane / 8)) * 8;
    };
    auto fetch = [&](int s) {
      const int64_t k = (int64_t)s * KS;
      if (s < full) {
#pragma unroll
        for (int i = 0; i < OPS; ++i) reg[i] = load16(from[i] + k);
      } else {
#pragma unroll
        for (int i = 0; i < OPS; ++i) {
          reg[i] = u32x4{0, 0, 0, 0};
          if (left(i, (int)k) >= 8) reg[i] = load16(from[i] + k);
        }
        if (p.K % 8) {
#pragma unroll
          for (int i = 0; i < OPS; ++i)
            if (left(i, (int)k) > 0 && left(i, (int)k) < 8) reg[i] = load16_head(from[i] + k, left(i, (int)k));
        }
      }
    };
    auto put = [&](int slot) {
#pragma unroll
      for (int i = 0; i < OPS; ++i) *(u32x4 *)(lora_smem + slot * STAGE + into[i] + lane * 16) = reg[i];
    };
    if (!SMALL) group_barrier();   // (the ring and the sums of the piece before are read)
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
      __bf16 h[LORA_TERMS][4];
      split<LORA_TERMS>(f, h);
      char *to = (char *)w.h + ((((int64_t)(t.group + i) * p.n_slices + s) * kt + r / 32) * LORA_TERMS) * 1024 +
                 (r / 8 % 4 * 16 + c16) * 16 + r % 8 * 2;
#pragma unroll
      for (int k = 0; k < LORA_TERMS; ++k) {
        *(bf16x4 *)(to + k * 1024) = bf16x4{h[k][0], h[k][1], h[k][2], h[k][3]};
        // (a block whose upper half no rank tile fills)
        if (q - s * lt == lt - 1 && lt % 2) *(u32x2 *)(to + k * 1024 + 512) = u32x2{0, 0};
      }
    };
    // where a piece's sums stand: small [K slice][tile][rank tile][lane], planned a workgroup's first and last piece
    auto small_at = [&](int q) { return w.partial + ((((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * qt + q) * 64 + lane) * 4; };
    auto piece_at = [&](int who, int i, int j) {
      const int64_t at = who * 2 + (who * run < unit * stages);
      return w.partial + ((at * (RT * NT) + j * RT + i) * 64 + lane) * 4;
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
    const bool whole = s0 == 0 && s1 == stages;
    if (wk == 0) {
#pragma unroll
      for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < NW; ++j) {
          const int rg = wr * RW + i, q = q0 + wn * NW + j;
          if (q >= live || rg * 16 >= t.n) continue;
          const f32x4 v = acc[i][j];
          if (SMALL) {
            *(f32x4 *)small_at(q) = v;
          } else if (whole) {
            finish(rg, q, v);
          } else {
            // (written through to device scope, so that the piece that arrives last can read it: see below)
            uint64_t *to = (uint64_t *)piece_at(me, rg, wn * NW + j);
            __hip_atomic_store(to, __builtin_bit_cast(uint64_t, u32x2{__float_as_uint(v[0]), __float_as_uint(v[1])}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(to + 1, __builtin_bit_cast(uint64_t, u32x2{__float_as_uint(v[2]), __float_as_uint(v[3])}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
        }
    }
    if (SMALL) return;
    if (!whole) {
      // The piece that arrives last at the unit's word adds all pieces' sums, in order, and leaves the operands.
      const int lo = unit * stages / run, hi = ((unit + 1) * stages - 1) / run;
      wait_loads<0>();   // (stores count as well)
      group_barrier();
      int *is_last = (int *)lora_smem;
      if (threadIdx.x == 0)
        *is_last = __hip_atomic_fetch_add(w.arrivals + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(hi - lo);
      __syncthreads();
      if (*is_last) {
        // (a wavefront's fragments of two pieces are asked for together: the loads are what this takes)
        constexpr int MINE = (RT * NT + LORA_WAVES - 1) / LORA_WAVES;
        f32x4 v[MINE];
#pragma unroll
        for (int f = 0; f < MINE; ++f) v[f] = f32x4{0, 0, 0, 0};
        for (int who = lo; who <= hi; who += 2) {
          u32x4 got[2][MINE];
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int f = 0; f < MINE; ++f) {
              const int at = wave + f * LORA_WAVES < RT * NT ? wave + f * LORA_WAVES : RT * NT - 1;
              const uint64_t *src = (const uint64_t *)piece_at(who + k <= hi ? who + k : hi, at % RT, at / RT);
              const u32x2 a = __builtin_bit_cast(u32x2, __hip_atomic_load(src, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
              const u32x2 b = __builtin_bit_cast(u32x2, __hip_atomic_load(src + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
              got[k][f] = u32x4{a[0], a[1], b[0], b[1]};
            }
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int f = 0; f < MINE; ++f)
              if (who + k <= hi) v[f] += __builtin_bit_cast(f32x4, got[k][f]);
        }
#pragma unroll
        for (int f = 0; f < MINE; ++f) {
          const int at = wave + f * LORA_WAVES, i = at % RT, q = q0 + at / RT;
          if (at < RT * NT && q < live && i * 16 < t.n) finish(i, q, v[f]);
        }
      }
    }
    ++unit;
  } while (true);
}

// ---------------------------------------------------------------------------------------------------------------
namespace {

// elements of K in a stage of the shrink launch: a stage is 16 .. 24 KiB whatever the tile's shape
constexpr int lora_ks(int rt, int nt) { return rt + nt <= 3 ? 256 : rt + nt <= 6 ? 128 : 64; }

int64_t lora_clamp(int64_t v, int64_t lo, int64_t hi) { return v > hi ? (hi < lo ? lo : hi) : v < lo ? lo : v; }

// most K slices of a small call: see lora_shape
int64_t lora_small_slices(int64_t stages) { return lora_clamp(stages >= 16 ? stages / 4 : stages, 1, 16); }

LoraShape lora_shape(const ZmiLora &p) {
  LoraShape s = {};
  s.small = p.T <= LORA_SMALL_T || (p.T <= LORA_SMALL_MOST && p.n_slots <= LORA_SMALL_SLOTS && p.rank * p.n_slices <= LORA_SMALL_RANKS);
  const int64_t ids = p.T < p.n_slots + 1 ? p.T : p.n_slots + 1;
  const int qt = p.n_slices * ((p.rank + 15) / 16);
  // (small calls: four rank tiles fit the live ones of a smaller adapter better, and take fewer K slices: 48 rows, three slices
  // of rank 64, both launches 22.2 us with eight, 20.8 with four)
  s.nt = qt >= 8 && !s.small ? 8 : qt > 2 ? 4 : qt;
  s.ny = (qt + s.nt - 1) / s.nt;
  // Tall tiles read A less often, low ones leave fewer pieces of a tile to join: half as many row groups as rank tiles, more
  // while there are two tiles a workgroup, and no more than the slots' rows fill on average (2048 rows of K = 4096, 1 / 2 / 4
  // groups: rank 8 8.1 / 9.0 / 11.2 us, rank 64 15.1 / 12.9 / 15.5; 8192 rows of K = 14336, rank 128: 132 / 95 / 78).
  const int64_t avg = p.T / ids;
  const int most = s.small || avg < 20 ? 1 : avg < 48 ? 2 : 4;
  s.rt = s.nt / 2 < 1 ? 1 : s.nt / 2 < most ? s.nt / 2 : most;
  while (s.rt < most && p.T / (32 * s.rt) * s.ny >= 512) s.rt *= 2;
  const auto tiles_of = [&](int rt) { return ids + (p.T - ids) / (16 * rt); };
  // Low ones again where there are few: 256 workgroups cut less than 64 units into more than four pieces each, which one
  // workgroup joins (4 / 2 / 1 groups at rank 128: 322 rows of K = 1120 in one slot 17.3 / 12.1 / 9.6 us, 976 of 10368 in 12
  // 27.4 / 21.6 / 20.4, 2048 of 4096 in 4 20.3 / 17.2 / 16.6; 2 / 1 at rank 64: 1024 of 4096 in 8 12.8 / 9.3; where there are
  // 64 it turns: two slices of rank 32, 2048 of 4096 in 4, 12.9 / 15.1).
  while (s.rt > 1 && tiles_of(s.rt) * s.ny < 64) s.rt /= 2;
  s.tiles = tiles_of(s.rt);
  s.groups = ids + (p.T - ids) / 16;
  const int64_t stages = (p.K + lora_ks(s.rt, s.nt) - 1) / lora_ks(s.rt, s.nt);
  // small: K slices of four stages or more (of one where K has few: 301 rows of K = 1001 7.6 us in four slices, 8.6 in one)
  // while there are less than two workgroups a compute unit (48 rows, 64 slots, three slices of rank 64 in eights of rank
  // tiles, both launches: 256 workgroups 23.8 us, 512 22.4, 1024 28.5)
  s.ks = (int)lora_clamp(512 / (s.tiles * s.ny), 1, lora_small_slices(stages));
  // planned: a workgroup a compute unit (two share what one already gets through: 512 workgroups 90 us against 82 for 8192
  // rows of K = 14336 at rank 128, 33 against 21 us for 2048 rows of K = 4096), runs of LORA_RUN stages or more (of two up
  // to 128 workgroups)
  const int64_t all = s.tiles * s.ny * stages, few = lora_clamp(all / 2, 8, 128);
  s.grid = (int)lora_clamp(all / LORA_RUN, few, 256) / 8 * 8;
  s.dma = p.ldx % 8 == 0 && p.a_ld % 8 == 0 && p.a_slot % 8 == 0 && (uintptr_t)p.x % 16 == 0 && (uintptr_t)p.a % 16 == 0;
  s.kt = p.rank <= 32 ? 1 : p.rank <= 64 ? 2 : p.rank <= 128 ? 4 : 8;
  // columns of an expand lane: eight, where the registers hold B of so many and every slice's columns are whole eights (f16,
  // whose B takes two terms, up to rank 32, four / eight: 2593 rows of 5104 columns at rank 32 25.6 / 20.9 us, 1416 of 9480 at
  // rank 1 21.5 / 17.0, 1937 of 2792 at rank 24 13.9 / 15.9; with rank 64 eight would gain nothing: 4096 of 4096 24.8 / 25.4,
  // 600 of 4096 11.2 / 13.0)
  bool eights = !s.small && p.dt_dst != ZMI_DT_F32 && s.kt <= (p.dt_x == ZMI_DT_BF16 ? 4 : 1);
  for (int i = 0; i < p.n_slices; ++i) eights &= p.N[i] % 8 == 0;
  s.nj = s.kt == 8 ? 2 : eights ? 8 : 4;
  s.col_blocks = 0;
  const int cols = LORA_WAVES * 16 * s.nj;
  for (int i = 0; i < p.n_slices; ++i) s.col_blocks += (p.N[i] + cols - 1) / cols;
  // (two expand workgroups a compute unit; a run's B is loaded once a slot)
  s.runs = lora_clamp(512 / s.col_blocks, 1, s.groups);
  return s;
}

size_t pad256(size_t n) { return (n + 255) / 256 * 256; }

// workspace of a small call with that many pairs of a tile and a K slice
size_t lora_small_bytes(const ZmiLora &p, const LoraShape &s, int64_t parts) {
  return pad256((size_t)s.tiles * 80) + pad256((size_t)parts * p.n_slices * ((p.rank + 15) / 16) * 1024);
}

// the parts of the workspace; base null: only the size is wanted
size_t lora_layout(const ZmiLora &p, const LoraShape &s, char *base, ZmiLoraPlan *w) {
  size_t at = 0;
  auto take = [&](size_t n) { char *q = base + at; at += pad256(n); return q; };
  const size_t qt = (size_t)p.n_slices * ((p.rank + 15) / 16);
  ZmiLoraPlan l = {};
  if (!s.small) {
    l.header = (int32_t *)take(16);
    l.tiles = (int32_t *)take((size_t)s.tiles * 16);
    l.group_slot = (int32_t *)take((size_t)s.groups * 8);
    l.order = (int32_t *)take((size_t)s.groups * 64);
    l.place = (int32_t *)take(p.T > LORA_PLAN_KEEP * 256 ? (size_t)p.T * 4 : 0);
    l.n_arrivals = (int32_t)(s.tiles * s.ny);
    l.arrivals = (uint32_t *)take((size_t)l.n_arrivals * 4);
    l.h = take((size_t)s.groups * p.n_slices * ((p.rank + 31) / 32) * LORA_TERMS * 1024);
    l.partial = (float *)take((size_t)s.grid * 2 * s.rt * s.nt * 1024);
  } else {
    l.tiles = (int32_t *)take((size_t)s.tiles * 80);
    l.partial = (float *)take((size_t)s.ks * s.tiles * qt * 1024);
  }
  if (w) *w = l;
  return at;
}

template <bool F16, int RT, int NT, int WR, int WN, bool SMALL>
hipError_t launch_shrink_as(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream) {
  constexpr int KS = lora_ks(RT, NT), STAGE = (RT + NT) * 32 * KS, D = STAGE <= 18432 ? 4 : 3;
  static_assert(LORA_WAVES / (WR * WN) * WR * WN == LORA_WAVES && D * STAGE <= 80 * 1024, "two workgroups a compute unit");
  const dim3 grid = SMALL ? dim3((unsigned)s.tiles, (unsigned)s.ny, (unsigned)s.ks) : dim3((unsigned)s.grid), block(LORA_WAVES * 64);
  if (s.dma) {
    const auto kernel = zmi_lora_shrink_kernel<F16, RT, NT, KS, WR, WN, D, true, SMALL>;
    const hipError_t e = zmi_func_smem_once((const void *)kernel, D * STAGE);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, grid, block, D * STAGE, stream, p, w, s.ny);
  } else {
    const auto kernel = zmi_lora_shrink_kernel<F16, RT, NT, KS, WR, WN, D, false, SMALL>;
    hipLaunchKernelGGL(kernel, grid, block, 2 * STAGE, stream, p, w, s.ny);
  }
  return hipGetLastError();
}

template <bool F16, int RT, bool SMALL>
hipError_t launch_shrink(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream) {
  constexpr int R2 = RT >= 2 ? 2 : 1;
  if (s.nt == 1) return launch_shrink_as<F16, RT, 1, RT, 1, SMALL>(p, w, s, stream);
  if (s.nt == 2) return launch_shrink_as<F16, RT, 2, RT, RT == 2 ? 2 : 1, SMALL>(p, w, s, stream);
  if constexpr (!SMALL)
    if (s.nt == 8) return launch_shrink_as<F16, RT, 8, R2, 4 / R2, SMALL>(p, w, s, stream);
  return launch_shrink_as<F16, RT, 4, R2, 4 / R2, SMALL>(p, w, s, stream);
}

template <bool F16>
hipError_t launch_any_shrink(const ZmiLora &p, const ZmiLoraPlan &w, const LoraShape &s, hipStream_t stream) {
  return s.small ? launch_shrink<F16, 1, true>(p, w, s, stream) : s.rt == 1 ? launch_shrink<F16, 1, false>(p, w, s, stream)
       : s.rt == 2 ? launch_shrink<F16, 2, false>(p, w, s, stream) : launch_shrink<F16, 4, false>(p, w, s, stream);
}

}  // namespace

// What no call of up to p.T rows needs more than.  Fewer rows may be cut into more parts of K, and into more or taller tiles: the
// parts of the workspace are taken for the most that there can be.
size_t zmi_lora_workspace_bound(const ZmiLora &p) {
  if (p.T <= 0) return 0;
  ZmiLora q = p;
  size_t bytes = 0;
  for (int32_t T : {LORA_SMALL_T, LORA_SMALL_MOST}) {
    q.T = T < p.T ? T : p.T;
    const LoraShape s = lora_shape(q);
    if (!s.small) continue;
    // (K slices times tiles: all slices of few tiles, 512 workgroups, or one slice)
    const int64_t most = lora_small_slices((p.K + lora_ks(1, s.nt) - 1) / lora_ks(1, s.nt)), parts = lora_clamp(512 / s.ny, s.tiles, s.tiles * most);
    const size_t n = lora_small_bytes(q, s, parts);
    bytes = n > bytes ? n : bytes;
  }
  LoraShape s = lora_shape(p);
  if (!s.small) {
    s.rt = 4;
    s.tiles = s.groups;
    s.grid = 256;
    const size_t n = lora_layout(p, s, nullptr, nullptr);
    bytes = n > bytes ? n : bytes;
  }
  return bytes;
}

size_t zmi_lora_workspace_bytes(const ZmiLora &p) { return p.T > 0 ? lora_layout(p, lora_shape(p), nullptr, nullptr) : 0; }

hipError_t zmi_launch_lora(const ZmiLora &p, hipStream_t stream, const char **name) {
  if (p.T <= 0) return hipSuccess;
  if (!p.workspace || p.n_slots > ZMI_LORA_MAX_SLOTS || p.n_slices > 4) return hipErrorInvalidValue;
  const LoraShape s = lora_shape(p);
  if (s.runs > 65535 || s.ny > 65535) return hipErrorInvalidValue;
  ZmiLoraPlan w;
  lora_layout(p, s, (char *)p.workspace, &w);
  hipError_t e = hipSuccess;
  if (!s.small) {
    // (a row of counts per wavefront and four words of every slot in LDS)
    const int waves = p.n_slots < 1024 ? 16 : p.n_slots < 2048 ? 8 : 4, smem = (waves * 4 + 16) * (p.n_slots + 1);
    e = zmi_func_smem_once((const void *)zmi_lora_plan_kernel, (4 * 4 + 16) * (ZMI_LORA_MAX_SLOTS + 1));
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(zmi_lora_plan_kernel, dim3(1), dim3(1024), smem, stream, p, w, 16 * s.rt, waves);
    e = hipGetLastError();
  }
  if (e == hipSuccess) e = p.dt_x == ZMI_DT_F16 ? launch_any_shrink<true>(p, w, s, stream) : launch_any_shrink<false>(p, w, s, stream);
  if (e == hipSuccess) e = lora_launch_expand(p, w, s, stream);
  *name = s.small ? "lora_small" : "lora_planned";
  return e;
}
