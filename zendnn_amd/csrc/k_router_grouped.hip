// MoE router with sigmoid or softmax scores, a bias for the choice, groups of experts (gfx950); see zmi_lowoha.h.
//
//   * s_e = sigmoid(x_e) or softmax(x)_e, v_e = s_e + bias_e;
//   * group values: the largest v, or the sum of the two largest; the best topk_group groups stay;
//   * the topk best v among their experts, weights from s.
//
// One wavefront per token, 4 tokens per workgroup; lane l holds experts J l .. J l + J - 1.  A round of the choice is a
// maximum over the wavefront's keys (DPP, no LDS), a ballot per held expert, and the lowest lane and expert that hold it.
//
// Two experts of one token can lie nearer to each other than f32 tells apart (256 experts leave gaps of 1e-3 on average,
// so one token in some hundreds has two chosen or bordering values within f32's error), and ids have to be those of
// exact values.  The choice is therefore made on f32 values while every gap that decides it -- between one chosen expert
// and the next, the last and the best that is left, the last group and the best that is left -- is wider than what
// the f32 values can be off by; a token where one is not is chosen again by the same rounds on 64-bit values.  Without a
// bias experts are ordered by their logits, exactly, and no score is computed but those of the chosen.
//
// What bounds it: instructions.  8192 tokens of 256 f32 logits (sigmoid, bias, 4 of 8 groups, 8 experts) take 12.8 us and
// 621 vector instructions a token, 32768 of 512 (softmax, bias, 10 experts) 38 us and 761, where the bytes alone would
// take 2 and 14 us; at four clocks an instruction and 2.4 GHz that would be 8 and 41 us.  Short batches are a launch and one
// token's chain: 4 us.  Logits with many equal values under an equal bias have most tokens chosen twice: 8192 x 256 bf16
// with a zero bias 19.6 us, with a random one 13.0.
#include <type_traits>

#include "zmi_device.h"
#include "zmi_launch.h"

#define RGK_WAVES 4

namespace {

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t rgk_dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint64_t rgk_dpp(uint64_t v) {
  return rgk_dpp<CTRL, ROWS>((uint32_t)v) | (uint64_t)rgk_dpp<CTRL, ROWS>((uint32_t)(v >> 32)) << 32;
}

// maximum over the wavefront (lanes that a step does not reach get 0, the least value)
__device__ __forceinline__ uint32_t rgk_wave_max(uint32_t v) {
  v = max(v, rgk_dpp<0x111>(v));        // row_shr 1, 2, 4, 8: lane 15 of each row of 16
  v = max(v, rgk_dpp<0x112>(v));
  v = max(v, rgk_dpp<0x114>(v));
  v = max(v, rgk_dpp<0x118>(v));
  v = max(v, rgk_dpp<0x142, 0xa>(v));   // row_bcast 15 into rows 1 and 3
  v = max(v, rgk_dpp<0x143, 0xc>(v));   // row_bcast 31 into rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint64_t rgk_wave_max(uint64_t v) {
  const uint32_t hi = rgk_wave_max((uint32_t)(v >> 32));
  return (uint64_t)hi << 32 | rgk_wave_max((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
}

__device__ __forceinline__ double rgk_wave_sum(double v) {
  auto step = [&](uint64_t u) { v += __longlong_as_double((long long)u); };
  auto bits = [&] { return (uint64_t)__double_as_longlong(v); };
  step(rgk_dpp<0x111>(bits()));
  step(rgk_dpp<0x112>(bits()));
  step(rgk_dpp<0x114>(bits()));
  step(rgk_dpp<0x118>(bits()));
  step(rgk_dpp<0x142, 0xa>(bits()));
  step(rgk_dpp<0x143, 0xc>(bits()));
  const uint64_t u = bits();
  return __longlong_as_double((long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)u, 63) |
                                          (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), 63) << 32));
}

// exp(d) for d <= 0 (NaN stays), as zmi_expf without what only overflow needs; 0 below -200
__device__ __forceinline__ float rgk_exp_down(float d) {
  const float l2e_hi = 1.44269502162933349609375f, l2e_lo = 1.925963033500011e-08f;
  d = d < -200.0f ? -200.0f : d;   // (infinities would meet in the correction)
  const float t = d * l2e_hi;
  const float r = __builtin_fmaf(d, l2e_lo, __builtin_fmaf(d, l2e_hi, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, r * 0.693147182464599609375f, e);
}

// exp(d) in 64 bits, to 2^-31.7 of its value: exp(n ln 2) exp(r) with |r| <= ln 2 / 2, whose series ends at r^8 / 8!  (what the
// weights need and no more: 64 x 64 logits 3.33 us, with the library's exp 3.45)
__device__ __forceinline__ double rgk_exp64(double d) {
  d = d < -1100.0 ? -1100.0 : d > 1100.0 ? 1100.0 : d;   // (beyond are 0 and infinity; NaN stays)
  const double n = __builtin_rint(d * 1.4426950408889634), r = __builtin_fma(n, -0.6931471805599453, d), r2 = r * r;
  const double low = __builtin_fma(__builtin_fma(r, 1.0 / 6, 0.5), r2, 1.0 + r);
  const double high = __builtin_fma(__builtin_fma(r, 1.0 / 5040, 1.0 / 720), r2, __builtin_fma(r, 1.0 / 120, 1.0 / 24));
  const double r4 = r2 * r2;
  return __builtin_ldexp(__builtin_fma(__builtin_fma(r4, 1.0 / 40320, high), r4, low), (int)n);
}

// value -> unsigned key in the values' order; -0 == +0; NaN 1, below every number (0: nothing)
__device__ __forceinline__ uint32_t rgk_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return x != x ? 1u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t rgk_key(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return x != x ? 1u : u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ float rgk_value(uint32_t k) { return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ double rgk_value(uint64_t k) { return __longlong_as_double((long long)(k >> 63 ? k ^ 0x8000000000000000ull : ~k)); }

// The DEPTH largest of a lane's J keys in descending order in front of the others, equal ones in ascending j (neighbours are
// exchanged only when out of order); returns the j of each, four bits apiece, the first in the lowest bits, and ones behind
// them.
template <int J, int DEPTH, class K>
__device__ __forceinline__ uint32_t rgk_sort(K (&key)[J]) {
  // (a vector, not an array: choosing between two elements of an array becomes an indexed read, a chain of comparisons)
  typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
  u32x8 at = {0, 1, 2, 3, 4, 5, 6, 7};
  uint32_t queue = DEPTH < 8 ? ~0u << (4 * DEPTH % 32) : 0u;
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
#pragma unroll
    for (int j = J - 2; j >= d; --j) {
      const bool swap = key[j + 1] > key[j];
      const K hi = max(key[j], key[j + 1]), lo = min(key[j], key[j + 1]);
      const uint32_t a = at[j], b = at[j + 1];
      key[j] = hi; key[j + 1] = lo;
      at[j] = swap ? b : a;
      at[j + 1] = swap ? a : b;
    }
#pragma unroll
  for (int j = 0; j < DEPTH; ++j) queue |= at[j] << (4 * j);
  return queue;
}

// The two largest of two lanes, from the two largest of each.
template <int CTRL, class K>
__device__ __forceinline__ void rgk_pair(K &a, K &b) {
  const K c = rgk_dpp<CTRL>(a), d = rgk_dpp<CTRL>(b);
  b = max(min(a, c), max(b, d));
  a = max(a, c);
}

// The rounds of the choice, on V's keys: the largest first key of a lane, of the lowest lane that has it.  A lane gives up to
// DEPTH of its J; false where the one behind them might have been chosen, or where a gap that decides is not wide enough.
template <int J, int DEPTH, class V, class K>
__device__ __forceinline__ bool rgk_rounds(const ZmiRouterGrouped &p, K (&key)[J], float score, int *mine) {
  const int lane = threadIdx.x % 64;
  uint32_t queue = rgk_sort<J, DEPTH>(key);
  uint32_t order = 0;   // float values: lane r keeps the r-th key
  for (int r = 0; r < p.topk; ++r) {
    const K top = rgk_wave_max(key[0]);
    const int at = __builtin_ctzll(__ballot(key[0] == top));
    const int e = at * J + (__builtin_amdgcn_readlane((int)queue, at) & 15);
    if (lane == r) { *mine = e; order = (uint32_t)top; }
    if (lane == at) {
#pragma unroll
      for (int j = 0; j + 1 < DEPTH; ++j) key[j] = key[j + 1];
      key[DEPTH - 1] = 0;
      queue = DEPTH < 8 ? (uint32_t)((int32_t)queue >> 4) : queue >> 4;
    }
  }
  if (DEPTH < J) {
    const bool empty = (queue & 15) == 15;
    if (__ballot(empty)) {
      K hidden = 0;
#pragma unroll
      for (int j = DEPTH; j < J; ++j) hidden = max(hidden, key[j]);
      if (empty) key[0] = hidden;
      if (__ballot(empty && hidden >= (K)(uint32_t)__builtin_amdgcn_readlane((int)order, p.topk - 1))) return false;
    }
  }
  if (std::is_same<V, float>::value && p.bias) {
    const uint32_t rest = (uint32_t)rgk_wave_max(key[0]), below = (uint32_t)__shfl_down((int)order, 1, 64);
    const uint32_t next = lane == p.topk - 1 ? rest : below;
    const float a = rgk_value(order), b = rgk_value(next);
    const bool close = lane < p.topk && next && !(a - b > 0x1p-19f * score + 0x1p-23f * (__builtin_fabsf(a) + __builtin_fabsf(b)));
    if (__ballot(close)) return false;
  }
  return true;
}

// The choice.  key: what experts are ordered by, v: the values that groups are valued by (top2); both of V's type.  Lane r
// gets the r-th expert.
//
// Float keys (with a bias) and v are f32 values of scores up to `score`: false when a gap that decides is not wide enough.  What
// the f32 scores of two experts are off by, in half steps of 2^-24 `score`, all of them the other way: sigmoids 7 each
// (exponential 4, addition 1, reciprocal 2); softmax scores 5.4 each (exponential 4, product 1, x - m in front of it 0.4 at the
// most) and 13 of their difference (the sum, and its inverse), 19 together.  32 are asked for, and for two groups of two
// experts 64, where at most 38 meet; rounding a value adds half an ulp of it, which is asked for twice.
// Values below the one compared with can be off by more where they are larger, but then they are negative and far below.
template <int J, int SORT, class V, class K>
__device__ __forceinline__ bool rgk_choose(const ZmiRouterGrouped &p, K (&key)[J], const V (&v)[J], float score, void *scratch, int *mine) {
  const int lane = threadIdx.x % 64, e0 = lane * J, n = p.E - e0, per = p.per;
  if (p.topk_group < p.n_group) {
    K a = 0, b = 0;   // a lane's, then its group's, two largest
    const bool in_lanes = p.lane_shift >= 0;
    if (in_lanes) {
      const int lanes = 1 << p.lane_shift;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const K k = !p.top2 ? key[j] : j < n ? rgk_key(v[j]) : (K)0;
        b = max(b, min(a, k));
        a = max(a, k);
      }
      // (steps inside rows of 16 lanes: swap neighbours, pairs, mirror halves of eight, mirror the row)
      if (lanes > 1) rgk_pair<0xb1>(a, b);
      if (lanes > 2) rgk_pair<0x4e>(a, b);
      if (lanes > 4) rgk_pair<0x141>(a, b);
      if (lanes > 8) rgk_pair<0x140>(a, b);
    } else {
      K *all = (K *)scratch;
#pragma unroll
      for (int j = 0; j < J; ++j) all[e0 + j] = p.top2 ? rgk_key(v[j]) : key[j];
      // (one wavefront writes and reads its own slice: the order of its LDS instructions is all that is needed)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (lane < p.n_group)
        for (int i = 0; i < per; ++i) {
          const K k = all[lane * per + i];
          b = max(b, min(a, k));
          a = max(a, k);
        }
    }
    // group g is held by lanes [g << w, (g + 1) << w)
    const int w = in_lanes ? p.lane_shift : 0, g = lane >> w;
    K gk = g < p.n_group ? (p.top2 ? rgk_key(rgk_value(a) + rgk_value(b)) : a) : (K)0, last = 0;
    uint64_t groups = 0;
    for (int r = 0; r < p.topk_group; ++r) {
      last = rgk_wave_max(gk);
      const int i = __builtin_ctzll(__ballot(gk == last)) >> w;
      groups |= 1ull << i;
      if (g == i) gk = 0;
    }
    if (std::is_same<V, float>::value && (p.bias || p.top2)) {
      // the best that is left may be as good as the last one taken (a sum is off by twice as much, and by its rounding)
      const float next = (float)rgk_value(rgk_wave_max(gk)), taken = (float)rgk_value(last);
      float size = __builtin_fabsf((float)rgk_value(a)) + (p.top2 ? __builtin_fabsf((float)rgk_value(b)) : 0.0f);
      if (g >= p.n_group || !(size < __builtin_inff())) size = 0.0f;
      size = __uint_as_float(rgk_wave_max(__float_as_uint(size)));
      if (!(taken - next > 0x1p-18f * score + 0x1p-21f * size)) return false;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int of = in_lanes ? g : (int)(((float)(e0 + j) + 0.5f) * p.inv_per);
      if (j < n && !((groups >> of) & 1u)) key[j] = 0;
    }
  }
  return rgk_rounds<J, std::is_same<V, float>::value ? SORT : J, V>(p, key, score, mine);
}

}  // namespace

template <int J, bool SIGMOID, int SORT>   // SORT: experts that a lane sorts for the choice on f32 values
__global__ __launch_bounds__(RGK_WAVES * 64) void zmi_moe_router_grouped_kernel(ZmiRouterGrouped p) {
  __shared__ double scratch[RGK_WAVES][64 * J];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int t = blockIdx.x * RGK_WAVES + wave;
  if (t >= p.T) return;   // (whole wavefronts; nothing below synchronizes across wavefronts)
  const int e0 = lane * J, n = p.E - e0;   // this lane's experts: e0 .. e0 + min(J, n) - 1
  const int64_t row = (int64_t)t * p.ldl;
  float x[J], bias[J];
  // (lanes at the end read the last expert's word in the place of what is not there)
  if (p.logits_dt == ZMI_DT_F32) {
    const float *f = (const float *)p.logits + row;
    if (n >= J) {
      __builtin_memcpy(x, f + e0, J * 4);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) x[j] = f[j < n ? e0 + j : p.E - 1];
    }
  } else {
    const uint16_t *f = (const uint16_t *)p.logits + row;
    uint16_t h[J];
    if (n >= J) {
      __builtin_memcpy(h, f + e0, J * 2);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) h[j] = f[j < n ? e0 + j : p.E - 1];
    }
    const bool bf16 = p.logits_dt == ZMI_DT_BF16;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const float a = zmi_bf16_to_f32(h[j]), b = zmi_f16_to_f32(h[j]);
      x[j] = bf16 ? a : b;
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j) bias[j] = 0.0f;
  if (p.bias) {
    if (n >= J) {
      __builtin_memcpy(bias, p.bias + e0, J * 4);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) bias[j] = p.bias[j < n ? e0 + j : p.E - 1];
    }
  }
  uint32_t key[J];
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (j >= n) x[j] = -__builtin_inff();
  // ---- softmax: the row's maximum and sum ----
  float m = 0.0f, v[J];
  double sum = 0.0;
  if (!SIGMOID) {
    float top = x[0];
#pragma unroll
    for (int j = 1; j < J; ++j) top = fmaxf(top, x[j]);   // (skips NaN; a NaN logit reaches the sum below)
    m = rgk_value(rgk_wave_max(rgk_key(top)));
    float part[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      // (equal to the maximum is 1, whatever it is, and -inf is 0; NaN stays)
      v[j] = rgk_exp_down(x[j] - m);
      v[j] = x[j] == m ? 1.0f : v[j];
      v[j] = x[j] == -__builtin_inff() ? 0.0f : v[j];
      part[j] = v[j];
    }
    // (a lane's terms are added in f32, at most three roundings deep, the lanes' sums in 64 bits)
#pragma unroll
    for (int w = J / 2; w >= 1; w /= 2)
#pragma unroll
      for (int j = 0; j < w; ++j) part[j] += part[j + w];
    sum = rgk_wave_sum((double)part[0]);
  }
  float score = 0.0f;   // the largest score there can be, where values are f32 scores
  if (p.bias || (p.top2 && p.topk_group < p.n_group)) {
    const float top = SIGMOID ? 1.0f : sum == 0.0 ? 0.0f : 1.0f / (float)sum;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      v[j] = (SIGMOID ? zmi_sigmoid(x[j]) : v[j] * top) + bias[j];
      if (p.bias) key[j] = j < n ? rgk_key(v[j]) : 0u;
    }
    score = top;
  }
  if (!p.bias) {
#pragma unroll
    for (int j = 0; j < J; ++j) key[j] = j < n ? rgk_key(x[j]) : 0u;
  }
  int mine = 0;
  if (!rgk_choose<J, SORT>(p, key, v, score, scratch[wave], &mine)) {
    double v64[J];
    uint64_t key64[J];
    double z = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const double e = exp(SIGMOID ? -(double)x[j] : (double)x[j] - (double)m);
      v64[j] = SIGMOID ? 1.0 / (1.0 + e) : x[j] == -__builtin_inff() ? 0.0 : x[j] == m ? 1.0 : e;
      z += v64[j];
    }
    if (!SIGMOID) z = rgk_wave_sum(z);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (!SIGMOID) v64[j] = z == 0.0 ? 0.0 : v64[j] / z;
      v64[j] += (double)bias[j];
      key64[j] = j >= n ? 0u : p.bias ? rgk_key(v64[j]) : rgk_key((double)x[j]);
    }
    rgk_choose<J, SORT>(p, key64, v64, 0.0f, scratch[wave], &mine);
  }
  // ---- weights, in 64 bits: y - m rounded to f32 would be off by more the further an expert lies below the best ----
  double s = 0.0;
  if (lane < p.topk) {
    const float y = zmi_ld_f32(p.logits, p.logits_dt, row + mine);
    const double e = rgk_exp64(SIGMOID ? -(double)y : (double)y - (double)m);
    s = SIGMOID ? 1.0 / (1.0 + e) : y == -__builtin_inff() ? 0.0 : y == m ? 1.0 : e;
  }
  const double z = p.renormalize ? rgk_wave_sum(s) : SIGMOID ? 1.0 : sum;
  if (lane < p.topk) {
    p.topk_ids[(int64_t)t * p.topk + lane] = mine;
    p.topk_weights[(int64_t)t * p.topk + lane] = z == 0.0 ? 0.0f : (float)(s / z * (double)p.scale);
  }
}

namespace {

template <int J, int SORT = J>
void rgk_launch(const ZmiRouterGrouped &p, hipStream_t stream) {
  const dim3 grid((unsigned)((p.T + RGK_WAVES - 1) / RGK_WAVES)), block(RGK_WAVES * 64);
  if (p.sigmoid) hipLaunchKernelGGL((zmi_moe_router_grouped_kernel<J, true, SORT>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((zmi_moe_router_grouped_kernel<J, false, SORT>), grid, block, 0, stream, p);
}

}  // namespace

hipError_t zmi_launch_moe_router_grouped(ZmiRouterGrouped p, hipStream_t stream) {
  if (p.T <= 0) return hipSuccess;
  if (p.E <= 0 || p.E > 512 || p.n_group <= 0 || p.n_group > 64 || p.E % p.n_group || p.topk_group <= 0 ||
      p.topk_group > p.n_group || p.topk <= 0 || p.topk > 64 || p.topk > p.topk_group * (p.E / p.n_group))
    return hipErrorInvalidValue;
  // a group that fills 1, 2, 4, 8 or 16 whole lanes is valued in registers, others through LDS
  const int J = p.E <= 64 ? 1 : p.E <= 128 ? 2 : p.E <= 256 ? 4 : 8, lanes = p.E / p.n_group / J;
  p.per = p.E / p.n_group;
  p.inv_per = 1.0f / (float)p.per;   // (e + 0.5) times it truncates to e / per for every e < 512
  p.lane_shift = p.per % J == 0 && lanes <= 16 && (lanes & (lanes - 1)) == 0 ? __builtin_ctz(lanes) : -1;
  // Of eight experts a lane sorts three, unless too many tokens would have four of their best in one lane, be short of the fourth
  // and chosen again: topk^4 / 24 sets of four, each in one of the live lanes with 1 / lanes^3; at more than one token in 128
  // a lane sorts all eight, with a bias, where that costs more, at one in 16 (16384 x 512 softmax, three / eight: topk 10
  // 20.7 / 21.7 us, 16 25.8 / 25.2, 32 44.3 / 35.8, 64 116.7 / 56.3; with a bias 16 25.9 / 29.2, 32 41.0 / 44.3, 64 107 / 74; 8
  // experts of one group of 64 29.5 / 25.9, of two 25.6 / 26.8, 12 of two 32.6 / 30.4).
  const int64_t live = p.topk_group * p.per / 8 + 1, sets = (int64_t)p.topk * (p.topk - 1) * (p.topk - 2) * (p.topk - 3) / 24;
  if (J == 1) rgk_launch<1>(p, stream);
  else if (J == 2) rgk_launch<2>(p, stream);
  else if (J == 4) rgk_launch<4>(p, stream);
  else if (sets * (p.bias ? 16 : 128) > live * live * live) rgk_launch<8>(p, stream);
  else rgk_launch<8, 3>(p, stream);
  return hipGetLastError();
}
