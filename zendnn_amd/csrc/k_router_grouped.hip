// MoE router with sigmoid or softmax scores, a bias for the choice, groups of experts (gfx950); see zmi_lowoha.h.
//
//   * s_e = sigmoid(x_e) or softmax(x)_e, v_e = s_e + bias_e;
//   * group values: the largest v, or the sum of the two largest; the best topk_group groups stay;
//   * the topk best v among their experts, weights from s.
//
// One wavefront per token, 4 tokens per workgroup; lane l holds experts l, l + 64, ... (at most 8).  Two experts of one
// token can lie nearer to each other than f32 tells apart (256 experts leave gaps of 1e-3 on average, so one token in
// some thousands has two chosen or bordering values within an f32 ulp), hence scores and values in 64 bits.
#include "zmi_device.h"
#include "zmi_launch.h"

#define RGK_WAVES 4
#define RGK_PER_LANE 8

namespace {

// double -> unsigned key whose unsigned order is the value order; -0 == +0; NaN lowest
__device__ __forceinline__ uint64_t rgk_key(double x) {
  if (x != x) return 0u;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// (key, index) of the wavefront's best: largest key, then lowest index; index < 0: nothing to offer
__device__ __forceinline__ void rgk_best(uint64_t &k, int &i) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) {
    const uint64_t ok = __shfl_xor((unsigned long long)k, s, 64);
    const int oi = __shfl_xor(i, s, 64);
    if (oi >= 0 && (i < 0 || ok > k || (ok == k && oi < i))) { k = ok; i = oi; }
  }
}

__device__ __forceinline__ double rgk_sum(double v) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) v += __shfl_xor(v, s, 64);
  return v;
}

}  // namespace

__global__ __launch_bounds__(RGK_WAVES * 64) void zmi_moe_router_grouped_kernel(ZmiRouterGrouped p) {
  __shared__ double value[RGK_WAVES][64 * RGK_PER_LANE];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int t = blockIdx.x * RGK_WAVES + wave;
  if (t >= p.T) return;   // (whole wavefronts; nothing below synchronizes across wavefronts)
  float x[RGK_PER_LANE];
#pragma unroll
  for (int j = 0; j < RGK_PER_LANE; ++j) {
    const int e = lane + 64 * j;
    x[j] = e < p.E ? zmi_ld_f32(p.logits, p.logits_dt, (int64_t)t * p.ldl + e) : -__builtin_inff();
  }
  // ---- scores ----
  double s[RGK_PER_LANE];
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < RGK_PER_LANE; ++j) s[j] = 1.0 / (1.0 + exp(-(double)x[j]));
  } else {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < RGK_PER_LANE; ++j) m = fmaxf(m, x[j]);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < RGK_PER_LANE; ++j) {
      // (a row's largest logit may be infinite: equal to the maximum is 1 whatever it is, -inf is 0)
      s[j] = x[j] == -__builtin_inff() ? 0.0 : x[j] == m ? 1.0 : exp((double)x[j] - (double)m);
      sum += s[j];
    }
    sum = rgk_sum(sum);
#pragma unroll
    for (int j = 0; j < RGK_PER_LANE; ++j) s[j] = sum == 0.0 ? 0.0 : s[j] / sum;
  }
  // ---- values: without a bias the logits' own order ----
  double v[RGK_PER_LANE];
  uint64_t key[RGK_PER_LANE];
#pragma unroll
  for (int j = 0; j < RGK_PER_LANE; ++j) {
    const int e = lane + 64 * j;
    v[j] = p.bias && e < p.E ? s[j] + (double)p.bias[e] : s[j];
    key[j] = rgk_key(p.bias ? v[j] : (double)x[j]);
  }
  uint64_t groups = ~0ull;   // bit g: group g may be chosen from
  const int per = p.E / p.n_group;
  if (p.topk_group < p.n_group) {
    const bool by_logit = !p.bias && !p.top2;
#pragma unroll
    for (int j = 0; j < RGK_PER_LANE; ++j)
      if (lane + 64 * j < p.E) value[wave][lane + 64 * j] = by_logit ? (double)x[j] : v[j];
    // (one wavefront writes and reads its own slice: the order of its LDS instructions is all that is needed)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    uint64_t gk = 0;
    if (lane < p.n_group) {
      double b1 = value[wave][lane * per], b2 = -__builtin_inf();
      bool second = false;
      for (int i = 1; i < per; ++i) {
        const double a = value[wave][lane * per + i];
        if (rgk_key(a) > rgk_key(b1)) { b2 = b1; b1 = a; }
        else if (!second || rgk_key(a) > rgk_key(b2)) b2 = a;
        second = true;
      }
      gk = rgk_key(p.top2 ? b1 + b2 : b1);
    }
    groups = 0;
    for (int r = 0; r < p.topk_group; ++r) {
      uint64_t k = gk;
      int i = lane < p.n_group && !((groups >> lane) & 1u) ? lane : -1;
      rgk_best(k, i);
      groups |= 1ull << i;
    }
  }
  // ---- topk rounds ----
  unsigned live = 0;
#pragma unroll
  for (int j = 0; j < RGK_PER_LANE; ++j) {
    const int e = lane + 64 * j;
    if (e < p.E && ((groups >> (e / per)) & 1u)) live |= 1u << j;
  }
  double sel = 0.0, mine = 0.0;
  for (int r = 0; r < p.topk; ++r) {
    uint64_t k = 0;
    int i = -1;
    double sv = 0.0;
#pragma unroll
    for (int j = 0; j < RGK_PER_LANE; ++j)
      if (((live >> j) & 1u) && (i < 0 || key[j] > k)) { k = key[j]; i = lane + 64 * j; sv = s[j]; }
    rgk_best(k, i);
    if (i % 64 == lane) live &= ~(1u << (i / 64));
    sv = __shfl(sv, i % 64, 64);
    sel += sv;
    if (lane == r) mine = sv;
    if (lane == 0) p.topk_ids[(int64_t)t * p.topk + r] = i;
  }
  if (p.renormalize) mine = sel == 0.0 ? 0.0 : mine / sel;
  if (lane < p.topk) p.topk_weights[(int64_t)t * p.topk + lane] = (float)(mine * (double)p.scale);
}

hipError_t zmi_launch_moe_router_grouped(const ZmiRouterGrouped &p, hipStream_t stream) {
  if (p.T <= 0) return hipSuccess;
  if (p.E <= 0 || p.E > 64 * RGK_PER_LANE || p.n_group <= 0 || p.n_group > 64 || p.E % p.n_group || p.topk_group <= 0 ||
      p.topk_group > p.n_group || p.topk <= 0 || p.topk > 64 || p.topk > p.topk_group * (p.E / p.n_group))
    return hipErrorInvalidValue;
  hipLaunchKernelGGL(zmi_moe_router_grouped_kernel, dim3((unsigned)((p.T + RGK_WAVES - 1) / RGK_WAVES)), dim3(RGK_WAVES * 64), 0,
                     stream, p);
  return hipGetLastError();
}
