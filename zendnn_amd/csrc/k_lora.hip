// Low-rank adapters of many requests beside a shared projection (gfx950); see zmi_lowoha.h.
//
//   h[t][s, r] = sum_k x[t][k] A[a][s rank + r][k],  dst[t][n] = base[t][n] + scales[a] sum_r h[t][s, r] B_s[a][n][r]
//
// with a = slot_ids[t].  Two launches: the first computes h in f32, a wavefront per element; the second a thread per
// element of dst.
#include "zmi_device.h"
#include "zmi_launch.h"

namespace {

__device__ __forceinline__ int lora_rank(const ZmiLora &p, int slot) {
  if (!p.ranks) return p.rank;
  const int r = p.ranks[slot];
  return r < 0 ? 0 : r > p.rank ? p.rank : r;
}

}  // namespace

__global__ __launch_bounds__(256) void zmi_lora_shrink_kernel(ZmiLora p) {
  const int lane = threadIdx.x % 64;
  const int64_t t = blockIdx.x;
  const int slot = p.slot_ids[t];
  if ((unsigned)slot >= (unsigned)p.n_slots) return;
  const int rank = lora_rank(p, slot), rt = p.n_slices * p.rank;
  for (int i = threadIdx.x / 64; i < rt; i += 4) {
    if (i % p.rank >= rank) continue;
    float acc = 0.0f;
    for (int k = lane; k < p.K; k += 64)
      acc = __builtin_fmaf(zmi_ld_f32(p.x, p.dt_x, t * p.ldx + k), zmi_ld_f32(p.a, p.dt_x, slot * p.a_slot + i * p.a_ld + k), acc);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) acc += __shfl_xor(acc, d, 64);
    if (lane == 0) p.h[t * rt + i] = acc;
  }
}

__global__ __launch_bounds__(256) void zmi_lora_expand_kernel(ZmiLora p, int n_cols) {
  const int64_t t = blockIdx.x;
  int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= n_cols) return;
  const int64_t at = t * p.ld_dst + col;
  float y = p.base ? zmi_ld_f32(p.base, p.dt_dst, t * p.ld_base + col) : 0.0f;
  const int slot = p.slot_ids[t];
  if ((unsigned)slot < (unsigned)p.n_slots) {
    int s = 0;
    while (col >= p.N[s]) col -= p.N[s++];
    const int rank = lora_rank(p, slot);
    float acc = 0.0f;
    for (int r = 0; r < rank; ++r)
      acc = __builtin_fmaf(p.h[t * (p.n_slices * p.rank) + s * p.rank + r],
                           zmi_ld_f32(p.b[s], p.dt_x, slot * p.b_slot[s] + col * p.b_ld[s] + r), acc);
    y = __builtin_fmaf(acc, p.scales ? p.scales[slot] : 1.0f, y);
  } else if (p.base == p.dst) {
    return;
  }
  if (p.dt_dst == ZMI_DT_F32) ((float *)p.dst)[at] = y;
  else if (p.dt_dst == ZMI_DT_BF16) ((__bf16 *)p.dst)[at] = (__bf16)y;
  else ((_Float16 *)p.dst)[at] = (_Float16)y;
}

size_t zmi_lora_workspace_bytes(const ZmiLora &p) { return (size_t)p.T * p.n_slices * p.rank * sizeof(float); }

hipError_t zmi_launch_lora(const ZmiLora &p, hipStream_t stream, const char **name) {
  if (p.T <= 0) return hipSuccess;
  int64_t n_cols = 0;
  for (int s = 0; s < p.n_slices; ++s) n_cols += p.N[s];
  hipLaunchKernelGGL(zmi_lora_shrink_kernel, dim3((unsigned)p.T), dim3(256), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(zmi_lora_expand_kernel, dim3((unsigned)p.T, (unsigned)((n_cols + 255) / 256)), dim3(256), 0, stream, p,
                     (int)n_cols);
  *name = "lora";
  return hipGetLastError();
}
