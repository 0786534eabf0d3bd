// zmi_lora_direct: low-rank adapters of many requests beside a shared projection (no counterpart in the reference).
#include <cstring>

#include "../../include/zmi_lowoha.h"
#include "zmi_api.h"

namespace zmi {
namespace {

bool half_type(int32_t dt) { return dt == ZMI_DT_BF16 || dt == ZMI_DT_F16; }

// The sizes and types alone (what zmi_lora_workspace_size goes by): status, with the error text set when refused.
int32_t lora_check_sizes(const zmi_lora_t &l) {
  if (l.T < 0 || l.K <= 0 || l.rank <= 0 || l.n_slices <= 0 || l.n_slots <= 0) { set_error("lora: bad sizes"); return ZMI_FAILURE; }
  if (l.rank > 256 || l.n_slices > ZMI_LORA_MAX_SLICES || l.n_slots > ZMI_LORA_MAX_SLOTS) { set_error("lora: at most rank 256, 4 slices, 4096 slots"); return ZMI_UNIMPLEMENTED; }
  int64_t cols = 0;
  for (int s = 0; s < l.n_slices; ++s) {
    if (l.N[s] <= 0) { set_error("lora: bad sizes"); return ZMI_FAILURE; }
    cols += l.N[s];
  }
  if (cols > 1 << 30) { set_error("lora: too many columns"); return ZMI_UNIMPLEMENTED; }
  // (tiles x rank tile sets x stages of K stay below 2^31: 20.5 k x 8 x 8192)
  if (l.T > 1 << 20 || l.K > 1 << 19) { set_error("lora: at most 2^20 rows, K at most 2^19"); return ZMI_UNIMPLEMENTED; }
  if (!half_type(l.dt_x)) { set_error("lora: dt_x must be bf16 or f16"); return ZMI_UNIMPLEMENTED; }
  if (!half_type(l.dt_dst) && l.dt_dst != ZMI_DT_F32) { set_error("lora: dt_dst must be bf16, f16 or f32"); return ZMI_UNIMPLEMENTED; }
  return ZMI_SUCCESS;
}

// n_slots x rows x cols elements, slot stride and row stride as given, on addresses of whole elements
bool lora_weights_ok(const void *p, int64_t ld, int64_t slot, int64_t n_slots, int64_t rows, int64_t cols) {
  if (!p || (uintptr_t)p % 2 || ld < cols) return false;
  return n_slots == 1 || slot >= (rows - 1) * ld + cols;
}

// Whether a row of base and a row of dst share bytes: T rows of `cols` elements of `size` bytes each.
bool lora_rows_meet(const void *base, int64_t ld_base, const void *dst, int64_t ld_dst, int64_t T, int64_t cols, int64_t size) {
  typedef __int128 wide;   // (strides may be anything)
  const wide b0 = (uintptr_t)base, d0 = (uintptr_t)dst, base_step = (wide)ld_base * size, dst_step = (wide)ld_dst * size, bytes = cols * size;
  if (b0 + (T - 1) * base_step + bytes <= d0 || d0 + (T - 1) * dst_step + bytes <= b0) return false;
  if (base_step == dst_step || T == 1) {
    // base's row j lies (j - i) steps and b0 - d0 from dst's row i: less than a row apart for the step below or above only
    const wide k = T == 1 ? 0 : (d0 - b0) / base_step;
    for (wide i = k - 1; i <= k + 1; ++i)
      if (i > -(wide)T && i < T) {
        const wide apart = b0 - d0 + i * base_step;
        if (apart < bytes && -apart < bytes) return true;
      }
    return false;
  }
  for (int64_t i = 0, j = 0; i < T && j < T;) {   // (both in ascending order)
    const wide b = b0 + j * base_step, d = d0 + i * dst_step;
    if (b + bytes <= d) ++j;
    else if (d + bytes <= b) ++i;
    else return true;
  }
  return false;
}

ZmiLora lora_flat(const zmi_lora_t &l) {
  ZmiLora p;
  std::memset(&p, 0, sizeof(p));
  p.T = l.T; p.K = l.K; p.rank = l.rank; p.n_slices = l.n_slices; p.n_slots = l.n_slots;
  p.dt_x = l.dt_x; p.dt_dst = l.dt_dst;
  p.x = l.x; p.ldx = l.ldx; p.slot_ids = l.slot_ids;
  p.a = l.a; p.a_ld = l.a_ld; p.a_slot = l.a_slot;
  for (int s = 0; s < l.n_slices; ++s) { p.N[s] = l.N[s]; p.b[s] = l.b[s]; p.b_ld[s] = l.b_ld[s]; p.b_slot[s] = l.b_slot[s]; }
  p.ranks = l.ranks; p.scales = l.scales;
  p.base = l.base; p.ld_base = l.ld_base; p.dst = l.dst; p.ld_dst = l.ld_dst;
  return p;
}

}  // namespace
}  // namespace zmi

using namespace zmi;

extern "C" {

void zmi_lora_params_init(zmi_lora_t *l) {
  if (!l) return;
  std::memset(l, 0, sizeof(*l));
  l->n_slices = 1;
  l->dt_x = l->dt_dst = ZMI_DT_BF16;
}

uint64_t zmi_lora_workspace_size(const zmi_lora_t *l) {
  clear_error();
  if (!l) { set_error("lora: null argument"); return 0; }
  if (lora_check_sizes(*l) != ZMI_SUCCESS) return 0;
  return zmi_lora_workspace_bound(lora_flat(*l));
}

int32_t zmi_lora_direct(const zmi_lora_t *l) {
  clear_error();
  if (!l) { set_error("lora: null argument"); return ZMI_FAILURE; }
  if (int32_t st = lora_check_sizes(*l); st != ZMI_SUCCESS) return st;
  if (l->T == 0) return ZMI_SUCCESS;
  if (!l->x || !l->slot_ids || !l->dst) { set_error("lora: null argument"); return ZMI_FAILURE; }
  int64_t cols = 0;
  const int64_t dst_size = l->dt_dst == ZMI_DT_F32 ? 4 : 2;
  if (!lora_weights_ok(l->a, l->a_ld, l->a_slot, l->n_slots, (int64_t)l->n_slices * l->rank, l->K)) { set_error("lora: a is null, misaligned, or its strides are smaller than what they step over"); return ZMI_FAILURE; }
  for (int s = 0; s < l->n_slices; ++s) {
    if (!lora_weights_ok(l->b[s], l->b_ld[s], l->b_slot[s], l->n_slots, l->N[s], l->rank)) { set_error("lora: b is null, misaligned, or its strides are smaller than what they step over"); return ZMI_FAILURE; }
    cols += l->N[s];
  }
  if (l->ldx < l->K || l->ld_dst < cols || (l->base && l->ld_base < cols)) { set_error("lora: row stride smaller than the row"); return ZMI_FAILURE; }
  if (l->base == l->dst && l->ld_base != l->ld_dst) { set_error("lora: base at dst's address needs dst's row stride"); return ZMI_FAILURE; }
  if (l->base && l->base != l->dst &&
      lora_rows_meet(l->base, l->ld_base, l->dst, l->ld_dst, l->T, cols, dst_size)) {
    set_error("lora: base and dst overlap in part (base is dst itself or apart from it)");
    return ZMI_FAILURE;
  }
  if ((uintptr_t)l->x % 2 || (uintptr_t)l->dst % dst_size || (uintptr_t)l->base % dst_size || (uintptr_t)l->slot_ids % 4 ||
      (uintptr_t)l->ranks % 4 || (uintptr_t)l->scales % 4 || (uintptr_t)l->workspace % 16) {
    set_error("lora: an address is not a multiple of its element's size (workspace: 16 bytes)");
    return ZMI_FAILURE;
  }
  note_operand(l->x); note_operand(l->slot_ids); note_operand(l->a); note_operand(l->dst); note_operand(l->base);
  note_operand(l->ranks); note_operand(l->scales); note_operand(l->workspace);
  for (int s = 0; s < l->n_slices; ++s) note_operand(l->b[s]);
  ZmiLora p = lora_flat(*l);
  const size_t need = zmi_lora_workspace_bytes(p);
  if (l->workspace && l->workspace_bytes < need) { set_error("lora: workspace smaller than zmi_lora_workspace_size()"); return ZMI_FAILURE; }
  if (!ensure_device()) return ZMI_FAILURE;
  if (need) {
    void *ws = l->workspace;
    if (!ws) {
      // (a captured call would leave the arena's address in the graph, where later calls move or reuse it)
      hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
      if (!hip_ok(hipStreamIsCapturing(stream(), &cs), "hipStreamIsCapturing")) return ZMI_FAILURE;
      if (cs != hipStreamCaptureStatusNone) { set_error("lora: a call under stream capture needs the caller's workspace"); return ZMI_FAILURE; }
      if (!arena().begin(Arena::padded(need))) return ZMI_FAILURE;
      ws = arena().alloc(need);
    }
    p.workspace = ws;
  }
  const char *name = "lora";
  if (!hip_ok(zmi_launch_lora(p, stream(), &name), "lora launch")) return ZMI_FAILURE;
  set_kernel_name(name);
  return ZMI_SUCCESS;
}

}  // extern "C"
