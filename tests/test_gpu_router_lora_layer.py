"""GPU test of a served mixture-of-experts layer with per-request adapters, as a program would call it: a fused
query / key / value projection (matmul_direct) with its adapters added in place, the gate projection with f32 logits and
its adapters, the router, the experts.  Each step is held against the definition on the values that the step before it left."""
import numpy as np
import pytest
import torch

from zendnn_amd import capi, lowoha
from tests import gpu_helpers as H
from tests import moe_helpers as MH
from tests.test_gpu_lora import Case
from tests.test_gpu_router_grouped import REL_TOL, expect

pytestmark = pytest.mark.gpu


def project(rng, x, N, dst_dt):
    """A dynamically quantized projection of bf16 rows (matmul_direct)."""
    T, K = x.shape
    w = H.to_dev(H.gen_weights(rng, K, N))
    ws = H.to_dev(rng.uniform(1e-4, 2e-4, N).astype(np.float32))
    p = lowoha.MatmulParams(src=capi.DT_BF16, wei=capi.DT_S8, dst=dst_dt, compute=capi.DT_S8)
    p.dynamic_quant = True
    p.src_scale = lowoha.QuantParam(None, capi.DT_F32, (T, 1))
    p.wei_scale = lowoha.QuantParam(ws, capi.DT_F32, (1, N))
    dst = torch.zeros((T, N), dtype=torch.float32 if dst_dt == capi.DT_F32 else torch.bfloat16, device=H.DEV)
    st = lowoha.matmul_direct("r", False, False, T, N, K, 1.0, x, K, w, N, None, 0.0, dst, N, False, p)
    assert st == capi.SUCCESS, lowoha.last_error()
    return dst


@pytest.mark.parametrize("T", [1, 12, 200])
def test_layer(zo, T):
    rng = np.random.default_rng(T)
    E, topk = 8, 2
    moe = MH.make_case(3, T, 256, 64, E, topk)
    d = MH.DeviceMoe(moe)
    x = H.to_dev(moe.x)
    # projections and their adapters
    for N, dst, code in (([256, 64, 64], torch.bfloat16, capi.DT_BF16), ([E], torch.float32, capi.DT_F32)):
        y = project(rng, x, sum(N), code)
        c = Case(T + len(N), T, 256, N, 8, 5, torch.bfloat16, dst)
        c.x, c.base = x, y.clone()
        want, tol = c.want(c.base)
        assert lowoha.lora_direct(x, c.ids, c.a, c.b, y, y, c.ranks, c.scales) == capi.SUCCESS, lowoha.last_error()
        c.compare(y, want, tol)
    # the router on the adapted logits, then the experts
    bias = (rng.standard_normal(E) * 0.05).astype(np.float32)
    st, ids, w = lowoha.moe_router_grouped(y, topk, capi.SCORE_SIGMOID, H.to_dev(bias), 4, 2, capi.GROUP_TOP2_SUM, True, 1.0)
    assert st == capi.SUCCESS, lowoha.last_error()
    want_ids, want_w = expect(y.double().cpu().numpy(), topk, capi.SCORE_SIGMOID, bias, 4, 2, True, True, 1.0)
    assert np.array_equal(H.to_host(ids), want_ids)
    assert np.all(np.abs(H.to_host(w) - want_w) <= REL_TOL * want_w)
    c = moe
    c.ids, c.w = want_ids, H.to_host(w)
    c.rows_of = [[] for _ in range(E)]
    for t in range(T):
        for k in range(topk):
            e = int(c.ids[t, k])
            c.slot[t, k] = (e, len(c.rows_of[e]))
            c.rows_of[e].append(t)
    blobs13, blobs2 = [H.prepack(t, c.H, 2 * c.I) for t in d.w13], [H.prepack(t, c.I, c.H) for t in d.w2]
    st = lowoha.moe_fused_device(x, ids, w, blobs13, blobs2, d.s13, d.s2, c.I, capi.ACT_SILU_AND_MUL, d.out)
    assert st == capi.SUCCESS, lowoha.last_error()
    MH.check_moe_out(H.to_host(d.out), MH.oracle_moe(zo, c, list(range(T))), flipped_rows=1)
