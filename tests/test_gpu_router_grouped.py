"""GPU tests of zmi_moe_router_grouped (through the C ABI): ids bit-exact and weights to 1e-6 relative against the
definition in float64 on the host.

The weights' tolerance, in half steps of 2^-24: a score's exponential is within 2 ulp (4 half steps), the terms of a
softmax's sum are too, and a lane adds up to eight of them in f32, three roundings deep (7 together); sums over lanes and
over the chosen, the division and the scale are in 64 bits, and the result is rounded once: 4 + 7 + 1 = 12 half steps,
7.2e-7.
"""
import numpy as np
import pytest
import torch

from zendnn_amd import capi, lowoha
from tests import gpu_helpers as H

pytestmark = pytest.mark.gpu

REL_TOL = 1e-6


def expect(logits, topk, scoring, bias=None, n_group=1, topk_group=1, top2=False, renormalize=False, scale=1.0):
    """logits: float64 [T, E] holding the values the GPU reads."""
    T, E = logits.shape
    with np.errstate(over="ignore", invalid="ignore"):
        if scoring == capi.SCORE_SIGMOID:
            s = 1.0 / (1.0 + np.exp(-logits))
        else:
            m = np.max(logits, axis=1, keepdims=True)
            e = np.where(logits == -np.inf, 0.0, np.where(logits == m, 1.0, np.exp(logits - m)))
            z = e.sum(axis=1, keepdims=True)
            s = np.where(z == 0, 0.0, e / np.where(z == 0, 1.0, z))
    v = s + bias.astype(np.float64) if bias is not None else s
    order = v if bias is not None else logits
    live = np.ones((T, E), dtype=bool)
    if topk_group < n_group:
        per = E // n_group
        by = (v if top2 else order).reshape(T, n_group, per)
        top = -np.sort(-by, axis=2)
        g = top[:, :, 0] + top[:, :, 1] if top2 else top[:, :, 0]
        kept = np.argsort(-g, axis=1, kind="stable")[:, :topk_group]
        ok = np.zeros((T, n_group), dtype=bool)
        np.put_along_axis(ok, kept, True, axis=1)
        live = np.repeat(ok, per, axis=1)
    # (a chosen set among the live experts: stable descending, the others behind all of them)
    ids = np.zeros((T, topk), dtype=np.int32)
    for t in range(T):
        cand = np.nonzero(live[t])[0]
        ids[t] = cand[np.argsort(-order[t, cand], kind="stable")][:topk]
    w = np.take_along_axis(s, ids.astype(np.int64), axis=1)
    if renormalize:
        z = w.sum(axis=1, keepdims=True)
        w = np.where(z == 0, 0.0, w / np.where(z == 0, 1.0, z))
    return ids, w * scale


def check(x, topk, scoring, bias=None, n_group=1, topk_group=1, top2=False, renormalize=False, scale=1.0):
    """x: a GPU tensor as the call gets it."""
    b = H.to_dev(bias) if bias is not None else None
    st, ids, w = lowoha.moe_router_grouped(x, topk, scoring, b, n_group, topk_group,
                                           capi.GROUP_TOP2_SUM if top2 else capi.GROUP_MAX, renormalize, scale)
    assert st == capi.SUCCESS, lowoha.last_error()
    assert lowoha.last_kernel().startswith("moe_router_grouped")
    want_ids, want_w = expect(x.double().cpu().numpy(), topk, scoring, bias, n_group, topk_group, top2, renormalize, scale)
    got_ids, got_w = H.to_host(ids), H.to_host(w)
    bad = np.nonzero((got_ids != want_ids).any(axis=1))[0]
    assert not len(bad), (bad[:4], got_ids[bad[:2]], want_ids[bad[:2]])
    assert np.all(np.abs(got_w - want_w) <= REL_TOL * np.abs(want_w) + 2.0 ** -149)
    return got_ids, got_w


def gen(seed, T, E, dt=torch.float32, std=1.5, pad=0):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((T, E + pad)) * std + rng.standard_normal(E + pad) * 0.7).astype(np.float32)
    return H.to_dev(x).to(dt)[:, :E], (rng.standard_normal(E) * 0.05).astype(np.float32)


@pytest.mark.parametrize("T,E,topk,n_group,topk_group", [
    (1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (1, 8, 8, 2, 2), (3, 4, 2, 2, 1), (5, 64, 6, 1, 1), (64, 64, 6, 8, 3), (65, 63, 5, 9, 2),
    (7, 60, 10, 5, 2), (33, 65, 4, 1, 1), (130, 128, 8, 4, 2), (19, 160, 6, 8, 3), (40, 512, 64, 1, 1), (9, 512, 64, 64, 8),
    (513, 256, 8, 8, 4), (300, 384, 8, 1, 1), (17, 500, 7, 50, 3), (6, 128, 64, 64, 32), (31, 257, 3, 1, 1), (21, 16, 4, 4, 4)])
@pytest.mark.parametrize("scoring", [capi.SCORE_SIGMOID, capi.SCORE_SOFTMAX])
@pytest.mark.parametrize("biased,top2,renormalize", [(True, True, True), (True, False, False), (False, False, True), (False, True, False)])
def test_random_logits(T, E, topk, n_group, topk_group, scoring, biased, top2, renormalize):
    x, bias = gen(T * 7 + E, T, E)
    if E // n_group < 2 and n_group > 1:
        top2 = False
    check(x, topk, scoring, bias if biased else None, n_group, topk_group, top2, renormalize, 2.5)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,E,pad,offset", [(77, 64, 16, 0), (40, 256, 5, 1), (9, 61, 3, 3), (100, 512, 0, 0), (200, 128, 0, 0)])
def test_types_row_strides_and_offsets(dt, T, E, pad, offset):
    """Rows of a wider buffer and rows that start at odd elements of it."""
    x, bias = gen(T + E, T, E, dt, pad=pad)
    if offset:
        x = torch.empty(T * (E + pad) + offset, dtype=dt, device=H.DEV)[offset:].view(T, E + pad)[:, :E].copy_(x)
    check(x, 8, capi.SCORE_SIGMOID, bias, renormalize=True)
    check(x, 8, capi.SCORE_SOFTMAX, None, renormalize=False)


@pytest.mark.parametrize("scoring", [capi.SCORE_SIGMOID, capi.SCORE_SOFTMAX])
@pytest.mark.parametrize("E,n_group,topk_group", [(64, 1, 1), (256, 8, 4), (96, 6, 2)])
def test_equal_values_go_to_the_lower_expert_and_group(scoring, E, n_group, topk_group):
    rng = np.random.default_rng(E)
    x = (rng.integers(-2, 3, size=(200, E)) * 0.5).astype(np.float32)
    x[0] = 1.25
    x[1] = np.where(rng.random(E) < 0.5, 0.0, -0.0)
    x[2] = -3.0
    x[2, E - 1] = 7.0
    for bias in (None, np.zeros(E, dtype=np.float32), np.full(E, 0.25, dtype=np.float32)):
        for top2 in (False, True):
            ids, _ = check(H.to_dev(x), 8, scoring, bias, n_group, topk_group, top2)
            assert ids[0].tolist() == list(range(8)) and ids[1].tolist() == list(range(8)) and ids[2, 0] == E - 1


@pytest.mark.parametrize("scoring", [capi.SCORE_SIGMOID, capi.SCORE_SOFTMAX])
@pytest.mark.parametrize("spread", [1e-2, 1e-4, 1e-6])
def test_values_nearer_than_32_bits_can_tell(scoring, spread):
    """Distinct f32 logits whose scores (and sums with the bias) collide in f32: the choice is that of 64 bits."""
    rng = np.random.default_rng(int(1 / spread))
    T, E = 64, 256
    x = (rng.random((T, E)) * spread).astype(np.float32)
    bias = np.full(E, 0.37, dtype=np.float32)
    check(H.to_dev(x), 16, scoring, bias, renormalize=True)
    check(H.to_dev(x), 16, scoring, bias, 8, 4, True)
    check(H.to_dev(x), 16, scoring, bias, 8, 4, False)
    check(H.to_dev(x), 16, scoring, None, 8, 4, True)
    x[:, ::3] = x[:, :1]                 # and values that are equal, among them
    check(H.to_dev(x), 16, scoring, bias, 8, 2, True)


def test_a_long_batch_of_close_calls():
    """Enough tokens that some have two values within an f32 ulp at the border of the choice."""
    x, bias = gen(5, 20000, 256)
    check(x, 8, capi.SCORE_SIGMOID, bias, 8, 4, True, True, 2.5)
    check(x, 8, capi.SCORE_SOFTMAX, bias * 0.01, 1, 1, False, True)


@pytest.mark.parametrize("scoring", [capi.SCORE_SIGMOID, capi.SCORE_SOFTMAX])
@pytest.mark.parametrize("biased", [False, True])
def test_masked_experts_and_rows(scoring, biased):
    E = 64
    x, bias = gen(9, 8, E)
    b = bias if biased else None
    low = torch.finfo(torch.float32).min
    x[0, 5:] = -float("inf")             # fewer live experts than topk
    x[1] = -float("inf")                 # none
    x[2, ::2] = -float("inf")
    x[3] = low                           # a mask of the type's lowest value on every expert ...
    x[4, 3:] = low                       # ... and on most
    x[5, 7] = float("inf")
    x[6, 1:] = 100.0                     # saturated scores
    x[6, 0] = 101.0
    x[7] = torch.linspace(-300.0, 300.0, E)
    for renormalize in (False, True):
        ids, w = check(x, 8, scoring, b, renormalize=renormalize)
        assert np.isfinite(w).all()
        check(x, 8, scoring, b, 8, 3, True, renormalize=renormalize)
        check(x, 8, scoring, b, 8, 3, False, renormalize=renormalize)
    if scoring == capi.SCORE_SOFTMAX:
        assert (w[1] == 0).all()         # nothing left: no weight


def test_experts_disabled_by_their_bias():
    x, bias = gen(4, 50, 64)
    bias[::2] = -np.inf
    ids, _ = check(x, 8, capi.SCORE_SIGMOID, bias)
    assert (ids % 2 == 1).all()
    check(x, 8, capi.SCORE_SIGMOID, bias, 8, 2, False)
    check(x, 40, capi.SCORE_SIGMOID, bias)                      # more than are enabled
    bias[5] = np.inf
    ids, _ = check(x, 8, capi.SCORE_SOFTMAX, bias)
    assert (ids[:, 0] == 5).all()


def test_nan_logits_are_chosen_last():
    x, bias = gen(2, 6, 32)
    x[0, 7] = float("nan")
    x[1, 3:] = float("nan")
    x[2] = float("nan")
    for b in (None, H.to_dev(bias)):
        st, ids, w = lowoha.moe_router_grouped(x, 4, capi.SCORE_SIGMOID, b)
        assert st == capi.SUCCESS
        ids, w = H.to_host(ids), H.to_host(w)
        assert 7 not in ids[0] and np.isfinite(w[0]).all()
        assert set(ids[1, :3]) == {0, 1, 2} and ids[1, 3] == 3 and np.isnan(w[1, 3]) and np.isfinite(w[1, :3]).all()
        assert ids[2].tolist() == [0, 1, 2, 3] and np.isnan(w[2]).all()
    # every id stays in range and distinct whatever the row holds, in groups too
    st, ids, w = lowoha.moe_router_grouped(x, 8, capi.SCORE_SOFTMAX, H.to_dev(bias), 4, 2, capi.GROUP_TOP2_SUM, True)
    ids = np.sort(H.to_host(ids), axis=1)
    assert st == capi.SUCCESS and ids.min() >= 0 and ids.max() < 32 and (ids[:, 1:] != ids[:, :-1]).all()


def test_without_groups_and_bias_it_is_the_softmax_router():
    x, _ = gen(8, 333, 128, torch.bfloat16)
    st, ids, w = lowoha.moe_router_grouped(x, 6, capi.SCORE_SOFTMAX, renormalize=True)
    st2, ids2, w2 = lowoha.moe_router_topk(x, 6, True)
    assert st == st2 == capi.SUCCESS and torch.equal(ids, ids2)
    assert ((w - w2).abs() <= 2 * REL_TOL * w2).all()


def test_empty_batch_and_rows_behind_the_batch():
    st, ids, w = lowoha.moe_router_grouped(torch.empty(0, 64, device=H.DEV), 6)
    assert st == capi.SUCCESS and ids.shape == (0, 6)
    import ctypes as C
    x, _ = gen(3, 5, 64)
    ids = torch.full((9, 6), -7, dtype=torch.int32, device=H.DEV)
    w = torch.full((9, 6), -7.0, device=H.DEV)
    r = capi.MoeRouterT()
    capi.load().zmi_moe_router_params_init(C.byref(r))
    r.T, r.E, r.topk, r.logits, r.ldl = 5, 64, 6, x.data_ptr(), 64
    r.topk_ids, r.topk_weights = ids[2:].data_ptr(), w[2:].data_ptr()
    assert capi.load().zmi_moe_router_grouped(C.byref(r)) == capi.SUCCESS
    torch.cuda.synchronize()
    for o in (ids, w):
        assert (o[:2] == -7).all() and (o[7:] == -7).all() and (o[2:7] != -7).all()


def test_captured_and_replayed_on_another_stream():
    x, bias = gen(6, 100, 256)
    b = H.to_dev(bias)
    call, ids, w = lowoha.prepared_moe_router_grouped(x, 8, capi.SCORE_SIGMOID, b, 8, 4, capi.GROUP_TOP2_SUM, True, 2.5)
    s = torch.cuda.Stream()
    lib = capi.load()
    try:
        with torch.cuda.stream(s):
            lib.zmi_set_stream(s.cuda_stream)
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=s):
                assert call() == capi.SUCCESS, lowoha.last_error()
    finally:
        lib.zmi_set_stream(None)
    for k in range(4):
        y, _ = gen(60 + k, 100, 256)
        x.copy_(y)
        ids.fill_(-1)
        g.replay()
        torch.cuda.synchronize()
        want_ids, want_w = expect(y.double().cpu().numpy(), 8, capi.SCORE_SIGMOID, bias, 8, 4, True, True, 2.5)
        assert np.array_equal(H.to_host(ids), want_ids)
        assert np.all(np.abs(H.to_host(w) - want_w) <= REL_TOL * want_w)


def test_logits_far_apart_in_memory():
    """Row offsets beyond 2^31 elements."""
    stride = (1 << 30) + 12345
    buf = torch.empty(2 * stride + 64, dtype=torch.bfloat16, device=H.DEV)
    x = buf.as_strided((3, 64), (stride, 1))
    y, bias = gen(1, 3, 64, torch.bfloat16)
    x.copy_(y)
    check(x, 6, capi.SCORE_SIGMOID, bias, 8, 4, True, True)
