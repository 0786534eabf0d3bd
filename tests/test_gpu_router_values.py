"""GPU tests of zmi_moe_router_grouped where experts lie far below the best one, and where many of few are chosen.

The weights' tolerance in half steps of 2^-24, whatever the logits' spread.  A chosen expert's exponential is taken in 64 bits.
A softmax's sum has, relative to itself: its terms' 2 ulp (4), the rounding of x - m in front of each (half an ulp of it, so
sum p |x - m|: at most u - 1 where 511 exp(-u) = u - 1, 3.9 for 512 experts), a lane's three additions (3).  The division and
the scale are in 64 bits and the result is rounded once (1): 12 half steps, 7.2e-7, without renormalization, and 1 with it."""
import numpy as np
import pytest
import torch

from zendnn_amd import capi, lowoha
from tests import gpu_helpers as H
from tests.test_gpu_router_grouped import expect

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24


def check(x, topk, scoring, bias=None, n_group=1, topk_group=1, top2=False, renormalize=False, scale=1.0):
    b = H.to_dev(bias) if bias is not None else None
    st, ids, w = lowoha.moe_router_grouped(x, topk, scoring, b, n_group, topk_group, capi.GROUP_TOP2_SUM if top2 else capi.GROUP_MAX,
                                           renormalize, scale)
    assert st == capi.SUCCESS, lowoha.last_error()
    want_ids, want_w = expect(x.double().cpu().numpy(), topk, scoring, bias, n_group, topk_group, top2, renormalize, scale)
    assert np.array_equal(H.to_host(ids), want_ids)
    steps = np.abs(H.to_host(w) - want_w) / (STEP * np.abs(want_w) + 2.0 ** -150)
    allowed = 1.01 if renormalize or scoring == capi.SCORE_SIGMOID else 12   # (0.01: what 64 bits leave)
    assert steps.max() <= allowed, (steps.max(), want_w.flat[steps.argmax()])


@pytest.mark.parametrize("scoring", [capi.SCORE_SOFTMAX, capi.SCORE_SIGMOID])
@pytest.mark.parametrize("spread", [1.5, 5.0, 10.0, 20.0, 40.0])
@pytest.mark.parametrize("T,E,topk", [(200, 512, 64), (200, 256, 32), (100, 64, 64), (100, 100, 16)])
@pytest.mark.parametrize("renormalize", [False, True])
def test_weights_of_experts_far_below_the_best(scoring, spread, T, E, topk, renormalize):
    rng = np.random.default_rng(int(spread * 10) + E)
    x = (rng.standard_normal((T, E)) * spread).astype(np.float32)
    check(H.to_dev(x), topk, scoring, None, renormalize=renormalize, scale=1.5)
    bias = (rng.standard_normal(E) * 0.05).astype(np.float32)
    check(H.to_dev(x), topk, scoring, bias, renormalize=renormalize)


@pytest.mark.parametrize("E", [8, 64, 512])
def test_weights_where_the_roundings_of_x_minus_m_add_up(E):
    """One expert ahead of equal others, at the distance where their share of the sum times it is largest."""
    u = 4.88 if E == 512 else 3.0 if E == 64 else 1.5
    rng = np.random.default_rng(E)
    x = (rng.random((300, E)).astype(np.float32) * 1e-3 + np.float32(1.7)).astype(np.float32)
    x[:, 3] += np.float32(u)
    check(H.to_dev(x), min(E, 64), capi.SCORE_SOFTMAX)
    check(H.to_dev(-x), min(E, 64), capi.SCORE_SOFTMAX)


@pytest.mark.parametrize("scoring", [capi.SCORE_SOFTMAX, capi.SCORE_SIGMOID])
@pytest.mark.parametrize("E", [512, 500, 300])
@pytest.mark.parametrize("topk", [4, 8, 10, 12, 16, 32, 64])
@pytest.mark.parametrize("together", [2, 3, 4, 5, 8, 11])
def test_best_experts_next_to_each_other(scoring, E, topk, together):
    """More than 256 experts stand in eights: tokens whose best ones share an eight, at its start and across its end."""
    rng = np.random.default_rng(E + topk + together)
    x = rng.standard_normal((48, E)).astype(np.float32)
    bias = (rng.standard_normal(E) * 0.01).astype(np.float32)
    for t in range(48):
        at = min((t * 8 + (0 if t % 3 else 3)) % E, E - together)
        x[t, at:at + together] += np.float32(4.0)
        if t % 4 == 0:      # two such places, one of them at the border of the choice
            at = (at + E // 2) % (E - together)
            x[t, at:at + together] = np.sort(x[t])[-topk] + rng.permutation(together).astype(np.float32) * np.float32(1e-2)
        if t % 5 == 0:      # equal ones
            x[t, at:at + together] = x[t, at]
    for b in (None, bias, np.zeros(E, dtype=np.float32)):
        check(H.to_dev(x), topk, scoring, b, renormalize=True)


@pytest.mark.parametrize("E,n_group,topk_group,topk", [(512, 8, 1, 8), (512, 8, 1, 64), (512, 64, 2, 16), (512, 64, 1, 8), (320, 64, 1, 5),
                                                       (320, 64, 3, 12), (500, 50, 2, 20), (300, 4, 1, 40), (512, 8, 2, 4), (512, 8, 2, 33)])
@pytest.mark.parametrize("scoring", [capi.SCORE_SOFTMAX, capi.SCORE_SIGMOID])
@pytest.mark.parametrize("biased", [False, True])
def test_many_of_the_experts_of_few_groups(E, n_group, topk_group, topk, scoring, biased):
    rng = np.random.default_rng(E + topk)
    x = rng.standard_normal((64, E)).astype(np.float32)
    bias = (rng.standard_normal(E) * 0.05).astype(np.float32) if biased else None
    check(H.to_dev(x), topk, scoring, bias, n_group, topk_group, False, True)
    check(H.to_dev(x), topk, scoring, bias, n_group, topk_group, True, False)
    x = np.round(x * 4) / 4          # many equal values
    check(H.to_dev(x.astype(np.float32)), topk, scoring, bias, n_group, topk_group, True, True)
