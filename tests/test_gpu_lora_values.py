"""GPU tests of the values of zmi_lora_direct: infinite and huge operands, and the precision that h is held in."""
import pytest
import torch

from zendnn_amd import capi, lowoha
from tests import gpu_helpers as H
from tests.test_gpu_lora import BF, F32, HF, Case

pytestmark = pytest.mark.gpu

INF = float("inf")


def definition(c, base):
    """dst of a Case in float64 on the host, the products of the second step one by one: infinities meet only what the
    definition lets them meet."""
    ids, x = c.ids.cpu(), c.x.cpu().double()
    y = base.cpu().double() if base is not None else torch.zeros(c.T, sum(c.N), dtype=torch.float64)
    for t in range(c.T):
        s, col = int(ids[t]), 0
        if not 0 <= s < c.S:
            continue
        r = int(c.ranks[s]) if c.ranks is not None else c.rank
        for i, n in enumerate(c.N):
            h = c.a[s, i * c.rank:i * c.rank + r].cpu().double() @ x[t]
            y[t, col:col + n] += float(c.scales[s]) * (c.b[i][s, :, :r].cpu().double() * h).sum(1)
            col += n
    return y


def same_kind(got, want):
    """NaN where the definition has NaN, its infinities where it has them."""
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    odd = torch.isinf(want)
    assert torch.equal(torch.isinf(got), odd) and torch.equal(got[odd], want[odd])


# (calls without and with a launch that sorts the rows; one, two and more blocks of 32 ranks)
CALLS = [(3, 192, [96], 8), (40, 200, [72, 40], 33), (300, 192, [96], 100), (600, 192, [136, 64], 16), (700, 136, [96], 64),
         (600, 72, [44], 128), (530, 72, [44], 200)]


@pytest.mark.parametrize("T,K,N,rank", CALLS)
@pytest.mark.parametrize("dt,dst", [(BF, BF), (HF, HF), (BF, F32), (HF, F32), (HF, BF)])
def test_infinite_adapters(T, K, N, rank, dt, dst):
    """An infinite (or NaN) element of B in slots that rows use: +-inf or NaN in its column alone."""
    c = Case(T + rank, T, K, N, rank, 3, dt, dst, mixed=False)
    c.scales = c.scales.abs() + 0.25
    clean = c.check("other").clone()
    for i, b in enumerate(c.b):
        b[0, 3, 1] = INF
        b[1, 5, rank - 1] = -INF
        b[1, 17, 0] = INF
        b[1, 17, 2] = INF
        b[2, 30, 0] = float("nan")
    y = definition(c, c.base)
    assert torch.isinf(y).any() and torch.isnan(y).any() and torch.isfinite(y).any()
    assert c.call(c.base) == capi.SUCCESS, lowoha.last_error()
    same_kind(c.dst, y)
    whole = torch.isfinite(y).to(H.DEV)
    assert torch.equal(c.dst[whole], clean[whole])   # the other columns keep their bits


@pytest.mark.parametrize("T,K,N,rank", CALLS)
@pytest.mark.parametrize("dt,dst", [(BF, BF), (HF, HF), (BF, F32), (HF, F32), (BF, HF)])
def test_infinite_rows(T, K, N, rank, dt, dst):
    """An infinite x: h is infinite, and so is what positive B makes of it; rows beside it keep their bits."""
    c = Case(T * rank, T, K, N, rank, 3, dt, dst, mixed=False, none=0.0)
    c.scales = c.scales.abs() + 0.25
    c.a.abs_().add_(2.0 ** -10)
    for b in c.b:
        b.abs_().add_(2.0 ** -10)
        b[:, 2] = 0.0                                # (0 * inf)
        b[:, 3, 1:] *= -1.0                          # (inf - inf)
    c.check("dst")
    clean = c.dst.clone()
    c.x[1, 5], c.x[2, K - 1] = INF, -INF
    y = definition(c, c.base)
    assert (y[1] == INF).any() and (y[2] == -INF).any() and torch.isnan(y[1]).any()
    c.dst.copy_(c.base)
    assert c.call(c.dst) == capi.SUCCESS, lowoha.last_error()
    same_kind(c.dst, y)
    keep = [t for t in range(T) if t not in (1, 2)]
    assert torch.equal(c.dst[keep], clean[keep])


@pytest.mark.parametrize("T", [2, 700])
@pytest.mark.parametrize("dst", [BF, F32])
def test_h_between_the_largest_bf16_and_the_largest_f32(T, dst):
    """h = (2 - 2^-9) 2^127 is finite, its nearest bf16 is not; with B = 2^-100 the result is an ordinary number."""
    c = Case(7, T, 64, [40], 8, 2, BF, dst, mixed=False, none=0.0, scales=False)
    c.x.zero_()
    c.a.zero_()
    sign = torch.where(torch.arange(T, device=H.DEV) % 2 == 0, 1.0, -1.0)
    c.x[:, 0], c.x[:, 1] = (sign * (2 - 2.0 ** -7) * 2.0 ** 63).to(BF), (sign * 3 * 2.0 ** 59).to(BF)
    c.a[:, :, 0], c.a[:, :, 1] = 2.0 ** 64, 2.0 ** 59
    c.b = [torch.zeros_like(c.b[0])]
    c.b[0][:, :, 3] = 2.0 ** -100
    assert c.call(None) == capi.SUCCESS, lowoha.last_error()
    want = (sign.double() * (2 - 2.0 ** -9) * 2.0 ** 27).to(dst)[:, None].expand(-1, 40)
    assert torch.equal(c.dst, want)

@pytest.mark.parametrize("T", [1, 40, 300, 700])
@pytest.mark.parametrize("dt,dst", [(BF, BF), (BF, HF), (BF, F32), (HF, HF), (HF, BF), (HF, F32)])
def test_h_keeps_24_bits(T, dt, dst):
    """h of 22 bits, exact in f32, next to a base that cancels all but its lowest ones: what is left is exact, and dst is its
    rounding."""
    c = Case(T, T, 64, [40], 8, 2, dt, dst, mixed=False, none=0.0, scales=False)
    g = torch.Generator(device=H.DEV)
    g.manual_seed(T)
    c.x.zero_()
    c.x[:, 0], c.x[:, 1], c.x[:, 2] = 1.0, 2.0 ** -8, 2.0 ** -15
    a = 1.0 + torch.randint(0, 128, (2, 8, 64), generator=g, device=H.DEV) / 128.0   # 8 bits: h has 1 + 22 of them
    c.a.copy_(a)
    c.b[0].zero_()
    rank_of = torch.randint(0, 8, (2, 40), generator=g, device=H.DEV)
    c.b[0].scatter_(2, rank_of[:, :, None], 1.0)
    h = c.x[:, :3].double()[:, None, :] * c.a.double()[c.ids.long()][:, :, :3]
    h = torch.gather(h.sum(2), 1, rank_of[c.ids.long()])
    assert torch.equal(h, h.float().double())
    c.base.copy_(-h)                                 # (rounded to dst's type)
    want = (h + c.base.double()).to(dst)
    assert c.call(c.base) == capi.SUCCESS, lowoha.last_error()
    assert torch.equal(c.dst, want), float((c.dst.double() - want.double()).abs().max())


@pytest.mark.parametrize("T", [40, 700])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("others", [0.0, 1.0])
def test_rows_that_are_not_finite_from_some_rank_on(T, dt, others):
    """One infinite (or NaN) element of x per row, which A's row r reads with weight 2 and the others with `others`: at 0 their h
    is NaN in front of, between and behind what rank r holds, at 1 all of h is infinite."""
    c = Case(T, T, 192, [40], 37, 3, dt, F32, mixed=False, none=0.0)
    c.scales = c.scales.abs() + 0.25
    c.b[0].abs_().add_(2.0 ** -6)
    c.x[:, 5] = 0.0
    clean, rows = c.x.clone(), [1, 17, T - 1]
    for value in (float("nan"), INF, -INF):
        for r in (0, 7, 8, 31, 32, 36):
            c.x.copy_(clean)
            c.x[rows, 5] = value
            c.a[:, :, 5] = others
            c.a[:, r, 5] = 2.0
            y = definition(c, None)
            assert not torch.isfinite(y[rows]).any()
            assert c.call(None) == capi.SUCCESS, lowoha.last_error()
            same_kind(c.dst, y)
