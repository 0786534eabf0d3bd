"""GPU tests of zmi_lora_direct's tile shapes over a K that goes several times round their LDS rings, and of what a row's bits
depend on."""
import pytest
import torch

from zendnn_amd import capi, lowoha
from tests import gpu_helpers as H
from tests.test_gpu_lora import BF, F32, HF, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,pad", [(BF, 0), (HF, 0), (BF, 5), (HF, 3)])
@pytest.mark.parametrize("T,K,N,rank", [
    (20000, 1048, [16], 16), (20000, 1300, [24], 9),     # two row groups, one rank tile: stages of 256
    (33000, 648, [8], 8), (33000, 712, [16], 16),        # four, one: of 128
    (20000, 776, [16], 32), (33000, 776, [8], 32),       # two and four, two
    (20000, 648, [8], 64), (33000, 392, [8], 64), (33000, 456, [8, 8], 32),   # two and four, four
    (8192, 392, [8], 128)])                              # four, eight
def test_tile_shapes_of_a_long_k(T, K, N, rank, dt, pad):
    Case(T + rank, T, K, N, rank, 2, dt, mixed=False, pad=pad, w_pad=pad).check("other")


@pytest.mark.parametrize("T,K,N,rank,S,dt,dst", [
    (24, 4096, [200, 64], 16, 3, BF, BF), (300, 1024, [192], 16, 3, HF, HF), (100, 520, [64], 64, 40, BF, F32),
    (700, 1024, [264], 32, 4, BF, BF), (2048, 4096, [96], 8, 16, BF, F32), (2300, 2056, [128], 128, 3, HF, HF)])
def test_a_row_has_the_same_bits_whatever_the_other_rows_hold(T, K, N, rank, S, dt, dst):
    """Same sizes and slot ids, every other row's x and base replaced (some by what is not finite): calls with and without a
    sorting launch, units cut into several pieces that meet in any order of arrival."""
    c = Case(T, T, K, N, rank, S, dt, dst)
    c.check("other")
    first = c.dst.clone()
    g = torch.Generator(device=H.DEV)
    g.manual_seed(T)
    for k in range(8):
        other = torch.rand(T, generator=g, device=H.DEV) < 0.5
        x, base = c.x.clone(), c.base.clone()
        c.x[other] = (torch.randn(int(other.sum()), K, generator=g, device=H.DEV) * 3).to(dt)
        c.base[other] = 0.0
        c.x[other.nonzero()[:, 0][::7], k] = float("inf" if k % 2 else "nan")
        assert c.call(c.base) == capi.SUCCESS, lowoha.last_error()
        assert torch.equal(c.dst[~other], first[~other])
        c.x.copy_(x)
        c.base.copy_(base)
    assert c.call(c.base) == capi.SUCCESS and torch.equal(c.dst, first)
