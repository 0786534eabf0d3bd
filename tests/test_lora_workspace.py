"""Tests of zmi_lora_workspace_size: a workspace for T rows serves every shorter batch."""
import random

import pytest
import torch

from zendnn_amd import capi, lowoha
from tests.test_cabi_host import fake_pointers
from tests.test_router_lora_host import ADDR, lora


def sizes(rng):
    n = [rng.choice([1, 40, 512, 4097]) for _ in range(rng.randint(1, 4))]
    K, rank = rng.choice([1, 63, 520, 4096, 14336, 1 << 19]), rng.choice([1, 8, 16, 33, 64, 128, 256])
    return dict(K=K, ldx=K, rank=rank, N=tuple(n), n_slots=rng.choice([1, 3, 16, 17, 300, 4096]), a_ld=K, a_slot=len(n) * rank * K,
                b_ld=rank, b_slot=rank * 4097, dt_x=rng.choice([capi.DT_BF16, capi.DT_F16]),
                dt_dst=rng.choice([capi.DT_BF16, capi.DT_F32]))


@fake_pointers
@pytest.mark.parametrize("seed", range(40))
def test_size_grows_with_the_batch_and_serves_shorter_ones(seed):
    rng = random.Random(seed)
    kw, last = sizes(rng), 0
    rows = sorted({1, 2, 16, 127, 128, 129, 511, 512, 513, 2047, 2048, 2049, 8193, 40000, 1 << 20, *(rng.randint(1, 3000) for _ in range(200))})
    for i, T in enumerate(rows):
        size = lora(True, T=T, **kw)
        assert size >= last, (kw, T)
        last = size
        for t in {T, *rng.sample(rows[:i + 1], min(i + 1, 6))}:
            st, err = lora(T=t, workspace=ADDR, workspace_bytes=size, **kw)
            assert st == capi.FAILURE and "64 KiB" in err, (kw, T, t, err)   # (every other rule is passed)
    assert lora(True, T=0, **kw) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rank,S", [(8, 3), (64, 40)])
def test_one_workspace_for_batches_of_all_lengths(rank, S):
    from tests.test_gpu_lora import Case
    size = None
    for T in (700, 1, 24, 128, 129, 300, 513, 699):
        c = Case(T, T, 2048, [72, 8], rank, S)
        if size is None:
            size = lowoha.lora_workspace_size(c.x, c.ids, c.a, c.b, c.dst)
            ws = torch.empty(size + 256, dtype=torch.uint8, device="cuda:0")
        ws.fill_(0xff)
        y, tol = c.want(c.base)
        assert c.call(c.base, workspace=ws[:size]) == capi.SUCCESS, lowoha.last_error()
        c.compare(c.dst, y, tol)
        assert (ws[size:] == 0xff).all()
