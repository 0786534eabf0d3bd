"""CPU tests of the refusals of zmi_moe_router_grouped and zmi_lora_direct, of their defaults and of the workspace size.
Every call here is refused before anything touches an address."""
import ctypes as C

import pytest

from zendnn_amd import capi, lowoha
from tests.test_cabi_host import fake_pointers

ADDR = 0x1000   # (in the first 64 KiB: a call that passes every other rule is refused for its addresses)


def router(**kw):
    r = capi.MoeRouterT()
    capi.load().zmi_moe_router_params_init(C.byref(r))
    r.T, r.E, r.topk, r.ldl = 4, 64, 6, 64
    r.logits = r.topk_ids = r.topk_weights = ADDR
    for k, v in kw.items():
        setattr(r, k, v)
    return capi.load().zmi_moe_router_grouped(C.byref(r)), lowoha.last_error()


def lora(_size=False, N=(32,), b=ADDR, b_ld=8, b_slot=32 * 8, **kw):
    l = capi.LoraT()
    capi.load().zmi_lora_params_init(C.byref(l))
    l.T, l.K, l.rank, l.n_slices, l.n_slots = 4, 64, 8, len(N), 3
    l.x = l.slot_ids = l.a = l.dst = ADDR
    l.ldx, l.a_ld, l.a_slot, l.ld_dst = 64, 64, len(N) * 8 * 64, sum(N)
    for i, n in enumerate(N[:capi.LORA_MAX_SLICES]):
        l.N[i], l.b[i], l.b_ld[i], l.b_slot[i] = n, b, b_ld, b_slot
    for k, v in kw.items():
        setattr(l, k, v)
    lib = capi.load()
    if _size:
        return lib.zmi_lora_workspace_size(C.byref(l))
    return lib.zmi_lora_direct(C.byref(l)), lowoha.last_error()


def test_defaults():
    r, l = capi.MoeRouterT(), capi.LoraT()
    capi.load().zmi_moe_router_params_init(C.byref(r))
    capi.load().zmi_lora_params_init(C.byref(l))
    assert (r.n_group, r.topk_group, r.scale, r.logits_dt, r.scoring, r.group_score) == (1, 1, 1.0, capi.DT_F32, 0, 0)
    assert (l.n_slices, l.dt_x, l.dt_dst, l.base, l.workspace) == (1, capi.DT_BF16, capi.DT_BF16, None, None)


@fake_pointers
@pytest.mark.parametrize("kw,status,text", [
    (dict(T=-1), capi.FAILURE, "bad arguments"), (dict(E=0), capi.FAILURE, "bad arguments"),
    (dict(topk=0), capi.FAILURE, "bad arguments"), (dict(ldl=63), capi.FAILURE, "bad arguments"),
    (dict(n_group=0), capi.FAILURE, "bad arguments"), (dict(n_group=-2), capi.FAILURE, "bad arguments"),
    (dict(E=513, ldl=513), capi.UNIMPLEMENTED, "512"), (dict(E=512, ldl=512, topk=65), capi.UNIMPLEMENTED, "64"),
    (dict(E=65, ldl=65, n_group=65), capi.UNIMPLEMENTED, "64 groups"),
    (dict(n_group=5), capi.FAILURE, "divide"), (dict(n_group=4, topk_group=5), capi.FAILURE, "topk_group"),
    (dict(n_group=4, topk_group=0), capi.FAILURE, "topk_group"), (dict(n_group=16, topk_group=1), capi.FAILURE, "topk exceeds"),
    (dict(E=5, ldl=5), capi.FAILURE, "topk exceeds"),
    (dict(scoring=2), capi.FAILURE, "scoring"), (dict(group_score=-1), capi.FAILURE, "group_score"),
    (dict(n_group=64, topk_group=8, group_score=capi.GROUP_TOP2_SUM), capi.FAILURE, "groups of two"),
    (dict(logits_dt=capi.DT_S8), capi.FAILURE, "f32, bf16 or f16"),
    (dict(logits=None), capi.FAILURE, "null"), (dict(topk_ids=None), capi.FAILURE, "null"),
    (dict(topk_weights=None), capi.FAILURE, "null"),
    (dict(logits=ADDR + 2), capi.FAILURE, "multiple"), (dict(bias=ADDR + 1), capi.FAILURE, "multiple"),
    (dict(), capi.FAILURE, "64 KiB"), (dict(logits=ADDR + 2, logits_dt=capi.DT_BF16), capi.FAILURE, "64 KiB"),
    (dict(T=0, logits=None, topk_ids=None, topk_weights=None), capi.SUCCESS, "")])
def test_router_refusals(kw, status, text):
    st, err = router(**kw)
    assert st == status and text in err, err


@fake_pointers
@pytest.mark.parametrize("kw,status,text", [
    (dict(T=-1), capi.FAILURE, "bad sizes"), (dict(K=0), capi.FAILURE, "bad sizes"), (dict(rank=0), capi.FAILURE, "bad sizes"),
    (dict(n_slots=0), capi.FAILURE, "bad sizes"), (dict(n_slices=0), capi.FAILURE, "bad sizes"),
    (dict(N=(32, 0)), capi.FAILURE, "bad sizes"), (dict(N=(8,) * 5), capi.UNIMPLEMENTED, "4 slices"),
    (dict(rank=257), capi.UNIMPLEMENTED, "256"), (dict(n_slots=4097), capi.UNIMPLEMENTED, "slots"),
    (dict(N=(0x7fffffff, 0x7fffffff)), capi.UNIMPLEMENTED, "columns"),
    (dict(T=(1 << 20) + 1), capi.UNIMPLEMENTED, "rows"), (dict(K=(1 << 19) + 1), capi.UNIMPLEMENTED, "2^19"),
    (dict(dt_x=capi.DT_F32), capi.UNIMPLEMENTED, "dt_x"), (dict(dt_dst=capi.DT_S8), capi.UNIMPLEMENTED, "dt_dst"),
    (dict(x=None), capi.FAILURE, "null"), (dict(slot_ids=None), capi.FAILURE, "null"), (dict(dst=None), capi.FAILURE, "null"),
    (dict(a=None), capi.FAILURE, "a is null"), (dict(a_ld=63), capi.FAILURE, "a is null"),
    (dict(a_slot=8 * 64 - 1), capi.FAILURE, "a is null"), (dict(a_slot=-8 * 64), capi.FAILURE, "a is null"),
    (dict(a=ADDR + 1), capi.FAILURE, "a is null"),
    (dict(b=None), capi.FAILURE, "b is null"), (dict(b_ld=7), capi.FAILURE, "b is null"), (dict(b_slot=255), capi.FAILURE, "b is null"),
    (dict(ldx=63), capi.FAILURE, "row stride"), (dict(ld_dst=31), capi.FAILURE, "row stride"),
    (dict(N=(32, 32), ld_dst=63), capi.FAILURE, "row stride"),
    (dict(base=ADDR + 16, ld_base=31), capi.FAILURE, "row stride"), (dict(base=ADDR, ld_base=40), capi.FAILURE, "dst's row stride"),
    (dict(x=ADDR + 1), capi.FAILURE, "multiple"), (dict(dst=ADDR + 1), capi.FAILURE, "multiple"),
    (dict(dst=ADDR + 2, dt_dst=capi.DT_F32), capi.FAILURE, "multiple"), (dict(slot_ids=ADDR + 2), capi.FAILURE, "multiple"),
    (dict(ranks=ADDR + 1), capi.FAILURE, "multiple"), (dict(scales=ADDR + 2), capi.FAILURE, "multiple"),
    (dict(workspace=ADDR + 8, workspace_bytes=1 << 30), capi.FAILURE, "multiple"),
    (dict(), capi.FAILURE, "64 KiB"), (dict(n_slots=1, a_slot=0, b_slot=0), capi.FAILURE, "64 KiB"),
    (dict(T=0, x=None, slot_ids=None, dst=None, a=None), capi.SUCCESS, "")])
def test_lora_refusals(kw, status, text):
    st, err = lora(**kw)
    assert st == status and text in err, err


@fake_pointers
def test_a_workspace_that_is_too_small_is_refused():
    big = dict(T=300, K=4096, ldx=4096, a_ld=4096, a_slot=8 * 4096)
    need = lora(True, **big)
    assert need > 0
    st, err = lora(workspace=ADDR, workspace_bytes=need - 1, **big)
    assert st == capi.FAILURE and "workspace" in err
    st, err = lora(workspace=ADDR, workspace_bytes=need, **big)
    assert st == capi.FAILURE and "64 KiB" in err


def test_workspace_size_of_refused_sizes_is_zero():
    assert lora(True, rank=0) == 0 and lora(True, T=-1) == 0 and lora(True, dt_x=capi.DT_S8) == 0
    assert capi.load().zmi_lora_workspace_size(None) == 0
    assert capi.load().zmi_lora_direct(None) == capi.FAILURE and "null" in lowoha.last_error()
    assert capi.load().zmi_moe_router_grouped(None) == capi.FAILURE


def test_python_wrappers_refuse_tensors_they_cannot_describe():
    import torch
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="not on the GPU"):
        lowoha.moe_router_grouped(x, 2)
    with pytest.raises(ValueError, match="dtype"):
        lowoha.moe_router_grouped(x.to(torch.int8), 2)
    with pytest.raises(ValueError, match="dtype"):
        lowoha.lora_direct(x.float(), torch.zeros(4, dtype=torch.int32), x, x, x)
    with pytest.raises(ValueError, match="slices"):
        lowoha.lora_direct(x, torch.zeros(4, dtype=torch.int32), x, [], x)


@fake_pointers
def test_router_batches_longer_than_a_launch_are_refused():
    for T in ((1 << 25) + 1, 0x7fffffff):
        st, err = router(T=T)
        assert st == capi.UNIMPLEMENTED and "2^25" in err
    st, err = router(T=1 << 25)
    assert st == capi.FAILURE and "64 KiB" in err
