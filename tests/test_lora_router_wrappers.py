"""Tests of what the Python wrappers of zmi_lora_direct and zmi_moe_router_grouped refuse ahead of the call."""
import pytest
import torch

from zendnn_amd import capi, lowoha


def operands(dev="cpu"):
    t = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device=dev)   # noqa: E731
    return dict(x=t(4, 64), slot_ids=t(4, dt=torch.int32), a=t(3, 8, 64), b=t(3, 32, 8), dst=t(4, 32))


def test_a_workspace_that_is_not_one_piece_is_refused():
    """An expanded view has more elements than memory behind it, a strided one other bytes than its own between them."""
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(1 << 30), torch.zeros(1, 4, dtype=torch.uint8).expand(1 << 20, 4),
               torch.zeros(64, 2, dtype=torch.uint8)[:, 0], torch.zeros(8, 8, dtype=torch.uint8).t()):
        for fn in (lowoha.lora_direct, lowoha.prepared_lora):
            with pytest.raises(ValueError, match="workspace"):
                fn(**operands(), workspace=ws)


def test_sizes_that_32_bits_do_not_hold_are_refused():
    """(the argument block would take them modulo 2^32)"""
    far = torch.zeros(1, 1, dtype=torch.bfloat16).expand((1 << 32) + 4, 1)
    with pytest.raises(ValueError, match="2\\^31"):
        lowoha.moe_router_grouped(far, 1)
    with pytest.raises(ValueError, match="2\\^31"):
        lowoha.lora_direct(**operands() | dict(x=far))


@pytest.mark.gpu
def test_tensors_on_another_device_than_the_current_one_are_refused(monkeypatch):
    """(the library launches on the current one)"""
    args = operands("cuda:0")
    assert lowoha.lora_direct(**args) == capi.SUCCESS
    assert lowoha.moe_router_grouped(args["x"], 2)[0] == capi.SUCCESS
    torch.cuda.synchronize()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        lowoha.lora_direct(**args)
    with pytest.raises(ValueError, match="current device"):
        lowoha.moe_router_grouped(args["x"], 2)
