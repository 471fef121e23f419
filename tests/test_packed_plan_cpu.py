"""prefill_packed with a plan: lengths that only begin where the plan's do are refused before anything is launched."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


def fake(shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="cuda:0")


def same_start(t):
    """t's own storage address, whatever view of it is asked (a fake tensor has none)."""
    return 4096


@pytest.mark.parametrize("which", ["cu strided", "cu int64", "cu too long", "lens strided", "lens int64"])
def test_other_views_of_the_plans_lengths(monkeypatch, which):
    from atflash import _lib, ops
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("reached the library"))
    monkeypatch.setattr(torch.Tensor, "data_ptr", same_start)
    with FakeTensorMode():
        cu, lens = fake(4), fake(3)
        plan = ops.PackedPlan.__new__(ops.PackedPlan)
        plan.cu_seqlens, plan.seq_lens, plan.batch, plan.total_q, plan.max_seq_len, plan.num_q_heads = cu, lens, 3, 9, 64, 4
        plan.tiles = fake(8)
        if which == "cu strided":
            cu = fake(8)[::2]
        elif which == "cu int64":
            cu = fake(4, torch.int64)
        elif which == "cu too long":
            cu = fake(5)
        elif which == "lens strided":
            lens = fake(6)[::2]
        else:
            lens = fake(3, torch.int64)
        q, kv = fake((9, 4, 128), torch.bfloat16), fake((8, 2, 2, 2048), torch.bfloat16)
        with pytest.raises(ValueError):
            ops.prefill_packed(q, kv, fake((3, 4)), cu, lens, 64, None, 0.1, None, 0, plan)
