"""flash_attn_packed as a registered operator, as its siblings are: fake outputs, the kernel's bits, a compiled function
without a graph break."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF = torch.bfloat16


def test_fake():
    from atflash import ops  # noqa: F401
    with FakeTensorMode():
        q, k = (torch.empty((10, h, 128), dtype=BF, device="cuda") for h in (6, 2))
        cu = torch.empty(3, dtype=torch.int32, device="cuda")
        out, lse = torch.ops.atflash.flash_attn_packed(q[:, ::1], k, k, cu, 10, [9] * 8, 0.1, None, 0)
        assert out.shape == q.shape and out.dtype == BF and lse.shape == (6, 10) and lse.dtype == torch.float32


@pytest.mark.gpu
def test_registered_and_compiled(dev):
    from atflash import ops
    g = torch.Generator(device=dev).manual_seed(1)
    q, k, v = (torch.randn((300, h, 128), generator=g, device=dev).to(BF) for h in (6, 2, 2))
    cu = torch.tensor([0, 40, 300], dtype=torch.int32, device=dev)
    args = (q, k, v, cu, 260, None, 128 ** -0.5, None, 0)
    want = ops.flash_attn_packed(*args)
    got = torch.ops.atflash.flash_attn_packed(*args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    torch.library.opcheck(torch.ops.atflash.flash_attn_packed, args, test_utils=("test_schema", "test_faketensor"))

    @torch.compile(backend="aot_eager", fullgraph=True)
    def twice(q, k, v, cu):
        out, lse = torch.ops.atflash.flash_attn_packed(q, k, v, cu, 260, None, 128 ** -0.5, None, 0)
        return out * 2, lse
    out, lse = twice(q, k, v, cu)
    assert torch.equal(out, want[0] * 2) and torch.equal(lse, want[1])
