"""Log probabilities beside NaN of every kind: quiet and signalling ones of both signs rank as -inf does and take no other logit with
them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
NANS = {"bf16": (torch.bfloat16, torch.int16, (0x7fa0, -0x60, 0x7f81, 0x7fc0, -1)),
        "fp16": (torch.float16, torch.int16, (0x7d00, -0x300, 0x7c01, 0x7e00, -1)),
        "fp32": (torch.float32, torch.int32, (0x7fa00000, -0x600000, 0x7f800001, 0x7fc00000, -1))}


@pytest.mark.parametrize("R,V", [(4, 90), (4, 9000), (600, 9000), (3, 40001)])
@pytest.mark.parametrize("kind", list(NANS))
def test_no_nan_hides_a_logit(dev, kind, R, V):
    """A row for every kind of NaN and every place of the largest logits within 16 bytes beside it."""
    from atflash import ops
    dt, whole, bits = NANS[kind]
    E = 4 if kind == "fp32" else 8
    g = torch.Generator(device=dev).manual_seed(V)
    x = torch.randn((R, V), generator=g, device=dev).to(dt)
    cpu = x.cpu()
    for r in range(R):
        best, at = r % E, (r // E) % E
        base = (V // 2 + 7 * r % (V // 4)) // E * E
        cpu[r, base + best] = 50.0
        cpu[r, base + (best + 1) % E] = 40.0
        cpu[r, r % E] = 30.0
        cpu.view(whole)[r, base + at] = bits[r % len(bits)]        # (may take a place of theirs)
        cpu.view(whole)[r, (r + 1) % E] = bits[(r + 2) % len(bits)]
        cpu.view(whole)[r, V - 1] = bits[(r + 1) % len(bits)]
    x.view(whole).copy_(cpu.view(whole))
    assert torch.equal(x.view(whole).cpu(), cpu.view(whole))
    ranked = torch.where(cpu.isnan(), -float("inf"), cpu.double())
    for top in (1, 5, 20):
        logp, ent, vals, ids = ops.token_logprobs(x, torch.zeros(R, dtype=torch.int64, device=dev), top)
        want = torch.sort(ranked, dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(ids.cpu(), want), (ids.cpu() != want).any(1).nonzero()[:, 0].tolist()[:9]
        assert torch.isnan(logp).all() and torch.isnan(ent).all() and torch.isnan(vals).all()


@pytest.mark.parametrize("kind", list(NANS))
def test_nan_beside_masks(dev, kind):
    """Rows of -inf, the type's lowest value, NaN and a few logits."""
    from atflash import ops
    dt, whole, bits = NANS[kind]
    V = 5000
    cpu = torch.full((6, V), float("-inf"), dtype=dt)
    cpu[3:] = torch.finfo(dt).min
    for r in range(6):
        cpu[r, 100:4900:97] = torch.arange(len(range(100, 4900, 97))).to(dt)
        cpu.view(whole)[r, 101:4900:97] = bits[r % len(bits)]
        cpu.view(whole)[r, 99:4900:97 * 2] = bits[(r + 1) % len(bits)]
    ranked = torch.where(cpu.isnan(), -float("inf"), cpu.double())
    x = torch.empty((6, V), dtype=dt, device=dev)
    x.view(whole).copy_(cpu.view(whole))
    for top in (1, 20, 64):
        ids = ops.token_logprobs(x, None, top)[3]
        assert torch.equal(ids.cpu(), torch.sort(ranked, dim=-1, descending=True, stable=True).indices[:, :top])
