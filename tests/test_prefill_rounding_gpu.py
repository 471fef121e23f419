"""With RoPE at load, a prompt alone (the 128-row kernel) and among others (the 256-row kernel) gets the same bits: both
round a rotated query element alike."""
import pytest
import torch

from helpers import D, gpu_qkv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,seed", [(700, 1), (700, 2), (513, 3), (1000, 4)])
def test_a_prompt_alone_and_among_others(dev, n, seed):
    from atflash import interface
    hq, hkv, many = 28, 4, 12
    inv = 1e7 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    cs = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous().to(dev)
    q, k, v = gpu_qkv(many, n, hq, hkv, dev, seed)
    out, lse = interface._flash_attn_fwd(q, k, v, rope=cs)
    for b in range(many):
        o, l1 = interface._flash_attn_fwd(q[b:b + 1], k[b:b + 1], v[b:b + 1], rope=cs)
        assert torch.equal(o[0], out[b]) and torch.equal(l1[0], lse[b])
