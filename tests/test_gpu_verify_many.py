"""The verification step's operators on more rows than the work-items of one
grid (2^32) hold waves or workgroups for."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L,D,R", [
    ((1 << 25) + 70, 6, 4),       # any layout: a wave a head's row, 2^26 + 140 of them
    ((1 << 26) + 70, 16, 16),     # vectors: a wave a token
])
def test_norm_rope(gpu, L, D, R):
    """Rows all along the call as on their own."""
    from dropkv_amd import ops
    g = torch.Generator(device=gpu).manual_seed(D)
    q, k = (torch.randn(1, 1, L, D, generator=g, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    cos, sin = (torch.randn(1, R, generator=g, device=gpu).expand(L, R) for _ in range(2))
    w = torch.randn(D, generator=g, device=gpu)
    qo, ko = ops.norm_rope(q, k, cos, sin, q_weight=w)
    for lo in (0, L // 2 - 40, (1 << 25) - 40, L - 80):
        part = slice(lo, lo + 80)
        qp, kp = ops.norm_rope(q[:, :, part].clone(), k[:, :, part].clone(), cos[:80], sin[:80], q_weight=w)
        assert torch.equal(qo[:, :, part], qp) and torch.equal(ko[:, :, part], kp), lo
    # (No row is left out: a turned row of random numbers is no row of zeros.)
    for t in (qo, ko):
        for rows in t[0, 0].split(1 << 24):
            assert (rows != 0).any(-1).all()


@pytest.mark.parametrize("top", [0, 1, 2])
def test_token_logprobs(gpu, top):
    """A workgroup a row, 2^24 + 5 rows of three logits: rows all along the call
    as on their own."""
    from dropkv_amd import ops
    N, V = (1 << 24) + 5, 3
    g = torch.Generator(device=gpu).manual_seed(top)
    x = torch.randn(N, V, generator=g, device=gpu)
    tokens = torch.randint(0, V, (N,), generator=g, device=gpu)
    got = ops.token_logprobs(x, tokens, top=top)
    lp = torch.log_softmax(x.double(), -1)
    want = [lp.gather(1, tokens[:, None])[:, 0], -(lp.exp() * lp).sum(-1)]
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    # (Values below 20 in size: a few roundings of fp32 each.)
    for a, b in zip(got[:3], (*want, lp.gather(1, ids))):
        assert ((a.double() - b).abs() <= 2.0 ** -24 * 64).all()
    assert torch.equal(got.top_ids, ids)
