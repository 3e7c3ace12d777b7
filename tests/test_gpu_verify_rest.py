"""What is left of p where a draft failed: tokens of equal probability in both models have
nothing left, to the last bit, and the token that is drawn is one that has."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T", [2, 18])  # (in one kernel, and in three)
def test_equal_probabilities_leave_nothing(gpu, T, dtype):
    """The draft model has two tokens' logits exchanged, and everything else alike: sums of the
    same weights, the two added to one another first.  So p = q elsewhere, and only the
    token that the draft has too little of is left, also for u_0 = 0, which takes the
    first token with any weight."""
    from dropkv_amd import ops
    B, V, per = 64, 40, 16 // torch.empty(0, dtype=dtype).element_size()
    g = torch.Generator(device=gpu).manual_seed(T)
    x = torch.full((B, T, V), float("-inf"), device=gpu)
    x[..., :3 * per] = torch.randn(B, T, 3 * per, generator=g, device=gpu) * 2
    low, high = 3 * per, 3 * per + 1  # (of one thread's loads, which holds no others)
    x[..., low], x[..., high] = 1.0, 2.5
    x = x.to(dtype)
    y = x[:, :-1].clone()
    y[..., low], y[..., high] = 2.5, 1.0
    tokens = torch.full((B, T), low, dtype=torch.int64, device=gpu)
    u = torch.full((B, T), 0.9, device=gpu)
    u[:, 0] = 0.0
    for temperature in (0.6, 0.7, 1.0, 1.3):
        got = ops.verify_drafts(x, tokens, u, y, temperature)
        # (Node 1 stands while 0.9 q < p, and q is e^(1.5 / temperature) times p.)
        assert (got.accepted == 1).all()
        assert (got.choice[:, 0] == high).all(), (temperature, (got.choice[:, 0] != high).sum())
        assert (got.choice[:, 1:] == -1).all()
        want = torch.log_softmax(x[:, 0].double() / temperature, dim=-1)[:, high]
        torch.testing.assert_close(got.logprobs[:, 0].double(), want, rtol=2.0 ** -22, atol=2.0 ** -22)
