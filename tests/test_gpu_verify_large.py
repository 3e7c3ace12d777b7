"""The verification step's operators on tensors whose offsets pass 32 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [2, 40])
def test_tree_attention_of_a_long_cache(gpu, T):
    """2^23 rows of 128 to a head, the most that fit: 2 GiB a head, 8 GiB in
    all.  All rows are zeros but a few that the queries single out (their logits
    are 60 above the others: the others' share is 2^23 e^-60)."""
    from dropkv_amd import ops
    B, Hkv, g, D, C = 1, 2, 2, 128, 1 << 23
    kc, vc = (torch.zeros(B, Hkv, C, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    rows = [0, C // 2 + 3, C - 1]
    for i, r in enumerate(rows):
        kc[:, :, r, i] = 60.0
        vc[:, 0, r], vc[:, 1, r] = float(i + 1), float(10 * i + 5)
    q = torch.zeros(B, Hkv * g, T, D, dtype=torch.bfloat16, device=gpu)
    want = torch.zeros(B, T, Hkv * g, device=gpu)
    for t in range(T):
        q[:, :, t, t % 3] = 1.0
        want[:, t, :g], want[:, t, g:] = float(t % 3 + 1), float(10 * (t % 3) + 5)
    kn = torch.zeros(B, Hkv, T, D, dtype=torch.bfloat16, device=gpu)
    n = torch.tensor([C], dtype=torch.int32, device=gpu)
    out = ops.tree_attention(q, kn, kn, kc, vc, n, 1.0)
    assert torch.equal(out.float(), want[..., None].expand_as(out))
    n.fill_(C - 1)    # without the last row, its queries see zeros alone
    out = ops.tree_attention(q, kn, kn, kc, vc, n, 1.0)
    assert (out[:, 2::3].abs() < 1e-3).all() and torch.equal(out[:, 0], want[:, 0, :, None].expand(B, Hkv * g, D))


def test_commit_into_long_caches(gpu):
    from dropkv_amd import ops
    N, B, H, T, D, C = 3, 1, 1, 4, 128, 1 << 23
    kc = torch.zeros(N, B, H, C, D, dtype=torch.bfloat16, device=gpu)
    kn, vn = (torch.randn(N, B, H, T, D, device=gpu).bfloat16() for _ in range(2))
    tok = torch.arange(T, device=gpu)[None]
    par = torch.arange(-1, T - 1, dtype=torch.int32, device=gpu)
    n = torch.tensor([[C - 4], [5], [C - 9]], dtype=torch.int32, device=gpu)
    vc = torch.zeros_like(kc)
    path, acc = ops.tree_commit(tok, par, tok + 1, kn, vn, kc, vc, n)
    assert acc.tolist() == [T]
    for l in range(N):
        r = int(n[l, 0])
        assert torch.equal(kc[l, 0, 0, r:r + T], kn[l, 0, 0]) and torch.equal(vc[l, 0, 0, r:r + T], vn[l, 0, 0])
        kc[l, 0, 0, r:r + T] = 0
    assert not kc.any()


def test_logprobs_of_many_rows(gpu):
    """15000 x 151936 logits, 4.6 GB: the last rows as on their own."""
    from dropkv_amd import ops
    N, V = 15000, 151936
    x = torch.zeros(N, V, dtype=torch.bfloat16, device=gpu)
    x[-40:] = torch.randn(40, V, device=gpu).bfloat16()
    t = torch.arange(N, device=gpu)
    for top in (1, 6):
        got = ops.token_logprobs(x, t, top=top)
        own = ops.token_logprobs(x[-40:].clone(), t[-40:], top=top)
        assert torch.equal(got.top_ids[-40:], own.top_ids)
        # (another cut into segments: sums in another order)
        for a, b in zip(got[:3], own[:3]):
            torch.testing.assert_close(a[-40:], b, rtol=1e-5, atol=1e-5)
        assert torch.equal(got.top_ids[:-40], torch.arange(top, device=gpu).expand(N - 40, top))


def test_norm_rope_of_far_rows(gpu):
    """Rows of one buffer 2^32 elements apart."""
    from dropkv_amd import ops
    D = 128
    buf = torch.zeros((1 << 32) + (1 << 14), dtype=torch.bfloat16, device=gpu)
    far = buf.as_strided((2, 1, 3, D), (1 << 32, D, D, 1))
    far.copy_(torch.randn(2, 1, 3, D, device=gpu))
    near = far.contiguous()
    cos, sin = torch.randn(3, D, device=gpu), torch.randn(3, D, device=gpu)
    a, b = ops.norm_rope(far, far, cos, sin)
    c, d = ops.norm_rope(near, near, cos, sin)
    assert torch.equal(a, c) and torch.equal(b, d)
    ops.norm_rope(near, near, cos, sin, q_out=far, k_out=d)
    assert torch.equal(far, c)
