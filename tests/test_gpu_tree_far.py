"""Attention of drafted tokens at logits so large that fp32 holds them, times
the scale, to whole numbers or less (``dropkv_tree_attention``).

The products q . k are small whole numbers here, exact in fp32, and different
ones are at least one scale apart: the weights of a row are equal for the keys
of its largest product and 0 for the others (e^-scale), so the answer is the
mean of these keys' values.  Their sum is exact in fp32 (values of two bits,
fewer than 2^20 keys) but for the weight that they share: held in two parts, it
is off by 2^-16 of itself against the one that is summed.  Parts' weights are
equal, too, since their maxima are.  The quotient and the store round once each."""

import pytest
import torch

pytestmark = pytest.mark.gpu

# Rows of a KV head, by kernel and by the number of parts.
SHAPES = [(1, 2, 1, 900), (1, 4, 3, 40), (1, 8, 5, 2000), (1, 8, 12, 700), (1, 16, 20, 1500), (200, 8, 20, 300)]


def reference(s, v):
    """Mean of the values of each row's largest products: s [H, T, n], v [H, n, D]."""
    best = (s == s.amax(-1, keepdim=True)).double()
    return best @ v.double() / best.sum(-1, keepdim=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,T,n", SHAPES)
@pytest.mark.parametrize("scale", [3e4, 1e6, 3.7e7, 1e9, 1e30])
@pytest.mark.parametrize("shift", [-900, 0, 900])
def test_large_products(gpu, dtype, D, B, H, T, n, scale, shift):
    """Products between -8 and 8 from a whole number on, which falls from key to key
    or rises (the reference moves, or stays)."""
    from dropkv_amd import ops
    g = torch.Generator().manual_seed(n + T)
    q, k = torch.zeros(1, H, T, D), torch.zeros(1, 1, n + T, D)
    q[..., 0], q[..., 1] = 1.0, torch.randint(-2, 3, (1, H, T), generator=g).float()
    q[..., 2] = 30.0
    k[..., 0] = torch.randint(-4, 5, (1, 1, n + T), generator=g).float()
    k[..., 1] = torch.randint(-2, 3, (1, 1, n + T), generator=g).float()
    k[..., 2] = shift / 30
    v = torch.randint(-2, 2, (1, 1, n + T, D), generator=g).float()
    mask = torch.ones(T, T, dtype=torch.bool).tril()
    s = (q[0].double() @ k[0, 0].double().t()).masked_fill(
        ~torch.cat([torch.ones(T, n, dtype=torch.bool), mask], -1), -torch.inf)
    want = reference(s, v[0].expand(H, -1, -1)).transpose(0, 1)[None]
    many = lambda x: x.to(dtype).to(gpu).repeat(B, 1, 1, 1)
    got = ops.tree_attention(many(q), many(k[:, :, n:]), many(v[:, :, n:]), many(k[:, :, :n]), many(v[:, :, :n]),
                             torch.tensor([n], dtype=torch.int32, device=gpu), scale)
    assert (got == got[:1]).all()
    got = got[:1].cpu().double()
    half = torch.finfo(dtype).eps / 2
    # (Values of at most 2: the weight, and fp32's roundings of the quotient and the join.)
    assert ((got - want).abs() <= want.abs() * half + 2.0 ** -15 + 2.0 ** -21).all(), float((got - want).abs().max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,T", [(2, 3), (8, 20)])
def test_rows_without_keys_beside_large_products(gpu, dtype, H, T):
    """A row that sees nothing and one whose only logit is -inf: zeros; the rows
    beside them as ever."""
    from dropkv_amd import ops
    D, n = 64, 0
    q = torch.zeros(1, H, T, D, dtype=dtype)
    q[..., 0] = 100.0
    k = torch.zeros(1, 1, T, D, dtype=dtype)
    k[..., 0] = 90.0
    k[:, :, 1, 1] = -torch.inf
    q[..., 1] = 1.0
    v = torch.arange(T, dtype=torch.float32)[:, None].expand(T, D)[None, None].to(dtype)
    mask = torch.eye(T, dtype=torch.bool)
    mask[0] = False
    mask[2:, 0] = True
    cache = torch.zeros(1, 1, 8, D, dtype=dtype, device=gpu)
    for scale in (0.1, 1e6, 1e30):
        got = ops.tree_attention(q.to(gpu), k.to(gpu), v.to(gpu), cache, cache,
                                 torch.tensor([n], dtype=torch.int32, device=gpu), scale, mask=mask.to(gpu)).cpu()
        assert (got[:, :2] == 0).all(), scale
        for t in range(2, T):     # two equal products: the mean of their values
            assert (got[:, t] == torch.tensor(t / 2).to(dtype)).all(), (scale, t)
