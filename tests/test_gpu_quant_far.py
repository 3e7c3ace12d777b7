"""Attention over a cache in 8 bits where logits are so large that fp32 holds no fraction of
them: the keys that a query singles out, and no others, make its output."""

import math

import pytest
import torch

import quant_ref as R
from test_gpu_quant import BF, FP, F8, I8, counts, generator

pytestmark = pytest.mark.gpu

N = 64 * 5 + 20


def singled_out(gpu, B, T, D, dtype, store, where, power, n):
    """(inputs, expected, mean of |v|).  Query class c has its own D / 4 dimensions, and two
    keys (one where there is room for one) hold the same there, so that their logits are
    equal, of about 2^power in powers of two.  The other keys' are at most half of it, which
    is far beyond what fp32 rounds."""
    Hq, Hkv, w = 8, 2, D // 4
    g = generator(gpu, T + D)
    scale = D ** -0.5
    amp = (torch.arange(4, device=gpu) * -0.06 + 1) * math.sqrt(2.0 ** power / (scale * math.log2(math.e) * w))
    amp = amp.to(dtype).float()
    classes = 4 if where != "new" or T >= 8 else 1
    pattern = torch.zeros(4, D, device=gpu)
    for c in range(4):
        pattern[c, c * w:(c + 1) * w] = amp[c]
    of = (torch.arange(B, device=gpu)[:, None, None] + torch.arange(Hq, device=gpu)[:, None] + torch.arange(T, device=gpu)) % classes
    q = pattern[of].to(dtype)                                                       # [B, Hq, T, D]
    k, kn = ((torch.rand(B, Hkv, r, D, generator=g, device=gpu) - 0.5) * amp[0] for r in (max(n, 1), T))
    v, vn = (torch.randn(B, Hkv, r, D, generator=g, device=gpu).to(dtype) for r in (max(n, 1), T))
    held = {"block": R.held(v[:, :, :n], store), "tail": v.double(), "new": vn.double()}[where]
    first = {"block": (64 + 9, 192 + 50), "tail": (n // 64 * 64 + 2, n // 64 * 64 + 11), "new": (0, 4)}[where]
    if classes == 1:
        first = first[:1]
    ref = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=gpu)
    mean = torch.zeros_like(ref)
    at = of.transpose(1, 2)[..., None]                                              # [B, T, Hq, 1]
    for c in range(classes):
        for f in first:
            (kn if where == "new" else k)[:, :, f + c] = pattern[c]
            row = held[:, :, f + c].repeat_interleave(Hq // Hkv, 1)[:, None]        # [B, 1, Hq, D]
            ref += torch.where(at == c, row, 0.0) / len(first)
            mean += torch.where(at == c, row.abs(), 0.0) / len(first)
    mask = torch.ones(T, T, dtype=torch.bool, device=gpu)
    return (q, k.to(dtype), v, kn.to(dtype), vn, mask, scale), ref, mean


# (Rows of a workgroup: 16, 32, 64, 64, 128, 256.)
@pytest.mark.parametrize("B,T", [(1, 1), (1, 8), (1, 16), (16, 60), (16, 150), (64, 150)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("where", ["block", "tail", "new"])
def test_far_logits(gpu, where, dtype, D, B, T):
    """Equal logits have equal weights, so what is left is the rounding of the weights and of
    the output (``R.tolerance`` without the logits' share)."""
    from dropkv_amd import ops
    for store in (I8, F8):
        for power in (22.7, 25.5, 28.0, 30.0, 32.0):
            for n in ((N, 0) if where == "new" else (N,)):
                (q, k, v, kn, vn, mask, scale), ref, mean = singled_out(gpu, B, T, D, dtype, store, where, power, n)
                cache = ops.quant_cache(B, 2, N, D, dtype=dtype, store=store, device=gpu)
                ops.quant_append(cache, k, v, counts(gpu, 0), counts=counts(gpu, *[n] * B))
                got = ops.quant_attention(q, kn, vn, cache, counts(gpu, n), scale, mask=mask)
                tol = R.tolerance(ref, mean, 0.0, dtype, D, once=4 * T > 64 and dtype is BF)
                err = (got.double() - ref).abs()
                assert torch.isfinite(got).all() and (err <= tol).all(), (store, power, n, float((err / tol).max()))
