"""Keys in 16 bits whose weights are small, and whose values are all that a row's output is
made of: the key of the largest weight has none.  The weights hold 16 bits there too."""

import pytest
import torch

import quant_ref as R
from test_gpu_quant import BF, FP, I8, counts, generator

pytestmark = pytest.mark.gpu


# (Rows of a workgroup: 16, 32, 64, 64, 128, 256.)
@pytest.mark.parametrize("B,T", [(1, 2), (1, 8), (1, 16), (16, 60), (16, 150), (64, 150)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n", [0, 138])
def test_small_weights(gpu, n, dtype, D, B, T):
    """Logits of 30 for the first 16-bit key, 16 to 18 for the others, 0 for those in blocks;
    the bound is ``R.tolerance``."""
    from dropkv_amd import ops
    Hq, Hkv, N = 8, 2, max(n, 1)
    g = generator(gpu, T + D + n)
    a = torch.rand(B, Hkv, N + T, generator=g, device=gpu) * 2 + 16
    v = torch.randn(B, Hkv, N + T, D, generator=g, device=gpu) * 1000
    first = 128 if n else N  # (rows of n = 0 are not stored: the new ones begin at N)
    a[:, :, :first] = 0
    a[:, :, first], v[:, :, first] = 30, 0
    k = torch.zeros(B, Hkv, N + T, D, device=gpu)
    k[..., 0] = a
    k, v = k.to(dtype), v.to(dtype)
    q = torch.zeros(B, Hq, T, D, dtype=dtype, device=gpu)
    q[..., 0] = 1
    mask = torch.ones(T, T, dtype=torch.bool, device=gpu)
    cache = ops.quant_cache(B, Hkv, 320, D, dtype=dtype, store=I8, device=gpu)
    ops.quant_append(cache, k[:, :, :n], v[:, :, :n], counts(gpu, 0))
    kn, vn = k[:, :, N:], v[:, :, N:]
    got = ops.quant_attention(q, kn, vn, cache, counts(gpu, n), 1.0, mask=mask)
    ref, mean, size = R.attend(q, k, v, kn, vn, [n] * B, 1.0, mask, I8)
    # (2^-25: half a step of fp16 below its normal numbers.)
    tol = R.tolerance(ref, mean, size, dtype, D, once=4 * T > 64 and dtype is BF) + 2.0 ** -25
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())
