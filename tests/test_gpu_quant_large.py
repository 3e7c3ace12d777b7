"""The cache in 8 bits and the sampled verification on tensors whose offsets pass 32
bits, large batches and long lists of parts."""

import pytest
import torch

import quant_ref as R
from test_gpu_quant import attention_case, check_attention, counts, generator, rows
from test_gpu_verify_drafts import case as drafts_case, check as check_drafts, reference as drafts_reference

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("store", R.STORES)
def test_attention_over_a_long_cache(gpu, store):
    """2^23 rows of 128 to a head, the most that fit.  All rows are zeros but a few that
    the queries single out (their logits are 60 above the others: the others' share is
    2^23 e^-60), and those are whole multiples of their block's step."""
    from dropkv_amd import ops
    Hkv, g, D, C = 2, 2, 128, 1 << 23
    kc, vc = (torch.zeros(1, Hkv, C, D, dtype=BF, device=gpu) for _ in range(2))
    for i, r in enumerate([0, C // 2 + 3, C - 1]):
        kc[:, :, r, i] = 60.0
        vc[:, 0, r], vc[:, 1, r] = float(i + 1), float(10 * i + 5)
    cache = ops.quant_cache(1, Hkv, C, D, store=store, device=gpu)
    ops.quant_append(cache, kc[:, :, :C - 1], vc[:, :, :C - 1], counts(gpu, 0))
    for n in (C - 1, C):
        if n == C:
            ops.quant_append(cache, kc[:, :, n - 1:], vc[:, :, n - 1:], counts(gpu, n - 1))
        for T in (1, 7, 30, 200):  # (a workgroup of 16, 16, 64 and 256 rows)
            q = torch.zeros(1, Hkv * g, T, D, dtype=BF, device=gpu)
            want = torch.zeros(1, T, Hkv * g, device=gpu)
            for t in range(T):
                q[:, :, t, t % 3] = 1.0
                want[:, t, :g], want[:, t, g:] = float(t % 3 + 1), float(10 * (t % 3) + 5)
            kn = torch.zeros(1, Hkv, T, D, dtype=BF, device=gpu)
            out = ops.quant_attention(q, kn, kn, cache, counts(gpu, n), 1.0).float()
            if n < C:  # the last row is not there: its queries see zeros alone
                assert (out[:, 2::3].abs() < 1e-3).all()
                want[:, 2::3], out[:, 2::3] = 0, 0
            assert torch.equal(out, want[..., None].expand_as(out)), (n, T)
    k, v = ops.quant_read(cache, counts(gpu, C), 65, C - 65)
    assert torch.equal(k, kc[:, :, C - 65:]) and torch.equal(v, vc[:, :, C - 65:])


def test_layers_of_long_caches(gpu):
    """Rows behind the last ones of layers whose buffers begin past 2^31 bytes."""
    from dropkv_amd import ops
    N, D, C, L = 3, 128, 1 << 23, 100
    g = generator(gpu, 1)
    k, v = rows(g, N, 1, 1, L, D), rows(g, N, 1, 1, L, D)
    cache = ops.quant_cache(1, 1, C, D, layers=N, device=gpu)
    n = [C - 100, 5, C - 9]
    ops.quant_append(cache, k, v, counts(gpu, *n)[:, None])
    after = counts(gpu, C, 105, C)[:, None]
    for first, l in ((C - 128, 0), (0, 1), (C - 128, 2)):
        got = ops.quant_read(cache, after, 128, first)
        for x, y in zip((k, v), got):
            z = torch.zeros(1, 1, 128 if l != 1 else 105, D, dtype=BF, device=gpu)
            at, m = (n[l] - first, min(L, C - n[l]))
            z[:, :, at:at + m] = x[l, :, :, :m]
            want = R.held(z, torch.int8)
            assert not y[l, :, :, z.shape[2]:].any()
            err = (y[l, :, :, :z.shape[2]].double() - want).abs()
            assert (err <= (R.HALF[BF] + 2.0 ** -22) * want.abs() + 2.0 ** -25).all(), l


@pytest.mark.parametrize("T", [1, 20, 70])
def test_operands_far_apart(gpu, T):
    """Queries and new rows of one buffer 2^32 elements apart."""
    from dropkv_amd import ops
    n = [90, 130]
    q, k, v, kn, vn, cache, mask, scale = attention_case(gpu, 2, 1, 64, T, n, BF, torch.int8)
    want = ops.quant_attention(q, kn, vn, cache, counts(gpu, *n), scale, mask=mask)
    buf = torch.zeros((1 << 32) + (1 << 18), dtype=BF, device=gpu)
    far = []
    at = 0
    for x in (q, kn, vn):
        y = buf[at:].as_strided(x.shape, (1 << 32, *x.stride()[1:]))
        y.copy_(x)
        far.append(y)
        at += x[0].numel()
    out = buf[at:].as_strided((2, T, 2, 64), (1 << 32, 128, 64, 1))
    ops.quant_attention(*far, cache, counts(gpu, *n), scale, out=out, mask=mask)
    assert torch.equal(out, want)
    ops.quant_append(cache, far[1], far[2], counts(gpu, *n))
    other = ops.quant_cache(2, 1, cache.capacity, 64, device=gpu)
    ops.quant_append(other, torch.cat([k, k[:, :, :0]], 2), v, counts(gpu, 0), counts=counts(gpu, *n))
    ops.quant_append(other, kn, vn, counts(gpu, *n))
    rows_after = counts(gpu, *(x + T for x in n))
    for x, y in zip(ops.quant_read(cache, rows_after, 64), ops.quant_read(other, rows_after, 64)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T", [1, 5, 12, 40])
def test_many_sequences(gpu, T, dtype):
    """More sequences than the parts are dealt out for by length."""
    n = [(37 * i * i) % 400 for i in range(70)]
    case = attention_case(gpu, 4, 2, 64, T, n, dtype, torch.int8, mask=None)
    check_attention(gpu, *case, n)


@pytest.mark.parametrize("T", [1, 2, 8, 20, 60])
def test_one_long_sequence_among_short_ones(gpu, T):
    """Most of the parts go to one sequence."""
    n = [0, 1, 20011, 64, 0, 5, 63, 128]
    case = attention_case(gpu, 8, 2, 128, T, n, BF, torch.float8_e4m3fn, mask=None)
    check_attention(gpu, *case, n)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("store", R.STORES)
def test_large_logits_of_many_rows(gpu, dtype, store):
    """Logits up to 10^9 (bf16), where a row's largest changes from block to block."""
    from dropkv_amd import ops
    T, n = 150, [1500, 700]
    q, k, v, kn, vn, cache, mask, scale = attention_case(gpu, 8, 2, 64, T, n, dtype, store)
    q, k, kn = q * 100, k * 100, kn * 100
    if dtype is BF:
        q, k, kn = q * 64, k * 64, kn * 64
    ops.quant_append(cache, k, v, counts(gpu, 0), counts=counts(gpu, *n))
    got = ops.quant_attention(q, kn, vn, cache, counts(gpu, *n), scale, mask=mask)
    assert torch.isfinite(got).all()
    assert got.abs().max() <= max(v.abs().max(), vn.abs().max()) * (1 + 2.0 ** -7)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("B,T,V", [(1500, 3, 120), (2, 3, 300001), (1, 20, 600000)])
def test_drafts_of_large_batches_and_vocabularies(gpu, B, T, V, draft):
    from dropkv_amd import ops
    x, tok, u, y = drafts_case(gpu, B, T, V, BF, draft)
    check_drafts(ops.verify_drafts(x, tok, u, y), drafts_reference(x, tok, u, y, 1.0), x, 1.0)


@pytest.mark.parametrize("B,T", [(4000, 8), (1000, 29)])
def test_drafts_of_many_rows(gpu, B, T):
    """More than 2^32 logits: the last sequences as on their own."""
    from dropkv_amd import ops
    V = 151936
    x = torch.zeros(B, T, V, dtype=BF, device=gpu)
    own, tok_own, u_own, _ = drafts_case(gpu, 4, T, V, BF, False)
    u_own[:, 1:] *= 1e-4
    x[-4:] = own
    tok = torch.randint(0, V, (B, T), device=gpu)
    u = torch.rand(B, T, device=gpu)
    tok[-4:], u[-4:] = tok_own, u_own
    got, want = ops.verify_drafts(x, tok, u), ops.verify_drafts(own, tok_own, u_own)
    assert torch.equal(got.choice[-4:], want.choice) and torch.equal(got.accepted[-4:], want.accepted)
    torch.testing.assert_close(got.logprobs[-4:], want.logprobs, rtol=2.0 ** -22, atol=2.0 ** -22)
    # Equal logits: a token stands with a probability of 1 / V, and the next one is
    # the u_0 V-th, past the one that failed.
    assert got.accepted[:-4].float().mean() < 1.01
    first = (got.accepted[:-4] == 1).nonzero()[:, 0]
    at = (u[first, 0].double() * (V - 1)).floor().long()
    at += at >= tok[first, 1]
    assert ((got.choice[first, 0] - at).abs() <= 1).all()
