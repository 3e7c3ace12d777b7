"""A cache in 8 bits: rows quantised as they are written, read back, and attention
over them, against their definitions in 64 bits."""

import pytest
import torch

import quant_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
I8, F8 = R.STORES


def rows(gen, *shape, dtype=BF, scale=1.0, channels=True):
    x = torch.randn(*shape, generator=gen, device=gen.device) * scale
    if channels:
        x = x * torch.exp(torch.randn(*shape[:-2], 1, shape[-1], generator=gen, device=gen.device))
    return x.to(dtype)


def generator(gpu, seed):
    return torch.Generator(device=gpu).manual_seed(seed)


def counts(gpu, *n):
    return torch.tensor(n, dtype=torch.int32, device=gpu)


def stored(cache):
    """The stored values [.., H, capacity, D] (float64) of K and V, as rows."""
    k = cache.k.double()
    v = cache.v.double().transpose(-1, -2).flatten(-3, -2)
    return k, v


def check_cache(cache, k, v, n):
    """Everything that a cache holds after rows k, v [B, H, >= n[b], D]."""
    store, dtype = cache.k.dtype, cache.k_tail.dtype
    for x, q, s, tail in ((k, stored(cache)[0], cache.k_scale, cache.k_tail), (v, stored(cache)[1], cache.v_scale, cache.v_tail)):
        for b, nb in enumerate(n):
            full = nb // 64
            if full:
                want, scale = R.quantise(x[b, :, :full * 64].unflatten(1, (full, 64)), store)
                assert torch.equal(q[b, :, :full * 64], want.flatten(1, 2)), b
                torch.testing.assert_close(s[b, :, :full].double(), scale, rtol=2.0 ** -24, atol=0, equal_nan=True)
            assert not s[b, :, full:].any() and not q[b, :, full * 64:].any()
            at = torch.arange(full * 64, nb, device=x.device)
            assert torch.equal(tail[b][:, at % 128].view(torch.int16), x[b][:, at].to(dtype).view(torch.int16)), b


@pytest.mark.parametrize("store", R.STORES)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [1, 63, 64, 65, 200, 1000])
def test_append_to_an_empty_cache(gpu, L, D, dtype, store):
    from dropkv_amd import ops
    g = generator(gpu, L + D)
    k, v = rows(g, 2, 3, L, D, dtype=dtype), rows(g, 2, 3, L, D, dtype=dtype, channels=False)
    cache = ops.quant_cache(2, 3, L, D, dtype=dtype, store=store, device=gpu)
    ops.quant_append(cache, k, v, counts(gpu, 0))
    check_cache(cache, k, v, [L, L])
    # Read back: the rows as they are held, rounded once.
    kk, vv = ops.quant_read(cache, counts(gpu, L), L)
    for x, y in ((k, kk), (v, vv)):
        want = R.held(x, store)
        assert ((y.double() - want).abs() <= (R.HALF[dtype] + 2.0 ** -22) * want.abs() + 2.0 ** -25).all()
        assert torch.equal(y[:, :, L // 64 * 64:], x[:, :, L // 64 * 64:])


@pytest.mark.parametrize("store", R.STORES)
@pytest.mark.parametrize("lengths", [[1] * 130, [63, 1, 64, 1, 62, 130], [200, 7, 1], [5, 256, 3]])
def test_pieces_of_any_length_give_the_same_cache(gpu, lengths, store):
    from dropkv_amd import ops
    g = generator(gpu, sum(lengths))
    n = sum(lengths)
    k, v = rows(g, 2, 2, n, 64), rows(g, 2, 2, n, 64)
    cache = ops.quant_cache(2, 2, n + 70, 64, store=store, device=gpu)
    at = 0
    for L in lengths:
        ops.quant_append(cache, k[:, :, at:at + L], v[:, :, at:at + L], counts(gpu, at))
        at += L
    check_cache(cache, k, v, [n, n])


@pytest.mark.parametrize("store", R.STORES)
def test_ties_and_signs(gpu, store):
    """Whole and half multiples of the step, of both signs, and -0."""
    from dropkv_amd import ops
    x = torch.zeros(1, 1, 64, 64)
    x[..., 0, 0] = 127.0 if store is I8 else 448.0
    x[..., 1, :] = torch.arange(64) / 2 - 16
    x[..., 2, :] = -torch.arange(64) / 2
    x[..., 3, :] = torch.arange(64) * 2.0 ** -10
    x[..., 4, :] = -0.0
    x[..., 5, :] = (torch.arange(64) + 16.5) * 2
    for f in (1.0, 2.0 ** -20, 2.0 ** 60, 2.0 ** 119, 2.0 ** -100):
        y = (x * f).to(BF).to(gpu)
        cache = ops.quant_cache(1, 1, 64, 64, store=store, device=gpu)
        ops.quant_append(cache, y, y, counts(gpu, 0))
        check_cache(cache, y, y, [64])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("store", R.STORES)
def test_every_value_against_every_size(gpu, store, dtype):
    """Blocks of many largest magnitudes, each with values spread over all signs and
    exponents of the type."""
    from dropkv_amd import ops
    g = generator(gpu, 5)
    n = 400
    bits = torch.randint(0, 1 << 16, (1, 1, n * 64, 64), generator=g, device=gpu, dtype=torch.int32).to(torch.int16)
    x = bits.view(dtype)
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    # (Magnitudes below a block's own.)
    top = torch.exp2(torch.rand(n, generator=g, device=gpu) * 24 - 12) * (1 + torch.rand(n, generator=g, device=gpu))
    top = top.repeat_interleave(64)[None, None, :, None]
    x = torch.where(x.abs() > top, (torch.frexp(x.float())[0] * top).to(dtype), x)
    cache = ops.quant_cache(1, 1, n * 64, 64, dtype=dtype, store=store, device=gpu)
    ops.quant_append(cache, x, x, counts(gpu, 0))
    check_cache(cache, x, x, [n * 64])


@pytest.mark.parametrize("store", R.STORES)
def test_blocks_without_a_scale(gpu, store):
    """All zeros, magnitudes below 2^-100, and values that are not finite: zeros and
    NaN, of their own block alone."""
    from dropkv_amd import ops
    g = generator(gpu, 9)
    x = rows(g, 1, 2, 64 * 6 + 3, 64)
    x[:, :, :64] = 0
    x[:, :, 64:128] *= 2.0 ** -110
    x[:, 0, 130, 5] = float("inf")
    x[:, 0, 200, 6] = float("nan")
    x[:, 1, 270, 7] = float("-inf")
    x[:, :, -1, 0] = float("nan")  # in the tail: kept
    n = x.shape[2]
    cache = ops.quant_cache(1, 2, n, 64, store=store, device=gpu)
    ops.quant_append(cache, x, x, counts(gpu, 0))
    check_cache(cache, x, x, [n])
    for y in ops.quant_read(cache, counts(gpu, n), n):
        want = R.held(x, store)
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        assert not y[:, :, :128].any()
        assert torch.equal(y[:, :, -3:].view(torch.int16), x[:, :, -3:].view(torch.int16))


@pytest.mark.parametrize("layers", [None, 3])
@pytest.mark.parametrize("L", [8, 64, 150])
def test_paths_counts_and_layers(gpu, L, layers):
    """Each sequence appends rows of its own path behind its own length, in every
    layer; what a count leaves out is not touched."""
    from dropkv_amd import ops
    g = generator(gpu, L)
    B, H, D, C = 4, 2, 128, 640
    n = [0, 61, 64, 130]
    take = [0, min(L, 5), L, min(L, 64)]
    lead = (B,) if layers is None else (layers, B)
    old_k, old_v = rows(g, *lead, H, 192, D, dtype=FP), rows(g, *lead, H, 192, D, dtype=FP)
    new_k, new_v = rows(g, *lead, H, L, D, dtype=FP), rows(g, *lead, H, L, D, dtype=FP)
    cache = ops.quant_cache(B, H, C, D, dtype=FP, store=I8, layers=layers, device=gpu)
    n_rows = counts(gpu, *n) if layers is None else counts(gpu, *n).repeat(layers, 1)
    ops.quant_append(cache, old_k, old_v, torch.zeros_like(n_rows), counts=counts(gpu, *n))
    path = torch.full((B, L), -7, dtype=torch.int32, device=gpu)
    for b, t in enumerate(take):
        path[b, :t] = torch.randperm(L, generator=g, device=gpu)[:t].sort().values
    ops.quant_append(cache, new_k, new_v, n_rows, path=path, counts=counts(gpu, *take))
    for i in range(layers or 1):
        one = cache if layers is None else cache.layer(i)
        ok, ov, nk, nv = (t if layers is None else t[i] for t in (old_k, old_v, new_k, new_v))
        total = [a + t for a, t in zip(n, take)]
        want = []
        for o, w in ((ok, nk), (ov, nv)):
            x = torch.zeros(B, H, max(total), D, dtype=FP, device=gpu)
            for b in range(B):
                x[b, :, :n[b]] = o[b, :, :n[b]]
                x[b, :, n[b]:total[b]] = w[b][:, path[b, :take[b]].long()]
            want.append(x)
        check_cache(one, *want, total)


@pytest.mark.parametrize("n,L", [(0, 40), (61, 5), (70, 64), (127, 1)])
def test_the_same_append_again(gpu, n, L):
    from dropkv_amd import ops
    g = generator(gpu, n)
    k, v = rows(g, 1, 2, n + L, 64), rows(g, 1, 2, n + L, 64)
    cache = ops.quant_cache(1, 2, 256, 64, device=gpu)
    if n:
        ops.quant_append(cache, k[:, :, :n], v[:, :, :n], counts(gpu, 0))
    for _ in range(3):
        ops.quant_append(cache, k[:, :, n:], v[:, :, n:], counts(gpu, n))
        check_cache(cache, k, v, [n + L])


def test_rows_past_the_capacity_are_dropped(gpu):
    from dropkv_amd import ops
    g = generator(gpu, 3)
    k, v = rows(g, 3, 2, 300, 64), rows(g, 3, 2, 300, 64)
    cache = ops.quant_cache(3, 2, 128, 64, device=gpu)
    guard = [t.clone() for t in cache]
    ops.quant_append(cache, k, v, counts(gpu, 128, 500, -1))
    for t, w in zip(cache, guard):
        assert torch.equal(t.view(torch.uint8), w.view(torch.uint8))
    ops.quant_append(cache, k, v, counts(gpu, 0, 0, 0))
    check_cache(cache, k, v, [128, 128, 128])
    cache = ops.quant_cache(3, 2, 128, 64, device=gpu)
    ops.quant_append(cache, k[:, :, :100], v[:, :, :100], counts(gpu, 0))
    ops.quant_append(cache, k[:, :, 100:], v[:, :, 100:], counts(gpu, 100))
    check_cache(cache, k, v, [128, 128, 128])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("store", R.STORES)
def test_read_ranges(gpu, store, dtype):
    """Any range of rows, zeros behind the last, from sequences of their own lengths."""
    from dropkv_amd import ops
    g = generator(gpu, 4)
    n = [0, 37, 128, 333]
    k, v = rows(g, 4, 2, 333, 128, dtype=dtype), rows(g, 4, 2, 333, 128, dtype=dtype)
    cache = ops.quant_cache(4, 2, 400, 128, dtype=dtype, store=store, device=gpu)
    ops.quant_append(cache, k, v, counts(gpu, 0), counts=counts(gpu, *n))
    for first, L in ((0, 448), (0, 1), (63, 2), (64, 64), (100, 150), (320, 13), (330, 118), (447, 1), (448, 0)):
        outs = ops.quant_read(cache, counts(gpu, *n), L, first)
        for x, y in zip((k, v), outs):
            assert y.shape == (4, 2, L, 128) and y.dtype is dtype
            for b in range(4):
                want = torch.zeros(2, 448, 128, dtype=torch.float64, device=gpu)
                want[:, :n[b]] = R.held(x[b, :, :n[b]], store)
                want = want[:, first:first + L]
                assert ((y[b].double() - want).abs() <= (R.HALF[dtype] + 2.0 ** -22) * want.abs() + 2.0 ** -25).all(), (first, b)


def test_strided_rows(gpu):
    """Projections [B, L, H, D] seen as [B, H, L, D], at odd offsets, and one row for
    all heads."""
    from dropkv_amd import ops
    g = generator(gpu, 6)
    L, H, D = 150, 3, 64
    wide = rows(g, 2, L, H * D + 1)
    k = wide[:, :, 1:].unflatten(-1, (H, D)).transpose(1, 2)
    v = rows(g, 2, 1, L, D).expand(2, H, L, D)
    cache = ops.quant_cache(2, H, L, D, device=gpu)
    ops.quant_append(cache, k, v, counts(gpu, 0))
    check_cache(cache, k, v, [L, L])
    cache = ops.quant_cache(2, H, D, 64, device=gpu)
    k = rows(g, 2, H, D, 64).transpose(2, 3)  # the last axis not contiguous
    ops.quant_append(cache, k, k, counts(gpu, 0))
    check_cache(cache, k, k, [64, 64])


# --- attention ------------------------------------------------------------------

def tree(gen, B, T):
    mask = torch.zeros(B, T, T, dtype=torch.bool, device=gen.device)
    mask[:, 0, 0] = True
    for i in range(1, T):
        p = torch.randint(0, i, (B,), generator=gen, device=gen.device)
        mask[:, i] = mask[torch.arange(B, device=gen.device), p]
        mask[:, i, i] = True
    return mask


def attention_case(gpu, Hq, Hkv, D, T, n, dtype, store, mask="tree", seed=0, C=None, scale=None):
    from dropkv_amd import ops
    g = generator(gpu, seed + T + D)
    B, N = len(n), max(max(n), 1)
    q = rows(g, B, Hq, T, D, dtype=dtype, channels=False)
    k, v = rows(g, B, Hkv, N, D, dtype=dtype), rows(g, B, Hkv, N, D, dtype=dtype, channels=False)
    kn, vn = rows(g, B, Hkv, T, D, dtype=dtype), rows(g, B, Hkv, T, D, dtype=dtype, channels=False)
    cache = ops.quant_cache(B, Hkv, C or N + T, D, dtype=dtype, store=store, device=gpu)
    for t in cache:  # what is not stored must not count
        t.view(torch.uint8).fill_(0xff)
    ops.quant_append(cache, k, v, counts(gpu, 0), counts=counts(gpu, *n))
    m = tree(g, B, T) if mask == "tree" else mask
    return q, k, v, kn, vn, cache, m, scale or D ** -0.5


def check_attention(gpu, q, k, v, kn, vn, cache, mask, scale, n, **kw):
    from dropkv_amd import ops
    got = ops.quant_attention(q, kn, vn, cache, counts(gpu, *n), scale, mask=mask, **kw)
    D, M = q.shape[3], q.shape[1] // k.shape[1] * q.shape[2]
    ref, mean, size = R.attend(q, k, v, kn, vn, n, scale, mask, cache.k.dtype)
    tol = R.tolerance(ref, mean, size, q.dtype, D, once=M > 64 and q.dtype is BF)
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), float((err / tol).max())
    return got


@pytest.mark.parametrize("store", R.STORES)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 64), (14, 2, 64), (32, 8, 128), (16, 1, 128)])
@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 130, 1000])
def test_one_token(gpu, n, Hq, Hkv, D, dtype, store):
    case = attention_case(gpu, Hq, Hkv, D, 1, [n], dtype, store, mask=None)
    check_attention(gpu, *case, [n])


@pytest.mark.parametrize("store", R.STORES)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("T", [2, 5, 16, 17, 40, 64, 65, 100, 256])
def test_drafted_tokens(gpu, T, Hq, Hkv, D, dtype, store):
    n = [200, 0, 447]
    case = attention_case(gpu, Hq, Hkv, D, T, n, dtype, store)
    check_attention(gpu, *case, n)


@pytest.mark.parametrize("T", [1, 7, 33, 90])
def test_a_batch_of_unequal_lengths(gpu, T):
    n = [5000, 3, 64, 1999, 0, 129, 640, 63]
    case = attention_case(gpu, 8, 2, 128, T, n, BF, I8, mask=None)
    check_attention(gpu, *case, n)


@pytest.mark.parametrize("T", [1, 6, 20, 130])
def test_one_count_for_all(gpu, T):
    from dropkv_amd import ops
    n = [333, 333]
    case = attention_case(gpu, 8, 4, 64, T, n, FP, F8)
    q, k, v, kn, vn, cache, mask, scale = case
    a = check_attention(gpu, *case, n)
    b = ops.quant_attention(q, kn, vn, cache, counts(gpu, 333), scale, mask=mask)
    torch.testing.assert_close(a, b, rtol=2.0 ** -10, atol=2.0 ** -12)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T", [1, 4, 30, 120])
def test_rows_that_see_nothing(gpu, T, dtype):
    """Tokens whose mask is empty over an empty cache: zeros; not over a cache with rows."""
    g = generator(gpu, T)
    mask = tree(g, 2, T)
    mask[:, T // 2] = False
    n = [0, 100]
    case = attention_case(gpu, 4, 2, 64, T, n, dtype, I8, mask=mask)
    got = check_attention(gpu, *case, n)
    assert not got[0, T // 2].any() and got[1, T // 2].any()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T", [3, 24, 80])
def test_values_that_are_not_finite(gpu, T, dtype):
    """New rows that are not finite reach the tokens that see them alone; a block that
    holds one comes out as NaN for its sequence's head."""
    from dropkv_amd import ops
    n = [70, 70]
    q, k, v, kn, vn, cache, mask, scale = attention_case(gpu, 4, 2, 64, T, n, dtype, I8)
    clean = ops.quant_attention(q, kn, vn, cache, counts(gpu, *n), scale, mask=mask)
    kx, vx = kn.clone(), vn.clone()
    kx[0, 0, T - 1] = float("nan")
    vx[0, 1, 1, 5] = float("inf")
    vx[1, 0, T - 1, 6] = float("nan")
    got = ops.quant_attention(q, kx, vx, cache, counts(gpu, *n), scale, mask=mask)
    for b in range(2):
        for h in range(4):
            for t in range(T):
                bad = torch.zeros(64, dtype=torch.bool, device=gpu)
                if b == 0 and h < 2 and mask[b, t, T - 1]:
                    bad[:] = True
                if b == 0 and h >= 2 and mask[b, t, 1]:
                    bad[5] = True
                if b == 1 and h < 2 and mask[b, t, T - 1]:
                    bad[6] = True
                assert torch.equal(torch.isfinite(got[b, t, h]), ~bad), (b, h, t)
                if b == 0 and h < 2 and not mask[b, t, T - 1]:
                    assert torch.equal(got[b, t, h], clean[b, t, h])
    # Stored: a block of its own, and a row of the tail.
    for at, block in ((3, True), (66, False)):
        k2 = k.clone()
        k2[1, 1, at, 2] = float("nan")
        ops.quant_append(cache, k2, v, counts(gpu, 0), counts=counts(gpu, *n))
        got = ops.quant_attention(q, kn, vn, cache, counts(gpu, *n), scale, mask=mask)
        assert torch.isnan(got[1, :, 2:]).all() and torch.isfinite(got[1, :, :2]).all() and torch.isfinite(got[0]).all()


@pytest.mark.parametrize("T", [1, 5, 40, 70])
def test_scales_of_all_sizes(gpu, T):
    """Blocks whose scales differ by many orders, zeros and blocks below 2^-100 among
    them."""
    g = generator(gpu, T)
    q, k, v, kn, vn, cache, mask, scale = attention_case(gpu, 8, 2, 64, T, [64 * 9 + 5], BF, I8)
    from dropkv_amd import ops
    f = torch.tensor([1, 1e-3, 0, 3e4, 1e-35, 1e-8, 1e8, 1, 1e-20, 1.0], device=gpu).repeat_interleave(64)[:k.shape[2], None]
    v = (v.float() * f).to(BF)
    k = (k.float() * f.clamp(max=1)).to(BF)
    ops.quant_append(cache, k, v, counts(gpu, 0))
    check_attention(gpu, q, k, v, kn, vn, cache, mask, scale, [64 * 9 + 5])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T", [1, 9, 30, 80])
def test_large_logits(gpu, T, dtype):
    """Logits up to 10^9 (bf16): no weight leaves the type's range."""
    from dropkv_amd import ops
    q, k, v, kn, vn, cache, mask, scale = attention_case(gpu, 4, 2, 64, T, [300], dtype, F8)
    q, k, kn = q * 100, k * 100, kn * 100
    if dtype is BF:
        q, k, kn = q * 64, k * 64, kn * 64
    ops.quant_append(cache, k, v, counts(gpu, 0))
    got = ops.quant_attention(q, kn, vn, cache, counts(gpu, 300), scale, mask=mask)
    assert torch.isfinite(got).all()
    assert got.abs().max() <= max(v.abs().max(), vn.abs().max()) * (1 + 2.0 ** -7)


@pytest.mark.parametrize("T", [1, 12, 50, 140])
def test_strides(gpu, T):
    """q as a projection, new rows as views of a longer buffer at odd offsets, a mask
    and an output by strides."""
    from dropkv_amd import ops
    n = [150, 90]
    q, k, v, kn, vn, cache, mask, scale = attention_case(gpu, 8, 2, 128, T, n, BF, I8)
    want = ops.quant_attention(q, kn, vn, cache, counts(gpu, *n), scale, mask=mask)
    q2 = q.transpose(1, 2).contiguous().transpose(1, 2)
    big = torch.full((2, 2, T + 3, 131), 7.0, dtype=BF, device=gpu)
    big[:, :, 2:T + 2, 1:129] = kn
    m2 = mask.transpose(1, 2).contiguous().transpose(1, 2)
    out = torch.full((2, 8, T, 128), 3.0, dtype=BF, device=gpu).transpose(1, 2)
    ws = ops.quant_workspace(2, 8, 2, 128, T, cache.k.shape[2], gpu)
    got = ops.quant_attention(q2, big[:, :, 2:T + 2, 1:129], vn, cache, counts(gpu, *n), scale, out, ws, m2)
    assert got is out and torch.equal(got, want)


@pytest.mark.parametrize("T", [1, 10, 70])
def test_graph_replays(gpu, T):
    """Append, attention and read captured together, replayed with other counts."""
    from dropkv_amd import ops
    n = [100, 61]
    q, k, v, kn, vn, cache, mask, scale = attention_case(gpu, 8, 2, 64, T, n, BF, I8, C=640)
    n_rows = counts(gpu, *n)

    def step():
        out = ops.quant_attention(q, kn, vn, cache, n_rows, scale, mask=mask)
        ops.quant_append(cache, kn, vn, n_rows)
        return out, *ops.quant_read(cache, n_rows, 400)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    keep = [t.clone() for t in cache]
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for t, w in zip(cache, keep):
        t.view(torch.uint8).copy_(w.view(torch.uint8))
    for _ in range(3):
        before = [t.clone() for t in cache]
        graph.replay()
        got = [t.clone() for t in outs]
        after = [t.clone() for t in cache]
        for t, w in zip(cache, before):
            t.view(torch.uint8).copy_(w.view(torch.uint8))
        for a, b in zip(got, step()):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        for a, b in zip(after, cache):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        n_rows += T
        torch.cuda.synchronize()


def test_two_streams(gpu):
    """Calls on two streams at once keep their workspaces apart."""
    from dropkv_amd import ops
    cases = [attention_case(gpu, 8, 2, 128, 9, [3000], BF, s, seed=i) for i, s in enumerate(R.STORES)]

    def call(c):
        q, k, v, kn, vn, cache, mask, scale = c
        return ops.quant_attention(q, kn, vn, cache, counts(gpu, 3000), scale, mask=mask)

    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x, want[i])
