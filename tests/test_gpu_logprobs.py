"""Log probabilities, entropy and top tokens (``dropkv_token_logprobs``)
against the formulas in 64 bits.

Tolerance.  With d = x - m (one rounding), e^d is off by 2^-24 |d log2 e| + 2^-22
relative (the product's rounding, the exponential's), a term |d| of weight
e^d by at most 2^-22 in the sums, and each of the additions adds 2^-24: a
thread adds V / 256 terms or fewer one after the other, and 20 partial sums.
ln s and the final differences add 4 roundings of the values' magnitudes."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(x, tokens, top):
    """(logprob, entropy, top logprobs, top ids) in 64 bits, on the CPU."""
    d = x.double()
    lp = torch.log_softmax(d, -1)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    t = tokens.clamp(0, x.shape[-1] - 1)
    out = torch.where(tokens < 0, torch.zeros(()).double(), lp.gather(-1, t[..., None])[..., 0])
    out = torch.where(tokens >= x.shape[-1], torch.full_like(out, math.nan), out)
    order = torch.where(d.isnan(), torch.full_like(d, math.inf), d)   # (rows with NaN hold no +inf here)
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :top]
    return out, ent, lp.gather(-1, ids), ids


def close(got, want, V):
    want = want.float().double()   # (a difference of two values near fp32's largest is -inf in fp32)
    tol = (V / 256 + 40) * 2.0 ** -24 * 2 + 4 * 2.0 ** -24 * want.abs().clamp(min=1) + 2.0 ** -20
    same = (got.double() == want) | (got.isnan() & want.isnan())
    return (same | ((got.double() - want).abs() <= tol)).all()


def check(gpu, x, top, tokens=None):
    from dropkv_amd import ops
    lead, V = x.shape[:-1], x.shape[-1]
    if tokens is None:
        tokens = torch.randint(0, V, lead, generator=torch.Generator().manual_seed(V))
    want = reference(x, tokens, top)
    got = ops.token_logprobs(x.to(gpu), tokens.to(gpu), top=top)
    for g, w, name in zip(got, want, ("logprob", "entropy", "top_logprobs")):
        assert g.shape == w.shape and close(g.cpu(), w, V), name
    assert torch.equal(got.top_ids.cpu(), want[3])
    return got


@pytest.mark.parametrize("N,V,top,dtype", [
    (1, 151936, 5, torch.bfloat16),
    (3, 151936, 1, torch.bfloat16),
    (3, 32000, 32, torch.float16),
    (5, 32001, 20, torch.bfloat16),       # rows at odd addresses
    (2, 4096, 8, torch.float32),
    (2, 4097, 8, torch.float32),
    (2, 300001, 32, torch.float32),       # blocks of several selection rounds
    (1, 600000, 20, torch.bfloat16),
    (20, 151936, 7, torch.bfloat16),      # segments joined by a second kernel
    (20, 151936, 1, torch.float16),
    (20, 50000, 0, torch.bfloat16),
    (7, 1, 1, torch.float32),
    (4, 31, 31, torch.bfloat16),
    (4, 8, 0, torch.float16),
    (300, 9001, 3, torch.float16),        # segments of several tiles
    (2100, 5003, 20, torch.bfloat16),     # rows whole
    (2100, 700, 1, torch.bfloat16),
])
def test_rows(gpu, N, V, top, dtype):
    g = torch.Generator().manual_seed(N + V)
    x = torch.randn(N, V, generator=g) * 3
    hot = torch.randint(0, V, (N, 5), generator=g)
    x.scatter_add_(1, hot, torch.rand(N, 5, generator=g) * 12)
    check(gpu, x.to(dtype), top)


@pytest.mark.parametrize("V,top", [(20000, 20), (20000, 32), (20000, 1), (9000, 2)])
@pytest.mark.parametrize("N", [2, 2500])
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "two values", "steps"])
def test_orders(gpu, V, top, N, order):
    """Orders that make the list of candidates overflow or tie throughout."""
    base = {"rising": torch.arange(V) / 64.0, "falling": -torch.arange(V) / 64.0, "equal": torch.full((V,), 2.5),
            "two values": (torch.arange(V) % 97 == 5).float() * 3, "steps": (torch.arange(V) // 3000).float()}[order]
    from dropkv_amd import ops
    x = base.float().expand(2, V).contiguous()
    want = reference(x, torch.tensor([0, V - 1]), top)
    xs, ts = x[:1].expand(N, V), torch.zeros(N, dtype=torch.int64)     # (every row the same, read by stride 0)
    got = ops.token_logprobs(xs.to(gpu) if N < 10 else x[:1].to(gpu).expand(N, V), ts.to(gpu), top=top)
    for g, w in zip(got[:3], want[:3]):
        assert close(g.cpu(), w[:1].expand(N, *w.shape[1:]), V)
    assert torch.equal(got.top_ids.cpu(), want[3][:1].expand(N, top))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("top", [0, 1, 4])
def test_masked_logits(gpu, dtype, top):
    """-inf and the type's lowest value among the logits, rows of nothing
    else, and single survivors."""
    V = 10000
    g = torch.Generator().manual_seed(top)
    x = torch.randn(8, V, generator=g)
    low = torch.finfo(dtype).min
    x[0, torch.rand(V, generator=g) < 0.9] = -math.inf
    x[1, torch.rand(V, generator=g) < 0.9] = low
    x[2] = -math.inf
    x[3] = low
    x[4] = -math.inf
    x[4, 7777] = 1.5
    x[5, :9990] = -math.inf
    x[6] = low
    x[6, 9999] = torch.finfo(dtype).max
    x = x.to(dtype)
    tokens = torch.tensor([0, 1, 2, 3, 7777, 0, 9999, -100])
    from dropkv_amd import ops
    want = reference(x, tokens, top)
    got = ops.token_logprobs(x.to(gpu), tokens.to(gpu), top=top)
    for i in range(8):
        if i == 2:      # only -inf: nothing is defined
            assert got.logprob[2].isnan() and got.entropy[2].isnan() and got.top_logprobs[2].isnan().all()
        else:
            for g_, w in zip(got[:3], want[:3]):
                if not (dtype == torch.float32 and i == 6):
                    assert close(g_[i].cpu(), w[i], V), i
    assert torch.equal(got.top_ids.cpu(), want[3])
    assert float(got.logprob[6]) == 0 and float(got.entropy[6]) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [0, 1, 4])
@pytest.mark.parametrize("N", [1, 2100])
def test_huge_logits(gpu, dtype, top, N):
    """Logits near and beyond 1e38, of either sign, rising and falling through it
    within a thread's share: differences that large leave weight to the largest
    alone, or to its equals."""
    V, big = 20000, 3e38
    line = lambda lo, hi: torch.linspace(lo, hi, V, dtype=torch.float64).float()     # (its span is beyond fp32)
    rows = [line(-big, -9e37), line(-9e37, -big), line(-big, big), line(big, 9e37),
            torch.full((V,), -2e38), torch.full((V,), 9e37), torch.full((V,), 1e30)]
    rows[4][[5, 4101, 9000]] = -1.5e38
    rows[5][[17, 8209]] = 1.1e38
    rows[6][4096:] = -3.3e38
    x = torch.stack(rows).to(dtype)
    tokens = torch.tensor([0, 0, V - 1, 0, 5, 8209, 100])
    want = reference(x, tokens, top)
    from dropkv_amd import ops
    for i in range(len(rows)):
        got = ops.token_logprobs(x[i:i + 1].to(gpu).expand(N, V), tokens[i:i + 1].to(gpu).expand(N), top=top)
        for g, w, name in zip(got[:3], want[:3], ("logprob", "entropy", "top_logprobs")):
            assert close(g.cpu(), w[i:i + 1].expand(N, *w.shape[1:]), V), (i, name)
        assert torch.equal(got.top_ids.cpu(), want[3][i:i + 1].expand(N, top)), i


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [50.0, 300.0, -4000.0])
@pytest.mark.parametrize("N", [1, 2100])
def test_logits_far_from_zero(gpu, dtype, shift, N):
    """What is said of a row does not lose by where its logits lie."""
    V = 30000
    x = (torch.randn(V, generator=torch.Generator().manual_seed(3)) * 4 + shift).to(dtype)[None]
    tokens = torch.tensor([77])
    want = reference(x, tokens, 3)
    from dropkv_amd import ops
    got = ops.token_logprobs(x.to(gpu).expand(N, V), tokens.to(gpu).expand(N), top=3)
    for g, w, name in zip(got[:3], want[:3], ("logprob", "entropy", "top_logprobs")):
        assert close(g.cpu(), w.expand(N, *w.shape[1:]), V), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("value", [-1.7, 0.3, math.nan, -60000.0])
@pytest.mark.parametrize("V,N,top", [(20000, 3, 32), (150001, 1, 20), (3000, 2500, 7), (90, 4, 32), (700, 2, 31)])
def test_equal_logits(gpu, dtype, value, V, N, top):
    """More equals than the list of candidates holds, of either sign, a few
    larger ones among them: the lowest places come first."""
    x = torch.full((V,), value, dtype=dtype)
    more = [V // 2, V // 3, V - 1]
    if value == value:
        x[more] = 2.0
        want = sorted(more)
    else:
        x[more] = 2.0        # NaN is above them
        want = []
    rest = [i for i in range(top + 6) if i not in more]
    from dropkv_amd import ops
    got = ops.token_logprobs(x.to(gpu).expand(N, V), top=top)
    assert torch.equal(got.top_ids.cpu(), torch.tensor((want + rest)[:top]).expand(N, top))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("top", [1, 6])
@pytest.mark.parametrize("N", [1, 2100])
def test_zeros_of_either_sign(gpu, dtype, top, N):
    """-0 and 0 are equals: the lowest places come first."""
    V = 5000
    x = torch.full((1, V), -2.0, dtype=dtype)
    x[0, 3:4000:5] = 0.0
    x[0, 3:4000:10] = -0.0
    from dropkv_amd import ops
    got = ops.token_logprobs(x.to(gpu).expand(N, V), top=top)
    assert torch.equal(got.top_ids.cpu(), torch.arange(3, 3 + 5 * top, 5).expand(N, top))


@pytest.mark.parametrize("top", [1, 6])
def test_nan_and_inf(gpu, top):
    """NaN or +inf anywhere: the row is NaN; NaN ranks above all, ties and NaN
    by the lowest place; other rows are untouched."""
    from dropkv_amd import ops
    V = 13000
    x = torch.randn(4, V, generator=torch.Generator().manual_seed(1))
    clean = ops.token_logprobs(x.to(gpu), torch.zeros(4, dtype=torch.int64, device=gpu), top=top)
    x[1, 12999] = math.nan
    x[1, 600] = -math.nan
    x[2, 5000] = math.inf
    got = ops.token_logprobs(x.to(gpu), torch.zeros(4, dtype=torch.int64, device=gpu), top=top)
    for a, b in zip(got, clean):
        assert torch.equal(a[[0, 3]], b[[0, 3]])
    assert got.entropy[1:3].isnan().all() and got.logprob[1:3].isnan().all()
    want = reference(x, torch.zeros(4, dtype=torch.int64), top)[3]
    assert torch.equal(got.top_ids.cpu(), want)


def test_tokens_outside_and_shapes(gpu):
    from dropkv_amd import ops
    x = torch.randn(2, 3, 500, generator=torch.Generator().manual_seed(0)).bfloat16()
    t = torch.tensor([[-1, 499, 500], [0, -100, 2 ** 40]])
    got = check(gpu, x, 2, t)
    assert float(got.logprob[0, 0]) == 0 and got.logprob[0, 2].isnan() and got.logprob[1, 2].isnan()
    # Rows by stride, an axis that is not contiguous, a single row, none.
    big = torch.randn(4, 2, 600, generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu)
    part = big[:, 1, 3:503]
    assert torch.equal(ops.token_logprobs(part, top=2).entropy, ops.token_logprobs(part.clone(), top=2).entropy)
    turned = part.t().contiguous().t()
    assert torch.equal(ops.token_logprobs(turned, top=2).top_ids, ops.token_logprobs(part, top=2).top_ids)
    one = ops.token_logprobs(part[0], torch.tensor(4, device=gpu), top=2)
    assert one.logprob.shape == () and one.top_ids.shape == (2,)
    none = ops.token_logprobs(part[:0], top=3)
    assert none.logprob is None and none.top_ids.shape == (0, 3)


def test_two_streams(gpu):
    """Calls on two streams at once keep their workspaces apart."""
    from dropkv_amd import ops
    xs = [torch.randn(3, 100000 + 7 * i, generator=torch.Generator().manual_seed(i)).to(gpu) for i in range(2)]
    want = [ops.token_logprobs(x, top=9) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.token_logprobs(xs[i], top=9))
    torch.cuda.synchronize()
    for w, rs in zip(want, got):
        for r in rs:
            assert all(torch.equal(a, b) for a, b in zip(r[1:], w[1:]))


def test_in_a_graph(gpu):
    from dropkv_amd import ops
    x = torch.randn(8, 30001, device=gpu).bfloat16()
    t = torch.zeros(8, dtype=torch.int64, device=gpu)
    ops.token_logprobs(x, t, top=7)
    torch.cuda.synchronize()
    graphs, res = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res.append(ops.token_logprobs(x, t, top=7))
        graphs.append(gr)
    for step in range(3):
        x.normal_()
        t.add_(111)
        for gr in graphs:
            gr.replay()
        want = ops.token_logprobs(x, t, top=7)
        torch.cuda.synchronize()
        for r in res:
            assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_refusals(gpu):
    from dropkv_amd import ops
    x = torch.zeros(3, 100, device=gpu)
    t = torch.zeros(3, dtype=torch.int64, device=gpu)
    for args, kw in [((x.long(), t), {}), ((x, t.int()), {}), ((x, t[:2]), {}), ((x, t), dict(top=101)),
                     ((x, t), dict(top=33)), ((x, t), dict(top=-1)), ((x, t.cpu()), {}), ((x.cpu(), None), {}),
                     ((x.clone().requires_grad_(), t), {})]:
        with pytest.raises(RuntimeError):
            ops.token_logprobs(*args, **kw)
