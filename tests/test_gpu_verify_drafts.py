"""Drafted chains verified by sampling, against the definition in 64 bits: which
tokens stand, the token drawn after them, log probabilities."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def reference(logits, tokens, uniforms, draft_logits, temperature):
    B, T, V = logits.shape
    choice = torch.full((B, T), -1, dtype=torch.int64)
    accepted = torch.zeros(B, dtype=torch.int32)
    lps = torch.zeros(B, T, dtype=torch.float64)
    tok, u = tokens.tolist(), uniforms.double().tolist()
    for b in range(B):
        i = 0
        while True:
            lp = torch.log_softmax(logits[b, i].double() / temperature, -1)
            p = lp.exp()
            x = tok[b][i + 1] if i + 1 < T else -1
            w = p
            if 0 <= x < V:
                if draft_logits is None:
                    q = torch.zeros_like(p)
                    q[x] = 1
                else:
                    q = torch.softmax(draft_logits[b, i].double() / temperature, -1)
                if u[b][i + 1] * float(q[x]) < float(p[x]):
                    choice[b, i], lps[b, i] = x, lp[x]
                    i += 1
                    continue
                rest = (p - q).clamp(min=0)
                w = rest if float(rest.sum()) > 0 else p
            if not math.isfinite(float(w.sum())):
                lps[b, i] = float("nan")
            else:
                c = w.cumsum(0)
                over = torch.nonzero((c > u[b][0] * c[-1]) & (w > 0))
                x = int(over[0]) if len(over) else int(torch.nonzero(w > 0)[-1])
                choice[b, i], lps[b, i] = x, lp[x]
            accepted[b] = i + 1
            break
    return choice, accepted, lps


def case(gpu, B, T, V, dtype, draft=True, seed=0, err=0.5, temperature=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed + 7 * T + V)
    x = torch.randn(B, T, V, generator=g, device=gpu) * 3
    near = (x[:, :-1] + err * torch.randn(B, T - 1, V, generator=g, device=gpu)).to(dtype)
    tokens = torch.randint(0, V, (B, T), generator=g, device=gpu)
    if T > 1:
        w = torch.softmax(near.float() / temperature, -1)
        tokens[:, 1:] = torch.multinomial(w.view(-1, V), 1, generator=g).view(B, T - 1)
    u = torch.rand(B, T, generator=g, device=gpu)
    return x.to(dtype), tokens, u, (near if draft else None)


def check(got, want, logits, temperature):
    choice, accepted, lps = want
    assert torch.equal(got.accepted.cpu(), accepted)
    assert torch.equal(got.choice.cpu(), choice)
    # One rounding of the difference to fp32, one of the result's own, and the logarithm's.
    lp = got.logprobs.cpu().double()
    torch.testing.assert_close(lp, lps, rtol=2.0 ** -22, atol=2.0 ** -22, equal_nan=True)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (2, 1, 50), (3, 2, 2), (5, 4, 7), (4, 8, 500), (2, 5, 4096), (2, 5, 4097),
                                   (7, 6, 32003), (1, 8, 151936), (3, 17, 9001), (2, 256, 301), (600, 3, 64)])
def test_against_the_definition(gpu, B, T, V, dtype, draft):
    from dropkv_amd import ops
    for temperature in (1.0, 0.7):
        x, tok, u, y = case(gpu, B, T, V, dtype, draft, temperature=temperature)
        got = ops.verify_drafts(x, tok, u, y, temperature)
        check(got, reference(x, tok, u, y, temperature), x, temperature)


@pytest.mark.parametrize("draft", [True, False])
def test_edges_of_the_random_numbers(gpu, draft):
    """u of 0 lets every token with any probability stand and draws the first one with
    any weight; u next to 1, 1 and NaN the last one."""
    from dropkv_amd import ops
    x, tok, u, y = case(gpu, 6, 4, 333, F32, draft)
    x[:, :, :3] = -math.inf
    x[:, :, -2:] = -math.inf
    tok.clamp_(3, 330)
    for first, rest in ((0.0, 0.0), (0.0, 1 - 2.0 ** -24), (1 - 2.0 ** -24, 1 - 2.0 ** -24), (1 - 2.0 ** -24, 0.0), (1.0, 1.0)):
        u[:, 0], u[:, 1:] = first, rest
        check(ops.verify_drafts(x, tok, u, y), reference(x, tok, u, y, 1.0), x, 1.0)
    u[:] = float("nan")
    got = ops.verify_drafts(x, tok, u, y)
    assert (got.accepted == 1).all() and (got.choice[:, 0] >= 3).all() and (got.choice[:, 0] < 331).all()


def test_equal_distributions_always_stand(gpu):
    from dropkv_amd import ops
    x, tok, u, _ = case(gpu, 8, 9, 1000, BF)
    u.clamp_(max=1 - 2.0 ** -24)
    got = ops.verify_drafts(x, tok, u, x[:, :-1])
    assert (got.accepted == 9).all() and torch.equal(got.choice[:, :-1], tok[:, 1:])


def test_tokens_that_end_a_chain(gpu):
    """A negative token, or one past the vocabulary: the chain before it stands by
    itself, and the next token is drawn from all of p."""
    from dropkv_amd import ops
    x, tok, u, y = case(gpu, 6, 5, 200, BF)
    tok[0, 1], tok[1, 2], tok[2, 4], tok[3, 3], tok[4, 1:] = -1, -5, -1, 200, 1 << 40
    tok[:, 0] = -3  # not read
    check(ops.verify_drafts(x, tok, u, y), reference(x, tok, u, y, 1.0), x, 1.0)
    check(ops.verify_drafts(x, tok, u), reference(x, tok, u, None, 1.0), x, 1.0)


def test_rows_that_are_not_finite(gpu):
    from dropkv_amd import ops
    x, tok, u, y = case(gpu, 6, 3, 777, F32)
    u[:, 1:] = 0
    x[0, 0, 5] = math.inf
    x[1, 0, 6] = math.nan
    x[2, 0] = -math.inf
    x[3, 2, 9] = math.nan
    y[4, 0, 3] = math.nan
    y[5, 1, 2] = math.inf
    tok[5, 2] = 10
    got = ops.verify_drafts(x, tok, u, y)
    assert got.accepted.tolist()[:5] == [1, 1, 1, 3, 1]
    for b, i in ((0, 0), (1, 0), (2, 0), (3, 2)):
        assert int(got.choice[b, i]) == -1 and math.isnan(float(got.logprobs[b, i]))
    # A draft row that is not finite: its token falls, and p itself is sampled.
    assert torch.equal(got.choice[4, :1].cpu(), reference(x[4:5, :1], tok[4:5, :1], u[4:5, :1], None, 1.0)[0][0])
    assert torch.isfinite(got.logprobs[4:]).all()


@pytest.mark.parametrize("temperature", [0.02, 0.3, 5.0, 1000.0])
def test_temperatures(gpu, temperature):
    from dropkv_amd import ops
    x, tok, u, y = case(gpu, 8, 6, 5000, BF, temperature=temperature)
    got = ops.verify_drafts(x, tok, u, y, temperature)
    choice, accepted, lps = reference(x, tok, u, y, temperature)
    assert torch.equal(got.choice.cpu(), choice) and torch.equal(got.accepted.cpu(), accepted)
    torch.testing.assert_close(got.logprobs.cpu().double(), lps, rtol=2.0 ** -22, atol=2.0 ** -22)


def test_tokens_are_distributed_as_the_models(gpu):
    """One node drafted from q, judged and replaced: the first new token over 200,000
    chains has the model's distribution (each frequency within 5 standard deviations)."""
    from dropkv_amd import ops
    N, V, temperature = 65000, 12, 0.9
    g = torch.Generator(device=gpu).manual_seed(3)
    one, draft = torch.randn(V, generator=g, device=gpu) * 1.5, torch.randn(V, generator=g, device=gpu) * 1.5
    p, q = (torch.softmax(t / temperature, -1) for t in (one, draft))
    count = torch.zeros(V, dtype=torch.float64, device=gpu)
    for _ in range(3):
        x = one.expand(N // 2, 2, V).contiguous()
        for _ in range(2):
            n = N // 2
            tok = torch.multinomial(q, n, replacement=True, generator=g)
            got = ops.verify_drafts(x, torch.stack([tok, tok], 1), torch.rand(n, 2, generator=g, device=gpu),
                                    draft.expand(n, 1, V).contiguous(), temperature)
            count += torch.bincount(got.choice[:, 0], minlength=V)
    total = count.sum()
    dev = torch.sqrt(total * p.double() * (1 - p.double()))
    assert ((count - total * p.double()).abs() < 5 * dev).all()


def test_strides(gpu):
    from dropkv_amd import ops
    x, tok, u, y = case(gpu, 3, 5, 1001, BF)
    want = ops.verify_drafts(x, tok, u, y)
    big = torch.zeros(3, 7, 1005, dtype=BF, device=gpu)
    big[:, 1:6, 3:1004] = x
    dr = torch.zeros(4, 3, 1001, dtype=BF, device=gpu)
    dr.copy_(y.transpose(0, 1))
    got = ops.verify_drafts(big[:, 1:6, 3:1004], tok.t().contiguous().t(), u, dr.transpose(0, 1))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    got = ops.verify_drafts(x.transpose(1, 2).contiguous().transpose(1, 2), tok, u, y)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_graph_replays_and_streams(gpu):
    from dropkv_amd import ops
    x, tok, u, y = case(gpu, 4, 6, 20000, BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.verify_drafts(x, tok, u, y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.verify_drafts(x, tok, u, y)
    for seed in range(4):
        x2, tok2, u2, y2 = case(gpu, 4, 6, 20000, BF, seed=seed + 1)
        for a, b in ((x, x2), (tok, tok2), (u, u2), (y, y2)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        check(out, reference(x2, tok2, u2, y2, 1.0), x2, 1.0)
        with torch.cuda.stream(side):
            other = ops.verify_drafts(x2, tok2, u2, y2)
        torch.cuda.synchronize()
        assert torch.equal(other.choice, out.choice)


@pytest.mark.parametrize("temperature,top", [(1e-6, 2.0 ** 17), (3e-9, 100.0), (3e-9, -100.0), (1e-12, 100.0), (1e-12, 1.0),
                                             (1e-29, 3.0), (2e-5, 2.0 ** 12), (1e-3, 2.0 ** 17)])
def test_temperatures_next_to_zero(gpu, temperature, top):
    """Logits a step of fp32 below the largest, where that is thousands of powers of two:
    the largest ones share all of the probability."""
    from dropkv_amd import ops
    step = abs(top) * 2.0 ** -23
    k = torch.randint(1, 4, (4, 3, 5000), generator=torch.Generator().manual_seed(1))
    k[:, :, 77::1000] = 0
    x = (top - k.double() * step * 2).float().to(gpu)
    gap = 2 * step / temperature
    u = torch.tensor([0.0, 0.9, 0.0]).repeat(4, 1).to(gpu)
    u[:, 0] = torch.tensor([0.0, 0.25, 0.65, 0.99])
    tok = torch.full((4, 3), 78, device=gpu)
    got = ops.verify_drafts(x, tok, u, None, temperature)
    if gap > 800:
        assert (got.accepted == 1).all() and got.choice[:, 0].tolist() == [77, 1077, 3077, 4077]
        torch.testing.assert_close(got.logprobs[:, 0].cpu().double(), torch.full((4,), -math.log(5.0), dtype=torch.float64),
                                   rtol=2.0 ** -22, atol=2.0 ** -22)
    else:  # (differences of a step are exact in 64 bits)
        lp = torch.log_softmax((x[:, 0].double() - top) / temperature, -1).gather(1, got.choice[:, :1].clamp(min=0))[:, 0]
        torch.testing.assert_close(got.logprobs[:, 0].double(), lp, rtol=2.0 ** -22, atol=2.0 ** -22)
