"""Attention of drafted tokens (``dropkv_tree_attention``) and the accepted
rows (``dropkv_tree_commit``) against the formulas in 64 bits on the CPU.

Tolerance of the attention.  Products of bf16 / fp16 values are exact in fp32,
so a logit is off by at most D 2^-24 |scale| |q| |k| =: d, a weight relative by
2 d (its own and the sum's) and by 2^-16 for P held in two parts and the
exponential; each addition of the sums over n keys adds 2^-24, one for 16 keys
at the most and one for a split.  The store adds half a step.

With more than 64 rows (g T) to a KV head P may be rounded once to the element type:
each weight is off by half a step, 2^-8 (bf16) or 2^-11 (fp16) of itself, and the
output by at most that of sum p |v|."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def make_tree(B, T, seed, window=6):
    """Random parents [B, T] and ancestor masks [B, T, T]."""
    g = torch.Generator().manual_seed(seed)
    parents = torch.zeros(B, T, dtype=torch.int64)
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    for i in range(T):
        if i:
            parents[:, i] = torch.randint(max(0, i - window), i, (B,), generator=g)
            mask[:, i] = mask[torch.arange(B), parents[:, i]]
        mask[:, i, i] = True
    return parents.to(torch.int32), mask


def reference(q, kn, vn, kc, vc, lens, mask, scale):
    """[B, T, Hq, D] in 64 bits, on the rows each token sees; and the bound."""
    B, Hq, T, D = q.shape
    g = Hq // kc.shape[1]
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    tol = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    for b, n in enumerate(lens):
        for h in range(Hq):
            k = torch.cat([kc[b, h // g, :n], kn[b, h // g]]).double()
            v = torch.cat([vc[b, h // g, :n], vn[b, h // g]]).double()
            for t in range(T):
                see = torch.cat([torch.ones(n, dtype=torch.bool), mask[b, t]])
                if not see.any():
                    continue
                ks, vs = k[see], v[see]
                s = ks @ q[b, h, t].double() * scale
                out[b, t, h] = torch.softmax(s, 0) @ vs
                d = D * 2.0 ** -24 * abs(scale) * q[b, h, t].double().norm() * ks.norm(dim=1).max()
                p = torch.softmax(s, 0)
                tol[b, t, h] = vs.abs().max() * (2 * d + 2.0 ** -16 + (n / 16 + T / 16 + 80) * 2.0 ** -24)
                if g * T > 64:
                    tol[b, t, h] = tol[b, t, h] + torch.finfo(q.dtype).eps / 2 * (p @ vs.abs())
    half = torch.finfo(q.dtype).eps / 2
    return out, tol * (1 + half) + half * out.abs()


def case(B, Hq, Hkv, D, T, C, dtype, seed, strided=False):
    g = torch.Generator().manual_seed(seed)

    def rnd(H, L):
        x = torch.randn(B, L, H, D, generator=g).to(dtype) if strided else torch.randn(B, H, L, D, generator=g).to(dtype)
        return x.transpose(1, 2) if strided else x

    return (rnd(Hq, T) * 1.5, rnd(Hkv, T), rnd(Hkv, T), torch.randn(B, Hkv, C, D, generator=g).to(dtype),
            torch.randn(B, Hkv, C, D, generator=g).to(dtype))


def check(gpu, B, Hq, Hkv, D, T, C, lens, dtype, mask="tree", strided=False, seed=0):
    from dropkv_amd import ops
    q, kn, vn, kc, vc = case(B, Hq, Hkv, D, T, C, dtype, seed, strided)
    m = make_tree(B, T, seed)[1] if mask == "tree" else torch.ones(T, T, dtype=torch.bool).tril().expand(B, T, T)
    scale = D ** -0.5
    ref, tol = reference(q, kn, vn, kc, vc, lens, m, scale)
    n_rows = torch.tensor(lens, dtype=torch.int32, device=gpu)
    kd, vd = kc.to(gpu), vc.to(gpu)
    got = ops.tree_attention(q.to(gpu), kn.to(gpu), vn.to(gpu), kd, vd, n_rows, scale,
                             mask=m.to(gpu) if mask == "tree" else None)
    err = (got.cpu().double() - ref).abs()
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)


@pytest.mark.parametrize("B,Hq,Hkv,D,T,C,lens,dtype", [
    (1, 14, 2, 64, 8, 700, [638], torch.bfloat16),        # Qwen2-0.5B heads
    (1, 32, 8, 128, 16, 420, [411], torch.bfloat16),      # Llama heads
    (2, 8, 2, 128, 5, 96, [33, 64], torch.float16),       # odd tree, lengths around whole tiles
    (3, 4, 4, 64, 1, 64, [0, 1, 63], torch.bfloat16),     # one token; an empty cache
    (2, 6, 2, 64, 33, 40, [0, 31], torch.float16),        # more drafted than a tile, capacity of no whole tile
    (1, 64, 8, 128, 64, 300, [257], torch.bfloat16),      # 512 rows a KV head
    (1, 2, 1, 64, 256, 100, [100], torch.bfloat16),       # the largest tree, a full buffer
    (4, 16, 16, 64, 7, 2100, [2100, 1, 1024, 2047], torch.float16),
    (1, 17, 1, 128, 3, 200, [150], torch.bfloat16),       # 17 query heads to one KV head
])
@pytest.mark.parametrize("mask", ["tree", "chain"])
def test_attention(gpu, B, Hq, Hkv, D, T, C, lens, dtype, mask):
    check(gpu, B, Hq, Hkv, D, T, C, lens, dtype, mask, seed=C + T)


@pytest.mark.parametrize("T", [1, 4, 27])
def test_attention_of_projections(gpu, T):
    """q, k_new and v_new as [B, T, H, D] seen as [B, H, T, D]."""
    check(gpu, 2, 14, 2, 64, T, 333, [300, 17], torch.bfloat16, strided=True, seed=T)


@pytest.mark.parametrize("B,Hq,Hkv,D,T,C,top", [
    (64, 4, 2, 64, 3, 3000, 3000),     # up to 16 rows: lengths 0 .. 3000, the most sequences dealt by length
    (65, 2, 1, 64, 2, 900, 900),       # one more: equal parts
    (12, 8, 2, 64, 9, 2500, 2500),     # up to 64 rows
    (9, 8, 1, 128, 13, 1900, 1900),    # up to 128
    (7, 16, 2, 64, 33, 1500, 1500),    # beyond: two chunks of rows
    (3, 16, 2, 64, 33, 4200, 70),      # short sequences in long buffers
])
def test_lengths_of_their_own(gpu, B, Hq, Hkv, D, T, C, top):
    """Sequences from empty to full, dealt out to the workgroups by length."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, top + 1, (B,), generator=g).tolist()
    lens[0], lens[-1] = 0, top
    if B > 10:      # a sample is compared; the reference walks row by row
        from dropkv_amd import ops
        q, kn, vn, kc, vc = case(B, Hq, Hkv, D, T, C, torch.bfloat16, 5)
        m = make_tree(B, T, 5)[1]
        got = ops.tree_attention(q.to(gpu), kn.to(gpu), vn.to(gpu), kc.to(gpu), vc.to(gpu),
                                 torch.tensor(lens, dtype=torch.int32, device=gpu), D ** -0.5, mask=m.to(gpu)).cpu()
        for b in (0, 1, B // 2, B - 2, B - 1):
            s = slice(b, b + 1)
            ref, tol = reference(q[s], kn[s], vn[s], kc[s], vc[s], lens[s], m[s], D ** -0.5)
            assert ((got[s].double() - ref).abs() <= tol).all(), b
    else:
        check(gpu, B, Hq, Hkv, D, T, C, lens, torch.bfloat16, seed=5)


def test_attention_unaligned(gpu):
    """Rows of q, k_new and v_new that start at no whole 16 bytes, a mask of
    other strides, one mask and one count for all sequences, out by strides."""
    from dropkv_amd import ops
    B, Hq, Hkv, D, T, C, n = 2, 8, 4, 64, 6, 128, 77
    q, kn, vn, kc, vc = case(B, Hq, Hkv, D, T, C, torch.bfloat16, 3)
    m = make_tree(1, T, 5)[1]
    ref, tol = reference(q, kn, vn, kc, vc, [n, n], m.expand(B, T, T), 0.2)

    def odd(x):
        big = torch.full((*x.shape[:-1], D + 3), 7.0, dtype=x.dtype, device=gpu)
        big[..., 1:1 + D] = x.to(gpu)
        return big[..., 1:1 + D]

    mt = m[0].t().contiguous().to(gpu).t()
    buf = torch.full((B, Hq, T, D), 3.0, dtype=torch.bfloat16, device=gpu)
    got = ops.tree_attention(odd(q), odd(kn), odd(vn), kc.to(gpu), vc.to(gpu),
                             torch.tensor([n], dtype=torch.int32, device=gpu), 0.2, out=buf.transpose(1, 2), mask=mt)
    assert got.data_ptr() == buf.data_ptr()
    assert ((got.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_see_nothing(gpu, dtype, D):
    """An empty cache and mask rows of zeros: zeros; the other rows as ever."""
    from dropkv_amd import ops
    B, Hq, Hkv, T, C = 1, 6, 2, 9, 64
    q, kn, vn, kc, vc = case(B, Hq, Hkv, D, T, C, dtype, 11)
    m = make_tree(B, T, 1)[1]
    m[:, 4] = False
    m[:, 8] = False
    ref, tol = reference(q, kn, vn, kc, vc, [0], m, 0.1)
    got = ops.tree_attention(q.to(gpu), kn.to(gpu), vn.to(gpu), kc.to(gpu), vc.to(gpu),
                             torch.zeros(1, dtype=torch.int32, device=gpu), 0.1, mask=m.to(gpu)).cpu()
    assert ((got.double() - ref).abs() <= tol).all()
    assert (got[:, [4, 8]] == 0).all()


@pytest.mark.parametrize("B,Hq,Hkv,D,T,C,dtype", [
    (48, 4, 4, 64, 70, 130, torch.float16),       # one part: its workgroup writes the output
    (24, 8, 4, 128, 70, 130, torch.bfloat16),
    (70, 12, 4, 64, 24, 65, torch.bfloat16),
    (48, 8, 4, 128, 100, 300, torch.float16),     # 200 rows of one workgroup
    (64, 8, 4, 128, 40, 1200, torch.bfloat16),
    (48, 8, 4, 64, 40, 1200, torch.bfloat16),     # two parts, the drafted keys with the last
    (48, 4, 4, 128, 100, 0, torch.bfloat16),      # no cache
])
@pytest.mark.parametrize("own", [True, False])
def test_many_heads(gpu, B, Hq, Hkv, D, T, C, dtype, own):
    """Heads enough to fill the GPU: few parts, the drafted keys in the last.  Rows
    that see nothing of an empty cache, a drafted value that is not finite and
    that one token sees, outputs in a buffer with room between the tokens."""
    from dropkv_amd import ops
    q, kn, vn, kc, vc = case(B, Hq, Hkv, D, T, C, dtype, 9)
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, C + 1, (B,), generator=g).tolist() if own else [max(0, C - 3)] * B
    if own:
        lens[0], lens[1] = 0, C
    m = make_tree(B, T, 9)[1]
    m[:, 5] = False
    m[:, :, 11] = False
    m[:, 11, 11] = True
    refs = {b: reference(q[b:b + 1], kn[b:b + 1], vn[b:b + 1], kc[b:b + 1], vc[b:b + 1], lens[b:b + 1], m[b:b + 1], 0.1)
            for b in (0, 1, B - 1)}
    vn[:, :, 11, 3] = math.inf
    out = torch.full((B, T, Hq, D + 8), 7.0, dtype=dtype, device=gpu)
    ops.tree_attention(q.to(gpu), kn.to(gpu), vn.to(gpu), kc.to(gpu), vc.to(gpu),
                       torch.tensor(lens if own else lens[:1], dtype=torch.int32, device=gpu), 0.1, mask=m.to(gpu),
                       out=out[..., :D])
    got = out.cpu()
    assert (got[..., D:] == 7).all()
    for b, (ref, tol) in refs.items():
        x = got[b:b + 1, ..., :D].double()
        assert torch.isposinf(x[:, 11, :, 3]).all(), b
        x[:, 11, :, 3] = ref[:, 11, :, 3]
        assert ((x - ref).abs() <= tol).all(), b


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("which", ["k", "v"])
def test_values_that_are_not_finite(gpu, value, which):
    """Rows that see a key that is not finite follow the formula; every other
    row, and whatever lies in the buffers past the stored rows, is untouched
    by it."""
    from dropkv_amd import ops
    B, Hq, Hkv, D, T, C, n = 2, 8, 2, 64, 40, 128, 50
    q, kn, vn, kc, vc = case(B, Hq, Hkv, D, T, C, torch.bfloat16, 21)
    kc[:, :, n:] = math.nan
    vc[:, :, n:] = math.inf
    m = make_tree(B, T, 4)[1]
    m[:, :, 7] = False
    m[:, 7, 7] = True
    m[:, :, 35] = False            # seen by nobody
    ref, tol = reference(q, kn, vn, kc, vc, [n] * B, m, 0.125)
    clean = ref.clone()
    unseen = m.clone()
    unseen[:, 7, 7] = False
    gone, gone_tol = reference(q, kn, vn, kc, vc, [n] * B, unseen, 0.125)
    x = kn if which == "k" else vn
    x[:, :, 7, 5] = value
    x[:, :, 35] = value
    ref, _ = reference(q, kn, vn, kc, vc, [n] * B, m, 0.125)
    got = ops.tree_attention(q.to(gpu), kn.to(gpu), vn.to(gpu), kc.to(gpu), vc.to(gpu),
                             torch.full((B,), n, dtype=torch.int32, device=gpu), 0.125, mask=m.to(gpu)).cpu().double()
    rest = [t for t in range(T) if t != 7]
    assert ((got[:, rest] - clean[:, rest]).abs() <= tol[:, rest]).all()
    if which == "v":
        cols = [d for d in range(D) if d != 5]
        assert ((got[:, 7][..., cols] - clean[:, 7][..., cols]).abs() <= tol[:, 7][..., cols]).all()
        g5, r5 = got[:, 7, :, 5], ref[:, 7, :, 5]
        assert torch.equal(g5.isnan(), r5.isnan()) and torch.equal(g5[~g5.isnan()], r5[~r5.isnan()])
    else:
        # q . k is +inf, -inf or NaN by the sign of q: +inf and NaN give NaN,
        # and with -inf the key has no weight: the row is that of a token that
        # does not see it, bound included.
        nan = ref[:, 7].isnan().all(-1)
        assert torch.equal(got[:, 7].isnan().all(-1), nan)
        assert ((got[:, 7] - gone[:, 7]).abs() <= gone_tol[:, 7])[~nan].all()


def test_many_small_weights_fp16(gpu):
    """A key far ahead of 20,000 others whose weights are each below fp16's
    smallest number, and together a tenth of the answer."""
    from dropkv_amd import ops
    n, D, T = 20000, 64, 2
    q = torch.zeros(1, 1, T, D, dtype=torch.float16)
    q[..., 0] = 1
    kc = torch.zeros(1, 1, n, D, dtype=torch.float16)
    kc[:, :, 0, 0] = 12.0          # e^12 against 20,000 ones: weights 6e-6 of the maximum
    kc[:, :, 1:, 0] = -0.2
    vc = torch.ones(1, 1, n, D, dtype=torch.float16)
    vc[:, :, 0] = 0
    kn, vn = torch.full((1, 1, T, D), -1.0, dtype=torch.float16), torch.zeros(1, 1, T, D, dtype=torch.float16)
    m = torch.ones(1, T, T, dtype=torch.bool).tril()
    for scale in (1.0, 1.4):       # weights down to 4e-8
        ref, tol = reference(q, kn, vn, kc, vc, [n], m, scale)
        got = ops.tree_attention(q.to(gpu), kn.to(gpu), vn.to(gpu), kc.to(gpu), vc.to(gpu),
                                 torch.tensor([n], dtype=torch.int32, device=gpu), scale)
        assert ((got.cpu().double() - ref).abs() <= tol).all(), scale


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hq,T", [(1, 2, 1), (1, 4, 10), (200, 4, 30), (200, 8, 20)])   # rows of each kernel
@pytest.mark.parametrize("step", [0.01, 0.05, 0.3, -0.05])
def test_rising_logits(gpu, dtype, B, Hq, T, step):
    """Logits that rise (or fall) from key to key, by a little or much per tile:
    the running maximum is behind or far behind."""
    from dropkv_amd import ops
    D, n = 64, 700
    g = torch.Generator().manual_seed(T)
    q = (torch.randn(1, Hq, T, D, generator=g) * 0.2)
    q[..., 0] = 4.0 + torch.rand(1, Hq, T, generator=g)
    kc = torch.randn(1, 1, n, D, generator=g) * 0.2
    kc[..., 0] = torch.arange(n) * (step / 4)
    vc, kn, vn = (torch.randn(1, 1, x, D, generator=g) for x in (n, T, T))
    q, kc, vc, kn, vn = (x.to(dtype) for x in (q, kc, vc, kn, vn))
    m = torch.ones(1, T, T, dtype=torch.bool).tril()
    ref, tol = reference(q, kn, vn, kc, vc, [n], m, 1.0)
    many = [x.to(gpu).repeat(B, 1, 1, 1) for x in (q, kn, vn, kc, vc)]
    got = ops.tree_attention(*many, torch.tensor([n], dtype=torch.int32, device=gpu), 1.0)
    assert (got == got[:1]).all()
    got = got[:1].cpu().double()
    assert ((got - ref).abs() <= tol).all(), float(((got - ref).abs() / tol).max())


def test_counts_out_of_range_stay_in_bounds(gpu):
    """A count past the capacity reads as the capacity, a negative one as 0."""
    from dropkv_amd import ops
    B, Hq, Hkv, D, T, C = 2, 4, 2, 64, 3, 70
    q, kn, vn, kc, vc = (x.to(gpu) for x in case(B, Hq, Hkv, D, T, C, torch.bfloat16, 8))
    run = lambda c: ops.tree_attention(q, kn, vn, kc, vc, torch.tensor(c, dtype=torch.int32, device=gpu), 0.1)
    assert torch.equal(run([C + 1000, -5]), run([C, 0]))


def test_attention_in_a_graph(gpu):
    """Captured once; replayed with other rows stored, other queries and other
    masks; two graphs with workspaces of their own; on a side stream."""
    from dropkv_amd import ops
    B, Hq, Hkv, D, T, C = 2, 14, 2, 64, 12, 900
    q, kn, vn, kc, vc = (x.to(gpu) for x in case(B, Hq, Hkv, D, T, C, torch.bfloat16, 2))
    m = make_tree(B, T, 1)[1].to(gpu)
    n = torch.tensor([700, 5], dtype=torch.int32, device=gpu)
    outs, graphs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.tree_attention(q, kn, vn, kc, vc, n, 0.125, mask=m)
    torch.cuda.synchronize()
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.tree_attention(q, kn, vn, kc, vc, n, 0.125, mask=m))
        graphs.append(gr)
    for step in range(4):
        n.copy_(torch.tensor([700 + 50 * step, 300 * step], dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)).to(q.dtype))
        m.copy_(make_tree(B, T, 50 + step)[1])
        for gr in graphs:
            gr.replay()
        want = ops.tree_attention(q, kn, vn, kc, vc, n, 0.125, mask=m)
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want), step


def test_two_streams(gpu):
    """Calls on two streams at once, with the streams' own workspaces."""
    from dropkv_amd import ops
    cases = [tuple(x.to(gpu) for x in case(1, 16, 2, 64, T, 2000, torch.bfloat16, T)) for T in (2, 40)]
    n = torch.tensor([1900], dtype=torch.int32, device=gpu)
    want = [ops.tree_attention(*c, n, 0.125) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.tree_attention(*cases[i], n, 0.125))
    torch.cuda.synchronize()
    for w, rs in zip(want, got):
        assert all(torch.equal(r, w) for r in rs)


def test_one_token_is_a_decode_step(gpu):
    """T = 1 agrees with the decode step on the same rows to a rounding."""
    from dropkv_amd import ops
    B, Hq, Hkv, D, C, n = 2, 32, 8, 128, 700, 611
    q, kn, vn, kc, vc = (x.to(gpu) for x in case(B, Hq, Hkv, D, 1, C, torch.bfloat16, 6))
    count = torch.tensor([n], dtype=torch.int32, device=gpu)
    got = ops.tree_attention(q, kn, vn, kc, vc, count, D ** -0.5)
    want = torch.empty_like(got)
    ops.decode_attention(q, kn, vn, kc, vc, count, D ** -0.5, want, ops.decode_workspace(B, Hq, Hkv, D, C, gpu))
    # Each is within half a step (relative 2^-9 of the value) of the same number, and their own errors below 1e-4.
    assert ((got.float() - want.float()).abs() <= want.float().abs() * 2.0 ** -8 + 2e-4).all()


# --- accepted rows ------------------------------------------------------------


def walk(tokens, parents, choice):
    path = [0]
    while True:
        kids = [i for i in range(path[-1] + 1, len(tokens))
                if parents[i] == path[-1] and tokens[i] == choice[path[-1]]]
        if not kids:
            return path
        path.append(kids[0])


@pytest.mark.parametrize("N,B,H,D,T,C,dtype", [
    (1, 1, 2, 64, 8, 40, torch.bfloat16),
    (3, 2, 8, 128, 64, 100, torch.float16),
    (24, 1, 2, 64, 1, 9, torch.bfloat16),
    (2, 3, 3, 20, 256, 300, torch.float32),    # rows of 80 bytes
    (2, 2, 1, 7, 100, 120, torch.bfloat16),    # rows of 14 bytes
])
@pytest.mark.parametrize("layers", [True, False])
def test_commit(gpu, N, B, H, D, T, C, dtype, layers):
    from dropkv_amd import ops
    if not layers:
        N = 1
    g = torch.Generator().manual_seed(T + N)
    parents = make_tree(B, T, T)[0]
    tokens = torch.randint(0, 3, (B, T), generator=g)      # few tokens: siblings with the same one
    choice = torch.randint(0, 3, (B, T), generator=g)
    if T > 4:
        parents[0, 3], parents[-1, 4] = -1, 200000000      # nodes out of the tree
    kn, vn = (torch.randn(N, B, T, H, D, generator=g).to(dtype).transpose(2, 3) for _ in range(2))
    kc, vc = (torch.randn(N, B, H, C, D, generator=g).to(dtype) for _ in range(2))
    n_rows = torch.randint(0, 8, (N, B), generator=g).to(torch.int32)
    want_k, want_v = kc.clone(), vc.clone()
    paths = [walk(tokens[b].tolist(), parents[b].tolist(), choice[b].tolist()) for b in range(B)]
    for l in range(N):
        for b in range(B):
            for i, node in enumerate(paths[b]):
                want_k[l, b, :, n_rows[l, b] + i] = kn[l, b, :, node]
                want_v[l, b, :, n_rows[l, b] + i] = vn[l, b, :, node]
    args = [x.to(gpu) for x in (tokens, parents, choice)]
    # (.to() would make the rows contiguous: keep them as projections.)
    kd, vd = (x.transpose(2, 3).to(gpu).transpose(2, 3) for x in (kn, vn))
    kcd, vcd, nd = kc.to(gpu), vc.to(gpu), n_rows.to(gpu)
    if layers:
        path, acc = ops.tree_commit(*args, kd, vd, kcd, vcd, nd)
    else:
        path, acc = ops.tree_commit(*args, kd[0], vd[0], kcd[0], vcd[0], nd[0])
    assert acc.tolist() == [len(p) for p in paths]
    assert path.tolist() == [p + [-1] * (T - len(p)) for p in paths]
    assert torch.equal(kcd.cpu(), want_k) and torch.equal(vcd.cpu(), want_v)
    assert torch.equal(nd.cpu(), n_rows)


def test_commit_chain_and_capacity(gpu):
    """A chain that stands whole, one tree for all sequences, one count; rows
    past the capacity and of a negative count are left out."""
    from dropkv_amd import ops
    B, H, D, T, C = 3, 2, 64, 256, 300
    tokens = torch.arange(T).expand(B, T).contiguous()
    choice = tokens + 1
    parents = torch.arange(-1, T - 1, dtype=torch.int32)
    kn, vn = torch.randn(B, H, T, D).bfloat16(), torch.randn(B, H, T, D).bfloat16()
    for n in (44, 45, 299, 300, 400, -1):
        kc, vc = torch.zeros(B, H, C, D).bfloat16().to(gpu), torch.zeros(B, H, C, D).bfloat16().to(gpu)
        path, acc = ops.tree_commit(tokens.to(gpu), parents.to(gpu), choice.to(gpu), kn.to(gpu), vn.to(gpu), kc, vc,
                                    torch.tensor([n], dtype=torch.int32, device=gpu))
        assert acc.tolist() == [T] * B and torch.equal(path.cpu(), torch.arange(T, dtype=torch.int32).expand(B, T))
        fit = max(0, min(T, C - n)) if n >= 0 else 0
        want = torch.zeros(B, H, C, D).bfloat16()
        if fit:
            want[:, :, n:n + fit] = kn[:, :, :fit]
        assert torch.equal(kc.cpu(), want)


def test_nothing_drafted_and_no_capacity(gpu):
    """T = 0 and B = 0 give empty tensors; buffers without a row leave the
    drafted tokens to one another; the walk needs a root and a layer."""
    from dropkv_amd import ops
    q, kn, vn, kc, vc = (x.to(gpu) for x in case(2, 4, 2, 64, 5, 70, torch.bfloat16, 8))
    n = torch.zeros(2, dtype=torch.int32, device=gpu)
    assert ops.tree_attention(q[:, :, :0], kn[:, :, :0], vn[:, :, :0], kc, vc, n, 0.1).shape == (2, 0, 4, 64)
    assert ops.tree_attention(q[:0], kn[:0], vn[:0], kc[:0], vc[:0], n[:1], 0.1).shape == (0, 5, 4, 64)
    got = ops.tree_attention(q, kn, vn, kc[:, :, :0].contiguous(), vc[:, :, :0].contiguous(), n, 0.1)
    assert torch.equal(got, ops.tree_attention(q, kn, vn, kc, vc, n, 0.1))
    tok = torch.zeros(2, 5, dtype=torch.int64, device=gpu)
    par = torch.zeros(5, dtype=torch.int32, device=gpu)
    path, acc = ops.tree_commit(tok[:0], par, tok[:0], kn[:0], vn[:0], kc[:0], vc[:0], n[:0])
    assert path.shape == (0, 5) and acc.shape == (0,)
    with pytest.raises(RuntimeError):
        ops.tree_commit(tok[:, :0], par[:0], tok[:, :0], kn[:, :, :0], vn[:, :, :0], kc, vc, n)
    with pytest.raises(RuntimeError):
        ops.tree_commit(tok, par, tok, kn[None][:0], vn[None][:0], kc[None][:0], vc[None][:0], n[None][:0])


def test_refusals(gpu):
    from dropkv_amd import ops
    B, Hq, Hkv, D, T, C = 2, 4, 2, 64, 3, 70
    q, kn, vn, kc, vc = (x.to(gpu) for x in case(B, Hq, Hkv, D, T, C, torch.bfloat16, 8))
    n = torch.zeros(B, dtype=torch.int32, device=gpu)
    good = dict(q=q, k_new=kn, v_new=vn, k_cache=kc, v_cache=vc, n_rows=n, scale=0.1)
    ops.tree_attention(**good)
    bad = [dict(q=q.float()), dict(k_new=kn.half()), dict(k_new=kn[:, :, :2]), dict(v_new=vn[:1]),
           dict(k_cache=kc[:, :, ::2]), dict(v_cache=vc[:, :1].contiguous()), dict(n_rows=n.long()),
           dict(n_rows=torch.zeros(3, dtype=torch.int32, device=gpu)), dict(mask=torch.ones(T, T, device=gpu)),
           dict(mask=torch.ones(T, T + 1, dtype=torch.bool, device=gpu)), dict(n_rows=n.cpu()),
           dict(workspace=torch.empty(16, dtype=torch.uint8, device=gpu)),
           dict(out=torch.empty(B, Hq, T, D, dtype=q.dtype, device=gpu)),
           dict(q=q.clone().requires_grad_())]
    for change in bad:
        with pytest.raises(RuntimeError):
            ops.tree_attention(**{**good, **change})
    tok = torch.zeros(B, T, dtype=torch.int64, device=gpu)
    par = torch.zeros(T, dtype=torch.int32, device=gpu)
    ok = dict(tokens=tok, parents=par, choice=tok, k_new=kn, v_new=vn, k_cache=kc, v_cache=vc, n_rows=n)
    for change in [dict(tokens=tok.int()), dict(parents=par.long()), dict(choice=tok[:1]), dict(k_new=kn[:, :, :2]),
                   dict(k_cache=kc.transpose(1, 2)), dict(n_rows=n.long()), dict(v_cache=vc.half()),
                   dict(n_rows=torch.zeros(1, B, dtype=torch.int32, device=gpu))]:
        with pytest.raises(RuntimeError):
            ops.tree_commit(**{**ok, **change})


def test_shared_workspace(gpu):
    """Calls that bring no workspace share the stream's with the layer-calls of
    the eviction, whose counters at its start every call leaves zero."""
    from dropkv_amd import ops
    ops.release_workspaces()
    g = torch.Generator().manual_seed(0)
    Q, K, V = (torch.randn(1, h, 4096, 64, generator=g).bfloat16().to(gpu) for h in (14, 2, 2))
    x = torch.randn(3, 50000, generator=g).to(gpu)
    q, kn, vn, kc, vc = (t.to(gpu) for t in case(1, 14, 2, 64, 8, 700, torch.bfloat16, 1))
    n = torch.tensor([600], dtype=torch.int32, device=gpu)
    calls = [lambda: ops.evict(Q, K, V, 8, 11, 400), lambda: (ops.tree_attention(q, kn, vn, kc, vc, n, 0.1),),
             lambda: ops.token_logprobs(x, top=9)[1:]]
    first = [tuple(t.clone() for t in c()) for c in calls]
    for _ in range(3):
        for c, want in zip(calls, first):
            for a, b in zip(c(), want):
                assert torch.equal(a, b)
            for ws in ops._shared_ws.values():
                assert not ws[:4096].any()
