"""The operators of a verification step of speculative decoding, as they are
timed: attention of drafted tokens over a compressed cache, the norms and
rotation of queries and keys, log probabilities of the answers, and the
accepted path's rows appended to the caches.

A case is a dict of plain values; ``op`` names the operator:

* ``tree``    ``ops.tree_attention``: T drafted tokens a sequence attend to a
              cache of ``n`` rows (``n - b * spread`` for sequence b) and to
              their ancestors in the tree;
* ``rope``    ``ops.norm_rope``: norms (where ``norm`` is set) and rotation of
              queries and keys, K and V put where the cache keeps them;
* ``logprob`` ``ops.token_logprobs``: log probability of a given token,
              entropy and the ``top`` best alternatives of each row of logits;
* ``commit``  ``ops.tree_commit``: the accepted path of each sequence's tree
              and its K/V rows appended to every layer's cache.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # The smallest call: eight drafted tokens over the compressed cache of
        # a Qwen2-0.5B layer after a 16K prompt.  Latency is all of it.
        dict(name="tree_qwen_8", op="tree", B=1, Hq=14, Hkv=2, D=64, T=8, n=1638, spread=0, room=282, dtype="bf16",
             shape="tree"),
        # A Llama-3.1-8B layer after a 32K prompt, a tree of 16 tokens.
        dict(name="tree_llama_16", op="tree", B=1, Hq=32, Hkv=8, D=128, T=16, n=3276, spread=0, room=116, dtype="bf16",
             shape="tree"),
        # A batch of sequences of their own lengths, an odd number of drafted
        # tokens, float16.
        dict(name="tree_batch_27", op="tree", B=8, Hq=32, Hkv=8, D=128, T=27, n=8003, spread=1009, room=509,
             dtype="fp16", shape="tree"),
        # Longer chains with one query head per KV head.
        dict(name="chain_mha_5", op="tree", B=4, Hq=16, Hkv=16, D=64, T=5, n=6553, spread=1, room=64, dtype="bf16",
             shape="chain"),
        # The largest: four long caches, eight query heads per KV head, wide trees.
        dict(name="tree_gqa8_64", op="tree", B=4, Hq=64, Hkv=8, D=128, T=64, n=26214, spread=3, room=310, dtype="bf16",
             shape="tree"),
        # The drafted tokens of one sequence in one layer: latency.
        dict(name="rope_step_8", op="rope", B=1, Hq=14, Hkv=2, D=64, L=8, dtype="bf16", norm=False, table=False),
        # A batch of prompts of an odd length, with norms for each head and
        # angles from a table.
        dict(name="rope_batch_7001", op="rope", B=4, Hq=32, Hkv=8, D=128, L=7001, dtype="fp16", norm=True, table=True),
        # One decoded token over the vocabulary of Qwen2: latency.
        dict(name="logprob_token", op="logprob", N=1, V=151936, top=5, dtype="bf16"),
        # The nodes of a batch of trees.
        dict(name="logprob_tree", op="logprob", N=216, V=151936, top=1, dtype="bf16"),
        # A prompt scored whole, with alternatives.
        dict(name="logprob_prompt", op="logprob", N=2047, V=151936, top=20, dtype="bf16"),
        # Accepted rows of small and of large trees into every layer's cache.
        dict(name="commit_qwen_8", op="commit", N=24, B=1, Hkv=2, D=64, T=8, n=1638, room=90, dtype="bf16"),
        dict(name="commit_batch_64", op="commit", N=32, B=8, Hkv=8, D=128, T=64, n=201, room=311, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi], odd as often as even."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = ((8, 2, 64), (14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 128), (16, 8, 64), (64, 8, 128), (16, 16, 64))


def draw(rng):
    op = rng.choice(("tree", "tree", "tree", "rope", "logprob", "logprob", "commit"))
    Hq, Hkv, D = rng.choice(_HEADS)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "tree":
        B, T, n = rng.choice((1, 1, 2, 4, 8)), _log(rng, 1, 100), _log(rng, 1, 60000)
        while B * Hkv * n * D * 4 > 1 << 29 or B * Hq * T * n * D > 1 << 34:
            n //= 2
        return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, D=D, T=T, n=n, spread=rng.choice((0, 1, n // 16)),
                    room=T + rng.randrange(0, 500), dtype=dtype, shape=rng.choice(("tree", "tree", "chain")))
    if op == "rope":
        B, L = rng.choice((1, 1, 2, 4)), _log(rng, 1, 9000)
        while B * L * (Hq + 2 * Hkv) * D > 1 << 27:
            L //= 2
        return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, D=D, L=L, dtype=rng.choice((dtype, dtype, "fp32")),
                    norm=rng.random() < 0.5, table=rng.random() < 0.5)
    if op == "logprob":
        N, V = _log(rng, 1, 3000), rng.choice((151936, 32000, _log(rng, 500, 200000)))
        while N * V > 3 << 26:
            N //= 2
        return dict(op=op, N=N, V=V, top=rng.choice((1, 1, 5, 8, 20)), dtype=rng.choice((dtype, dtype, "fp32")))
    N, B = rng.choice((1, 16, 24, 32)), rng.choice((1, 2, 4, 8))
    n, T = _log(rng, 1, 4000), _log(rng, 1, 100)
    while N * B * Hkv * (n + T) * D * 4 > 1 << 29:
        n //= 2
        T = (T + 1) // 2
    return dict(op="commit", N=N, B=B, Hkv=Hkv, D=D, T=T, n=n, room=T + rng.randrange(0, 90), dtype=dtype)


def _lens(c):
    """Rows stored for each sequence of a ``tree`` case."""
    return [max(0, c["n"] - b * c["spread"]) for b in range(c["B"])]


def _trees(c, g):
    """Parents [B, T] of random trees (a node's parent among the eight before
    it, the root at 0) or chains, and their ancestor masks [B, T, T] (host)."""
    B, T = c["B"], c["T"]
    parents = torch.zeros(B, T, dtype=torch.int64)
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    mask[:, 0, 0] = True
    for i in range(1, T):
        if c.get("shape", "tree") == "chain":
            parents[:, i] = i - 1
        else:
            parents[:, i] = torch.randint(max(0, i - 8), i, (B,), generator=g)
        mask[:, i] = mask[torch.arange(B), parents[:, i]]
        mask[:, i, i] = True
    return parents, mask


def _is(c, op):
    return c["op"] == op


def prepare(c, seed):
    dev = torch.device("cuda:0")
    host = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device=dev).manual_seed(seed + 1)
    dt = _DTYPES[c["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gpu, device=dev) * scale).to(dt)

    st = dict(case=c)
    if _is(c, "tree"):
        B, Hq, Hkv, D, T, C = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"], c["n"] + c["room"]
        st.update(q=normal(B, Hq, T, D, scale=1.5), k_new=normal(B, Hkv, T, D), v_new=normal(B, Hkv, T, D),
                  k=normal(B, Hkv, C, D), v=normal(B, Hkv, C, D),
                  n_rows=torch.tensor(_lens(c), dtype=torch.int32, device=dev))
        st["mask"] = _trees(c, host)[1].to(dev) if c["shape"] == "tree" else None
        if own:
            from dropkv_amd import ops
            st["ws"] = ops.tree_workspace(B, Hq, Hkv, D, T, C, dev)
            st["out"] = torch.empty(B, T, Hq, D, dtype=dt, device=dev)
    elif _is(c, "rope"):
        # Projections [B, L, H, D] seen as [B, H, L, D], as a decoder layer has them.
        B, Hq, Hkv, D, L = c["B"], c["Hq"], c["Hkv"], c["D"], c["L"]
        for name, H in (("q", Hq), ("k", Hkv), ("v", Hkv)):
            st[name] = normal(B, L, H, D, scale=2.0).transpose(1, 2)
        inv = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
        rows = 3 * L + 50 if c["table"] else L
        first = 0 if c["table"] else seed % 1000
        ang = torch.arange(first, first + rows, dtype=torch.float64, device=dev)[:, None] * inv
        ang = torch.cat([ang, ang], dim=-1)
        # A table of angles is kept in float32; a step's own rows come in the model's type.
        tt = torch.float32 if c["table"] else dt
        st["cos"], st["sin"] = ang.cos().to(tt), ang.sin().to(tt)
        if c["table"]:
            start = torch.randint(0, 2 * L + 50, (B, 1), generator=host)
            st["positions"] = (start + torch.arange(L)).to(dev)
        else:
            st["cos"], st["sin"], st["positions"] = st["cos"][None], st["sin"][None], None
        st["qw"] = (1 + 0.2 * normal(D).float()).to(dt) if c["norm"] else None
        st["kw"] = (1 + 0.2 * normal(D).float()).to(dt) if c["norm"] else None
    elif _is(c, "logprob"):
        N, V = c["N"], c["V"]
        # A few likely tokens over a broad floor.
        x = torch.randn(N, V, generator=gpu, device=dev) * 2
        hot = torch.randint(0, V, (N, 12), generator=gpu, device=dev)
        x.scatter_add_(1, hot, torch.rand(N, 12, generator=gpu, device=dev) * 14)
        st["logits"] = x.to(dt)
        st["tokens"] = torch.where(torch.rand(N, generator=gpu, device=dev) < 0.7, hot[:, 0],
                                   torch.randint(0, V, (N,), generator=gpu, device=dev))
    else:
        N, B, Hkv, D, T, C = c["N"], c["B"], c["Hkv"], c["D"], c["T"], c["n"] + c["room"]
        parents, _ = _trees(c, host)
        tokens = torch.randint(0, 151936, (B, T), generator=host)
        choice = torch.randint(0, 151936, (B, T), generator=host)
        for i in range(T - 1, 0, -1):  # most nodes settle on one of their children
            hit = torch.rand(B, generator=host) < 0.8
            b = torch.nonzero(hit).flatten()
            choice[b, parents[b, i]] = tokens[b, i]
        st.update(tokens=tokens.to(dev), parents=parents.to(torch.int32).to(dev), choice=choice.to(dev),
                  k_new=normal(N, B, Hkv, T, D), v_new=normal(N, B, Hkv, T, D),
                  k=normal(N, B, Hkv, C, D), v=normal(N, B, Hkv, C, D),
                  n_rows=torch.full((N, B), c["n"], dtype=torch.int32, device=dev)
                  - torch.arange(B, dtype=torch.int32, device=dev).clamp_max(c["n"]))
    return st


def run(st):
    c = st["case"]
    if _is(c, "tree"):
        return _tree_own(st) if own else _tree_plain(st)
    if _is(c, "rope"):
        return _rope_own(st) if own else _rope_plain(st)
    if _is(c, "logprob"):
        return _logprob_own(st) if own else _logprob_plain(st)
    return _commit_own(st) if own else _commit_plain(st)


# --- the framework's calls ---------------------------------------------------

def _tree_own(st):
    from dropkv_amd import ops
    return ops.tree_attention(st["q"], st["k_new"], st["v_new"], st["k"], st["v"], st["n_rows"],
                              st["case"]["D"] ** -0.5, st["out"], st["ws"], mask=st["mask"])


def _rope_own(st):
    from dropkv_amd import ops
    return ops.norm_rope(st["q"], st["k"], st["cos"], st["sin"], positions=st["positions"], q_weight=st["qw"],
                         k_weight=st["kw"], eps=1e-6, v=st["v"])


def _logprob_own(st):
    from dropkv_amd import ops
    return tuple(ops.token_logprobs(st["logits"], st["tokens"], top=st["case"]["top"]))


def _commit_own(st):
    from dropkv_amd import ops
    path, accepted = ops.tree_commit(st["tokens"], st["parents"], st["choice"], st["k_new"], st["v_new"], st["k"],
                                     st["v"], st["n_rows"])
    return path, accepted, st["k"], st["v"]


# --- plain forms ---------------------------------------------------------------

def _tree_plain(st):
    c = st["case"]
    B, Hq, Hkv, D, T, C = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"], st["k"].shape[2]
    g = Hq // Hkv
    dev = st["q"].device
    q = st["q"].float().reshape(B, Hkv, g * T, D)
    k = torch.cat([st["k"], st["k_new"]], dim=2).float()
    v = torch.cat([st["v"], st["v_new"]], dim=2).float()
    s = torch.matmul(q, k.transpose(-1, -2)) * D ** -0.5
    seen = torch.arange(C, device=dev) < st["n_rows"][:, None]
    mask = st["mask"]
    if mask is None:
        mask = torch.ones(T, T, dtype=torch.bool, device=dev).tril().expand(B, T, T)
    seen = torch.cat([seen[:, None].expand(B, T, C), mask], dim=-1)[:, None, None]
    s = s.view(B, Hkv, g, T, C + T).masked_fill(~seen, -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-3e38))
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, Hkv, g * T, C + T), v).view(B, Hkv, g, T, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.reshape(B, Hq, T, D).transpose(1, 2).to(st["q"].dtype).contiguous()


def _rope_plain(st):
    D = st["q"].shape[-1]
    cos, sin = st["cos"], st["sin"]
    if st["positions"] is not None:
        cos, sin = cos[st["positions"]], sin[st["positions"]]
    cos, sin = cos.float()[:, None], sin.float()[:, None]

    def one(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        half = torch.cat([-y[..., D // 2:], y[..., :D // 2]], dim=-1)
        return (y * cos + half * sin).to(x.dtype).contiguous()

    return one(st["q"], st["qw"]), one(st["k"], st["kw"]), st["v"].contiguous()


def _logprob_plain(st):
    x = st["logits"].float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    lse = m + torch.log(s)
    entropy = torch.log(s[:, 0]) - (e * d).sum(-1) / s[:, 0]
    del d, e
    logprob = (x.gather(1, st["tokens"][:, None]) - lse)[:, 0]
    ids = torch.arange(x.shape[1], device=x.device)
    values, best = [], []
    rest = x.clone() if x.data_ptr() == st["logits"].data_ptr() else x
    for _ in range(st["case"]["top"]):
        v = rest.amax(-1, keepdim=True)
        i = torch.where(rest == v, ids, x.shape[1]).amin(-1, keepdim=True)
        values.append(v - lse)
        best.append(i)
        rest.scatter_(1, i, -math.inf)
    return logprob, entropy, torch.cat(values, dim=1), torch.cat(best, dim=1)


def _commit_plain(st):
    tokens, parents, choice = st["tokens"], st["parents"].long(), st["choice"]
    B, T = tokens.shape
    N, _, Hkv, _, D = st["k"].shape
    match = tokens == choice.gather(1, parents)
    on = torch.zeros(B, T, dtype=torch.bool, device=tokens.device)
    on[:, 0] = True
    gone_on = torch.zeros_like(on)
    for i in range(1, T):
        p = parents[:, i:i + 1]
        go = on.gather(1, p) & match[:, i:i + 1] & ~gone_on.gather(1, p)
        on[:, i:i + 1] = go
        gone_on.scatter_(1, p, gone_on.gather(1, p) | go)
    accepted = on.sum(-1)
    nodes = torch.arange(T, device=tokens.device).expand(B, T)
    path = torch.where(on, nodes, T).sort(-1).values
    valid = path < T
    src = torch.where(valid, path, 0)[None, :, None, :, None].expand(N, B, Hkv, T, D)
    dst = (st["n_rows"].long()[:, :, None] + nodes)[:, :, None, :, None].expand(N, B, Hkv, T, D)
    keep = valid[None, :, None, :, None]
    for cache, new in ((st["k"], st["k_new"]), (st["v"], st["v_new"])):
        cache.scatter_(3, dst, torch.where(keep, new.gather(3, src), cache.gather(3, dst)))
    return torch.where(valid, path, -1).to(torch.int32), accepted.to(torch.int32), st["k"], st["v"]


# --- what a pass cannot do without -------------------------------------------------

def work(c):
    e = _BYTES[c["dtype"]]
    if _is(c, "tree"):
        B, Hq, Hkv, D, T = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"]
        rows = sum(_lens(c)) + B * T
        mask = B * T * T if c["shape"] == "tree" else 0
        return dict(bytes=2 * Hkv * rows * D * e + 2 * B * Hq * T * D * e + mask, flops=4 * Hq * T * rows * D)
    if _is(c, "rope"):
        B, L, D, heads = c["B"], c["L"], c["D"], c["Hq"] + 2 * c["Hkv"]
        table = 2 * D * L * (4 * B if c["table"] else e)
        return dict(bytes=2 * B * L * heads * D * e + table,
                    flops=B * L * (c["Hq"] + c["Hkv"]) * D * (7 if c["norm"] else 3))
    if _is(c, "logprob"):
        return dict(bytes=c["N"] * (c["V"] * e + 16 + 12 * c["top"]), flops=6 * c["N"] * c["V"])
    # (A path of three nodes, about what these trees accept, in every layer.)
    return dict(bytes=4 * c["N"] * c["B"] * c["Hkv"] * 3 * c["D"] * e + 24 * c["B"] * c["T"], flops=c["B"] * c["T"])


# --- the definitions in 64 bits ------------------------------------------------------

def exact(c, seed):
    st = prepare(c, seed)
    if _is(c, "tree"):
        return _tree_exact(c, st)
    if _is(c, "rope"):
        return _rope_exact(c, st)
    if _is(c, "logprob"):
        return _logprob_exact(c, st)
    return _commit_exact(c, st)


def _tree_exact(c, st):
    """Sequence by sequence and KV head by KV head, on the rows that are stored."""
    B, Hq, Hkv, D, T = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"]
    g = Hq // Hkv
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=st["q"].device)
    for b, n in enumerate(_lens(c)):
        hide = torch.zeros(T, n + T, dtype=torch.float64, device=out.device)
        if st["mask"] is None:
            hide[:, n:] = torch.triu(torch.full((T, T), -math.inf, dtype=torch.float64, device=out.device), 1)
        else:
            hide[:, n:][~st["mask"][b]] = -math.inf
        for h in range(Hkv):
            k = torch.cat((st["k"][b, h, :n], st["k_new"][b, h])).double()
            v = torch.cat((st["v"][b, h, :n], st["v_new"][b, h])).double()
            for hq in range(h * g, (h + 1) * g):
                logits = st["q"][b, hq].double() @ k.t() / math.sqrt(D) + hide
                weights = (logits - torch.logsumexp(logits, -1, keepdim=True)).exp()
                out[b, :, hq] = weights @ v
    return out


def _rope_exact(c, st):
    """As complex products: pair i is x_i + j x_{i+D/2}, turned by cos + j sin."""
    D = c["D"]
    cos, sin = st["cos"].double(), st["sin"].double()
    if st["positions"] is not None:
        cos, sin = cos[st["positions"]], sin[st["positions"]]
    turn = torch.complex(cos[..., :D // 2], sin[..., :D // 2])[:, None]
    outs = []
    for x, w in ((st["q"], st["qw"]), (st["k"], st["kw"])):
        y = x.double()
        if w is not None:
            y = w.double() * y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + 1e-6)
        z = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * turn
        outs.append(torch.cat((z.real, z.imag), dim=-1))
    return outs[0], outs[1], st["v"].double().contiguous()


def _logprob_exact(c, st):
    N, V, top = c["N"], c["V"], c["top"]
    outs = []
    for x16, t in zip(st["logits"].split(256), st["tokens"].split(256)):
        lp = torch.log_softmax(x16.double(), dim=-1)
        # Value and place as one whole number: larger values first, then lower places.
        bits = x16.float().view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 20) + (V - 1 - torch.arange(V, device=lp.device))
        ids = key.topk(top, dim=-1, sorted=True).indices
        outs.append((lp.gather(1, t[:, None])[:, 0], -(lp.exp() * lp).sum(-1), lp.gather(1, ids), ids))
    return tuple(torch.cat(o) for o in zip(*outs))


def _commit_exact(c, st):
    """Walked on the host."""
    tokens, parents, choice = (st[x].tolist() for x in ("tokens", "parents", "choice"))
    paths = []
    for tok, par, want in zip(tokens, parents, choice):
        path = [0]
        for i in range(1, c["T"]):
            if par[i] == path[-1] and tok[i] == want[path[-1]]:
                path.append(i)
        paths.append(path)
    for layer, counts in enumerate(st["n_rows"].tolist()):
        for b, n in enumerate(counts):
            for cache, new in ((st["k"], st["k_new"]), (st["v"], st["v_new"])):
                cache[layer, b, :, n:n + len(paths[b])] = new[layer, b][:, paths[b]]
    path = torch.tensor([p + [-1] * (c["T"] - len(p)) for p in paths], dtype=torch.int32)
    return path, torch.tensor([len(p) for p in paths], dtype=torch.int32), st["k"].double(), st["v"].double()
