"""The operators of decoding on a compressed cache held in 8 bits, as they are
timed: rows quantised as they are written, read back, attention over them, and
the verification of drafted tokens by sampling.

The cache holds blocks of 64 rows per KV head, each with one scale for K and one
for V (the block's largest magnitude over 127 for int8, over 448 for e4m3); the
rows of a block that is not full are kept in 16 bits.

A case is a dict of plain values; ``op`` names the operator:

* ``append``  ``ops.quant_append``: L rows (where ``path`` is set: the accepted
              ones of L drafted tokens) behind ``n - b`` stored rows of sequence
              b, in N layers at once; what was written is read back;
* ``read``    ``ops.quant_read``: the stored rows, in 16 bits;
* ``attend``  ``ops.quant_attention``: T tokens a sequence attend to a cache of
              ``n`` rows (``n - b * spread`` for sequence b) and to one another;
* ``verify``  ``ops.verify_drafts``: which tokens of a drafted chain stand, and
              the token after them, from given random numbers.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_STORES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_TOPS = {"int8": 127.0, "fp8": 448.0}
_BLOCK = 64


def listed():
    return [
        # The smallest call: the accepted ones of eight drafted tokens into every
        # layer of a Qwen2-0.5B cache after a 16K prompt.  Latency is all of it.
        dict(name="append_qwen_8", op="append", N=24, B=1, Hkv=2, D=64, n=1658, L=8, path=True, dtype="bf16",
             store="int8"),
        # The evicted rows of a Llama-3.1-8B layer's batch, after the prefill.
        dict(name="append_llama_3276", op="append", N=1, B=4, Hkv=8, D=128, n=0, L=3276, path=False, dtype="bf16",
             store="fp8"),
        # A long cache of a batch, written whole.
        dict(name="append_long", op="append", N=1, B=4, Hkv=8, D=128, n=0, L=26214, path=False, dtype="fp16",
             store="int8"),
        # A Qwen2-0.5B layer read back: latency.
        dict(name="read_qwen_1638", op="read", B=1, Hkv=2, D=64, n=1638, spread=0, dtype="bf16", store="int8"),
        # Sequences of their own lengths read back.
        dict(name="read_batch_8003", op="read", B=8, Hkv=8, D=128, n=8003, spread=1009, dtype="bf16", store="fp8"),
        # One token over the compressed cache of a Qwen2-0.5B layer: latency.
        dict(name="attend_qwen_1", op="attend", B=1, Hq=14, Hkv=2, D=64, T=1, n=1638, spread=0, room=282, dtype="bf16",
             store="int8", shape="chain"),
        # One token a sequence of a batch, sequences of their own lengths.
        dict(name="attend_batch_1", op="attend", B=8, Hq=32, Hkv=8, D=128, T=1, n=26214, spread=1009, room=509,
             dtype="fp16", store="int8", shape="chain"),
        # A Llama-3.1-8B layer after a 32K prompt, a tree of 16 tokens.
        dict(name="attend_llama_16", op="attend", B=1, Hq=32, Hkv=8, D=128, T=16, n=3276, spread=0, room=116,
             dtype="bf16", store="fp8", shape="tree"),
        # The largest: four long caches, eight query heads per KV head, wide trees.
        dict(name="attend_gqa8_64", op="attend", B=4, Hq=64, Hkv=8, D=128, T=64, n=26214, spread=3, room=310,
             dtype="bf16", store="int8", shape="tree"),
        # A chain of drafts from a lookup (no probabilities of their own): latency.
        dict(name="verify_lookup_8", op="verify", B=1, T=8, V=151936, dtype="bf16", draft=False, temperature=0.8),
        # A draft model's chains for a batch.
        dict(name="verify_batch_9", op="verify", B=8, T=9, V=151936, dtype="bf16", draft=True, temperature=1.0),
        # Many short chains over an odd vocabulary, logits in float32.
        dict(name="verify_many_6", op="verify", B=64, T=6, V=32003, dtype="fp32", draft=True, temperature=0.7),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi], odd as often as even."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = ((8, 2, 64), (14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 128), (16, 8, 64), (64, 8, 128), (16, 16, 64))


def draw(rng):
    op = rng.choice(("append", "append", "read", "attend", "attend", "attend", "verify", "verify"))
    Hq, Hkv, D = rng.choice(_HEADS)
    dtype, store = rng.choice(("bf16", "bf16", "fp16")), rng.choice(("int8", "fp8"))
    if op == "append":
        if rng.random() < 0.5:  # tokens behind stored rows
            N, B = rng.choice((1, 16, 24, 32)), rng.choice((1, 2, 4, 8))
            n, L = _log(rng, 8, 4000), _log(rng, 1, 64)
            while N * B * Hkv * (n + L) * D > 1 << 27:
                n = (n + 8) // 2
            return dict(op=op, N=N, B=B, Hkv=Hkv, D=D, n=n, L=L, path=rng.random() < 0.7, dtype=dtype, store=store)
        B, L = rng.choice((1, 2, 4, 8)), _log(rng, 100, 50000)
        while B * Hkv * L * D > 4 * 8 * 26214 * 128:
            L //= 2
        return dict(op=op, N=1, B=B, Hkv=Hkv, D=D, n=0, L=L, path=False, dtype=dtype, store=store)
    if op == "read":
        B, n = rng.choice((1, 2, 4, 8)), _log(rng, 30, 40000)
        while B * Hkv * n * D > 1 << 26:
            n //= 2
        return dict(op=op, B=B, Hkv=Hkv, D=D, n=n, spread=rng.choice((0, 1, n // 16)), dtype=dtype, store=store)
    if op == "attend":
        B, n = rng.choice((1, 1, 2, 4, 8)), _log(rng, 1, 60000)
        T = rng.choice((1, 1, _log(rng, 2, 100)))
        while B * Hkv * n * D * 4 > 1 << 30 or B * Hq * T * n * D > 1 << 34:
            n //= 2
        return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, D=D, T=T, n=n, spread=rng.choice((0, 1, n // 16)),
                    room=T + rng.randrange(0, 500), dtype=dtype, store=store, shape=rng.choice(("tree", "tree", "chain")))
    B, T, V = _log(rng, 1, 64), _log(rng, 1, 17), rng.choice((151936, 32000, _log(rng, 500, 200000)))
    while B * T * V > 64 * 6 * 32003:
        B, T = (B + 1) // 2, max(1, T - 1)
    return dict(op=op, B=B, T=T, V=V, dtype=rng.choice((dtype, dtype, "fp32")), draft=rng.random() < 0.6,
                temperature=rng.choice((0.6, 0.8, 1.0, 1.0, 1.3)))


def _lens(c):
    """Rows stored for each sequence."""
    return [max(0, c["n"] - b * c.get("spread", 1)) for b in range(c["B"])]


def _rooms(c):
    """Rows of the cache's buffers (whole blocks)."""
    return (c["n"] + c.get("room", c.get("L", 0)) + 2 * _BLOCK) // _BLOCK * _BLOCK


def _window(c):
    """Of an ``append`` case: the first row and the number of rows that it may have touched."""
    first = _lens(c)[-1] // _BLOCK * _BLOCK
    return first, c["n"] + c["L"] - first


def _tree_mask(c, g):
    """Ancestors [B, T, T] (host) of random trees (a node's parent among the eight before it)."""
    B, T = c["B"], c["T"]
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    mask[:, 0, 0] = True
    for i in range(1, T):
        parent = torch.randint(max(0, i - 8), i, (B,), generator=g)
        mask[:, i] = mask[torch.arange(B), parent]
        mask[:, i, i] = True
    return mask


def prepare(c, seed):
    dev = torch.device("cuda:0")
    host = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device=dev).manual_seed(seed + 1)
    dt = _DTYPES[c["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gpu, device=dev) * scale).to(dt)

    def keys(*shape):
        """Rows of keys: each channel of each head has a size of its own."""
        size = torch.exp(0.5 * torch.randn(*shape[:-2], 1, shape[-1], generator=gpu, device=dev))
        return (torch.randn(*shape, generator=gpu, device=dev) * size).to(dt)

    st = dict(case=c)
    if c["op"] == "verify":
        B, T, V = c["B"], c["T"], c["V"]
        # A few likely tokens over a broad floor; the drafts' logits are those, with errors.
        x = torch.randn(B, T, V, generator=gpu, device=dev) * 2
        hot = torch.randint(0, V, (B, T, 12), generator=gpu, device=dev)
        x.scatter_add_(2, hot, torch.rand(B, T, 12, generator=gpu, device=dev) * 14)
        st["logits"] = x.to(dt)
        near = x[:, :-1] + 0.4 * torch.randn(B, T - 1, V, generator=gpu, device=dev)
        del x
        st["draft_logits"] = near.to(dt) if c["draft"] else None
        tokens = torch.randint(0, V, (B, T), generator=gpu, device=dev)
        if T > 1:
            weights = torch.softmax(near.to(dt).float() / c["temperature"], dim=-1)
            tokens[:, 1:] = torch.multinomial(weights.view(-1, V), 1, generator=gpu).view(B, T - 1)
        st["tokens"] = tokens
        st["uniforms"] = torch.rand(B, T, generator=gpu, device=dev)
        return st

    N, B, Hkv, D = c.get("N", 1), c["B"], c["Hkv"], c["D"]
    rows, C = max(1, c["n"]), _rooms(c)
    st["n_rows"] = torch.tensor(_lens(c), dtype=torch.int32, device=dev)
    if c["op"] == "append":
        st["n_rows"] = st["n_rows"].repeat(N, 1)
    lead = (N, B) if c["op"] == "append" else (B,)
    st.update(_stored(c, keys(*lead, Hkv, rows, D), normal(*lead, Hkv, rows, D), st["n_rows"], C))
    if c["op"] == "append":
        L = c["L"]
        st["k_new"], st["v_new"] = keys(*lead, Hkv, L, D), normal(*lead, Hkv, L, D)
        st["path"] = st["counts"] = None
        count = torch.full((B,), L, dtype=torch.int32)
        if c["path"]:
            count = torch.randint(1, L + 1, (B,), generator=host).to(torch.int32)
            path = torch.full((B, L), -1, dtype=torch.int32)
            for b, k in enumerate(count.tolist()):
                path[b, :k] = torch.randperm(L, generator=host)[:k].sort().values
            st["path"], st["counts"] = path.to(dev), count.to(dev)
        st["n_after"] = st["n_rows"] + count.to(dev)
    elif c["op"] == "attend":
        Hq, T = c["Hq"], c["T"]
        st["q"] = normal(B, Hq, T, D)
        st["k_new"], st["v_new"] = keys(B, Hkv, T, D), normal(B, Hkv, T, D)
        st["mask"] = _tree_mask(c, host).to(dev) if c["shape"] == "tree" else None
        if own:
            from dropkv_amd import ops
            st["ws"] = ops.quant_workspace(B, Hq, Hkv, D, T, C, dev)
            st["out"] = torch.empty(B, T, Hq, D, dtype=dt, device=dev)
    return st


def _stored(c, k, v, n_rows, C):
    """The cache's state: the framework's own, or the plain one."""
    *lead, H, rows, D = k.shape
    if own:
        from dropkv_amd import ops
        cache = ops.quant_cache(lead[-1], H, C, D, dtype=k.dtype, store=_STORES[c["store"]],
                                layers=lead[0] if len(lead) == 2 else None, device=k.device)
        ops.quant_append(cache, k, v, torch.zeros_like(n_rows), counts=n_rows.view(-1, lead[-1])[0].contiguous())
        return dict(cache=cache)
    # Plain: [.., H, blocks, 64, D] in 8 bits, a scale a block, and the rows of the last two blocks in 16 bits
    # (row r at r % 128).
    st = {}
    n = n_rows[..., None, None, None].long()
    for name, x in (("k", k), ("v", v)):
        x = torch.cat([x, x.new_zeros(*lead, H, C - rows, D)], dim=-2) if rows < C else x
        r = torch.arange(C, device=x.device)[:, None]
        whole = torch.where(r < n // _BLOCK * _BLOCK, x, torch.zeros_like(x))
        st[name + "8"], st[name + "s"] = _quantise(whole.view(*lead, H, C // _BLOCK, _BLOCK, D), c["store"])
        i = torch.arange(2 * _BLOCK, device=x.device)[:, None]
        first = (n // _BLOCK) * _BLOCK
        row = (first + (i - first) % (2 * _BLOCK)).clamp(max=C - 1).expand(*lead, H, 2 * _BLOCK, D)
        st[name + "t"] = x.gather(-2, row)
    return st


def run(st):
    op = st["case"]["op"]
    if op == "append":
        return _append_own(st) if own else _append_plain(st)
    if op == "read":
        return _read_own(st) if own else _read_plain(st)
    if op == "attend":
        return _attend_own(st) if own else _attend_plain(st)
    return _verify_own(st) if own else _verify_plain(st)


# --- the framework's calls ---------------------------------------------------

def _append_own(st):
    from dropkv_amd import ops
    cache = st["cache"]
    ops.quant_append(cache, st["k_new"], st["v_new"], st["n_rows"], path=st["path"], counts=st["counts"])
    first, rows = _window(st["case"])
    k, v = ops.quant_read(cache, st["n_after"], rows, first)
    return k, v, cache.k_scale, cache.v_scale


def _read_own(st):
    from dropkv_amd import ops
    return ops.quant_read(st["cache"], st["n_rows"], max(1, st["case"]["n"]))


def _attend_own(st):
    from dropkv_amd import ops
    return ops.quant_attention(st["q"], st["k_new"], st["v_new"], st["cache"], st["n_rows"], st["case"]["D"] ** -0.5,
                               st["out"], st["ws"], mask=st["mask"])


def _verify_own(st):
    from dropkv_amd import ops
    return tuple(ops.verify_drafts(st["logits"], st["tokens"], st["uniforms"], draft_logits=st["draft_logits"],
                                   temperature=st["case"]["temperature"]))


# --- plain forms ---------------------------------------------------------------

def _quantise(x, store):
    """Blocks [.., 64, D] in 8 bits and their scales.  (In 64 bits: a value may lie on the border of two steps.)"""
    top = _TOPS[store]
    x = x.double()
    a = x.abs().amax(dim=(-2, -1))
    q = x * top / torch.where(a > 0, a, torch.ones_like(a))[..., None, None]
    q = torch.round(q).to(torch.int8) if store == "int8" else q.float().to(torch.float8_e4m3fn)
    return q, (a / top).float()


def _rows_plain(st, n, L, first):
    """Rows first .. first + L - 1 of K and V: from full blocks, from the 16-bit rows, and zeros behind the last."""
    outs = []
    dt = _DTYPES[st["case"]["dtype"]]
    for name in ("k", "v"):
        q, s, t = st[name + "8"], st[name + "s"], st[name + "t"]
        D = q.shape[-1]
        b0, b1 = first // _BLOCK, (first + L + _BLOCK - 1) // _BLOCK
        x = (q[..., b0:b1, :, :].float() * s[..., b0:b1, None, None]).to(dt).flatten(-3, -2)
        x = x[..., first - b0 * _BLOCK:first - b0 * _BLOCK + L, :]
        r = torch.arange(first, first + L, device=q.device)[:, None]
        nn = n[..., None, None, None].long()
        x = torch.where(r < nn // _BLOCK * _BLOCK, x, t.gather(-2, (r % (2 * _BLOCK)).expand(*t.shape[:-2], L, D)))
        outs.append(torch.where(r < nn, x, torch.zeros_like(x)))
    return outs


def _append_plain(st):
    c = st["case"]
    L, n = c["L"], st["n_rows"].long()
    N, B = n.shape
    dev = n.device
    count = torch.full((B,), L, device=dev) if st["counts"] is None else st["counts"].long()
    path = torch.arange(L, device=dev).expand(B, L) if st["path"] is None else st["path"].long().clamp(min=0)
    # The rows of the blocks that are touched, from the first one's on.
    blocks = (_BLOCK - 1 + L) // _BLOCK + 1
    i = torch.arange(blocks * _BLOCK, device=dev)
    base = n // _BLOCK * _BLOCK
    r = base[..., None] + i                                       # [N, B, rows]
    old, new = r < n[..., None], r < (n + count)[..., None]
    at = path.expand(N, B, L).gather(2, (r - n[..., None]).clamp(0, L - 1))
    end = n + count
    for name, x in (("k", st["k_new"]), ("v", st["v_new"])):
        q, s, t = st[name + "8"], st[name + "s"], st[name + "t"]
        H, D = x.shape[2], x.shape[-1]
        wide = (N, B, H, blocks * _BLOCK, D)
        fresh = x.gather(3, at[:, :, None, :, None].expand(wide))
        kept = t.gather(3, (r % (2 * _BLOCK))[:, :, None, :, None].expand(wide))
        rows = torch.where(old[:, :, None, :, None], kept, torch.where(new[:, :, None, :, None], fresh,
                                                                       torch.zeros_like(fresh)))
        qb, sb = _quantise(rows.view(N, B, H, blocks, _BLOCK, D), c["store"])
        j = (base // _BLOCK)[..., None] + torch.arange(blocks, device=dev)
        full = (j + 1) * _BLOCK <= end[..., None]
        to = j[:, :, None, :].expand(N, B, H, blocks)
        # (Blocks that are not full keep what they held.)
        have = q.view(torch.int8)
        to8 = to[..., None, None].expand(N, B, H, blocks, _BLOCK, D)
        have.scatter_(3, to8, torch.where(full[:, :, None, :, None, None], qb.view(torch.int8), have.gather(3, to8)))
        s.scatter_(3, to, torch.where(full[:, :, None, :], sb, s.gather(3, to)))
        # The rows of the last block, if it is not full.
        k = torch.arange(_BLOCK, device=dev)
        last = end // _BLOCK * _BLOCK
        place = (last[..., None] - base[..., None] + k).clamp(max=blocks * _BLOCK - 1)
        slot = ((last[..., None] + k) % (2 * _BLOCK))[:, :, None, :, None].expand(N, B, H, _BLOCK, D)
        mine = (last[..., None] + k < end[..., None])[:, :, None, :, None]
        t.scatter_(3, slot, torch.where(mine, rows.gather(3, place[:, :, None, :, None].expand(N, B, H, _BLOCK, D)),
                                        t.gather(3, slot)))
    first, rows = _window(c)
    k, v = _rows_plain(st, st["n_after"], rows, first)
    return k, v, st["ks"], st["vs"]


def _read_plain(st):
    return tuple(_rows_plain(st, st["n_rows"], max(1, st["case"]["n"]), 0))


def _attend_plain(st):
    c = st["case"]
    B, Hq, Hkv, D, T = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"]
    g, dev, n = Hq // Hkv, st["q"].device, st["n_rows"].long()
    C = max(1, c["n"])
    r = torch.arange(C, device=dev)[:, None]
    whole = r < (n // _BLOCK * _BLOCK)[:, None, None, None]
    kv = []
    for name in ("k", "v"):
        q8, s, t = st[name + "8"], st[name + "s"], st[name + "t"]
        x = (q8.float() * s[..., None, None]).flatten(2, 3)[:, :, :C]
        x = torch.where(whole, x, t.float().gather(2, (r % (2 * _BLOCK)).expand(B, Hkv, C, D)))
        kv.append(torch.cat([x, st[name + "_new"].float()], dim=2))
    k, v = kv
    q = st["q"].float().reshape(B, Hkv, g * T, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * D ** -0.5
    seen = torch.arange(C, device=dev) < n[:, None]
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


def _verify_plain(st):
    """In 64 bits: a random number may lie next to the border of two tokens."""
    c = st["case"]
    x, tokens, u, draft = st["logits"].double() / c["temperature"], st["tokens"], st["uniforms"].double(), st["draft_logits"]
    B, T, V = x.shape
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    p = p / total
    stands = torch.zeros(B, T, dtype=torch.bool, device=x.device)
    if T > 1:
        fed = tokens[:, 1:].clamp(min=0)[..., None]
        px = p[:, :-1].gather(2, fed)[..., 0]
        if draft is None:
            q = torch.zeros_like(p[:, :-1]).scatter_(2, fed, 1.0)
        else:
            y = draft.double() / c["temperature"]
            q = torch.exp(y - y.amax(-1, keepdim=True))
            q = q / q.sum(-1, keepdim=True)
        ok = (tokens[:, 1:] >= 0) & (u[:, 1:] * q.gather(2, fed)[..., 0] < px)
        stands[:, :-1] = ok.to(torch.int32).cumprod(1).bool()
    last = stands.sum(1)                                          # the node whose distribution is sampled
    rows = torch.arange(B, device=x.device)
    w = p[rows, last]
    if T > 1:
        drafted = (last < T - 1) & (tokens[rows, (last + 1).clamp(max=T - 1)] >= 0)
        rest = (w - q[rows, last.clamp(max=T - 2)]).clamp(min=0)
        w = torch.where((drafted & (rest.sum(-1) > 0))[:, None], rest, w)
    upto = torch.cumsum(w, dim=-1)
    token = (upto <= u[:, :1] * upto[:, -1:]).sum(-1).clamp(max=V - 1)
    nodes = torch.arange(T, device=x.device)
    choice = torch.cat([tokens[:, 1:], tokens[:, :1]], dim=1)
    choice = torch.where(nodes == last[:, None], token[:, None], torch.where(nodes < last[:, None], choice, -1))
    lp = (x.gather(2, choice.clamp(min=0)[..., None]) - lse)[..., 0]
    return choice, (last + 1).to(torch.int32), torch.where(choice >= 0, lp, 0.0).float()


# --- what a pass cannot do without -------------------------------------------------

def work(c):
    e = _BYTES[c["dtype"]]
    if c["op"] == "append":
        # (Half of a path's nodes, about.)
        rows = c["N"] * c["B"] * c["Hkv"] * (max(1, c["L"] // 2) if c["path"] else c["L"]) * c["D"]
        return dict(bytes=2 * rows * (e + 1 + e), flops=4 * rows)
    if c["op"] == "read":
        held = c["Hkv"] * sum(_lens(c)) * c["D"]
        return dict(bytes=2 * held + 2 * c["B"] * c["Hkv"] * max(1, c["n"]) * c["D"] * e, flops=2 * held)
    if c["op"] == "attend":
        B, Hq, Hkv, D, T = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"]
        blocks = sum(n // _BLOCK for n in _lens(c))
        near = sum(n % _BLOCK for n in _lens(c)) + B * T
        mask = B * T * T if c["shape"] == "tree" else 0
        return dict(bytes=2 * Hkv * (blocks * (_BLOCK * D + 4) + near * D * e) + 2 * B * Hq * T * D * e + mask,
                    flops=4 * Hq * T * (blocks * _BLOCK + near) * D)
    rows = c["B"] * (2 * c["T"] - 1 if c["draft"] else c["T"])
    return dict(bytes=rows * c["V"] * e + 24 * c["B"] * c["T"], flops=4 * rows * c["V"])


# --- the definitions in 64 bits ------------------------------------------------------

def exact(c, seed):
    st = _plain_state(c, seed)
    if c["op"] == "append":
        return _append_exact(c, st)
    if c["op"] == "read":
        return _read_exact(c, st)
    if c["op"] == "attend":
        return _attend_exact(c, st)
    return _verify_exact(c, st)


def _plain_state(c, seed):
    """The inputs, with the rows that are stored as they were before they were quantised (``k_rows``, ``v_rows``)."""
    global own, _stored
    mine, stored = own, _stored
    try:
        own, _stored = False, lambda c, k, v, n_rows, C: dict(k_rows=k, v_rows=v)
        return prepare(c, seed)
    finally:
        own, _stored = mine, stored


def _held(x, store):
    """What the rows [.., n, D] of one head are held as, and the scales of the full blocks."""
    n = x.shape[-2]
    whole = n // _BLOCK * _BLOCK
    out = x.double().clone()
    blocks = out[..., :whole, :].unflatten(-2, (whole // _BLOCK, _BLOCK)) if whole else None
    if blocks is None:
        return out, out.new_zeros(*x.shape[:-2], 0)
    scale = blocks.abs().amax((-1, -2)) / _TOPS[store]
    y = blocks / torch.where(scale > 0, scale, 1.0)[..., None, None]
    # (The quotient may be half an ulp of 64 bits off a tie: ties are found in units of 2^-30, to which they belong.)
    y = torch.round(y * 2 ** 30) * 2.0 ** -30
    if store == "int8":
        y = torch.round(y)
    else:  # e4m3: four significant bits, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        y = torch.round(y / step) * step
    out[..., :whole, :] = (y * scale[..., None, None]).flatten(-3, -2)
    return out, scale


def _append_exact(c, st):
    N, B, Hkv, D, L = c["N"], c["B"], c["Hkv"], c["D"], c["L"]
    first, rows = _window(c)
    outs = []
    for name in ("k", "v"):
        values = torch.zeros(N, B, Hkv, rows, D, dtype=torch.float64, device=st["k_new"].device)
        scales = torch.zeros(N, B, Hkv, _rooms(c) // _BLOCK, dtype=torch.float64, device=values.device)
        for b, n in enumerate(_lens(c)):
            new = st[name + "_new"][:, b]
            if st["path"] is not None:
                new = new[:, :, st["path"][b, :int(st["counts"][b])].long()]
            x, s = _held(torch.cat([st[name + "_rows"][:, b, :, :n], new], dim=2), c["store"])
            part = x[:, :, first:first + rows]
            values[:, b, :, :part.shape[2]] = part
            scales[:, b, :, :s.shape[-1]] = s
        outs += [values, scales]
    return outs[0], outs[2], outs[1], outs[3]


def _read_exact(c, st):
    outs = []
    for x in (st["k_rows"], st["v_rows"]):
        y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        for b, n in enumerate(_lens(c)):
            y[b, :, :n] = _held(x[b, :, :n], c["store"])[0]
        outs.append(y)
    return tuple(outs)


def _attend_exact(c, st):
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
            k, v = (torch.cat((_held(st[x + "_rows"][b, h, :n], c["store"])[0], st[x + "_new"][b, h].double()))
                    for x in ("k", "v"))
            for hq in range(h * g, (h + 1) * g):
                logits = st["q"][b, hq].double() @ k.t() / math.sqrt(D) + hide
                out[b, :, hq] = (logits - torch.logsumexp(logits, -1, keepdim=True)).exp() @ v
    return out


def _verify_exact(c, st):
    """Walked token by token on the host, a row of probabilities at a time."""
    B, T = c["B"], c["T"]
    choice = torch.full((B, T), -1, dtype=torch.int64)
    accepted = torch.zeros(B, dtype=torch.int32)
    logprob = torch.zeros(B, T, dtype=torch.float64)
    tokens, uniforms = st["tokens"].tolist(), st["uniforms"].tolist()
    for b in range(B):
        node = 0
        while True:
            lp = torch.log_softmax(st["logits"][b, node].double() / c["temperature"], dim=-1)
            weights = lp.exp()
            x = tokens[b][node + 1] if node + 1 < T else -1
            if x >= 0:
                if st["draft_logits"] is not None:
                    drafted = torch.softmax(st["draft_logits"][b, node].double() / c["temperature"], dim=-1)
                else:
                    drafted = torch.zeros_like(weights)
                    drafted[x] = 1.0
                if uniforms[b][node + 1] * float(drafted[x]) < float(weights[x]):
                    choice[b, node], logprob[b, node] = x, lp[x]
                    node += 1
                    continue
                rest = torch.relu(weights - drafted)
                weights = rest if float(rest.sum()) > 0 else weights
            upto = weights.cumsum(0)
            x = int(torch.searchsorted(upto, uniforms[b][0] * upto[-1:], right=True))
            x = min(x, c["V"] - 1)
            choice[b, node], logprob[b, node] = x, lp[x]
            accepted[b] = node + 1
            break
    return choice, accepted, logprob
