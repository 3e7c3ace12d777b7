"""The operators of a cache in 8 bits together: ``CompressedDecoder(cache_dtype=...)``
step by step, over trees and by sampling, against the decoder in 16 bits on the rows
that the 8 bits stand for."""

import copy

import pytest
import torch

import quant_ref as R

pytestmark = pytest.mark.gpu

TINY = dict(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=3,
            num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=8192)


@pytest.fixture(scope="module")
def tiny(gpu):
    from dropkv_amd.e2e_qwen2 import build_model, make_config
    cfg = make_config(**TINY)
    return cfg, build_model(cfg, gpu, dtype=torch.bfloat16, seed=0)


def prefilled(tiny, gpu, L=1500, batch=1, seed=21):
    from dropkv_amd import hf_cache
    from dropkv_amd.e2e_qwen2 import prefill, random_prompt
    cfg, model = tiny
    cache = hf_cache.DropKVCache(cfg, keep_ratio=0.1)
    return cache, prefill(model, random_prompt(cfg.vocab_size, L, batch=batch, seed=seed, device=gpu), cache)


def held(cache, store):
    """A copy of the cache whose full blocks are what 8 bits hold of them."""
    cache = copy.deepcopy(cache)
    for lay in cache.layers:
        lay.keys, lay.values = (R.held(x, store).to(x.dtype) for x in (lay.keys, lay.values))
    return cache


def pair(tiny, gpu, store, batch=1, tokens=160, **kw):
    """Decoders in 16 and in 8 bits on the same rows, and the first token."""
    from dropkv_amd.decode import CompressedDecoder
    cache, tok = prefilled(tiny, gpu, batch=batch)
    a = CompressedDecoder(tiny[1], held(cache, store), max_new_tokens=tokens, **dict(kw, tree_size=kw.get("tree_size") or 1))
    return a, CompressedDecoder(tiny[1], cache, max_new_tokens=tokens, cache_dtype=store, **kw), tok


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("store", R.STORES)
def test_steps(gpu, tiny, store, use_graph):
    """150 kept rows and up to 42 more, until the block of the last 22 fills up: logits
    as in 16 bits, to the rounding of activations (the decoder's other tests' bound);
    then 64 more, whose rows are what 8 bits hold of those in 16."""
    a, b, tok = pair(tiny, gpu, store, use_graph=use_graph)
    n0 = int(b.n_rows[0, 0])
    assert n0 == 150
    g = torch.Generator().manual_seed(0)
    toks = torch.randint(0, 1000, (110, 1, 1), generator=g).to(gpu)
    for i, t in enumerate([tok, *toks]):
        x, y = a.step(t).clone(), b.step(t).clone()
        if n0 + i < 191:
            torch.testing.assert_close(y.float(), x.float(), rtol=3e-2, atol=3e-2, msg=f"step {i}")
    n = n0 + 111
    assert b.n_rows.tolist() == [[n]] * 3 and torch.equal(a.pos, b.pos)
    # The first layer's rows depend on tokens and positions alone.
    whole = (n0 // 64 * 64)
    for x, y in zip(a.stored(0), b.stored(0)):
        assert x.shape == y.shape == (1, 2, n, 64)
        want = torch.cat([x[:, :, :whole].double(), R.held(x[:, :, whole:], store)], dim=2)
        assert ((y.double() - want).abs() <= (R.HALF[torch.bfloat16] + 2.0 ** -22) * want.abs()).all()


@pytest.mark.parametrize("store", R.STORES)
def test_graph_and_eager_give_the_same_bits(gpu, tiny, store):
    """Steps, trees and sampled chains in turn, over several blocks."""
    from dropkv_amd.decode import CompressedDecoder
    cache, tok = prefilled(tiny, gpu, batch=2)
    decs = [CompressedDecoder(tiny[1], cache, 300, use_graph=u, tree_size=9, cache_dtype=store) for u in (False, True)]
    g = torch.Generator(device=gpu).manual_seed(5)
    for rnd in range(9):
        t = (9, 5, 7)[rnd % 3]
        drafts = torch.randint(0, 1000, (2, t), generator=g, device=gpu)
        drafts[:, :1] = tok
        if rnd % 3 == 0:
            outs = [d.step(tok).clone() for d in decs]
            assert torch.equal(*outs)
            tok = outs[0][:, -1].argmax(-1, keepdim=True)
            continue
        if rnd % 3 == 1:
            parents = [-1, 0, 0, 1, 2]
            args = ()
        else:
            parents = range(-1, t - 1)
            args = (torch.rand(2, t, generator=g, device=gpu) * 0.02, torch.randn(2, t - 1, 1000, generator=g, device=gpu).to(torch.bfloat16), 1.5)
        for d in decs:
            d.set_tree(parents)
        x, y = (d.verify(drafts, *args) for d in decs)
        torch.cuda.synchronize()
        for p, q in zip(x, y):
            assert torch.equal(p[:, :t] if p.dim() > 1 else p, q[:, :t] if q.dim() > 1 else q), rnd
        assert torch.equal(decs[0].n_rows, decs[1].n_rows) and torch.equal(decs[0].pos, decs[1].pos)
        tok = x.tokens.gather(1, x.accepted.long()[:, None] - 1)
    for i in range(3):
        for p, q in zip(decs[0].stored(i), decs[1].stored(i)):
            assert torch.equal(p, q)


@pytest.mark.parametrize("use_graph", [False, True])
def test_chain_of_right_tokens(gpu, tiny, use_graph):
    """Steps of one token, then the same tokens drafted as chains of eight, across the
    border of a block: what stands is what the steps gave, and so are the rows."""
    from dropkv_amd.decode import CompressedDecoder
    cache, tok = prefilled(tiny, gpu)
    a = CompressedDecoder(tiny[1], cache, 100, use_graph=use_graph, tree_size=8, cache_dtype="int8")
    b = CompressedDecoder(tiny[1], cache, 100, use_graph=use_graph, tree_size=8, cache_dtype="int8")
    toks = [tok]
    for _ in range(64):
        toks.append(a.step(toks[-1])[:, -1].argmax(-1, keepdim=True))
    line = torch.cat(toks, dim=1)
    at = 0
    while at < 56:
        v = b.verify(line[:, at:at + 8])
        k = int(v.accepted)
        assert v.path[0].tolist() == list(range(k)) + [-1] * (8 - k)
        best = v.logits[0].argmax(-1).tolist()
        want = 1
        while want < 8 and best[want - 1] == int(line[0, at + want]):
            want += 1
        assert k == want and v.tokens[0, :k].tolist() == best[:k]
        at += k
        if best[k - 1] != int(line[0, at]):
            break  # (two logits as near as their rounding)
    n = int(b.n_rows[0, 0])
    assert n == 150 + at
    for x, y in zip(a.stored(0), b.stored(0)):
        done = n // 64 * 64  # (blocks that both have filled up)
        assert torch.equal(x[:, :, :done], y[:, :, :done])


@pytest.mark.parametrize("cache_dtype", [None, "fp8"])
@pytest.mark.parametrize("use_graph", [False, True])
def test_verify_by_sampling(gpu, tiny, use_graph, cache_dtype):
    """The nodes that stand are those of ``ops.verify_drafts`` on the forward's own
    logits; their rows are appended, and the next forward sees them: its logits are those
    of a decoder that was fed the tokens one by one."""
    from dropkv_amd import ops
    from dropkv_amd.decode import CompressedDecoder
    B, T = 2, 6
    cache, tok = prefilled(tiny, gpu, batch=B)
    d = CompressedDecoder(tiny[1], cache, 200, use_graph=use_graph, tree_size=8, cache_dtype=cache_dtype)
    one = CompressedDecoder(tiny[1], cache, 200, use_graph=False, tree_size=1, cache_dtype=cache_dtype)
    d.set_tree(range(-1, T - 1))
    g = torch.Generator(device=gpu).manual_seed(2)
    lines = [tok]
    for rnd in range(4):
        near = torch.randn(B, T - 1, 1000, generator=g, device=gpu).to(torch.bfloat16)
        drafts = torch.cat([tok, torch.randint(0, 1000, (B, T - 1), generator=g, device=gpu)], dim=1)
        u = torch.rand(B, T, generator=g, device=gpu)
        if rnd < 2:
            u[:, 1:] *= 0.3 ** rnd  # (some stand)
        pos = d.pos.clone()
        v = d.verify(drafts, uniforms=u, draft_logits=near if rnd % 2 else None, temperature=1.3)
        want = ops.verify_drafts(v.logits[:, :T], drafts, u, near if rnd % 2 else None, 1.3)
        assert torch.equal(v.accepted, want.accepted) and torch.equal(v.tokens[:, :T], want.choice)
        assert torch.equal(v.logprobs[:, :T], want.logprobs)
        assert torch.equal(d.pos, pos + v.accepted[:, None].long())
        assert torch.equal(d.n_rows.long(), (150 + d.pos[:, 0] - d.logical).expand(3, B))
        for b in range(B):
            k = int(v.accepted[b])
            assert v.path[b].tolist() == list(range(k)) + [-1] * (8 - k)
        tok = v.tokens.gather(1, v.accepted.long()[:, None] - 1)
        lines.append((v.tokens.clone(), v.accepted.clone()))
    out = d.step(tok).clone()
    for b in range(B):
        # Sequence b alone, token by token (the other one is fed whatever).
        one = CompressedDecoder(tiny[1], cache, 200, use_graph=False, tree_size=1, cache_dtype=cache_dtype)
        feed = [int(lines[0][b])] + [int(t) for toks, k in lines[1:] for t in toks[b, :int(k[b])]]
        for t in feed:
            x = one.step(torch.full((B, 1), t, device=gpu))
        torch.testing.assert_close(out[b].float(), x[b].float(), rtol=3e-2, atol=3e-2)


def test_refusals(gpu, tiny):
    from dropkv_amd.decode import CompressedDecoder
    cache, tok = prefilled(tiny, gpu)
    with pytest.raises(ValueError, match="cache_dtype"):
        CompressedDecoder(tiny[1], cache, 8, cache_dtype="int4")
    d = CompressedDecoder(tiny[1], cache, 8, use_graph=False, tree_size=4, cache_dtype="int8")
    plain = CompressedDecoder(tiny[1], cache, 8, use_graph=False, cache_dtype="int8")
    with pytest.raises(RuntimeError, match="tree_size"):
        plain.verify(tok)
    d.set_tree([-1, 0, 0])
    drafts, u = tok.expand(1, 3).contiguous(), torch.rand(1, 3, device=gpu)
    with pytest.raises(ValueError, match="chain"):
        d.verify(drafts, uniforms=u)
    d.set_tree([-1, 0, 1])
    for kw in (dict(temperature=0.5), dict(draft_logits=torch.zeros(1, 2, 1000, dtype=torch.bfloat16, device=gpu))):
        with pytest.raises(ValueError, match="uniforms"):
            d.verify(drafts, **kw)
    with pytest.raises(ValueError, match="uniforms"):
        d.verify(drafts, uniforms=u[:, :2])
    for kw in (dict(temperature=0.0), dict(draft_logits=torch.zeros(1, 3, 1000, dtype=torch.bfloat16, device=gpu))):
        with pytest.raises(RuntimeError, match="verify_drafts"):
            d.verify(drafts, uniforms=u, **kw)
    assert int(d.pos) == d.logical
    for _ in range(8):
        plain.step(tok)
    with pytest.raises(RuntimeError, match="capacity"):
        plain.step(tok)


@pytest.mark.parametrize("fields", [{}, {"cache_dtype": None}, {"cache_dtype": "int8"}])
def test_the_command(gpu, fields):
    """The end-to-end command's function, also from callers that name no cache dtype."""
    import argparse
    from dropkv_amd import e2e_qwen2
    res = e2e_qwen2.run(argparse.Namespace(prompt=512, decode=4, layers=2, keep_ratio=0.1, window=8, kernel_size=11, reps=1,
                                           warmup=0, seed=0, compare=False, **fields))["dropkv"]
    assert res["logical_length"] == 516 and res["stored_kv_rows_layer0"] == 51 + 4
    assert ("int8" in res["decode"]) == ("int8" in fields.values())
