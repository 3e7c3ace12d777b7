"""A run of the verification step's operators together: the decoder's
``verify`` over trees and chains of drafted tokens, against its own steps of
one token at a time on the same cache."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = dict(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=3,
            num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=8192)


@pytest.fixture(scope="module")
def tiny(gpu):
    from dropkv_amd.e2e_qwen2 import build_model, make_config
    cfg = make_config(**TINY)
    return cfg, build_model(cfg, gpu, dtype=torch.bfloat16, seed=0)


def prefilled(cfg, model, gpu, L=1024, batch=1, seed=21):
    from dropkv_amd import hf_cache
    from dropkv_amd.e2e_qwen2 import prefill, random_prompt
    cache = hf_cache.DropKVCache(cfg, keep_ratio=0.1)
    ids = random_prompt(cfg.vocab_size, L, batch=batch, seed=seed, device=gpu)
    return cache, prefill(model, ids, cache)


def decoder(tiny, gpu, tokens=64, batch=1, **kw):
    from dropkv_amd.decode import CompressedDecoder
    cache, tok = prefilled(*tiny, gpu, batch=batch)
    return CompressedDecoder(tiny[1], cache, max_new_tokens=tokens, **kw), tok


def test_step_of_a_tree_decoder(gpu, tiny):
    """One token at a time: the logits of the decoder without trees, to the
    rounding of the rotation, and the same rows stored."""
    a, tok = decoder(tiny, gpu)
    b, _ = decoder(tiny, gpu, tree_size=6)
    for t in range(5):
        x, y = a.step(tok).clone(), b.step(tok).clone()
        torch.testing.assert_close(y.float(), x.float(), rtol=3e-2, atol=3e-2, msg=f"step {t}")
        tok = x[:, -1].argmax(-1, keepdim=True)
    assert b.n_rows[:, 0].tolist() == a.n_rows.tolist() and torch.equal(a.pos, b.pos)
    n = int(a.n_rows[0])
    torch.testing.assert_close(b.k_buf[0][:, :, :n].float(), a.k_buf[0][:, :, :n].float(), rtol=2e-2, atol=2e-2)


@pytest.mark.parametrize("use_graph", [False, True])
def test_chain_of_right_tokens(gpu, tiny, use_graph):
    """The tokens that steps of one give are drafted as a chain: logits at
    every node as in the steps, and what stands is the longest prefix on which
    the verification's own best tokens agree."""
    a, tok = decoder(tiny, gpu, tree_size=8, use_graph=False)
    toks, logits = [tok], []
    for _ in range(8):
        logits.append(a.step(tok).clone())
        tok = logits[-1][:, -1].argmax(-1, keepdim=True)
        toks.append(tok)
    b, _ = decoder(tiny, gpu, tree_size=8, use_graph=use_graph)
    n0 = b.n_rows.clone()
    v = b.verify(torch.cat(toks[:8], dim=1))
    torch.testing.assert_close(v.logits.float(), torch.cat(logits, dim=1).float(), rtol=3e-2, atol=3e-2)
    best = v.logits[0].argmax(-1).tolist()
    want = [0]
    while want[-1] < 7 and best[want[-1]] == int(toks[want[-1] + 1]):
        want.append(want[-1] + 1)
    assert v.accepted.tolist() == [len(want)]
    assert v.path[0].tolist() == want + [-1] * (8 - len(want))
    assert v.tokens[0].tolist() == [best[i] for i in want] + [-1] * (8 - len(want))
    lp = torch.log_softmax(v.logits[0].double(), -1)
    torch.testing.assert_close(v.logprobs[0, :len(want)].double(), lp[want, [best[i] for i in want]], rtol=0, atol=1e-4)
    assert torch.equal(b.n_rows, n0 + len(want)) and int(b.pos) == b.logical + len(want)
    n = int(n0[0, 0])
    torch.testing.assert_close(b.k_buf[1][:, :, n:n + len(want)].float(), a.k_buf[1][:, :, n:n + len(want)].float(),
                               rtol=3e-2, atol=3e-2)


def test_tree_batch_and_graph(gpu, tiny):
    """Random trees for two sequences, some nodes left out, one round after
    another with trees of other shapes: graph and eager give the same bits, each
    node's logits are those of its path fed token by token, sequences advance on
    their own, and a step of one token follows."""
    B, T = 2, 9
    eager, tok = decoder(tiny, gpu, batch=B, tree_size=T, use_graph=False)
    graph, _ = decoder(tiny, gpu, batch=B, tree_size=T, use_graph=True)
    g = torch.Generator().manual_seed(1)
    moved = torch.zeros(B, dtype=torch.int64)
    for rnd in range(3):
        t = (9, 5, 7)[rnd]
        parents = torch.stack([torch.tensor([-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, t)])
                               for _ in range(B)])
        parents[1, 3] = -1
        drafts = torch.randint(0, tiny[0].vocab_size, (B, t), generator=g).to(gpu)
        drafts[:, :1] = tok
        for d in (eager, graph):
            d.set_tree(parents)
        a, b = eager.verify(drafts), graph.verify(drafts)
        torch.cuda.synchronize()
        for x, y in zip(a, b):
            x, y = (x[:, :t], y[:, :t]) if x.dim() > 1 else (x, y)
            assert torch.equal(x, y), rnd
        moved += a.accepted.cpu().long()
        assert torch.equal(eager.n_rows, graph.n_rows) and torch.equal(eager.pos, graph.pos)
        assert (eager.pos[:, 0].cpu() - eager.logical).tolist() == moved.tolist()
        last = (a.accepted.long() - 1)[:, None]
        tok = a.tokens.gather(1, last)
    x, y = eager.step(tok).clone(), graph.step(tok).clone()
    assert torch.equal(x, y)


def test_accepted_tree_path_continues_like_steps(gpu, tiny):
    """A tree that holds the right continuation on one of its branches, drafted
    twice: what is generated is what steps of one token give."""
    T = 7
    a, tok = decoder(tiny, gpu, tree_size=T)
    first = tok.clone()
    right = []
    for _ in range(6):
        tok = a.step(tok)[:, -1].argmax(-1, keepdim=True)
        right.append(int(tok))
    b, _ = decoder(tiny, gpu, tree_size=T)
    # Nodes 1 and 2 are the root's children, 2 the right one; 4 follows 2, 6 follows 4.
    b.set_tree([-1, 0, 0, 1, 2, 2, 4])
    wrong = [(r + 1) % tiny[0].vocab_size for r in right]
    v = b.verify(torch.tensor([[int(first), wrong[0], right[0], wrong[1], right[1], wrong[1], right[2]]], device=gpu))
    assert v.path[0].tolist()[:4] == [0, 2, 4, 6] and int(v.accepted) == 4
    assert v.tokens[0].tolist()[:4] == right[:4]
    n = int(a.n_rows[0, 0])
    torch.testing.assert_close(b.k_buf[2][:, :, n - 6:n - 2].float(), a.k_buf[2][:, :, n - 6:n - 2].float(), rtol=3e-2,
                               atol=3e-2)
    out = b.step(v.tokens[:, 3:4].clone())
    assert int(out[:, -1].argmax(-1)) == right[4]


def test_negative_tokens_never_stand(gpu, tiny):
    """Nodes left out filled with -1, and a node of the tree that holds it: the
    others come out as without them."""
    a, tok = decoder(tiny, gpu, tree_size=6)
    b, _ = decoder(tiny, gpu, tree_size=6, use_graph=False)
    c, _ = decoder(tiny, gpu, tree_size=6, use_graph=False)
    right = int(a.step(tok)[:, -1].argmax(-1))
    b.set_tree([-1, 0, 0, 2, -1, -1])
    c.set_tree([-1, 0, 0, 2, -1, -1])
    row = [int(tok), -1, right, (right + 1) % 1000, -1, -7]
    v = b.verify(torch.tensor([row], device=gpu))
    w = c.verify(torch.tensor([[max(x, 0) for x in row]], device=gpu))
    assert v.path[0].tolist()[:2] == [0, 2] and torch.equal(v.path, w.path)
    assert torch.equal(v.tokens, w.tokens) and torch.equal(v.logits, w.logits)
    assert int(v.path.max()) < 4


def test_capacity_and_refusals(gpu, tiny):
    d, tok = decoder(tiny, gpu, tokens=5, tree_size=4, use_graph=False)
    plain, _ = decoder(tiny, gpu, tokens=5, use_graph=False)
    for call in (lambda: plain.verify(tok), lambda: plain.set_tree([-1])):
        with pytest.raises(RuntimeError, match="tree_size"):
            call()
    for bad in ([-1, 1], [-1, 0, 2], [-1] * 5, [[-1, 0]] * 2, [-1, -2], [0.0, 0.0]):
        with pytest.raises(ValueError):
            d.set_tree(bad)
    with pytest.raises(ValueError):
        d.verify(tok)                                  # the tree is a chain of four
    d.set_tree([-1, -1])
    # A draft that is left out cannot stand: one token a call, whatever `steps` counted.
    for i in range(5):
        v = d.verify(torch.cat([tok, tok], dim=1))
        assert int(v.accepted) == 1 and v.path[0].tolist()[:2] == [0, -1]
        tok = v.tokens[:, :1].clone()
    with pytest.raises(RuntimeError, match="capacity"):
        d.verify(torch.cat([tok, tok], dim=1))
    with pytest.raises(RuntimeError, match="capacity"):
        d.step(tok)
