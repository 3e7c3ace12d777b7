"""Rounds of verification for a batch whose sequences accept unequal numbers of
tokens, each against a decoder without trees that is fed one token at a time:
shared by the test on the kernels and the one on the CPU."""

from types import SimpleNamespace

import torch

from dropkv_amd.decode import CompressedDecoder


class OneByOne:
    """One sequence of a prefilled cache, its tokens fed one at a time."""

    def __init__(self, model, cache, b, room):
        layers = cache.layers if hasattr(cache, "layers") else [
            SimpleNamespace(keys=k, values=v) for k, v in zip(cache.key_cache, cache.value_cache)]
        own = SimpleNamespace(layers=[SimpleNamespace(keys=x.keys[b:b + 1], values=x.values[b:b + 1]) for x in layers],
                              get_seq_length=cache.get_seq_length)
        self.dec = CompressedDecoder(model, own, max_new_tokens=room, use_graph=False)
        self.start = self.dec.n_rows.clone(), self.dec.pos.clone()

    def logits(self, tokens):
        """[len(tokens), vocab]: after each of ``tokens``, from the prefill on."""
        self.dec.n_rows.copy_(self.start[0])
        self.dec.pos.copy_(self.start[1])
        self.dec.steps = 0
        return torch.cat([self.dec.step(torch.tensor([[t]], device=self.dec.device))[0].clone() for t in tokens])


# Three rounds.  Parents of both sequences' trees, of which each inner node has
# two children, and the sequences whose trees hold the two likeliest tokens after
# each inner node; the others' hold the two least likely.
ROUNDS = [
    ([[-1, 0, 0, 1, 1, 2, 2], [-1, 0, 1, 1, 0, 4, 4]], (0,)),
    ([[-1, 0, 0, 1, 2, 1, 2], [-1, 0, 0, 2, 2, 1, 1]], (1,)),
    ([[-1, 0, 0, 2, 1, 2, 1], [-1, 0, 0, 1, 2, 2, 1]], (0, 1)),
]


def check(model, cache, first, use_graph, tol):
    """``first`` [2, 1]: the tokens after the prefill; ``tol``: of logits and rows
    (times their size, and on its own).  Whatever rounding makes of a near tie of
    the two likeliest tokens, a tree that holds both holds the path."""
    B, T = 2, 7
    dec = CompressedDecoder(model, cache, max_new_tokens=64, use_graph=use_graph, tree_size=T)
    refs = [OneByOne(model, cache, b, 64) for b in range(B)]
    fed = [[int(first[b])] for b in range(B)]     # the last of them at node 0
    n0, pos0 = dec.n_rows.clone(), dec.pos.clone()

    def close(a, b):
        return bool(((a.float() - b.float()).abs() <= tol * b.float().abs() + tol).all())

    apart = 0.0
    for parents, favoured in ROUNDS:
        drafts = torch.zeros(B, T, dtype=torch.int64)
        want = []
        for b in range(B):
            paths, rows = [fed[b]], []
            drafts[b, 0] = fed[b][-1]
            for i in range(T):
                if i:
                    up = parents[b][i]
                    rank = sum(parents[b][j] == up for j in range(1, i))
                    order = rows[up].argsort(descending=b in favoured)
                    drafts[b, i] = order[rank]
                    paths.append(paths[up] + [int(order[rank])])
                rows.append(refs[b].logits(paths[i])[-1])
            want.append(torch.stack(rows))
            apart = max(apart, float((rows[0] - rows[1]).abs().max()))
        dec.set_tree(parents)
        v = dec.verify(drafts.to(dec.device))
        logits = v.logits.clone()
        for b in range(B):
            for i in range(T):
                assert close(logits[b, i], want[b][i]), (b, i)
            best, path = logits[b].argmax(-1).tolist(), [0]
            while True:
                kids = [i for i in range(path[-1] + 1, T)
                        if parents[b][i] == path[-1] and int(drafts[b, i]) == best[path[-1]]]
                if not kids:
                    break
                path.append(kids[0])
            assert len(path) == (3 if b in favoured else 1), (b, path)
            rest = [-1] * (T - len(path))
            assert v.path[b].tolist() == path + rest and int(v.accepted[b]) == len(path)
            assert v.tokens[b].tolist() == [best[i] for i in path] + rest
            lp = torch.log_softmax(logits[b].double(), -1)[path, [best[i] for i in path]]
            assert ((v.logprobs[b, :len(path)].double() - lp).abs() <= 1e-4).all()
            fed[b] += [best[i] for i in path]
            assert (dec.n_rows[:, b] == n0[:, b] + len(fed[b]) - 1).all()
            assert int(dec.pos[b]) == int(pos0[b]) + len(fed[b]) - 1
    assert apart > 10 * tol      # (one node's logits are not another's)
    tok = torch.tensor([[f[-1]] for f in fed], device=dec.device)
    after = dec.step(tok)
    for b in range(B):
        assert close(after[b], refs[b].logits(fed[b])[-1:])
        n = int(dec.n_rows[0, b])
        for mine, ref in ((dec.k_buf, refs[b].dec.k_buf), (dec.v_buf, refs[b].dec.v_buf)):
            for x, y in zip(mine, ref):
                assert close(x[b, :, :n], y[0, :, :n])
