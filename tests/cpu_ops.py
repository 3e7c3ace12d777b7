"""The operators that a decoder calls, in PyTorch on the CPU, for tests of what
the decoder does around them.  They rotate with the model's own function."""

import torch
from transformers.models.qwen2 import modeling_qwen2

from dropkv_amd import ops

ROTARY = modeling_qwen2.apply_rotary_pos_emb


def norm_rope(q, k, cos, sin, v=None, k_out=None, v_out=None):
    q, k = ROTARY(q, k, cos, sin)
    k_out.copy_(k)
    v_out.copy_(v)
    return q, k_out, v_out


def tree_attention(q, k_new, v_new, k_cache, v_cache, n_rows, scale, workspace=None, mask=None):
    B, Hq, T, D = q.shape
    out = torch.zeros(B, T, Hq, D)
    for b in range(B):
        n = int(n_rows[b])
        seen = torch.ones(T, T, dtype=torch.bool).tril() if mask is None else mask[b]
        seen = torch.cat([torch.ones(T, n, dtype=torch.bool), seen], dim=-1)
        for h in range(Hq):
            g = h * k_cache.shape[1] // Hq
            k, v = torch.cat([k_cache[b, g, :n], k_new[b, g]]), torch.cat([v_cache[b, g, :n], v_new[b, g]])
            out[b, :, h] = (q[b, h] @ k.t() * scale).masked_fill(~seen, -torch.inf).softmax(-1) @ v
    return out


def token_logprobs(logits, top=1):
    lp = logits.log_softmax(-1).max(-1, keepdim=True)
    return ops.TokenLogprobs(None, None, lp.values, lp.indices)


def tree_commit(tokens, parents, choice, k_new, v_new, k_cache, v_cache, n_rows):
    B, T = tokens.shape
    path = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        nodes = [0]
        for i in range(1, T):
            if int(parents[b, i]) == nodes[-1] and tokens[b, i] == choice[b, nodes[-1]]:
                nodes.append(i)
        path[b, :len(nodes)] = torch.tensor(nodes, dtype=torch.int32)
        for l in range(len(k_cache)):
            n = int(n_rows[l, b])
            k_cache[l, b, :, n:n + len(nodes)] = k_new[l, b][:, nodes]
            v_cache[l, b, :, n:n + len(nodes)] = v_new[l, b][:, nodes]
    return path, (path >= 0).sum(-1).int()


def decode_attention(q, k_new, v_new, k_cache, v_cache, n_rows, scale, out, workspace):
    n = int(n_rows)
    k_cache[:, :, n:n + 1], v_cache[:, :, n:n + 1] = k_new, v_new
    out.copy_(tree_attention(q, k_new, v_new, k_cache, v_cache, n_rows.expand(q.shape[0]), scale))
    return out


def install(monkeypatch):
    """In place of the HIP ones."""
    for fn in (norm_rope, tree_attention, token_logprobs, tree_commit, decode_attention):
        monkeypatch.setattr(ops, fn.__name__, fn)
    for name in ("tree_workspace", "decode_workspace"):
        monkeypatch.setattr(ops, name, lambda *a: torch.empty(1, dtype=torch.uint8))
