"""Decode on the compressed cache: preallocated K/V buffers, a HIP attention
kernel that appends and attends in one launch, and a HIP graph per step.

The reference decodes eagerly: every step appends the new row with
``torch.cat`` (dropkv_cache.py:609-617, patches/dropkv_transformers.patch:
206-213) and the model's SDPA attends over the concatenation.  Here, after
the prefill has evicted, each layer's kept rows are copied once into a
buffer with room for ``max_new_tokens`` more rows; the model (the installed
Transformers' own forward) runs with an attention function that calls
``dropkv_decode_attention`` on those buffers, whose row count lives on the
device.  Nothing in a step depends on the host, so the whole forward is
captured once as a HIP graph and replayed per token.

With ``tree_size`` the decoder also verifies drafted tokens: one forward over
a tree (or chain) of them, a captured graph too, whose attention rotates
queries and keys and lays out the drafted rows (``dropkv_norm_rope``), attends
over the cache and the tree (``dropkv_tree_attention``), and whose end takes the
best token at every node (``dropkv_token_logprobs``) and appends the rows of the
path that stands to every layer's buffer (``dropkv_tree_commit``).  A chain of
drafted tokens may be verified by sampling instead, from given random numbers
(``dropkv_verify_drafts``).

With ``cache_dtype`` the rows are held in 8 bits with a scale for each block of 64
rows and head: half the bytes that a step reads of the cache, and half its memory but for
128 rows a head in 16 bits (``dropkv_quant_append``, ``dropkv_quant_attention``).
"""

from __future__ import annotations

import contextlib
import threading
from typing import NamedTuple, Optional

import torch

from . import ops
from .hf_query import rotary_deferral

ATTN_NAME = "dropkv_decode"
_active = threading.local()


def _decode_attention(module, query, key, value, attention_mask=None, scaling=None, dropout=0.0, **kwargs):
    """Attention function for the Transformers attention interface: one
    decode step of layer ``module.layer_idx`` on the active decoder's buffers.
    Returns ([B, 1, Hq, D], None)."""
    dec = getattr(_active, "decoder", None)
    if dec is None:
        raise RuntimeError("dropkv_decode attention used outside CompressedDecoder")
    if dec.drafts:
        return dec._tree_attention(module, query, key, value, scaling, kwargs.get("sliding_window")), None
    if query.shape[2] != 1:
        raise RuntimeError("dropkv_decode attention takes one query position per step")
    i = module.layer_idx
    B, Hq, _, D = query.shape
    out = torch.empty(B, 1, Hq, D, dtype=query.dtype, device=query.device)
    scale = scaling if scaling is not None else D ** -0.5
    ops.decode_attention(query, key, value, dec.k_buf[i], dec.v_buf[i], dec.n_rows[i:i + 1], scale, out, dec.ws)
    return out, None


# Configurations whose attention is the decoders' at the moment: by id, how many
# forwards need it, and what it was.  The last one out puts that back, in whatever
# order threads come and go.
_attn_users: dict = {}
_attn_lock = threading.Lock()


@contextlib.contextmanager
def _own_attention(cfg):
    with _attn_lock:
        use = _attn_users.setdefault(id(cfg), [0, cfg._attn_implementation])
        use[0] += 1
        if use[0] == 1:
            cfg._attn_implementation = ATTN_NAME
    try:
        yield
    finally:
        with _attn_lock:
            use[0] -= 1
            if use[0] == 0:
                cfg._attn_implementation = use[1]
                del _attn_users[id(cfg)]


def _register():
    from transformers import AttentionInterface
    if ATTN_NAME not in AttentionInterface._global_mapping:
        AttentionInterface.register(ATTN_NAME, _decode_attention)


class _StepCache:
    """The ``past_key_values`` of a decode step: K/V already live in the
    decoder's buffers, so ``update`` hands the new rows straight to the
    attention, which stores them."""

    is_compileable = False

    def __init__(self, logical: int):
        self.logical = logical

    def update(self, key_states, value_states, layer_idx, *args, **kwargs):
        return key_states, value_states

    def get_seq_length(self, layer_idx: int = 0) -> int:
        return self.logical


def _stored_kv(cache):
    if hasattr(cache, "layers"):
        return [(lay.keys, lay.values) for lay in cache.layers]
    return list(zip(cache.key_cache, cache.value_cache))


class Verified(NamedTuple):
    """What :meth:`CompressedDecoder.verify` returns, on the device.  With a
    graph the tensors are the graph's own, overwritten by the next call."""

    tokens: torch.Tensor    # [B, T] int64: the token after each node of the path, then -1
    logprobs: torch.Tensor  # [B, T] fp32: their log probabilities, then 0
    accepted: torch.Tensor  # [B] int32: nodes of the path (1 or more), so many new tokens
    path: torch.Tensor      # [B, T] int32: the nodes, then -1
    logits: torch.Tensor    # [B, T, vocab]: of every node


class CompressedDecoder:
    """Greedy-decode driver on a cache that a prefill filled (and evicted).

    ``cache`` is a :class:`dropkv_amd.hf_cache.DropKVCache` or a
    :class:`dropkv_amd.DropKVCache` after the prefill; its rows are copied
    into buffers of ``stored + max_new_tokens`` rows (rounded up to 64).
    RoPE positions continue from the cache's logical length.  With
    ``use_graph`` the forward is captured once and replayed per step.

    With ``tree_size`` T, :meth:`set_tree` and :meth:`verify` take up to T
    drafted tokens in one forward; sequences of a batch then advance by their
    own number of tokens.

    With ``cache_dtype`` (``"int8"``, ``"fp8"`` or the torch dtypes) the rows are held
    in 8 bits (``self.cache``, an :class:`ops.QuantCache` of all layers) in the place of
    ``k_buf`` / ``v_buf``.
    """

    _STORES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, torch.int8: torch.int8,
               torch.float8_e4m3fn: torch.float8_e4m3fn}

    def __init__(self, model, cache, max_new_tokens: int, use_graph: bool = True, tree_size: int = 0, cache_dtype=None):
        if cache_dtype is not None and cache_dtype not in self._STORES:
            raise ValueError(f"cache_dtype must be 'int8', 'fp8' or None, got {cache_dtype!r}")
        _register()
        self.model = model
        self.tree_size = int(tree_size)
        if not 0 <= self.tree_size <= 256:
            raise ValueError(f"tree_size must be in [0, 256], got {tree_size}")
        self._angles = None  # of a layer whose rotation was deferred, until its attention takes them
        kv = _stored_kv(cache)
        if not kv:
            raise ValueError("the cache holds no layers: run the prefill first")
        k0 = kv[0][0]
        self.device = k0.device
        B, Hkv, _, D = k0.shape
        stored = [k.shape[2] for k, _ in kv]
        # (A verification that starts below max_new_tokens may end past it.)
        self.capacity = (max(stored) + max_new_tokens + self.tree_size + 63) // 64 * 64
        self.max_new_tokens = max_new_tokens
        # Rows of a forward's own, which its end appends: of drafted tokens, or, with
        # rows in 8 bits, of a step's one token too.
        self.drafts = self.tree_size or (1 if cache_dtype is not None else 0)
        self.k_buf, self.v_buf = [], []
        self.cache: Optional[ops.QuantCache] = None
        if cache_dtype is not None:
            self.cache = ops.quant_cache(B, Hkv, self.capacity, D, dtype=k0.dtype, store=self._STORES[cache_dtype],
                                         layers=len(kv), device=self.device)
            self._layers = [self.cache.layer(i) for i in range(len(kv))]
            empty = torch.zeros(1, dtype=torch.int32, device=self.device)
            with torch.no_grad():
                for one, (k, v) in zip(self._layers, kv):
                    ops.quant_append(one, k, v, empty)
            # (A buffer without room: which drafts stand is asked of tree_commit, their
            # rows are appended by quant_append.)
            self._no_room = torch.zeros(B, 1, 1, D, dtype=k0.dtype, device=self.device)
            self._full = torch.ones(1, dtype=torch.int32, device=self.device)
        else:
            if self.tree_size:
                self._k_all = torch.empty(len(kv), B, Hkv, self.capacity, D, dtype=k0.dtype, device=self.device)
                self._v_all = torch.empty_like(self._k_all)
            for i, (k, v) in enumerate(kv):
                if self.tree_size:
                    kb, vb = self._k_all[i], self._v_all[i]
                else:
                    kb = torch.empty(B, Hkv, self.capacity, D, dtype=k.dtype, device=self.device)
                    vb = torch.empty_like(kb)
                kb[:, :, :k.shape[2]].copy_(k)
                vb[:, :, :v.shape[2]].copy_(v)
                self.k_buf.append(kb)
                self.v_buf.append(vb)
        self.n_rows = torch.tensor(stored, dtype=torch.int32, device=self.device)
        Hq = model.config.num_attention_heads
        self.logical = cache.get_seq_length()
        if self.drafts:
            T = self.drafts
            self.n_rows = self.n_rows[:, None].repeat(1, B)
            self._k_draft = torch.empty(len(kv), B, Hkv, T, D, dtype=k0.dtype, device=self.device)
            self._v_draft = torch.empty_like(self._k_draft)
            # (One token takes more splits than a tree of them.)
            workspace = ops.tree_workspace if self.cache is None else ops.quant_workspace
            self.ws = max((workspace(B, Hq, Hkv, D, t, self.capacity, self.device) for t in (1, T)),
                          key=torch.Tensor.numel)
        else:
            self.ws = ops.decode_workspace(B, Hq, Hkv, D, self.capacity, self.device)
        if self.tree_size:
            self._tree_tok = torch.zeros(B, T, dtype=torch.int64, device=self.device)
            self._tree_parents = torch.zeros(B, T, dtype=torch.int32, device=self.device)
            self._tree_depth = torch.zeros(B, T, dtype=torch.int64, device=self.device)
            self._tree_mask = torch.zeros(B, T, T, dtype=torch.bool, device=self.device)
            self._root = torch.zeros(1, dtype=torch.int32, device=self.device)
            self.set_tree(range(-1, T - 1))
        self.pos = torch.full((B, 1), self.logical, dtype=torch.int64, device=self.device)
        self.tok = torch.zeros(B, 1, dtype=torch.int64, device=self.device)
        self.steps = 0
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        self.logits: Optional[torch.Tensor] = None
        self.tree_graph: Optional[torch.cuda.CUDAGraph] = None
        self.verified: Optional[Verified] = None
        self.use_graph = bool(use_graph)
        self.logits_graph: Optional[torch.cuda.CUDAGraph] = None  # of a verification by sampling: the forward alone
        self._tree_logits_out: Optional[torch.Tensor] = None
        if use_graph:
            self._capture()

    @contextlib.contextmanager
    def _active(self):
        prev = getattr(_active, "decoder", None)
        _active.decoder = self
        try:
            with _own_attention(self.model.config), (
                    rotary_deferral(self._defer) if self.drafts else contextlib.nullcontext()):
                yield
        finally:
            _active.decoder = prev
            self._angles = None

    def _defer(self, cos, sin, *args, **kwargs) -> bool:
        """Take a layer's angles, for its attention function to rotate with; not
        in another layout."""
        mine = not args and not kwargs and getattr(_active, "decoder", None) is self
        self._angles = (cos, sin) if mine else None
        return mine

    def _tree_attention(self, module, query, key, value, scaling, sliding_window) -> torch.Tensor:
        """One layer of a forward over T tokens: rows into the drafts' buffers,
        then attention over cache and drafts.  [B, T, Hq, D]."""
        if sliding_window is not None:
            raise RuntimeError("a decoder with tree_size or cache_dtype takes no layers with a sliding window")
        i = module.layer_idx
        T, D = query.shape[2], query.shape[3]
        k_new, v_new = self._k_draft[i, :, :, :T], self._v_draft[i, :, :, :T]
        angles, self._angles = self._angles, None
        if angles is not None:
            query, _, _ = ops.norm_rope(query, key, *angles, v=value, k_out=k_new, v_out=v_new)
        else:  # a layer whose rotation was not deferred
            k_new.copy_(key)
            v_new.copy_(value)
        scale, mask = scaling if scaling is not None else D ** -0.5, self._tree_mask if T > 1 else None
        if self.cache is not None:
            return ops.quant_attention(query, k_new, v_new, self._layers[i], self.n_rows[i], scale, workspace=self.ws,
                                       mask=mask)
        return ops.tree_attention(query, k_new, v_new, self.k_buf[i], self.v_buf[i], self.n_rows[i], scale,
                                  workspace=self.ws, mask=mask)

    def _advance(self):
        """After a forward over one token: its row counts."""
        if self.cache is not None:
            ops.quant_append(self.cache, self._k_draft[:, :, :, :1], self._v_draft[:, :, :, :1], self.n_rows)
        elif self.tree_size:
            ops.tree_commit(self.tok, self._root, self.tok, self._k_draft[:, :, :, :1], self._v_draft[:, :, :, :1],
                            self._k_all, self._v_all, self.n_rows)
        self.n_rows.add_(1)
        self.pos.add_(1)

    def _commit(self, tokens, choice, store: bool = True):
        """The path of the drafted tokens that stands, its rows appended."""
        if self.cache is None:
            return ops.tree_commit(tokens, self._tree_parents, choice, self._k_draft, self._v_draft, self._k_all,
                                   self._v_all, self.n_rows)
        path, accepted = ops.tree_commit(tokens, self._tree_parents, choice, self._k_draft[0, :, :1],
                                         self._v_draft[0, :, :1], self._no_room, self._no_room, self._full)
        ops.quant_append(self.cache, self._k_draft, self._v_draft, self.n_rows, path=path,
                         counts=accepted if store else torch.zeros_like(accepted))
        return path, accepted

    @torch.no_grad()
    def _tree_logits(self) -> torch.Tensor:
        with self._active():
            # (A negative token has no embedding, and equals no best token.)
            return self.model(self._tree_tok.clamp(min=0), position_ids=self.pos + self._tree_depth,
                              past_key_values=_StepCache(self.logical), use_cache=True).logits

    @torch.no_grad()
    def _tree_forward(self, store: bool = True) -> Verified:
        """A forward over the drafted tokens, and the path of them that stands.
        The counts are not advanced."""
        logits = self._tree_logits()
        best = ops.token_logprobs(logits, top=1)
        choice = best.top_ids[..., 0]
        path, accepted = self._commit(self._tree_tok, choice, store)
        on, at = path >= 0, path.clamp(min=0).long()
        return Verified(torch.where(on, choice.gather(1, at), -1),
                        torch.where(on, best.top_logprobs[..., 0].gather(1, at), 0.0), accepted, path, logits)

    def _tree_advance(self, v: Verified):
        self.n_rows.add_(v.accepted)
        self.pos.add_(v.accepted[:, None])

    @torch.no_grad()
    def _forward(self) -> torch.Tensor:
        with self._active():
            out = self.model(self.tok, position_ids=self.pos, past_key_values=_StepCache(self.logical),
                             use_cache=True, logits_to_keep=1)
        return out.logits

    def _beside(self, run):
        """``run()`` on a stream of its own, between two waits."""
        side = torch.cuda.Stream(device=self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream(self.device).wait_stream(side)
        torch.cuda.synchronize(self.device)

    @torch.no_grad()
    def _capture(self):
        # One eager run on a side stream first (library workspaces, lazy
        # initialisation); it stores a row at n that the first replay rewrites (in 8
        # bits none: a block that it filled up would have lost the rows before it).
        def once():
            self._forward()
            if self.tree_size:
                self._tree_forward(store=self.cache is None)

        self._beside(once)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = self._forward()
            self._advance()
        if self.tree_size:
            self.tree_graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.tree_graph):
                self.verified = self._tree_forward()
                self._tree_advance(self.verified)

    @torch.no_grad()
    def step(self, token: torch.Tensor) -> torch.Tensor:
        """Logits [B, 1, vocab] of the next position after ``token`` [B, 1]."""
        self._check_room()
        self.tok.copy_(token)
        self.steps += 1
        if self.graph is not None:
            self.graph.replay()
            return self.logits
        logits = self._forward()
        self._advance()
        return logits

    def _check_room(self):
        # (After a verification `steps` is the most that may have been accepted:
        # the device is asked only once that much would not fit.)
        if self.steps >= self.max_new_tokens and self.tree_size:
            self.steps = int(self.pos.max()) - self.logical
        if self.steps >= self.max_new_tokens:
            raise RuntimeError(f"decode capacity of {self.max_new_tokens} new tokens reached")

    def set_tree(self, parents) -> None:
        """The tree of the next verifications: ``parents`` (whole numbers, a list
        or a tensor, [t] or [B, t], t <= tree_size) holds each node's parent, a
        lower node, or -1 for a node that is left out; node 0 is the root.  The
        tree is a chain of ``tree_size`` tokens at first."""
        if not self.tree_size:
            raise RuntimeError("the decoder was made without tree_size")
        B, T = self._tree_tok.shape
        p = torch.as_tensor(list(parents) if isinstance(parents, range) else parents, device="cpu")
        if p.dtype.is_floating_point or p.dtype == torch.bool or p.dim() not in (1, 2) or p.shape[-1] < 1:
            raise ValueError("parents must be whole numbers, [t] or [B, t]")
        t = p.shape[-1]
        if t > T or (p.dim() == 2 and p.shape[0] != B):
            raise ValueError(f"a tree has at most {T} nodes, one tree or {B} of them")
        p = p.to(torch.int64).expand(B, t).clone()
        p[:, 0] = -1
        if bool((p[:, 1:] < -1).any()) or bool((p >= torch.arange(t)).any()):
            raise ValueError("a node's parent is a lower node, or -1")
        full = torch.full((B, T), -1, dtype=torch.int64)
        full[:, :t] = p
        depth = torch.zeros(B, T, dtype=torch.int64)
        mask = torch.eye(T, dtype=torch.bool).repeat(B, 1, 1)
        rows = torch.arange(B)
        for i in range(1, t):
            up = full[:, i].clamp(min=0)
            child = full[:, i] >= 0
            depth[:, i] = torch.where(child, depth[rows, up] + 1, 0)
            mask[:, i] |= mask[rows, up] & child[:, None]
        self.tree_nodes = t
        self._is_chain = bool((full[:, :t] == torch.arange(-1, t - 1)).all())
        self._tree_parents.copy_(full.to(torch.int32))
        self._tree_depth.copy_(depth)
        self._tree_mask.copy_(mask)

    @torch.no_grad()
    def verify(self, tokens: torch.Tensor, uniforms: Optional[torch.Tensor] = None,
               draft_logits: Optional[torch.Tensor] = None, temperature: float = 1.0) -> Verified:
        """One forward over the tree: ``tokens`` [B, t], the last token of each
        sequence at node 0 and drafted ones at the others (a negative one never
        stands: it may fill a node that is left out).  From the root on the path
        follows the children that the model's best token agrees with; the rows of
        its nodes are appended and the positions advanced, by ``accepted`` tokens
        a sequence, of which the last is the model's own.

        With ``uniforms`` ([B, t] fp32 in [0, 1)) the tokens are judged and drawn by
        sampling instead, at ``temperature``, and the tree has to be a chain:
        ``draft_logits`` [B, t - 1, vocab] is what the drafts were drawn from, without
        it they are taken as given (:func:`ops.verify_drafts`)."""
        if not self.tree_size:
            raise RuntimeError("the decoder was made without tree_size")
        t = self.tree_nodes
        if tuple(tokens.shape) != (self._tree_tok.shape[0], t):
            raise ValueError(f"tokens must be [{self._tree_tok.shape[0]}, {t}], as the tree")
        if uniforms is None:
            if draft_logits is not None or temperature != 1.0:
                raise ValueError("draft_logits and temperature go with uniforms")
        elif not self._is_chain:
            raise ValueError("tokens are verified by sampling along a chain (set_tree(range(-1, t - 1)))")
        elif tuple(uniforms.shape) != tuple(tokens.shape):
            raise ValueError("uniforms must have the tokens' shape")
        self._check_room()
        self._tree_tok[:, :t].copy_(tokens)
        if uniforms is not None:
            return self._verify_sampled(t, uniforms, draft_logits, temperature)
        self.steps += t
        if self.tree_graph is not None:
            self.tree_graph.replay()
            return self.verified
        v = self._tree_forward()
        self._tree_advance(v)
        return v

    def _verify_sampled(self, t: int, uniforms, draft_logits, temperature) -> Verified:
        """The forward (a graph of its own, captured at the first call), then the chain
        judged and its rows appended."""
        if self.use_graph and self.logits_graph is None:
            self._beside(self._tree_logits)
            self.logits_graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.logits_graph):
                self._tree_logits_out = self._tree_logits()
        if self.logits_graph is not None:
            self.logits_graph.replay()
            logits = self._tree_logits_out
        else:
            logits = self._tree_logits()
        tokens = self._tree_tok
        choice, accepted, logprobs = ops.verify_drafts(logits[:, :t], tokens[:, :t], uniforms, draft_logits, temperature)
        T = tokens.shape[1]
        if t < T:
            choice = torch.nn.functional.pad(choice, (0, T - t), value=-1)
            logprobs = torch.nn.functional.pad(logprobs, (0, T - t))
        # (The nodes that stand are known: no other equals a choice.)
        on = torch.arange(T, device=tokens.device) < accepted[:, None]
        path, _ = self._commit(torch.where(on, tokens, -2), choice)
        self.steps += t
        v = Verified(choice, logprobs, accepted, path, logits)
        self._tree_advance(v)
        return v

    @torch.no_grad()
    def stored(self, layer: int):
        """Layer ``layer``'s rows (k, v) [B, Hkv, n, D], n the longest sequence's count
        (asked of the device): views of the buffers, or new tensors read back from 8
        bits, then zeros behind a shorter sequence's rows."""
        n = int(self.n_rows[layer].max())
        if self.cache is not None:
            return ops.quant_read(self._layers[layer], self.n_rows[layer], n)
        return self.k_buf[layer][:, :, :n], self.v_buf[layer][:, :, :n]

    @torch.no_grad()
    def generate(self, token: torch.Tensor, steps: int) -> torch.Tensor:
        """``steps`` greedy tokens [B, steps] after ``token``; stays on the device."""
        toks = []
        for _ in range(steps):
            logits = self.step(token)
            token = logits[:, -1].argmax(-1, keepdim=True)
            toks.append(token)
        return torch.cat(toks, dim=1)
