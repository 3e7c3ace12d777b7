"""Post-RoPE query capture for unpatched HF Transformers 5.x attention.

The reference's eviction needs the attention's rotated ``query_states`` at
cache-update time; its Transformers patch adds them to ``cache_kwargs`` in
``Qwen2Attention`` and ``LlamaAttention`` (patches/dropkv_transformers.patch:330,
:343).  The installed Transformers calls ``past_key_values.update(key, value,
layer_idx)`` right after ``apply_rotary_pos_emb``, so recording that
function's rotated query gives the cache the same tensor without patching
the library.
"""

from __future__ import annotations

import contextlib
import importlib
import threading
from typing import Optional

import torch

# Modeling modules whose attention the reference patch changes (patch:330, :343).
DEFAULT_MODELING_MODULES = (
    "transformers.models.qwen2.modeling_qwen2",
    "transformers.models.llama.modeling_llama",
)

_slot = threading.local()


def take_captured_query() -> Optional[torch.Tensor]:
    """The query recorded by the last rotary call on this thread (or None),
    cleared so that it is used by one cache update only."""
    q = getattr(_slot, "query", None)
    _slot.query = None
    return q


class _Hook:
    """A modeling module's ``apply_rotary_pos_emb``, wrapped while any block of any
    thread needs it.  Blocks of different threads end in any order, so none of
    them restores what it found: the last one does."""

    def __init__(self, mod):
        self.mod, self.users, self.captures = mod, 0, 0
        self.laid = []   # (wrapper, what it was laid on)

    def lay(self):
        orig = self.mod.apply_rotary_pos_emb
        if any(orig is wrapper for wrapper, _ in self.laid):
            return

        def apply_rotary_pos_emb(q, k, *args, **kwargs):
            deferred = getattr(_slot, "defer", None)
            if deferred is not None and deferred(*args, **kwargs):
                return q, k
            q_rot, k_rot = orig(q, k, *args, **kwargs)
            if self.captures:
                _slot.query = q_rot
            return q_rot, k_rot

        apply_rotary_pos_emb.__wrapped__ = orig
        self.laid.append((apply_rotary_pos_emb, orig))
        self.mod.apply_rotary_pos_emb = apply_rotary_pos_emb

    def lift(self):
        for wrapper, orig in reversed(self.laid):
            if self.mod.apply_rotary_pos_emb is not wrapper:   # (another's wrapper lies on it: it passes through)
                break
            self.mod.apply_rotary_pos_emb = orig


_hooks: dict = {}   # by id(module)
_hooks_lock = threading.Lock()


@contextlib.contextmanager
def _hooked(mods, captures: int):
    hooks = []
    try:
        with _hooks_lock:
            for mod in mods:
                hook = _hooks.get(id(mod)) or _Hook(mod)
                hook.lay()
                _hooks[id(mod)] = hook
                hook.users += 1
                hook.captures += captures
                hooks.append(hook)
        yield
    finally:
        with _hooks_lock:
            for hook in reversed(hooks):
                hook.users -= 1
                hook.captures -= captures
                if hook.users == 0:
                    hook.lift()
                    del _hooks[id(hook.mod)]


def _modules(modules):
    return [importlib.import_module(m) if isinstance(m, str) else m for m in modules]


@contextlib.contextmanager
def query_capture(*modules):
    """Record the post-RoPE query of every attention call made inside the
    block, for the ``DropKVLayer.update`` that follows it on the same thread.

    ``modules`` are modeling modules (or their dotted names) whose
    ``apply_rotary_pos_emb`` the attention looks up at call time; the default
    covers Qwen2 and Llama, the two models the reference patch changes.
    The original functions are restored on exit, also on error, once no other
    thread's block needs them wrapped.
    """
    try:
        with _hooked(_modules(modules or DEFAULT_MODELING_MODULES), 1):
            yield
    finally:
        _slot.query = None


@contextlib.contextmanager
def rotary_deferral(defer):
    """Leave the rotation of the thread's queries and keys to someone else where
    ``defer(cos, sin, ...)``, given what the model gives its rotary function after
    q and k, is true: they come back as they are.  Other threads rotate as ever."""
    prev = getattr(_slot, "defer", None)
    with _hooked(_modules(DEFAULT_MODELING_MODULES), 0):
        _slot.defer = defer
        try:
            yield
        finally:
            _slot.defer = prev
