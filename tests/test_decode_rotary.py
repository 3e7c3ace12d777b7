"""Who rotates queries and keys in a forward over drafted tokens, on the CPU: a
tiny Qwen2 model with the operators replaced by PyTorch ones that rotate with
the model's own function, so that a rotation left out, or done twice, shows in
the logits' bits.  Threads that capture queries meanwhile, and layers that
rotate in a way of their own, change nothing."""

import threading
from types import SimpleNamespace

import pytest
import torch

pytest.importorskip("transformers")

from transformers import DynamicCache  # noqa: E402
from transformers.models.qwen2 import modeling_qwen2  # noqa: E402

import cpu_ops  # noqa: E402
from cpu_ops import ROTARY as ORIG  # noqa: E402
from dropkv_amd import decode  # noqa: E402
from dropkv_amd.e2e_qwen2 import build_model, make_config, random_prompt  # noqa: E402
from dropkv_amd.hf_query import query_capture, take_captured_query  # noqa: E402

TINY = dict(vocab_size=200, hidden_size=256, intermediate_size=256, num_hidden_layers=3,
            num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=512)


@pytest.fixture(scope="module")
def tiny():
    cfg = make_config(**TINY)
    return cfg, build_model(cfg, "cpu", dtype=torch.float32, seed=0)


@pytest.fixture
def decoder(tiny, monkeypatch):
    """A decoder of chains of four on a prompt of 20 rows."""
    cpu_ops.install(monkeypatch)
    cfg, model = tiny
    cache = DynamicCache(config=cfg)
    with torch.no_grad():
        model(random_prompt(cfg.vocab_size, 20, seed=1), past_key_values=cache, use_cache=True, logits_to_keep=1)

    def make():
        return decode.CompressedDecoder(model, cache, max_new_tokens=16, use_graph=False, tree_size=4)

    return make


DRAFTS = torch.tensor([[3, 50, 17, 91]])


def between_layers(model, layer, do):
    return model.model.layers[layer].register_forward_pre_hook(lambda *a: do())


class Capturing:
    """Another thread's query_capture block, entered and left on request."""

    def __init__(self):
        self.enter, self.entered, self.leave = (threading.Event() for _ in range(3))
        self.thread = threading.Thread(target=self._run)
        self.thread.start()

    def _run(self):
        self.enter.wait(30)
        with query_capture():
            self.entered.set()
            self.leave.wait(30)

    def go_in(self):
        self.enter.set()
        assert self.entered.wait(30)

    def go_out(self):
        self.leave.set()
        self.thread.join(30)
        assert not self.thread.is_alive()


def same(a, b):
    assert torch.equal(a.logits, b.logits) and torch.equal(a.tokens, b.tokens)


@pytest.mark.parametrize("went_in", ["before", "during"])
@pytest.mark.parametrize("came_out", ["during", "after"])
def test_a_capture_of_another_thread_in_between(tiny, decoder, went_in, came_out):
    want_dec, dec, other = decoder(), decoder(), Capturing()
    want = want_dec.verify(DRAFTS)
    if went_in == "before":
        other.go_in()
    handles = []
    if went_in == "during":
        handles.append(between_layers(tiny[1], 1, other.go_in))
    if came_out == "during":
        handles.append(between_layers(tiny[1], 2, other.go_out))
    try:
        got = dec.verify(DRAFTS)
    finally:
        for h in handles:
            h.remove()
        other.enter.set()
        other.go_out()
    same(got, want)
    for a, b in zip(dec.k_buf, want_dec.k_buf):
        n = int(dec.n_rows[0, 0])
        assert torch.equal(a[:, :, :n], b[:, :, :n])
    # Nothing is left behind: neither a wrapper nor a recorded query.
    assert modeling_qwen2.apply_rotary_pos_emb is ORIG
    assert take_captured_query() is None


def test_nested_captures_and_a_verification_within(tiny, decoder):
    """A capture around a verification stays in force after it."""
    want, dec = decoder().verify(DRAFTS), decoder()
    with query_capture():
        with query_capture():
            same(dec.verify(DRAFTS), want)
        assert modeling_qwen2.apply_rotary_pos_emb is not ORIG
        q = torch.randn(1, 4, 2, 64)
        cos, sin = torch.randn(1, 2, 64), torch.randn(1, 2, 64)
        rotated, _ = modeling_qwen2.apply_rotary_pos_emb(q, q, cos, sin)
        assert take_captured_query() is rotated and torch.equal(rotated, ORIG(q, q, cos, sin)[0])
    assert modeling_qwen2.apply_rotary_pos_emb is ORIG


@pytest.mark.parametrize("own", ["arguments", "another function"])
def test_a_layer_that_rotates_by_itself(tiny, decoder, monkeypatch, own):
    """A rotary call that is not deferred after layers whose was: its queries and
    keys are not turned again."""
    want, dec = decoder().verify(DRAFTS), decoder()
    state = SimpleNamespace(layer=0)
    handles = [between_layers(tiny[1], i, lambda i=i: setattr(state, "layer", i)) for i in range(3)]

    attention = type(tiny[1].model.layers[0].self_attn)
    forward = attention.forward

    def in_its_own_way(self, *args, **kwargs):
        if state.layer == 0:
            return forward(self, *args, **kwargs)
        hooked = modeling_qwen2.apply_rotary_pos_emb
        # (Layer 1 and 2: another layout given, or a function that no one wraps.)
        other = (lambda q, k, cos, sin: hooked(q, k, cos, sin, unsqueeze_dim=1)) if own == "arguments" else ORIG
        modeling_qwen2.apply_rotary_pos_emb = other
        try:
            return forward(self, *args, **kwargs)
        finally:
            modeling_qwen2.apply_rotary_pos_emb = hooked

    monkeypatch.setattr(attention, "forward", in_its_own_way)
    try:
        same(dec.verify(DRAFTS), want)
    finally:
        for h in handles:
            h.remove()
    assert modeling_qwen2.apply_rotary_pos_emb is ORIG


@pytest.mark.parametrize("second", ["verify", "plain step"])
def test_two_decoders_of_one_model_in_two_threads(tiny, decoder, second):
    """One thread's forward ends in the middle of the other's, whose layers go on
    as they began; afterwards the model is as it was."""
    cfg, model = tiny
    before = cfg._attn_implementation

    def run(dec):
        return dec.verify(DRAFTS).logits if dec.tree_size else dec.step(DRAFTS[:, :1])

    def make():
        dec = decoder()
        if second == "verify":
            return dec
        cache = SimpleNamespace(layers=[SimpleNamespace(keys=k[:, :, :20], values=v[:, :, :20])
                                        for k, v in zip(dec.k_buf, dec.v_buf)], get_seq_length=lambda: 20)
        return decode.CompressedDecoder(model, cache, max_new_tokens=16, use_graph=False)

    want = [run(decoder()), run(make())]
    first, other, got = decoder(), make(), [None, None]
    inside, go_on = threading.Event(), threading.Event()   # the second's forward has begun; the first's is over
    ids = {}

    def wait(*a):
        me = threading.get_ident()
        if me == ids.get("first"):
            assert inside.wait(30)
        elif me == ids.get("second"):
            inside.set()
            assert go_on.wait(30)

    handle = model.model.layers[1].register_forward_pre_hook(wait)

    def in_thread(name, i, dec):
        ids[name] = threading.get_ident()
        got[i] = run(dec)

    a = threading.Thread(target=in_thread, args=("first", 0, first))
    b = threading.Thread(target=in_thread, args=("second", 1, other))
    try:
        a.start()
        b.start()
        a.join(60)
        go_on.set()
        b.join(60)
    finally:
        handle.remove()
    for g, w in zip(got, want):
        assert g is not None and torch.equal(g, w)
    assert cfg._attn_implementation == before and modeling_qwen2.apply_rotary_pos_emb is ORIG
