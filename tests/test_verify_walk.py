"""What the decoder makes of trees of drafted tokens (masks, depths, paths, rows
and positions of each sequence), on the CPU in fp32 with PyTorch operators.

Tolerance: the two sides add the same products in other orders, a few hundred
fp32 roundings (2^-24 each) through three layers of sums of at most 256 terms."""

import pytest
import torch

pytest.importorskip("transformers")

from transformers import DynamicCache  # noqa: E402

import cpu_ops  # noqa: E402
import verify_walk  # noqa: E402
from dropkv_amd import decode  # noqa: E402
from dropkv_amd.e2e_qwen2 import build_model, make_config, random_prompt  # noqa: E402

TINY = dict(vocab_size=200, hidden_size=256, intermediate_size=256, num_hidden_layers=3,
            num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=512)


@pytest.fixture(scope="module")
def tiny():
    cfg = make_config(**TINY)
    return cfg, build_model(cfg, "cpu", dtype=torch.float32, seed=0)


def prefilled(cfg, model):
    cache = DynamicCache(config=cfg)
    with torch.no_grad():
        out = model(random_prompt(cfg.vocab_size, 20, batch=2, seed=1), past_key_values=cache, use_cache=True,
                    logits_to_keep=1)
    return cache, out.logits[:, -1].argmax(-1, keepdim=True)


def test_unequal_paths(tiny, monkeypatch):
    cpu_ops.install(monkeypatch)
    cache, tok = prefilled(*tiny)
    verify_walk.check(tiny[1], cache, tok, False, 1e-4)


@pytest.mark.parametrize("planted", ["mask", "depth", "rows"])
def test_the_check_sees_mistakes(tiny, monkeypatch, planted):
    """A mask of ancestors without the grandparents, depths that are node numbers,
    counts that advance alike: each is found."""
    cpu_ops.install(monkeypatch)
    set_tree, advance = decode.CompressedDecoder.set_tree, decode.CompressedDecoder._tree_advance

    def wrong_tree(self, parents):
        set_tree(self, parents)
        if planted == "mask":
            eye = torch.eye(self.tree_size, dtype=torch.bool)
            up = torch.nn.functional.one_hot(self._tree_parents.clamp(min=0).long(), self.tree_size).bool()
            self._tree_mask.copy_(eye | up)
        if planted == "depth":
            self._tree_depth.copy_(torch.arange(self.tree_size))

    def wrong_advance(self, v):
        advance(self, v._replace(accepted=v.accepted.max().expand_as(v.accepted)) if planted == "rows" else v)

    monkeypatch.setattr(decode.CompressedDecoder, "set_tree", wrong_tree)
    monkeypatch.setattr(decode.CompressedDecoder, "_tree_advance", wrong_advance)
    cache, tok = prefilled(*tiny)
    with pytest.raises(AssertionError):
        verify_walk.check(tiny[1], cache, tok, False, 1e-4)
