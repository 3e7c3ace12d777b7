"""The decoder's ``verify`` for a batch whose sequences accept unequal numbers of
tokens, round after round: every node's logits are those of its path fed token
by token to a decoder without trees, and each sequence advances on its own."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = dict(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=3,
            num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=8192)


@pytest.mark.parametrize("evicted", [False, True])
@pytest.mark.parametrize("use_graph", [False, True])
def test_unequal_paths(gpu, use_graph, evicted):
    """After 20 rows, where a grandparent left out of a node's mask moves this
    model's logits by about 0.2 and a wrong depth by 0.1, and after 1024 of which a
    tenth are kept.  The tolerance is the one of the decoder's other tests: bf16
    activations rounded at other places."""
    import verify_walk
    from transformers import DynamicCache
    from dropkv_amd import hf_cache
    from dropkv_amd.e2e_qwen2 import build_model, make_config, prefill, random_prompt
    cfg = make_config(**TINY)
    model = build_model(cfg, gpu, dtype=torch.bfloat16, seed=0)
    if evicted:
        cache = hf_cache.DropKVCache(cfg, keep_ratio=0.1)
        tok = prefill(model, random_prompt(cfg.vocab_size, 1024, batch=2, seed=21, device=gpu), cache)
    else:
        cache = DynamicCache(config=cfg)
        with torch.no_grad():
            out = model(random_prompt(cfg.vocab_size, 20, batch=2, seed=21, device=gpu), past_key_values=cache,
                        use_cache=True, logits_to_keep=1)
        tok = out.logits[:, -1].argmax(-1, keepdim=True)
    verify_walk.check(model, cache, tok, use_graph, 3e-2)
