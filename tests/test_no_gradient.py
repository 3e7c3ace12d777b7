"""The verification-step operators have no gradient: inputs that need one, and
inputs that carry a tangent, are refused before anything is enqueued.  CPU only
(the device check, which comes first, is taken out)."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from dropkv_amd import ops


def calls():
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    n, t = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int64)
    return {
        "tree_attention": (dict(q=z(1, 4, 3, 64), k_new=z(1, 2, 3, 64), v_new=z(1, 2, 3, 64), k_cache=z(1, 2, 9, 64),
                                v_cache=z(1, 2, 9, 64), n_rows=n, scale=0.1, out=z(1, 3, 4, 64)),
                           ("q", "k_new", "v_new", "k_cache", "v_cache", "out")),
        "tree_commit": (dict(tokens=t, parents=t[0].int(), choice=t, k_new=z(1, 2, 3, 64), v_new=z(1, 2, 3, 64),
                             k_cache=z(1, 2, 9, 64), v_cache=z(1, 2, 9, 64), n_rows=n),
                        ("k_new", "v_new", "k_cache", "v_cache")),
        "norm_rope": (dict(q=z(1, 4, 3, 64), k=z(1, 2, 3, 64), cos=z(3, 64), sin=z(3, 64), q_weight=z(64),
                           k_weight=z(64), v=z(1, 2, 3, 64), q_out=z(1, 4, 3, 64), k_out=z(1, 2, 3, 64), v_out=z(1, 2, 3, 64)),
                      ("q", "k", "v", "cos", "sin", "q_weight", "k_weight", "q_out", "k_out", "v_out")),
        "token_logprobs": (dict(logits=z(2, 50)), ("logits",)),
    }


CASES = [(op, name) for op, (_, names) in calls().items() for name in names]


@pytest.fixture(autouse=True)
def no_device_check(monkeypatch):
    monkeypatch.setattr(ops, "_device_index", lambda name, *ts: 0)

    def enqueued(*args):
        raise AssertionError("reached the entry point")

    monkeypatch.setattr(ops, "_call", enqueued)


@pytest.mark.parametrize("op,name", CASES)
def test_inputs_that_need_a_gradient(op, name):
    values = calls()[op][0]
    with pytest.raises(RuntimeError, match="no gradient"):
        getattr(ops, op)(**{**values, name: values[name].requires_grad_()})


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("op,name", CASES)
def test_inputs_that_carry_a_tangent(op, name, grad):
    """Forward mode stays on under no_grad."""
    values = calls()[op][0]
    with torch.set_grad_enabled(grad), fwad.dual_level():
        dual = fwad.make_dual(values[name], torch.ones_like(values[name]))
        with pytest.raises(RuntimeError, match="no gradient"):
            getattr(ops, op)(**{**values, name: dual})


@pytest.mark.parametrize("op", calls())
def test_plain_inputs_beside_them(op, monkeypatch):
    """Under a dual level, or with gradients on, tensors without either go on."""
    monkeypatch.setattr(ops, "_stream_workspace", lambda nbytes, dev: torch.empty(nbytes, dtype=torch.uint8))
    with fwad.dual_level(), pytest.raises(AssertionError, match="reached the entry point"):
        getattr(ops, op)(**calls()[op][0])
