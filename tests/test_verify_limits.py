"""Limits of the verification-step entry points that keep a launch within one
grid and its writes within what the caller gave, and what they refuse beyond;
CPU only."""

import os

import pytest
import torch

from dropkv_amd import _lib, ops

FAKE = 1 << 20   # a pointer that is never dereferenced: the checks fail first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from dropkv_amd import _build
        _build.build()
    return _lib.load()


def args(name, **values):
    fields = [f.removesuffix(":d") for f in _lib.ARG_FIELDS[name].split()]
    return _lib.ARGS[name].pack(*[values.get(f, 0) for f in fields])


@pytest.mark.parametrize("N,B,H", [(1 << 12, 1 << 12, 1), (1, 1 << 24, 1), (3, 1 << 10, 1 << 13), (1 << 31, 1, 1),
                                   (1 << 40, 1 << 40, 1 << 40)])
def test_tree_commit(lib, N, B, H):
    """A workgroup of 256 for each of N * B * H heads: fewer than 2^24 of them."""
    good = dict(tokens=FAKE, parents=FAKE, choice=FAKE, path=FAKE, accepted=FAKE, k_new=FAKE, v_new=FAKE, k_cache=FAKE,
                v_cache=FAKE, n_rows=FAKE, elem_bytes=2, T=8, D=128, capacity=100)
    assert lib.dropkv_tree_commit(args("dropkv_tree_commit", **good, N=N, B=B, H=H), None) == 2
    assert "N*B*H too large" in lib.dropkv_last_error().decode()


def test_workspace_of_repeated_bytes(lib, monkeypatch):
    """A workspace whose bytes are fewer than its shape says, or lie apart, is
    refused before anything is enqueued."""
    monkeypatch.setattr(ops, "_device_index", lambda name, *ts: 0)

    def enqueued(*args):
        raise AssertionError("reached the entry point")

    monkeypatch.setattr(ops, "_call", enqueued)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    q, kn, kc, n = z(1, 4, 3, 64), z(1, 2, 3, 64), z(1, 2, 9, 64), torch.zeros(1, dtype=torch.int32)
    need = lib.dropkv_tree_workspace_bytes(1, 4, 2, 64, 3, 9)
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(need), torch.zeros(2 * need, dtype=torch.uint8)[::2]):
        assert ws.nbytes >= need
        with pytest.raises(RuntimeError, match="contiguous"):
            ops.tree_attention(q, kn, kn, kc, kc, n, 0.1, workspace=ws)
    with pytest.raises(AssertionError, match="reached the entry point"):
        ops.tree_attention(q, kn, kn, kc, kc, n, 0.1, workspace=torch.zeros(need // 4 + 1))
