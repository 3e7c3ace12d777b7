"""Limits of the verification-step entry points that keep a launch within one
grid, and what they refuse beyond; CPU only."""

import os

import pytest

from dropkv_amd import _lib

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
