"""Argument checks and workspace sizes of the verification-step entry points
(drafted-token attention, accepted rows, norms and rotation, log
probabilities): every refusal comes before anything is enqueued.  CPU only."""

import ctypes
import os

import pytest
import torch

from dropkv_amd import _lib, ops

FAKE = ctypes.c_void_p(1 << 20)   # never dereferenced: the checks fail first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from dropkv_amd import _build
        _build.build()
    return _lib.load()


def refused(lib, rc, code, msg):
    assert rc == code, (rc, lib.dropkv_last_error())
    assert msg in lib.dropkv_last_error().decode()


def test_tree_workspace(lib):
    size = lib.dropkv_tree_workspace_bytes
    assert size(1, 32, 8, 128, 16, 3392) > 0
    for bad in [(0, 32, 8, 128, 16, 100), (1, 30, 8, 128, 16, 100), (1, 32, 8, 96, 16, 100), (1, 32, 8, 128, 0, 100),
                (1, 32, 8, 128, 257, 100), (1, 32, 8, 128, 16, 0), (1, 32, 8, 128, 16, 1 << 24),
                (1 << 13, 32, 8, 128, 256, 100)]:
        assert size(*bad) == 0, bad


@pytest.mark.parametrize("change,code,msg", [
    (dict(q=None), 1, "null pointer"),
    (dict(ws=None), 1, "null pointer"),
    (dict(dtype=3), 1, "bf16 or fp16"),
    (dict(Hq=30), 1, "Hkv | Hq"),
    (dict(B=0), 1, "must be positive"),
    (dict(T=0), 2, "T must be in"),
    (dict(T=257), 2, "T must be in"),
    (dict(D=80), 2, "head dim 80"),
    (dict(C=0), 1, "capacity"),
    (dict(C=(1 << 23) + 1), 1, "capacity"),
    (dict(B=1 << 17), 2, "B*Hq*T"),
    (dict(n_sb=2), 1, "n_sb"),
    (dict(k=ctypes.c_void_p((1 << 20) + 8)), 1, "16-byte aligned"),
    (dict(ws_bytes=1000), 3, "workspace too small"),
])
def test_tree_attention(lib, change, code, msg):
    a = dict(q=FAKE, k=FAKE, ws=FAKE, dtype=1, B=1, Hq=32, Hkv=8, T=8, D=128, C=300, n_sb=0, ws_bytes=1 << 40)
    a.update(change)
    rc = lib.dropkv_tree_attention(a["q"], 0, 0, 0, FAKE, 0, 0, 0, FAKE, 0, 0, 0, a["k"], FAKE, FAKE, a["n_sb"], None,
                                   0, 0, 0, a["dtype"], a["B"], a["Hq"], a["Hkv"], a["T"], a["D"], a["C"], 0.1, FAKE,
                                   0, 0, 0, a["ws"], a["ws_bytes"], None)
    refused(lib, rc, code, msg)


@pytest.mark.parametrize("change,code,msg", [
    (dict(tok=None), 1, "null pointer"),
    (dict(eb=8), 1, "elem_bytes"),
    (dict(N=0), 1, "must be positive"),
    (dict(T=0), 2, "T must be in"),
    (dict(T=300), 2, "T must be in"),
    (dict(D=5000), 2, "too large"),
    (dict(N=1 << 20, B=1 << 12), 2, "too large"),
    (dict(p_sb=3), 1, "p_sb"),
    (dict(n_sb=-1), 1, "strides"),
])
def test_tree_commit(lib, change, code, msg):
    a = dict(tok=FAKE, eb=2, N=1, B=1, T=8, D=128, p_sb=0, n_sb=0)
    a.update(change)
    rc = lib.dropkv_tree_commit(a["tok"], FAKE, a["p_sb"], FAKE, FAKE, FAKE, FAKE, 0, 0, 0, 0, FAKE, 0, 0, 0, 0, FAKE,
                                FAKE, FAKE, 0, a["n_sb"], a["eb"], a["N"], a["B"], 8, a["T"], a["D"], 100, None)
    refused(lib, rc, code, msg)


@pytest.mark.parametrize("change,code,msg", [
    (dict(q=None), 1, "null pointer"),
    (dict(v=FAKE), 1, "v without"),
    (dict(dtype=4), 1, "bf16, fp16 or fp32"),
    (dict(c_dtype=2), 1, "c_dtype"),
    (dict(w=FAKE, w_dtype=2), 1, "w_dtype"),
    (dict(D=1), 2, "head dim"),
    (dict(D=4098), 2, "head dim"),
    (dict(R=63), 1, "R must be"),
    (dict(R=0), 1, "R must be"),
    (dict(R=66), 1, "R must be"),
    (dict(pos=FAKE, rows=0), 1, "c_rows"),
    (dict(eps=-1.0), 1, "eps"),
    (dict(eps=float("nan")), 1, "eps"),
    (dict(B=1 << 20, L=1 << 10), 2, "above"),
    (dict(Hkv=0), 1, "invalid shape"),
])
def test_norm_rope(lib, change, code, msg):
    a = dict(q=FAKE, v=None, dtype=1, c_dtype=3, w=None, w_dtype=0, pos=None, rows=10, B=1, Hkv=2, L=4, D=64, R=64,
             eps=1e-6)
    a.update(change)
    s = (ctypes.c_int64 * 3)()
    rc = lib.dropkv_norm_rope(a["q"], s, FAKE, s, FAKE, s, FAKE, s, a["v"], None, None, None, a["w"], None,
                              a["w_dtype"], FAKE, FAKE, a["c_dtype"], 0, 64, a["pos"], 0, a["rows"], a["dtype"],
                              a["B"], 8, a["Hkv"], a["L"], a["D"], a["R"], a["eps"], None)
    refused(lib, rc, code, msg)


def test_norm_rope_of_nothing(lib):
    s = (ctypes.c_int64 * 3)()
    assert lib.dropkv_norm_rope(FAKE, s, FAKE, s, FAKE, s, FAKE, s, None, None, None, None, None, None, 0, FAKE, FAKE,
                                3, 0, 64, None, 0, 0, 1, 2, 8, 2, 0, 64, 64, 1e-6, None) == 0


@pytest.mark.parametrize("change,code,msg", [
    (dict(x=None), 1, "null pointer"),
    (dict(tok=FAKE, lp=None), 1, "go together"),
    (dict(dtype=0), 1, "bf16, fp16 or fp32"),
    (dict(V=0), 1, "V must be positive"),
    (dict(V=(1 << 30) + 1), 2, "too large"),
    (dict(top=-1), 1, "top must be"),
    (dict(V=5, top=6), 1, "top must be"),
    (dict(top=33), 2, "above 32"),
    (dict(top=4, ids=None), 1, "null top"),
    (dict(ws=None), 3, "workspace too small"),
    (dict(ws_bytes=64), 3, "workspace too small"),
])
def test_token_logprobs(lib, change, code, msg):
    a = dict(x=FAKE, tok=None, lp=None, dtype=1, N=2, V=100000, top=4, ids=FAKE, ws=FAKE, ws_bytes=1 << 40)
    a.update(change)
    rc = lib.dropkv_token_logprobs(a["x"], a["V"], a["dtype"], a["N"], a["V"], a["tok"], a["top"], a["lp"], FAKE, FAKE,
                                   a["ids"], a["ws"], a["ws_bytes"], None)
    refused(lib, rc, code, msg)


def test_token_logprobs_workspace(lib):
    size = lib.dropkv_token_logprobs_workspace_bytes
    assert size(1, 151936, 5) > 0 and size(100000, 1000, 5) == 0
    for bad in [(0, 10, 1), (1, 0, 0), (1, 10, 11), (1, 100, 33), (1, 100, -1), (1, (1 << 30) + 1, 1)]:
        assert size(*bad) == 0, bad
    assert lib.dropkv_token_logprobs(None, 0, 1, 0, 5, None, 0, None, None, None, None, None, 0, None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8)
    q, k, c = torch.zeros(1, 4, 3, 64).bfloat16(), torch.zeros(1, 2, 3, 64).bfloat16(), torch.zeros(3, 64)
    n = torch.zeros(1, dtype=torch.int32)
    t = torch.zeros(1, 3, dtype=torch.int64)
    for call in (lambda: ops.token_logprobs(x), lambda: ops.norm_rope(q, k, c, c),
                 lambda: ops.tree_attention(q, k, k, k, k, n, 0.1),
                 lambda: ops.tree_commit(t, t[0].int(), t, k, k, k, k, n)):
        with pytest.raises(RuntimeError, match="cuda"):
            call()
