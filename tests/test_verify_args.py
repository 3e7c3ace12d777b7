"""Argument checks and workspace sizes of the verification-step entry points
(drafted-token attention, accepted rows, norms and rotation, log
probabilities): every refusal comes before anything is enqueued.  CPU only."""

import os
import re
import threading

import pytest
import torch

from dropkv_amd import _lib, ops

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dropkv_amd.h")
FAKE = 1 << 20   # a pointer that is never dereferenced: the checks fail first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from dropkv_amd import _build
        _build.build()
    return _lib.load()


def args(name, **values):
    """The argument structure of ``name``: the values given, else 0."""
    fields = [f.removesuffix(":d") for f in _lib.ARG_FIELDS[name].split()]
    assert not set(values) - set(fields), set(values) - set(fields)
    return _lib.ARGS[name].pack(*[values.get(f, 0) for f in fields])


def test_structures_match_the_header():
    """Fields of the header's structures, in order (arrays spelled out)."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    for name, fields in _lib.ARG_FIELDS.items():
        body = re.search(r"typedef struct \{([^}]*)\} " + name + "_args;", text).group(1)
        want = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            kind, names = re.match(r"((?:const )?\w+\s*\*?)\s*(.*)", decl, re.S).groups()
            for n in (x.strip() for x in names.split(",")):
                m = re.match(r"(\w+)\[(\d)\]", n)
                want += [(m.group(1), "q")] * int(m.group(2)) if m else [(n, "d" if kind.strip() == "double" else "q")]
        got = [f.removesuffix(":d") for f in fields.split()]
        assert len(got) == len(want), name
        for g, (w, kind) in zip(got, want):
            # (an element of x_s[] is spelled x_ and the axis)
            assert g == w or (w.endswith("_s") and g.startswith(w)) , (name, g, w)
        assert _lib.ARGS[name].format == "@" + "".join(k for _, k in want)
        assert _lib.ARGS[name].size == 8 * len(want)


def refused(lib, rc, code, msg):
    assert rc == code, (rc, lib.dropkv_last_error())
    assert msg in lib.dropkv_last_error().decode()


def test_tree_workspace(lib):
    size = lib.dropkv_tree_workspace_bytes
    assert size(1, 32, 8, 128, 16, 3392) > 0
    for bad in [(0, 32, 8, 128, 16, 100), (1, 30, 8, 128, 16, 100), (1, 32, 8, 96, 16, 100), (1, 32, 8, 128, 0, 100),
                (1, 32, 8, 128, 257, 100), (1, 32, 8, 128, 16, -1), (1, 32, 8, 128, 16, 1 << 24),
                (1 << 13, 32, 8, 128, 256, 100)]:
        assert size(*bad) == 0, bad


@pytest.mark.parametrize("change,code,msg", [
    (dict(q=0), 1, "null pointer"),
    (dict(workspace=0), 1, "null pointer"),
    (dict(dtype=3), 1, "bf16 or fp16"),
    (dict(Hq=30), 1, "Hkv | Hq"),
    (dict(B=0), 1, "must be positive"),
    (dict(T=0), 2, "T must be in"),
    (dict(T=257), 2, "T must be in"),
    (dict(D=80), 2, "head dim 80"),
    (dict(capacity=-1), 1, "capacity"),
    (dict(k_cache=0), 1, "null pointer"),
    (dict(capacity=(1 << 23) + 1), 1, "capacity"),
    (dict(B=1 << 17), 2, "B*Hq*T"),
    (dict(n_sb=2), 1, "n_sb"),
    (dict(scale=0.0), 1, "scale"),
    (dict(scale=-0.1), 1, "scale"),
    (dict(scale=float("nan")), 1, "scale"),
    (dict(scale=float("inf")), 1, "scale"),
    (dict(k_cache=FAKE + 8), 1, "16-byte aligned"),
    (dict(workspace_bytes=1000), 3, "workspace too small"),
    (dict(workspace_bytes=-1), 3, "workspace too small"),
])
def test_tree_attention(lib, change, code, msg):
    good = dict(q=FAKE, k_new=FAKE, v_new=FAKE, k_cache=FAKE, v_cache=FAKE, n_rows=FAKE, out=FAKE, workspace=FAKE,
                dtype=1, B=1, Hq=32, Hkv=8, T=8, D=128, capacity=300, scale=0.1, workspace_bytes=1 << 40)
    refused(lib, lib.dropkv_tree_attention(args("dropkv_tree_attention", **{**good, **change}), None), code, msg)


@pytest.mark.parametrize("change,code,msg", [
    (dict(tokens=0), 1, "null pointer"),
    (dict(elem_bytes=8), 1, "elem_bytes"),
    (dict(N=0), 1, "must be positive"),
    (dict(T=0), 2, "T must be in"),
    (dict(T=300), 2, "T must be in"),
    (dict(D=5000), 2, "too large"),
    (dict(N=1 << 20, B=1 << 12), 2, "too large"),
    (dict(p_sb=3), 1, "p_sb"),
    (dict(n_sb=-1), 1, "strides"),
])
def test_tree_commit(lib, change, code, msg):
    good = dict(tokens=FAKE, parents=FAKE, choice=FAKE, path=FAKE, accepted=FAKE, k_new=FAKE, v_new=FAKE, k_cache=FAKE,
                v_cache=FAKE, n_rows=FAKE, elem_bytes=2, N=1, B=1, H=8, T=8, D=128, capacity=100)
    refused(lib, lib.dropkv_tree_commit(args("dropkv_tree_commit", **{**good, **change}), None), code, msg)


ROPE = dict(q=FAKE, q_out=FAKE, k=FAKE, k_out=FAKE, cos=FAKE, sin=FAKE, c_dtype=3, c_sl=64, c_rows=10, dtype=1, B=1,
            Hq=8, Hkv=2, L=4, D=64, R=64, eps=1e-6)


@pytest.mark.parametrize("change,code,msg", [
    (dict(q=0), 1, "null pointer"),
    (dict(v=FAKE), 1, "null pointer"),
    (dict(dtype=4), 1, "bf16, fp16 or fp32"),
    (dict(c_dtype=2), 1, "c_dtype"),
    (dict(q_w=FAKE, w_dtype=2), 1, "w_dtype"),
    (dict(D=1), 2, "head dim"),
    (dict(D=4098), 2, "head dim"),
    (dict(R=63), 1, "R must be"),
    (dict(R=0), 1, "R must be"),
    (dict(R=66), 1, "R must be"),
    (dict(positions=FAKE, c_rows=0), 1, "c_rows"),
    (dict(eps=-1.0), 1, "eps"),
    (dict(eps=float("nan")), 1, "eps"),
    (dict(B=1 << 20, L=1 << 10), 2, "above"),
    (dict(Hkv=0), 1, "invalid shape"),
])
def test_norm_rope(lib, change, code, msg):
    refused(lib, lib.dropkv_norm_rope(args("dropkv_norm_rope", **{**ROPE, **change}), None), code, msg)


def test_norm_rope_of_nothing(lib):
    assert lib.dropkv_norm_rope(args("dropkv_norm_rope", **{**ROPE, "L": 0}), None) == 0


@pytest.mark.parametrize("change,code,msg", [
    (dict(logits=0), 1, "null pointer"),
    (dict(tokens=FAKE), 1, "go together"),
    (dict(dtype=0), 1, "bf16, fp16 or fp32"),
    (dict(V=0), 1, "V must be positive"),
    (dict(V=(1 << 30) + 1), 2, "too large"),
    (dict(top=-1), 1, "top must be"),
    (dict(V=5, top=6), 1, "top must be"),
    (dict(top=33), 2, "above 32"),
    (dict(top=4, top_ids=0), 1, "null top"),
    (dict(workspace=0), 3, "workspace too small"),
    (dict(workspace_bytes=64), 3, "workspace too small"),
])
def test_token_logprobs(lib, change, code, msg):
    good = dict(logits=FAKE, row_stride=100000, dtype=1, N=2, V=100000, top=4, entropy=FAKE, top_logprobs=FAKE,
                top_ids=FAKE, workspace=FAKE, workspace_bytes=1 << 40)
    refused(lib, lib.dropkv_token_logprobs(args("dropkv_token_logprobs", **{**good, **change}), None), code, msg)


def test_token_logprobs_workspace(lib):
    size = lib.dropkv_token_logprobs_workspace_bytes
    assert size(1, 151936, 5) > 0 and size(100000, 1000, 5) > 0 and size(100000, 1000, 1) == 0
    for bad in [(0, 10, 1), (1, 0, 0), (1, 10, 11), (1, 100, 33), (1, 100, -1), (1, (1 << 30) + 1, 1)]:
        assert size(*bad) == 0, bad
    assert lib.dropkv_token_logprobs(args("dropkv_token_logprobs", V=5, dtype=1), None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8)
    q, k, c = torch.zeros(1, 4, 3, 64).bfloat16(), torch.zeros(1, 2, 3, 64).bfloat16(), torch.zeros(3, 64)
    n = torch.zeros(1, dtype=torch.int32)
    t = torch.zeros(1, 3, dtype=torch.int64)
    for call in (lambda: ops.token_logprobs(x), lambda: ops.norm_rope(q, k, c, c),
                 lambda: ops.tree_attention(q, k, k, k, k, n, 0.1),
                 lambda: ops.tree_commit(t, t[0].int(), t, k, k, k, k, n)):
        with pytest.raises(RuntimeError, match="device"):
            call()


def test_threads_have_their_own_workspace(monkeypatch):
    """A call is several kernels: another thread's, on the same stream, may come
    between them."""
    monkeypatch.setattr(ops, "_shared_ws", {})
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "_evict_workspace", lambda nbytes, dev: torch.zeros(nbytes, dtype=torch.uint8))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    dev = torch.device("cuda", 0)
    mine, theirs = ops._stream_workspace(100, dev), []
    thread = threading.Thread(target=lambda: theirs.append(ops._stream_workspace(50, dev)))
    thread.start()
    thread.join()
    assert ops._stream_workspace(60, dev) is mine and theirs[0] is not mine
    assert ops._stream_workspace(200, dev).numel() == 200
