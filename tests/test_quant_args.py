"""Argument checks, workspace sizes and refusals of the entry points of a cache in 8
bits and of the verification by sampling: every refusal comes before anything is
enqueued.  CPU only."""

import os

import pytest
import torch
import torch.autograd.forward_ad as fwad

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
    assert not set(values) - set(fields), set(values) - set(fields)
    return _lib.ARGS[name].pack(*[values.get(f, 0) for f in fields])


def refused(lib, name, values, code, msg):
    rc = getattr(lib, name)(args(name, **values), None)
    assert rc == code, (rc, lib.dropkv_last_error())
    assert msg in lib.dropkv_last_error().decode()


CACHE = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, k_tail=FAKE, v_tail=FAKE, dtype=1, store=4, B=2, D=64,
             capacity=640)
CACHE_BAD = [
    (dict(k=0), 1, "null pointer"), (dict(v_tail=0), 1, "null pointer"), (dict(k_scale=0), 1, "null pointer"),
    (dict(dtype=3), 1, "bf16 or fp16"), (dict(store=1), 1, "int8 or e4m3"), (dict(store=6), 1, "int8 or e4m3"),
    (dict(D=96), 2, "head dim 96"), (dict(k=FAKE + 8), 1, "16-byte aligned"), (dict(v_tail=FAKE + 2), 1, "16-byte aligned"),
    (dict(v_scale=FAKE + 2), 1, "4-byte aligned"), (dict(B=0), 1, "must be positive"),
]
ROWS_BAD = [(dict(capacity=600), 1, "multiple of 64"), (dict(capacity=0), 1, "multiple of 64"),
            (dict(capacity=(1 << 24) + 64), 1, "2^30"), (dict(N=0), 1, "must be positive"), (dict(H=0), 1, "must be positive"),
            (dict(n_rows=0), 1, "null pointer"), (dict(n_sn=-1), 1, "n_rows")]


@pytest.mark.parametrize("change,code,msg", CACHE_BAD + ROWS_BAD + [
    (dict(k_new=0), 1, "null pointer"), (dict(L=-1), 1, "L out of range"), (dict(L=1 << 31), 1, "L out of range"),
    (dict(N=1 << 20, B=8), 2, "too large"), (dict(L=1 << 30), 2, "too large")])
def test_append(lib, change, code, msg):
    refused(lib, "dropkv_quant_append", dict(CACHE, k_new=FAKE, v_new=FAKE, n_rows=FAKE, N=1, H=2, L=5, **{}) | change, code, msg)


@pytest.mark.parametrize("change,code,msg", CACHE_BAD + ROWS_BAD + [
    (dict(k_out=0), 1, "null pointer"), (dict(v_out=FAKE + 4), 1, "outputs"), (dict(L=-1), 1, "outside"),
    (dict(row0=-1), 1, "outside"), (dict(row0=640), 1, "outside"), (dict(L=641), 1, "outside"),
    (dict(row0=(1 << 63) - 1), 1, "outside"), (dict(N=1 << 22), 2, "too large")])
def test_read(lib, change, code, msg):
    refused(lib, "dropkv_quant_read", dict(CACHE, n_rows=FAKE, k_out=FAKE, v_out=FAKE, N=1, H=2, L=5) | change, code, msg)


@pytest.mark.parametrize("change,code,msg", CACHE_BAD + [
    (dict(capacity=600), 1, "multiple of 64"), (dict(capacity=0), 1, "multiple of 64"),
    (dict(q=0), 1, "null pointer"), (dict(out=0), 1, "null pointer"), (dict(workspace=0), 1, "null pointer"),
    (dict(n_rows=0), 1, "null pointer"), (dict(n_sb=2), 1, "n_sb"), (dict(Hq=5), 1, "Hkv | Hq"), (dict(T=0), 2, "T must be in"),
    (dict(T=257), 2, "T must be in"), (dict(B=1 << 20, T=16), 2, "B*Hq*T"), (dict(scale=0.0), 1, "scale"),
    (dict(scale=float("nan")), 1, "scale"), (dict(scale=1e38), 1, "scale"), (dict(workspace_bytes=100), 3, "workspace too small"),
    (dict(workspace_bytes=-1), 3, "workspace too small")])
def test_attention(lib, change, code, msg):
    values = dict(CACHE, q=FAKE, k_new=FAKE, v_new=FAKE, n_rows=FAKE, Hq=4, Hkv=2, T=3, scale=0.1, out=FAKE, workspace=FAKE,
                  workspace_bytes=1 << 30)
    refused(lib, "dropkv_quant_attention", values | change, code, msg)


@pytest.mark.parametrize("change,code,msg", [
    (dict(logits=0), 1, "null pointer"), (dict(tokens=0), 1, "null pointer"), (dict(uniforms=0), 1, "null pointer"),
    (dict(choice=0), 1, "null pointer"), (dict(workspace=0), 1, "null pointer"), (dict(dtype=4), 1, "bf16, fp16 or fp32"),
    (dict(B=0), 1, "must be positive"), (dict(V=0), 1, "must be positive"), (dict(T=257), 2, "T must be"),
    (dict(V=(1 << 26) + 1), 2, "V too large"), (dict(B=1 << 16, T=2), 2, "B*(2*T-1)"), (dict(B=1 << 62), 2, "B*(2*T-1)"),
    (dict(B=200, V=1 << 26), 2, "B*V"), (dict(temperature=0.0), 1, "temperature"), (dict(temperature=-1.0), 1, "temperature"),
    (dict(temperature=float("inf")), 1, "temperature"), (dict(temperature=float("nan")), 1, "temperature"),
    (dict(temperature=1e-300), 1, "temperature"), (dict(workspace_bytes=64), 3, "workspace too small")])
def test_verify_drafts(lib, change, code, msg):
    values = dict(logits=FAKE, tokens=FAKE, uniforms=FAKE, dtype=1, B=2, T=3, V=1000, temperature=1.0, choice=FAKE,
                  accepted=FAKE, logprobs=FAKE, workspace=FAKE, workspace_bytes=1 << 30)
    refused(lib, "dropkv_verify_drafts", values | change, code, msg)


def test_workspaces(lib):
    size = lib.dropkv_quant_workspace_bytes
    assert size(1, 32, 8, 128, 16, 3392) > 0
    for bad in [(0, 32, 8, 128, 16, 64), (1, 30, 8, 128, 16, 64), (1, 32, 8, 96, 16, 64), (1, 32, 8, 128, 0, 64),
                (1, 32, 8, 128, 257, 64), (1, 32, 8, 128, 16, 63), (1, 32, 8, 128, 16, 1 << 24), (1 << 13, 32, 8, 128, 256, 64)]:
        assert size(*bad) == 0, bad
    size = lib.dropkv_verify_drafts_workspace_bytes
    assert size(2, 8, 151936, 1) > size(2, 8, 151936, 0) > 0
    for bad in [(0, 8, 100, 1), (1, 0, 100, 1), (1, 257, 100, 1), (1, 8, 0, 1), (1, 8, (1 << 26) + 1, 1)]:
        assert size(*bad) == 0, bad


# --- the wrappers ------------------------------------------------------------

@pytest.fixture
def no_device_check(monkeypatch):
    monkeypatch.setattr(ops, "_device_index", lambda name, *ts: 0)
    monkeypatch.setattr(ops, "_quant_device", lambda name, cache, *ts: 0)
    monkeypatch.setattr(ops, "_stream_workspace", lambda nbytes, dev: torch.empty(1, dtype=torch.uint8))

    def enqueued(*args):
        raise AssertionError("reached the entry point")

    monkeypatch.setattr(ops, "_call", enqueued)


def z(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, dtype=dtype)


def cache(**kw):
    return ops.quant_cache(2, 2, 100, 64, device="cpu", **kw)


def calls():
    n, i32 = torch.zeros(2, dtype=torch.int32), torch.int32
    return {
        "quant_append": dict(cache=cache(), k=z(2, 2, 3, 64), v=z(2, 2, 3, 64), n_rows=n, path=z(2, 3, dtype=i32),
                             counts=z(2, dtype=i32)),
        "quant_read": dict(cache=cache(), n_rows=n, rows=5, first=3),
        "quant_attention": dict(q=z(2, 4, 3, 64), k_new=z(2, 2, 3, 64), v_new=z(2, 2, 3, 64), cache=cache(), n_rows=n,
                                scale=0.1, out=z(2, 3, 4, 64), mask=z(2, 3, 3, dtype=torch.bool)),
        "verify_drafts": dict(logits=z(2, 3, 50), tokens=z(2, 3, dtype=torch.int64), uniforms=z(2, 3, dtype=torch.float32),
                              draft_logits=z(2, 2, 50)),
    }


WRONG = [
    ("quant_append", dict(k=z(2, 2, 3, 128)), "must be"), ("quant_append", dict(v=z(2, 2, 4, 64)), "must be"),
    ("quant_append", dict(k=z(2, 3, 64), v=z(2, 3, 64)), "must be"),
    ("quant_append", dict(k=z(2, 2, 3, 64, dtype=torch.float16)), "dtype"), ("quant_append", dict(n_rows=z(2)), "n_rows"),
    ("quant_append", dict(n_rows=z(3, dtype=torch.int32)), "n_rows"), ("quant_append", dict(n_rows=z(2, 1, dtype=torch.int32)), "n_rows"),
    ("quant_append", dict(counts=z(2, dtype=torch.int64)), "counts"), ("quant_append", dict(counts=z(1, dtype=torch.int32)), "counts"),
    ("quant_append", dict(path=z(2, 4, dtype=torch.int32)), "path"), ("quant_append", dict(path=z(2, 3, dtype=torch.int64)), "path"),
    ("quant_append", dict(cache=cache(layers=2)), "must be"),
    ("quant_read", dict(rows=126), "capacity"), ("quant_read", dict(first=-1), "capacity"), ("quant_read", dict(rows=-1), "capacity"),
    ("quant_read", dict(cache=cache(layers=2)), "n_rows"),
    ("quant_attention", dict(cache=cache(layers=2)), "one layer"), ("quant_attention", dict(cache=cache(dtype=torch.float16)), "dtype"),
    ("quant_attention", dict(q=z(2, 4, 64)), "q must be"), ("quant_attention", dict(q=z(1, 4, 3, 64)), "fit"),
    ("quant_attention", dict(v_new=z(2, 2, 4, 64)), "fit"), ("quant_attention", dict(n_rows=z(2)), "n_rows"),
    ("quant_attention", dict(mask=z(3, 3)), "mask"), ("quant_attention", dict(mask=z(1, 3, 3, dtype=torch.bool)), "mask"),
    ("quant_attention", dict(out=z(2, 4, 3, 64)), "out"), ("quant_attention", dict(workspace=z(4, 4).t()[:, ::2]), "contiguous"),
    ("verify_drafts", dict(logits=z(2, 50)), "logits"), ("verify_drafts", dict(logits=z(2, 3, 50, dtype=torch.float64)), "bf16"),
    ("verify_drafts", dict(tokens=z(2, 3, dtype=torch.int32)), "tokens"), ("verify_drafts", dict(tokens=z(2, 2, dtype=torch.int64)), "tokens"),
    ("verify_drafts", dict(uniforms=z(2, 3, dtype=torch.float64)), "uniforms"), ("verify_drafts", dict(draft_logits=z(2, 3, 50)), "draft_logits"),
    ("verify_drafts", dict(draft_logits=z(2, 2, 50, dtype=torch.float32)), "draft_logits"), ("verify_drafts", dict(temperature=0.0), "temperature"),
    ("verify_drafts", dict(temperature=float("nan")), "temperature"),
]


@pytest.mark.parametrize("op,change,msg", WRONG)
def test_wrong_arguments(no_device_check, op, change, msg):
    with pytest.raises(RuntimeError, match=msg):
        getattr(ops, op)(**{**calls()[op], **change})


@pytest.mark.parametrize("op", calls())
def test_right_arguments_go_on(no_device_check, op):
    with pytest.raises(AssertionError, match="reached the entry point"):
        getattr(ops, op)(**calls()[op])


@pytest.mark.parametrize("op", calls())
def test_inputs_that_need_a_gradient(no_device_check, op):
    values = calls()[op]
    for name, t in values.items():
        if not isinstance(t, torch.Tensor) or not t.is_floating_point():
            continue
        with pytest.raises(RuntimeError, match="no gradient"):
            getattr(ops, op)(**{**values, name: t.clone().requires_grad_()})
        with torch.no_grad(), fwad.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
            getattr(ops, op)(**{**values, name: fwad.make_dual(t, torch.ones_like(t))})


def test_tensors_elsewhere():
    """CPU tensors, and a cache on the CPU, are refused."""
    for op, values in calls().items():
        with pytest.raises(RuntimeError, match="one ROCm"):
            getattr(ops, op)(**values)


def test_caches(no_device_check):
    c = cache(layers=3)
    assert c.k.shape == (3, 2, 2, 128, 64) and c.v.shape == (3, 2, 2, 2, 64, 64) and c.capacity == 128
    assert c.k_tail.shape == (3, 2, 2, 128, 64) and c.k_scale.shape == (3, 2, 2, 2)
    one = c.layer(1)
    assert one.k.data_ptr() == c.k[1].data_ptr() and not one.layers
    with pytest.raises(RuntimeError, match="no axis"):
        one.layer(0)
    for kw in (dict(dtype=torch.float32), dict(store=torch.uint8), dict(layers=0)):
        with pytest.raises(RuntimeError, match="quant_cache"):
            cache(**kw)
    for shape in ((0, 2, 64, 64), (1, 0, 64, 64), (1, 1, 0, 64), (1, 1, 64, 96), (1, 1, (1 << 24) + 1, 64)):
        with pytest.raises(RuntimeError, match="quant_cache"):
            ops.quant_cache(*shape, device="cpu")
    parts = list(cache())
    for i, bad in ((0, z(2, 2, 100, 64, dtype=torch.int8)), (1, z(2, 2, 128, 64, dtype=torch.int8)), (2, z(2, 2, 2)),
                   (3, z(2, 2, 3, dtype=torch.float32)), (4, z(2, 2, 64, 64)), (5, z(2, 2, 128, 64, dtype=torch.float16)),
                   (0, parts[0].view(torch.float8_e4m3fn)), (0, parts[0].transpose(0, 1)),
                   (4, z(2, 2, 128, 64).requires_grad_())):
        with pytest.raises(RuntimeError, match="QuantCache"):
            ops.QuantCache(*(bad if j == i else t for j, t in enumerate(parts)))
