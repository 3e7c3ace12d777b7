"""Workspaces that begin anywhere, of which only the first DROPKV_SYNC_BYTES are zero: the
counters lie in those, and are zero again afterwards."""

import pytest
import torch

from dropkv_amd import _lib
from test_gpu_quant import BF, I8, attention_case, counts

pytestmark = pytest.mark.gpu


def call(name, gpu, need, offset, **values):
    """One call through the C ABI on a workspace at `offset` bytes, all ones behind its zeros."""
    fields = [f.split(":")[0] for f in _lib.ARG_FIELDS[name].split()]
    assert set(values) <= set(fields)
    buf = torch.full((need + 64,), 0xff, dtype=torch.uint8, device=gpu)
    ws = buf[offset:offset + need]
    ws[:_lib.SYNC_BYTES] = 0
    values.update(workspace=ws.data_ptr(), workspace_bytes=need)
    for _ in range(2):
        rc = getattr(_lib.load(), name)(_lib.ARGS[name].pack(*[values.get(f, 0) for f in fields]),
                                        torch.cuda.current_stream().cuda_stream)
        assert rc == 0, _lib.load().dropkv_last_error()
        torch.cuda.synchronize()
        assert not ws[:_lib.SYNC_BYTES].any()
    assert (buf[:offset] == 0xff).all() and (buf[offset + need:] == 0xff).all()


@pytest.mark.parametrize("offset", [0, 1, 4, 8, 15])
@pytest.mark.parametrize("B", [1024, 1023, 512, 256, 32, 1])
def test_verify_drafts(gpu, B, offset):
    """Rows of two workgroups each: the second to arrive draws the token."""
    from dropkv_amd import ops
    T, V = 2, 5000
    g = torch.Generator(device=gpu).manual_seed(B)
    x = torch.randn(B, T, V, generator=g, device=gpu).to(BF)
    tok = torch.randint(0, V, (B, T), generator=g, device=gpu)
    u = torch.rand(B, T, generator=g, device=gpu)
    want = ops.verify_drafts(x, tok, u)
    choice, accepted, lp = torch.empty_like(tok), torch.empty(B, dtype=torch.int32, device=gpu), torch.empty_like(u)
    need = _lib.load().dropkv_verify_drafts_workspace_bytes(B, T, V, 0)
    call("dropkv_verify_drafts", gpu, need, offset, logits=x.data_ptr(), x_sb=T * V, x_st=V, tokens=tok.data_ptr(),
         uniforms=u.data_ptr(), dtype=_lib.DROPKV_BF16, B=B, T=T, V=V, temperature=1.0, choice=choice.data_ptr(),
         accepted=accepted.data_ptr(), logprobs=lp.data_ptr())
    assert torch.equal(choice, want.choice) and torch.equal(accepted, want.accepted) and torch.equal(lp, want.logprobs)


@pytest.mark.parametrize("offset", [0, 1, 4, 8, 15])
@pytest.mark.parametrize("B,T", [(1, 1), (2, 3), (1, 20)])
def test_quant_attention(gpu, B, T, offset):
    """Parts joined by the last workgroup, and by a second kernel."""
    from dropkv_amd import ops
    n = [1000, 700][:B]
    q, k, v, kn, vn, cache, _, scale = attention_case(gpu, 8, 2, 128, T, n, BF, I8, mask=None)
    n_rows = counts(gpu, *n)
    want = ops.quant_attention(q, kn, vn, cache, n_rows, scale)
    out = torch.empty_like(want)
    need = _lib.load().dropkv_quant_workspace_bytes(B, 8, 2, 128, T, cache.capacity)
    names = "k v k_scale v_scale k_tail v_tail".split()
    call("dropkv_quant_attention", gpu, need, offset, q=q.data_ptr(), q_sb=q.stride(0), q_sh=q.stride(1), q_st=q.stride(2),
         k_new=kn.data_ptr(), kn_sb=kn.stride(0), kn_sh=kn.stride(1), kn_st=kn.stride(2), v_new=vn.data_ptr(),
         vn_sb=vn.stride(0), vn_sh=vn.stride(1), vn_st=vn.stride(2), **dict(zip(names, cache.pointers())),
         n_rows=n_rows.data_ptr(), n_sb=int(B > 1), dtype=cache.codes[0], store=cache.codes[1], B=B, Hq=8, Hkv=2, T=T, D=128,
         capacity=cache.capacity, scale=scale, out=out.data_ptr(), o_sb=out.stride(0), o_st=out.stride(1), o_sh=out.stride(2))
    assert torch.equal(out, want)
