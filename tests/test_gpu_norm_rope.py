"""Norms and rotation of queries and keys (``dropkv_norm_rope``) against the
formula in 64 bits.

Tolerance.  Each rotated value is a sum of two products; the norm's factor is
off by (D / 2 + 4) 2^-24 (the sum's additions, halved by the root, and the
root, quotient and products), a rotated value by 2 2^-24 of the two products'
magnitudes; the store adds half a step, and fp16 half its smallest number."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(x, cos, sin, w, eps):
    """x [B, H, L, D] and cos / sin [B, L, R] -> (z, bound) in 64 bits."""
    D, R = x.shape[-1], cos.shape[-1]
    y = x.double()
    rel = 0.0
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
        rel = (D / 2 + 6) * 2.0 ** -24
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = y[..., :R // 2], y[..., R // 2:R]
    z = torch.cat([a * c[..., :R // 2] - b * s[..., :R // 2], b * c[..., R // 2:] + a * s[..., R // 2:], y[..., R:]], -1)
    mag = torch.cat([(a * c[..., :R // 2]).abs() + (b * s[..., :R // 2]).abs(),
                     (b * c[..., R // 2:]).abs() + (a * s[..., R // 2:]).abs(), y[..., R:].abs()], -1)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    return z, mag * (rel + 2 * 2.0 ** -24) * 1.01 + z.abs() * torch.finfo(x.dtype).eps / 2 * 1.01 + tiny


def angles(L, R, seed, first=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.arange(first, first + L, dtype=torch.float64)[:, None] * torch.rand(R, generator=g, dtype=torch.float64)
    return a.cos().float(), a.sin().float()   # (the two halves differ: no value is taken for another)


@pytest.mark.parametrize("B,Hq,Hkv,L,D,R", [
    (1, 14, 2, 8, 64, 64),
    (1, 14, 2, 1, 64, 64),
    (2, 32, 8, 37, 128, 128),
    (1, 8, 8, 129, 128, 64),       # half of the head rotated
    (1, 4, 1, 5, 256, 256),
    (2, 3, 1, 11, 96, 96),         # lanes without values
    (2, 3, 1, 11, 80, 48),
    (1, 4, 2, 7, 192, 192),
    (1, 3, 1, 300, 48, 32),
    (1, 3, 2, 4, 16, 16),
    (1, 2, 1, 9, 240, 16),
    (2, 3, 1, 11, 100, 96),        # generic kernel
    (1, 2, 1, 3, 272, 272),
    (1, 5, 5, 4, 64, 24),          # a rotated width of no whole 16
    (1, 2, 2, 3, 6, 4),
    (1, 2, 1, 2, 1000, 998),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("norm", [False, True])
def test_rows(gpu, B, Hq, Hkv, L, D, R, dtype, norm):
    """Projections [B, L, H, D] seen as [B, H, L, D], each sequence's own rows
    of cos and sin, K and V into rows of cache buffers."""
    from dropkv_amd import ops
    g = torch.Generator().manual_seed(D + L)
    q, k, v = (torch.randn(B, L, H, D, generator=g).to(dtype).mul(3) for H in (Hq, Hkv, Hkv))
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    if not norm:
        qw = kw = None
    cs = [angles(L, R, b, 17 * b) for b in range(B)]
    cos, sin = torch.stack([c for c, _ in cs]).to(dtype), torch.stack([s for _, s in cs]).to(dtype)
    C, n = L + 9, 5
    kb = torch.full((B, Hkv, C, D), 7.0, dtype=dtype, device=gpu)
    vb = torch.full((B, Hkv, C, D), 7.0, dtype=dtype, device=gpu)
    put = lambda x: None if x is None else x.to(gpu)
    qo, ko, vo = ops.norm_rope(q.to(gpu).transpose(1, 2), k.to(gpu).transpose(1, 2), cos.to(gpu), sin.to(gpu),
                               q_weight=put(qw), k_weight=put(kw), eps=1e-5, v=v.to(gpu).transpose(1, 2),
                               k_out=kb[:, :, n:n + L], v_out=vb[:, :, n:n + L])
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        z, tol = reference(x.transpose(1, 2), cos, sin, w, 1e-5)
        err = (got.cpu().double() - z).abs()
        assert (err <= tol).all(), float((err / tol).max())
    assert torch.equal(vo.cpu(), v.transpose(1, 2)) and torch.equal(vb[:, :, n:n + L], vo)
    for buf in (kb, vb):
        assert (buf[:, :, :n] == 7).all() and (buf[:, :, n + L:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 80])
def test_table(gpu, dtype, D):
    """A float32 table by positions, far ones and outside ones among them; norm
    weights in float32, for the keys alone."""
    from dropkv_amd import ops
    B, Hq, Hkv, L, P = 2, 6, 3, 7, 90000
    g = torch.Generator().manual_seed(D)
    q, k = torch.randn(B, Hq, L, D, generator=g).to(dtype), torch.randn(B, Hkv, L, D, generator=g).to(dtype)
    kw = 1 + 0.3 * torch.randn(D, generator=g)
    cos, sin = angles(P, D, 3)
    pos = torch.tensor([[0, 1, 89999, 5, 5, 70000, 2], [3, -1, 90000, 4, 2 ** 40, 0, 89998]])
    qo, ko = ops.norm_rope(q.to(gpu), k.to(gpu), cos.to(gpu), sin.to(gpu), positions=pos.to(gpu), k_weight=kw.to(gpu))
    known = (pos >= 0) & (pos < P)
    at = torch.where(known, pos, 0)
    for got, x, w in ((qo.cpu().double(), q, None), (ko.cpu().double(), k, kw)):
        z, tol = reference(x, cos[at], sin[at], w, 1e-6)
        ok = known[:, None, :, None].expand_as(z)
        assert ((got - z).abs() <= tol)[ok].all()
        assert got[~ok].isnan().all()


def test_shared_rows_unaligned_and_in_place(gpu):
    """[L, R] and [1, L, R] rows for all sequences, rows at odd addresses, and
    outputs that are the inputs."""
    from dropkv_amd import ops
    B, Hq, Hkv, L, D = 2, 4, 2, 6, 64
    g = torch.Generator().manual_seed(0)
    big = torch.randn(B, Hq + Hkv, L, D + 2, generator=g).bfloat16()
    cos, sin = (x.bfloat16() for x in angles(L, D, 1))
    x = big[..., 1:1 + D]
    z, tol = reference(x, cos[None], sin[None], None, 0)
    for c, s in ((cos, sin), (cos[None], sin[None])):
        for odd in (False, True):
            xd = big.to(gpu)[..., 1:1 + D] if odd else x.contiguous().to(gpu)
            qd, kd = xd[:, :Hq], xd[:, Hq:]
            qo, ko = ops.norm_rope(qd, kd, c.to(gpu), s.to(gpu), q_out=qd, k_out=kd)
            assert qo.data_ptr() == qd.data_ptr()
            assert ((xd.cpu().double() - z).abs() <= tol).all()


def test_values_that_are_not_finite(gpu):
    """A row that holds NaN or infinity leaves the other rows alone, also the
    heads that share its wave."""
    from dropkv_amd import ops
    q = torch.randn(1, 8, 2, 64, generator=torch.Generator().manual_seed(0)).bfloat16()
    cos, sin = angles(2, 64, 1)
    w = torch.ones(64)
    clean = ops.norm_rope(q.to(gpu), q.to(gpu), cos.to(gpu), sin.to(gpu), q_weight=w.to(gpu))[0].cpu()
    q[0, 3, 1, 9] = float("nan")
    q[0, 5, 0, 63] = float("inf")
    got = ops.norm_rope(q.to(gpu), q.to(gpu), cos.to(gpu), sin.to(gpu), q_weight=w.to(gpu))[0].cpu()
    hit = torch.zeros(8, 2, dtype=torch.bool)
    hit[3, 1] = hit[5, 0] = True
    assert torch.equal(got[0][~hit], clean[0][~hit]) and got[0, 3, 1].isnan().all()


def test_empty_and_refusals(gpu):
    from dropkv_amd import ops
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=gpu)
    q, k, c = z(2, 4, 3, 64), z(2, 2, 3, 64), z(3, 64)
    qo, ko = ops.norm_rope(q[:, :, :0], k[:, :, :0], c[:0], c[:0])
    assert qo.shape == (2, 4, 0, 64) and ko.shape == (2, 2, 0, 64)
    good = dict(q=q, k=k, cos=c, sin=c)
    ops.norm_rope(**good)
    bad = [dict(q=q.float()), dict(k=k[:1]), dict(sin=c[:2]), dict(cos=c.half(), sin=c.half()),
           dict(cos=c[:, :63], sin=c[:, :63]), dict(cos=z(3, 128), sin=z(3, 128)), dict(v=q), dict(v_out=k),
           dict(positions=torch.zeros(3, dtype=torch.int32, device=gpu)),
           dict(positions=torch.zeros(4, dtype=torch.int64, device=gpu)), dict(q_weight=z(63)),
           dict(q_weight=z(64), k_weight=z(64, dtype=torch.float32)), dict(k_out=k[:1]), dict(eps=-1.0),
           dict(q_out=z(2, 4, 64, 3).transpose(2, 3)), dict(cos=c.cpu(), sin=c.cpu()),
           dict(q=q.clone().requires_grad_())]
    for change in bad:
        with pytest.raises(RuntimeError):
            ops.norm_rope(**{**good, **change})


def test_in_a_graph(gpu):
    from dropkv_amd import ops
    q, k, v = (torch.randn(1, H, 8, 64, device=gpu).bfloat16() for H in (14, 2, 2))
    cos, sin = (x.to(gpu) for x in angles(500, 64, 0))
    pos = torch.arange(8, device=gpu)
    kb = torch.zeros(1, 2, 8, 64, device=gpu).bfloat16()
    ops.norm_rope(q, k, cos, sin, positions=pos, v=v)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        qo, ko, vo = ops.norm_rope(q, k, cos, sin, positions=pos, v=v, k_out=kb)
    for step in range(3):
        pos.add_(60)
        q.normal_()
        gr.replay()
        want = ops.norm_rope(q, k, cos, sin, positions=pos)
        torch.cuda.synchronize()
        assert torch.equal(qo, want[0]) and torch.equal(kb, want[1]) and torch.equal(vo, v)
