"""The cache in 8 bits and the attention over it in 64 bits, from their
definitions (test infrastructure)."""

import torch

BLOCK = 64
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
STORES = [torch.int8, torch.float8_e4m3fn]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def rounded(y, store):
    """To the nearest stored value, ties to even."""
    if store is torch.int8:
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def quantise(x, store):
    """Stored values and scales of blocks [..., 64, D] (bf16 or fp16): x top has at most
    18 significant bits and a 11, so the quotient in 64 bits is a tie only where the
    exact one is, and on the right side of one elsewhere."""
    x = x.double()
    a = x.abs().amax((-2, -1))
    odd, none = ~torch.isfinite(a), a < 2.0 ** -100
    q = rounded(x * TOP[store] / torch.where(none | odd, 1.0, a)[..., None, None], store)
    q = torch.where((none | odd)[..., None, None], 0.0, q)
    return q, torch.where(odd, float("nan"), torch.where(none, 0.0, a / TOP[store]))


def held(x, store):
    """What rows [..., n, D] are held as: full blocks quantised, the rest as they are."""
    n = x.shape[-2] // BLOCK * BLOCK
    y = x.double().clone()
    if n:
        q, s = quantise(x[..., :n, :].unflatten(-2, (n // BLOCK, BLOCK)), store)
        y[..., :n, :] = (q * s[..., None, None]).flatten(-3, -2)
    return y


def attend(q, k, v, k_new, v_new, n, scale, mask, store):
    """(out, bound) [B, T, Hq, D] in 64 bits: k, v [B, Hkv, >= n, D] the rows that were
    appended, n a list.  The bound is that of an evaluation with fp32 logits, sums of
    them over D, and weights of `w` relative error: see ``tolerance``."""
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    g = Hq // Hkv
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device)
    mean = torch.zeros_like(out)       # sum p |v|
    size = torch.zeros(B, T, Hq, 1, dtype=torch.float64, device=q.device)  # largest sum |q k| scale
    if mask is None:
        mask = torch.ones(T, T, dtype=torch.bool, device=q.device).tril()
    for b in range(B):
        m = mask if mask.dim() == 2 else mask[b]
        seen = torch.cat([torch.ones(T, n[b], dtype=torch.bool, device=q.device), m], dim=1)
        for h in range(Hkv):
            kk = torch.cat([held(k[b, h, :n[b]], store), k_new[b, h].double()])
            vv = torch.cat([held(v[b, h, :n[b]], store), v_new[b, h].double()])
            for x in range(h * g, (h + 1) * g):
                qq = q[b, x].double()
                s = (qq @ kk.T * scale).masked_fill(~seen, float("-inf"))
                top = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
                p = torch.where(seen, p, 0.0)
                total = p.sum(-1, keepdim=True)
                w = torch.where(total > 0, p / total, 0.0)
                # (0 * inf of keys that are not seen is no part of the sum.)
                out[b, :, x] = w @ torch.where(torch.isfinite(vv), vv, 0.0) if not torch.isfinite(vv).all() else w @ vv
                mean[b, :, x] = w @ vv.abs().nan_to_num(posinf=0.0)
                size[b, :, x] = ((qq.abs() @ kk.abs().T) * scale).masked_fill(~seen, 0.0).nan_to_num(posinf=0.0).amax(-1, keepdim=True)
    return out, mean, size


def tolerance(ref, mean, size, dtype, D, once):
    """Half a step of the output; each weight: fp32 logits off by D + 4 roundings of
    their largest sum, the exponential and the sums by 2^-20, and rounded to 16 bits
    (or, `once`, to bf16), in the sum above and in that below."""
    weight = 2 * ((D + 4) * 2.0 ** -24 * size + 2.0 ** -20 + (2.0 ** -8 if once else 2.0 ** -16))
    return HALF[dtype] * ref.abs() + weight * mean + 1e-30
