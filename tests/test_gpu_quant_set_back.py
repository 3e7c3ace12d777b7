"""Counts of a cache in 8 bits that are set back as far as they may be: to a multiple of 64,
within the block that is not full, and to where the last append of up to 64 rows began."""

import pytest
import torch

import quant_ref as R
from test_gpu_quant import BF, check_cache, counts, generator, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store", R.STORES)
@pytest.mark.parametrize("pieces,back", [
    ((300,), 256), ((300,), 64), ((300,), 0), ((128,), 128), ((300,), 299), ((290, 5), 260), ((191, 1), 191),
    ((100, 64), 100), ((127, 64), 127), ((65, 63), 65), ((1, 64), 1), ((200, 40, 20), 240)])
def test_other_rows_from_there(gpu, pieces, back, store):
    """Rows behind the count are read and appended as if the ones that were there had never come."""
    from dropkv_amd import ops
    g = generator(gpu, back)
    D, H, new, C = 64, 2, 90, 512
    cache = ops.quant_cache(1, H, C, D, store=store, device=gpu)
    k, v = rows(g, 1, H, sum(pieces), D), rows(g, 1, H, sum(pieces), D)
    n = 0
    for p in pieces:
        ops.quant_append(cache, k[:, :, n:n + p], v[:, :, n:n + p], counts(gpu, n))
        n += p
    for x, got in zip((k, v), ops.quant_read(cache, counts(gpu, back), C)):
        assert not got[:, :, back:].any()
        want = R.held(x[:, :, :back], store)
        assert ((got[:, :, :back].double() - want).abs() <= (R.HALF[BF] + 2.0 ** -22) * want.abs() + 1e-30).all()
    k2, v2 = (torch.cat([x[:, :, :back], rows(g, 1, H, new, D)], 2) for x in (k, v))
    ops.quant_append(cache, k2[:, :, back:], v2[:, :, back:], counts(gpu, back))
    end = back + new
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):  # (blocks behind the last may hold what was there)
        at = (end // 64 * 64 if t is cache.k else end // 64)
        t.view(torch.uint8 if t.element_size() == 1 else t.dtype)[:, :, at:] = 0
    check_cache(cache, k2, v2, [end])
