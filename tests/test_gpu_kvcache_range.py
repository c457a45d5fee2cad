"""Quantised paged KV cache on the GPU at the ends of its range: magnitudes, small weights, bad pages, padding."""
import pytest
import torch

from tests import kv_reference as R
from tests.test_gpu_kvcache import DEV, DTYPES, check_attention, fill_random, gen, make_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_row_tiles_of_padding_alone(backend, nb, dim, dtype):
    """Row tiles without a key: kv_len 0, and hundreds of padding rows before the tokens.  Zeros, every
    time, whatever the queries hold; the other rows are as ever."""
    lens = [(700, 0), (650, 5), (300, 300), (515, 258)] * 3
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, dim, 16, (8, 4))
    fill_random(cache, 80)
    q = torch.randn((rows, 8, dim), generator=gen(81), device=DEV).to(DTYPES[dtype])
    first = check_attention(cache, batch, lens, q)
    at = 0
    for n, kv in lens:
        assert not first[at:at + max(0, n - kv)].any()
        at += n
    outs = [torch.full_like(q, 7.0) for _ in range(20)]
    for out in outs:
        cache.attention(batch, q, out=out)
    cache.status()
    assert all(torch.equal(out.double(), first) for out in outs)
