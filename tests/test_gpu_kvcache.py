"""Quantised paged KV cache on the GPU: append, read, attention against plain 64-bit forms."""
import math

import pytest
import torch

from tests import kv_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def make_batch(nb, lens, page, seed=0, extra_pages=3, num_pages=None, bad_fill=None):
    """Batch over shuffled pages; unused table entries hold bad_fill (default: a page beyond the pool)."""
    need = [-(-kv // page) for _, kv in lens]
    total = sum(need) + extra_pages
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    per = max(need + [1]) + 1
    table = torch.full((len(lens), per), total + 1000 if bad_fill is None else bad_fill, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    batch = nb.KvBatch(torch.tensor(starts, dtype=torch.int32, device=DEV),
                       torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV), table.to(DEV),
                       max([n for n, _ in lens] + [0]), max([kv for _, kv in lens] + [0]))
    return batch, total, starts[-1]


def fill_random(cache, seed, spread=0.0):
    """Any bytes as codes, scales of both magnitudes a model has; NaN where nothing was written is the test's own."""
    g = gen(seed)
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device=DEV, dtype=torch.uint8))
        s = 0.02 * torch.exp2(spread * (torch.rand(scales.shape, generator=g, device=DEV) - 0.5))
        if scales.shape[-1] == 1:
            scales.copy_(s)
        else:
            s = 12 * s
            s[..., 1] = torch.randn(s.shape[:-1], generator=g, device=DEV) * 0.3
            scales.copy_(s)


def check_attention(cache, batch, lens, q, window=0, sinks=0, scale=None, out=None):
    got = cache.attention(batch, q, scale=scale, window=window, sinks=sinks, out=out)
    cache.status()
    ref, spread, reach, floor = R.attention(q, cache, lens, batch.page_table, window, sinks, scale)
    n = sum(a for a, _ in lens)
    got, ref = got[:n].double(), ref[:n]
    nan = torch.isnan(ref)
    assert torch.equal(nan, torch.isnan(got))
    tol = R.tolerance(ref, spread[:n], reach[:n], floor[:n], q.dtype)
    over = torch.where(nan, torch.zeros_like(ref), (got - torch.where(nan, got, ref)).abs() / tol)
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{worst} times the tolerance at {torch.nonzero(over > 1)[:4].tolist()}"
    return got


# ---------------------------------------------------------------- append, read

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [(8, 8), (4, 4), (8, 4), (4, 8)])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_append_codes_and_read(backend, nb, dim, bits, dtype):
    lens = [(1, 1), (17, 40), (1, 33), (0, 5), (130, 130), (3, 19)]
    batch, pages, rows = make_batch(nb, lens, 16, seed=dim)
    cache = nb.PagedKvCache.empty(backend, pages, 3, dim, 16, bits)
    fill_random(cache, 5)
    before = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    g = gen(dim + sum(bits))
    x = [(torch.randn((rows, 3, dim), generator=g, device=DEV) + 1.5).to(DTYPES[dtype]) for _ in range(2)]
    x[0][0] = 0.0                      # a group of zeros
    x[1][1, :, :] = -2.25              # constant groups
    x[0][2] = x[0][2] * 1e-3
    x[1][3, 1, 5] = math.inf
    x[0][4, 2, 0] = math.nan
    x[0][5, 0] = (torch.arange(dim, device=DEV) % 16 * 2.0 - 15).to(DTYPES[dtype])  # ties of the 4-bit codes
    x[1][6, 0] = (torch.arange(dim, device=DEV) * 2.0 - dim + 0.5).to(DTYPES[dtype])
    cache.append(batch, x[0], x[1])
    got = cache.read(batch, rows, dtype=torch.float32)
    cache.status()
    where = []
    at = 0
    for b, (n, kv) in enumerate(lens):
        for i in range(n):
            t = kv - n + i
            where.append((int(batch.page_table[b, t // 16]), t % 16))
    pg, sl = torch.tensor(where, device=DEV).T
    for i, (codes, scales, bt) in enumerate(((cache.k_codes, cache.k_scales, bits[0]),
                                             (cache.v_codes, cache.v_scales, bits[1]))):
        want, scale, zero = R.quantise(x[i], bt)
        c, s = codes[pg, :, sl], scales[pg, :, sl]
        assert torch.equal(c, R.pack(want, bt))
        sz = scale if bt == 8 else torch.cat([scale, zero], -1)
        assert torch.equal(torch.isnan(s), torch.isnan(sz)) and torch.equal(torch.nan_to_num(s), torch.nan_to_num(sz))
        value = R.held(want, scale, zero, bt).float()
        assert torch.equal(torch.nan_to_num(got[i], nan=7e9), torch.nan_to_num(value, nan=7e9))
        # nothing else in the cache moved
        keep = torch.ones(codes.shape[:3], dtype=torch.bool, device=DEV)
        keep[pg, :, sl] = False
        assert torch.equal(codes[keep], before[2 * i][keep]) and torch.equal(scales[keep], before[2 * i + 1][keep])


@pytest.mark.parametrize("bits", [8, 4])
def test_append_extreme_scales(backend, nb, bits):
    """Groups from subnormal to near the largest f32; a 4-bit range beyond f32 is held as NaN."""
    lens = [(9, 9)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 1, 64, 16, (bits, bits))
    x = torch.randn((rows, 1, 64), generator=gen(1), device=DEV)
    for i, f in enumerate((1e-44, 1e-38, 1e-32, 1e-20, 1.0, 1e20, 1e30, 1e37, 1.2e38)):
        x[i] *= f
    x[8] = x[8].clamp(-3e38, 3e38)
    x[8, 0, 0], x[8, 0, 1] = 3e38, -3e38
    cache.append(batch, x, x)
    k, v = cache.read(batch, rows)
    cache.status()
    codes, scale, zero = R.quantise(x, bits)
    want = R.held(codes, scale, zero, bits).float()
    assert torch.equal(torch.nan_to_num(k, nan=7.0), torch.nan_to_num(want, nan=7.0))
    assert torch.equal(torch.nan_to_num(v, nan=7.0), torch.nan_to_num(want, nan=7.0))
    assert bool(torch.isnan(k[8]).all()) == (bits == 4)


def test_append_every_quotient_near_a_tie(backend, nb):
    """Values within a few f32 steps of the border between two codes take the nearer code."""
    rows = 256
    batch, pages, n = make_batch(nb, [(rows, rows)], 64)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 128, 64, (8, 4))
    g = gen(3)
    top = torch.rand((rows, 2, 1), generator=g, device=DEV) * 3 + 0.5
    step8 = (top.double() / 127).float()
    half = torch.randint(-126, 126, (rows, 2, 128), generator=g, device=DEV) + 0.5
    x8 = (half.double() * step8.double()).float()
    x8 += x8 * torch.randint(-3, 4, x8.shape, generator=g, device=DEV) * 2.0 ** -24
    x8[..., 0:1] = top
    span = torch.rand((rows, 2, 1), generator=g, device=DEV) * 3 + 0.5
    lo = torch.randn((rows, 2, 1), generator=g, device=DEV)
    x4 = (lo.double() + (torch.randint(0, 14, (rows, 2, 128), generator=g, device=DEV) + 0.5) * span.double() / 15).float()
    x4[..., 0:1], x4[..., 1:2] = lo, lo + span
    cache.append(batch, x8, x4)
    k, v = cache.read(batch, n)
    cache.status()
    for got, x, bits in ((k, x8, 8), (v, x4, 4)):
        assert torch.equal(got, R.held(*R.quantise(x, bits), bits).float())


def test_append_strided_and_broadcast_rows(backend, nb):
    lens = [(5, 20), (8, 8)]
    batch, pages, rows = make_batch(nb, lens, 32)
    cache = nb.PagedKvCache.empty(backend, pages, 4, 64, 32, (8, 8))
    qkv = torch.randn((rows, 12, 64), generator=gen(8), device=DEV).half()
    k, v = qkv[:, 4:8], qkv[:, 8:9].expand(rows, 4, 64)   # a slice of fused rows; one head for all
    cache.append(batch, k, v)
    fused = torch.zeros((4, rows, 64), device=DEV)
    out = fused.transpose(0, 1), torch.zeros((rows, 4, 64), device=DEV)  # heads outermost
    cache.read(batch, rows, out=out)
    cache.status()
    for got, x in zip(out, (k, v)):
        assert torch.equal(got, R.held(*R.quantise(x, 8), 8).float())


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [(8, 8), (4, 4), (8, 4), (4, 8)])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_decode(backend, nb, dim, bits, dtype):
    lens = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 1000), (1, 0), (0, 30)]
    batch, pages, rows = make_batch(nb, lens, 16, seed=dim)
    cache = nb.PagedKvCache.empty(backend, pages, 2, dim, 16, bits)
    fill_random(cache, dim)
    q = torch.randn((rows, 8, dim), generator=gen(9), device=DEV).to(DTYPES[dtype])
    check_attention(cache, batch, lens, q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [(8, 8), (4, 4), (8, 4), (4, 8)])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_chunk(backend, nb, dim, bits, dtype):
    lens = [(40, 40), (33, 301), (1, 77), (129, 129), (64, 512)]
    batch, pages, rows = make_batch(nb, lens, 32, seed=dim)
    cache = nb.PagedKvCache.empty(backend, pages, 2, dim, 32, bits)
    fill_random(cache, dim + 1)
    q = torch.randn((rows, 8, dim), generator=gen(10), device=DEV).to(DTYPES[dtype])
    check_attention(cache, batch, lens, q)


@pytest.mark.parametrize("heads", [(1, 1), (2, 2), (3, 1), (12, 4), (5, 1), (24, 4), (14, 2), (8, 1), (16, 1), (34, 2),
                                   (40, 1), (128, 1)])
@pytest.mark.parametrize("new", [1, 2, 5, 70])
def test_head_groups(backend, nb, heads, new):
    hq, hkv = heads
    lens = [(new, new + 150), (1, 9), (new, new)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, hkv, 64, 16, (8, 4))
    fill_random(cache, 2)
    q = torch.randn((rows, hq, 64), generator=gen(11), device=DEV).bfloat16()
    check_attention(cache, batch, lens, q)


WINDOWS = [(1, 0), (1, 1), (7, 3), (16, 16), (33, 4), (64, 0), (100, 67), (128, 130), (300, 1), (5000, 4), (2 ** 31 - 1, 9)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("new", [1, 3, 150])
def test_window_and_sinks(backend, nb, new, window, sinks):
    lens = [(new, 700), (new, max(new, 40)), (1, 3), (new, new + 1), (new, 1025)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 8))
    fill_random(cache, 3)
    q = torch.randn((rows, 8, 64), generator=gen(12), device=DEV).half()
    check_attention(cache, batch, lens, q, window, sinks)


@pytest.mark.parametrize("new", [1, 4, 200])
@pytest.mark.parametrize("page", [16, 64, 4096])
def test_long_context_is_split(backend, nb, new, page):
    lens = [(new, 9001)]
    batch, pages, rows = make_batch(nb, lens, page)
    cache = nb.PagedKvCache.empty(backend, pages, 1, 128, page, (8, 8))
    fill_random(cache, 4)
    q = (2 * torch.randn((rows, 4, 128), generator=gen(13), device=DEV)).bfloat16()
    check_attention(cache, batch, lens, q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 90])
def test_scales_far_apart(backend, nb, new, dtype):
    """Token scales over 2^16: weights and values keep their precision whatever the scale of the values."""
    lens = [(new, 500)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 4))
    fill_random(cache, 14)
    g = gen(15)
    cache.v_scales.mul_(torch.exp2(16 * torch.rand(cache.v_scales.shape[:-1], generator=g, device=DEV) - 8)[..., None])
    q = (3 * torch.randn((rows, 4, 64), generator=g, device=DEV)).to(DTYPES[dtype])
    check_attention(cache, batch, lens, q)


@pytest.mark.parametrize("new", [1, 80])
@pytest.mark.parametrize("factor", [1e-30, 1e-12, 1e12, 1e30])
def test_values_of_any_magnitude(backend, nb, new, factor):
    lens = [(new, 200)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 1, 64, 16, (8, 8))
    fill_random(cache, 16)
    cache.v_scales.mul_(factor)
    q = torch.randn((rows, 4, 64), generator=gen(17), device=DEV)
    check_attention(cache, batch, lens, q)


@pytest.mark.parametrize("new", [1, 80])
def test_sharp_and_flat_rows(backend, nb, new):
    """Scores up to hundreds (one key takes all), all zero (every key alike), rows of different scale side by side."""
    lens = [(new, 300)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 1, 64, 16, (8, 8))
    fill_random(cache, 18)
    q = torch.randn((rows, 4, 64), generator=gen(19), device=DEV)
    q[:, 0] *= 100
    q[:, 1] = 0
    q[:, 2] *= 1e-20
    check_attention(cache, batch, lens, q.bfloat16())
    check_attention(cache, batch, lens, q)


@pytest.mark.parametrize("new", [1, 3, 60])
def test_hidden_tokens_may_hold_anything(backend, nb, new):
    """NaN scales behind a sequence's end, and in tokens that a window hides from some rows or from all."""
    window, sinks = 24, 2
    lens = [(new, 205), (new, max(new, 21))]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 1, 64, 16, (4, 8))
    fill_random(cache, 20)
    page = lambda b, t: (int(batch.page_table[b, t // 16]), 0, t % 16)  # noqa: E731
    for b, (n, kv) in enumerate(lens):
        for t in list(range(kv, -(-kv // 16) * 16)) + [t for t in range(sinks, kv - n - window + 1)]:
            for s in (cache.k_scales, cache.v_scales):
                s[page(b, t)] = math.nan
    seen_by_some = lens[0][1] - window - 3 if new > 3 else None
    if seen_by_some:
        cache.v_scales[page(0, seen_by_some)] = math.nan
        cache.k_scales[page(0, seen_by_some - 1)] = math.nan
    q = torch.randn((rows, 4, 64), generator=gen(21), device=DEV).half()
    got = check_attention(cache, batch, lens, q, window, sinks)
    assert bool(torch.isnan(got).any()) == bool(seen_by_some)


@pytest.mark.parametrize("new", [1, 60])
def test_not_a_number_in_a_query_stays_in_its_row(backend, nb, new):
    lens = [(new, 100), (new, 64)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 8))
    fill_random(cache, 22)
    q = torch.randn((rows, 4, 64), generator=gen(23), device=DEV)
    q[0, 1, 3] = math.nan
    got = cache.attention(batch, q)
    cache.status()
    bad = torch.isnan(got).all(-1)
    assert bad[0, 1] and int(bad.sum()) == 1 and int(torch.isnan(got).any(-1).sum()) == 1


@pytest.mark.parametrize("new", [1, 50])
def test_evicted_pages_are_not_read(backend, nb, new):
    """Table entries of pages wholly outside the window may name pages that do not exist."""
    window, sinks, page = 40, 5, 16
    lens = [(new, 800), (new, 333)]
    batch, pages, rows = make_batch(nb, lens, page)
    for b, (n, kv) in enumerate(lens):
        first = kv - n - window + 1
        batch.page_table[b, 1:first // page] = 2 ** 31 - 1
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, page, (8, 8))
    fill_random(cache, 24)
    q = torch.randn((rows, 4, 64), generator=gen(25), device=DEV).half()
    check_attention(cache, batch, lens, q, window, sinks)  # status() finds nothing


@pytest.mark.parametrize("new", [4, 70])
def test_padding_before_a_sequence(backend, nb, new):
    """More new rows than tokens: the first rows are padding and give zeros."""
    lens = [(new, new - 3), (new, 0), (new, new)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 8))
    fill_random(cache, 26)
    k = torch.randn((rows, 2, 64), generator=gen(27), device=DEV)
    cache.append(batch, k, k)
    got, _ = cache.read(batch, rows)
    values = R.held(*R.quantise(k, 8), 8).float()
    values[:3] = 0
    values[new:2 * new] = 0
    assert torch.equal(got, values)
    q = torch.randn((rows, 4, 64), generator=gen(28), device=DEV)
    out = check_attention(cache, batch, lens, q)
    assert not out[:3].any() and not out[new:2 * new].any()


@pytest.mark.parametrize("new", [1, 50])
def test_rows_outside_are_left_alone(backend, nb, new):
    lens = [(new, 60), (new, 80)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 8))
    fill_random(cache, 29)
    q = torch.randn((rows + 7, 4, 64), generator=gen(30), device=DEV).half()
    out = torch.full_like(q, 3.5)
    check_attention(cache, batch, lens, q, out=out)
    assert bool((out[rows:] == 3.5).all())
    kv = tuple(torch.full((rows + 7, 2, 64), 2.5, device=DEV) for _ in range(2))
    before = cache.k_codes.clone()
    cache.read(batch, rows + 7, out=kv)
    assert bool((kv[0][rows:] == 2.5).all() and (kv[1][rows:] == 2.5).all())
    cache.append(batch, kv[0], kv[1])
    cache.status()
    changed = int((cache.k_codes != before).any(-1).sum())
    assert 0 < changed <= rows * 2  # the slots of the sequences' own rows and heads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_strided_queries_and_outputs(backend, nb, new, dtype):
    lens = [(new, 130), (new, 50)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 8))
    fill_random(cache, 31)
    qkv = torch.randn((rows, 12, 64), generator=gen(32), device=DEV).to(DTYPES[dtype])
    out = torch.zeros((8, rows, 72), device=DEV, dtype=DTYPES[dtype]).transpose(0, 1)[..., :64]
    q = qkv[:, :8]
    check_attention(cache, batch, lens, q, out=out)
    one = q[:, :1].expand(rows, 8, 64)
    check_attention(cache, batch, lens, one)


def test_shared_prefix_pages(backend, nb):
    """Two sequences that list the same pages read the same tokens."""
    lens = [(1, 64), (1, 64)]
    batch, pages, rows = make_batch(nb, lens, 16)
    batch.page_table[1] = batch.page_table[0]
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 8))
    fill_random(cache, 33)
    q = torch.randn((1, 4, 64), generator=gen(34), device=DEV).half().expand(2, 4, 64)
    out = check_attention(cache, batch, lens, q)
    assert torch.equal(out[0], out[1])


def test_score_scale(backend, nb):
    lens = [(1, 90), (50, 90)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 32, 16, (8, 8))
    fill_random(cache, 35)
    q = torch.randn((rows, 4, 32), generator=gen(36), device=DEV)
    for s in (1.0, 1e-6, 3.0):
        check_attention(cache, batch, lens, q, scale=s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[(1, 90), (1, 40)], [(1, 9000)] * 2, [(1, 90000)], [(2, 300), (70, 200), (300, 800)],
                                  [(40, 6000)], [(0, 0), (5, 3), (1, 1)]])
def test_output_in_place_of_the_queries(backend, nb, lens, dtype):
    """One part, parts of a cluster, parts in the workspace, and chunks of one part and of several."""
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 4))
    fill_random(cache, 37)
    q = torch.randn((rows, 8, 64), generator=gen(38), device=DEV).to(DTYPES[dtype])
    want = cache.attention(batch, q)
    got = q.clone()
    cache.attention(batch, got, out=got)
    cache.status()
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def test_same_call_same_bits(backend, nb):
    lens = [(1, 5000), (60, 3000), (2, 900)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 128, 16, (8, 4))
    fill_random(cache, 37)
    q = torch.randn((rows, 8, 128), generator=gen(38), device=DEV).bfloat16()
    a = cache.attention(batch, q)
    for _ in range(3):
        assert torch.equal(a, cache.attention(batch, q))
    cache.status()


@pytest.mark.parametrize("dim,bits", [(128, (8, 8)), (64, (8, 4)), (32, (4, 8))])
@pytest.mark.parametrize("new", [1, 40, 300])
def test_f32_stays_exact_over_long_contexts(backend, nb, new, dim, bits):
    """Sums over 20000 tokens whose values share a sign: an accumulator that rounds one way
    loses 3e-5 here.  2e-6: two key tiles are 32 products rounded one way, half a step of
    2^-23 each at most, of a sum that grows to its end (32 * 2^-24 / 2 = 1e-6), and S as much."""
    lens = [(new, 20011)] + [(1, 20011)] * 40
    batch, pages, rows = make_batch(nb, lens[:1], 64)
    table = batch.page_table.expand(41, -1).contiguous()
    starts = [0] + [new + i for i in range(41)]
    batch = nb.KvBatch(torch.tensor(starts, dtype=torch.int32, device=DEV),
                       torch.full((41,), 20011, dtype=torch.int32, device=DEV), table, new, 20011)
    cache = nb.PagedKvCache.empty(backend, pages, 4, dim, 64, bits)
    fill_random(cache, 50)
    if bits[1] == 8:
        cache.v_codes.copy_(cache.v_codes // 4 + 160)
    else:
        cache.v_scales[..., 1].abs_().add_(2.0)
    q = torch.randn((new + 40, 8, dim), generator=gen(51), device=DEV)
    out = cache.attention(batch, q)
    cache.status()
    for rows, ls in ((slice(0, new), [(new, 20011)]), (slice(new, new + 1), [(1, 20011)])):
        ref = R.attention(q[rows], cache, ls, table)[0]
        assert float((out[rows].double() - ref).norm() / ref.norm()) < 2e-6


@pytest.mark.parametrize("new", [1, 60])
def test_cache_beyond_32_bit_offsets(backend, nb, new):
    """Pages whose codes lie beyond 4 GB of the pool, written, read and attended."""
    pages = (1 << 32) // (8 * 16 * 128) + 2000
    cache = nb.PagedKvCache.empty(backend, pages, 8, 128, 16, (8, 8))
    lens = [(new, 150), (new, max(new, 33))]
    table = torch.stack([torch.arange(pages - 1, pages - 13, -1), torch.arange(pages - 20, pages - 32, -1)]).to(torch.int32)
    for b in range(2):
        ids = table[b].long().to(DEV)
        for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
            codes[ids] = torch.randint(0, 256, codes[ids].shape, generator=gen(60 + b), device=DEV, dtype=torch.uint8)
            scales[ids] = 0.02
    batch = nb.KvBatch(torch.tensor([0, new, 2 * new], dtype=torch.int32, device=DEV),
                       torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV), table.to(DEV), new, 150)
    x = torch.randn((2 * new, 48, 128), generator=gen(62), device=DEV).bfloat16()
    cache.append(batch, x[:, 32:40], x[:, 40:])
    k, _ = cache.read(batch, 2 * new)
    assert torch.equal(k, R.held(*R.quantise(x[:, 32:40], 8), 8).float())
    check_attention(cache, batch, lens, x[:, :32])
    assert not cache.k_codes[: pages - 40].any()


def test_nothing_to_do(backend, nb):
    """No sequences, no rows, sequences without new tokens."""
    cache = nb.PagedKvCache.empty(backend, 4, 2, 64)
    none = torch.zeros((0, 2, 64), device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for batch in (nb.KvBatch(i32(0), i32(), torch.zeros((0, 3), dtype=torch.int32, device=DEV), 0, 0),
                  nb.KvBatch(i32(0, 0, 0), i32(5, 0), torch.zeros((2, 3), dtype=torch.int32, device=DEV), 0, 5)):
        cache.append(batch, none, none)
        assert cache.read(batch, 0)[0].shape == (0, 2, 64)
        assert cache.attention(batch, torch.zeros((0, 4, 64), device=DEV)).shape == (0, 4, 64)
        rows = torch.full((3, 4, 64), 2.0, device=DEV)
        assert bool((cache.attention(batch, rows, out=rows.clone()) == 2.0).all())
    cache.status()


def test_one_long_chunk_among_single_tokens_f32(backend, nb):
    lens = [(1, 900)] * 5 + [(700, 1500)] + [(1, 40)] * 5 + [(33, 2000)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 8))
    fill_random(cache, 63)
    q = torch.randn((rows, 8, 64), generator=gen(64), device=DEV)
    check_attention(cache, batch, lens, q)


# ---------------------------------------------------------------- used together

@pytest.mark.parametrize("bits", [(8, 8), (4, 4)])
def test_prompt_then_decode_steps(backend, nb, bits):
    """A prompt in two chunks, then decode steps of a growing batch: append
    before attention each time, against the plain form over the whole cache."""
    g, page, hkv, hq, dim = gen(39), 16, 2, 8, 64
    cache = nb.PagedKvCache.empty(backend, 40, hkv, dim, page, bits)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(2, 20).to(DEV)
    steps = [[(100, 100), (0, 0)], [(45, 145), (130, 130)]] + [[(1, 146 + i), (1, 131 + i)] for i in range(4)]
    for lens in steps:
        rows = sum(n for n, _ in lens)
        batch = nb.KvBatch(torch.tensor([0, lens[0][0], rows], dtype=torch.int32, device=DEV),
                           torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV), table,
                           max(n for n, _ in lens), max(kv for _, kv in lens))
        x = torch.randn((rows, hq + 2 * hkv, dim), generator=g, device=DEV).bfloat16()
        cache.append(batch, x[:, hq:hq + hkv], x[:, hq + hkv:])
        check_attention(cache, batch, lens, x[:, :hq])


def test_window_equals_whole_context_when_it_covers_it(backend, nb):
    lens = [(1, 90), (30, 90)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 8))
    fill_random(cache, 40)
    q = torch.randn((rows, 4, 64), generator=gen(41), device=DEV).half()
    a, b = cache.attention(batch, q), cache.attention(batch, q, window=90)
    cache.status()
    assert torch.allclose(a.float(), b.float(), rtol=2e-3, atol=1e-3)


# ---------------------------------------------------------------- streams, graphs, faults

@pytest.mark.parametrize("new", [1, 60])
def test_captured_step_follows_its_tensors(backend, nb, new):
    """One captured append + attention, replayed with longer sequences and other pages."""
    lens = [(new, 200), (new, 130)]
    batch, pages, rows = make_batch(nb, lens, 16)
    batch = nb.KvBatch(batch.q_start, batch.kv_len, batch.page_table, new, 400)
    cache = nb.PagedKvCache.empty(backend, 64, 2, 64, 16, (8, 4))
    fill_random(cache, 42)
    batch.page_table.copy_(torch.arange(batch.page_table.numel(), device=DEV).view_as(batch.page_table) % 64)
    x = torch.randn((rows, 12, 64), generator=gen(43), device=DEV).half()
    out = torch.empty((rows, 8, 64), dtype=torch.float16, device=DEV)

    def step():
        cache.append(batch, x[:, 8:10], x[:, 10:])
        cache.attention(batch, x[:, :8], out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens in ([(new, 200), (new, 130)], [(new, 61), (new, 205)], [(new, 60), (new, 190)]):
        batch.kv_len.copy_(torch.tensor([kv for _, kv in lens], dtype=torch.int32))
        x.copy_(torch.randn(x.shape, generator=gen(lens[0][1]), device=DEV))
        graph.replay()
        cache.status()
        ref, spread, reach, floor = R.attention(x[:, :8], cache, lens, batch.page_table)
        assert bool(((out.double() - ref).abs() <= R.tolerance(ref, spread, reach, floor, out.dtype)).all())


def test_two_streams_at_once(backend, nb):
    lens = [(1, 4000), (40, 2000)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, 8))
    fill_random(cache, 44)
    q = [torch.randn((rows, 8, 64), generator=gen(45 + i), device=DEV).half() for i in range(2)]
    want = [cache.attention(batch, x) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.attention(batch, q[i]))
    torch.cuda.synchronize()
    cache.status()
    for i in range(2):
        assert all(torch.equal(want[i], x) for x in got[i])


@pytest.mark.parametrize("new", [1, 40])
def test_faulty_batches_are_skipped_and_reported(backend, nb, new):
    """What only the device can see: the sound sequence is served, the faulty one skipped, status() tells."""
    lens = [(new, 100), (new, 90)]
    cache = nb.PagedKvCache.empty(backend, 32, 2, 64, 16, (8, 8))
    fill_random(cache, 46)
    q = torch.randn((2 * new, 4, 64), generator=gen(47), device=DEV).half()
    k = torch.randn((2 * new, 2, 64), generator=gen(48), device=DEV).half()

    def batch(**change):
        t = dict(q_start=[0, new, 2 * new], kv_len=[100, 90], table=torch.arange(16).view(2, 8))
        t.update(change)
        return nb.KvBatch(torch.tensor(t["q_start"], dtype=torch.int32, device=DEV),
                          torch.tensor(t["kv_len"], dtype=torch.int32, device=DEV), t["table"].int().to(DEV), new, 100)
    good = batch()
    want = cache.attention(good, q)
    cache.status()
    page = torch.arange(16).view(2, 8)
    page[1, :] = 32
    negative = page.clone()
    negative[1] = -1
    for fault in (dict(table=page), dict(q_start=[0, new, 2 * new + 1]), dict(q_start=[0, new, 0]),
                  dict(kv_len=[100, 101]), dict(kv_len=[100, 2 ** 31 - 1]), dict(q_start=[0, new, -5]),
                  dict(table=negative)):
        bad = batch(**fault)
        out = torch.zeros_like(q)
        cache.attention(bad, q, out=out)
        assert torch.equal(out[:new], want[:new])
        with pytest.raises(nb.NexusError):
            cache.status()
        cache.status()  # reported once
        before = cache.k_codes.clone()
        cache.append(bad, k, k)
        with pytest.raises(nb.NexusError):
            cache.status()
        cache.k_codes.copy_(before)
        fill_random(cache, 46)


def test_status_refused_during_capture(backend, nb):
    batch, pages, rows = make_batch(nb, [(1, 20)], 16)
    cache = nb.PagedKvCache.empty(backend, pages, 1, 64)
    q = torch.zeros((1, 1, 64), device=DEV)
    cache.attention(batch, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attention(batch, q)
        with pytest.raises(nb.NexusError):
            cache.status()
    graph.replay()
    cache.status()


def test_refusals_of_the_binding(backend, nb):
    batch, pages, rows = make_batch(nb, [(1, 20)], 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64)
    ok = torch.zeros((1, 4, 64), device=DEV)
    for q in (ok.double(), ok[..., :32], ok[0], ok[:, :3], ok.cpu(), ok.transpose(1, 2)):
        with pytest.raises(nb.NexusError):
            cache.attention(batch, q)
    with pytest.raises(nb.NexusError):
        cache.attention(batch, ok, window=-1)
    with pytest.raises(nb.NexusError):
        cache.attention(batch, ok, scale=-1.0)
    with pytest.raises(nb.NexusError):
        cache.attention(batch, torch.zeros(1 * 4 * 64 + 1, device=DEV)[1:].view(1, 4, 64))  # not 16-byte aligned
    with pytest.raises(nb.NexusError):
        cache.attention(batch, ok, out=torch.zeros((1, 1, 64), device=DEV).expand(1, 4, 64))  # heads overlap
    with pytest.raises(nb.NexusError):
        cache.append(batch, ok, ok)  # four heads, the cache has two
    with pytest.raises(nb.NexusError):
        nb.KvBatch(batch.q_start.long(), batch.kv_len, batch.page_table, 1, 20)
    with pytest.raises(nb.NexusError):
        nb.PagedKvCache.empty(backend, 4, 2, 64, bits=(3, 8))
    with pytest.raises(nb.NexusError):
        cache = nb.PagedKvCache.empty(backend, 4, 2, 96)
        cache.attention(batch, torch.zeros((1, 4, 96), device=DEV))
