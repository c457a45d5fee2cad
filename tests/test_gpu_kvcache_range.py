"""Quantised paged KV cache on the GPU at the ends of its range: magnitudes, small weights, bad pages, padding, callers at once."""
import math
import threading

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


@pytest.mark.parametrize("new", [1, 60])
def test_a_sliced_page_table_ends_with_its_columns(backend, nb, new):
    """Columns of a wider table: a length beyond them is a fault, whatever stands behind them."""
    wide = torch.full((2, 40), 5, dtype=torch.int32, device=DEV)
    wide[:, 30:] = torch.randperm(20, generator=torch.Generator().manual_seed(2)).view(2, 10).to(torch.int32)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cache = nb.PagedKvCache.empty(backend, 24, 2, 64)
    fill_random(cache, 82)
    lens = [(new, 160), (new, 150)]
    batch = nb.KvBatch(i32(0, new, 2 * new), i32(160, 150), wide[:, 30:], new, 1000)
    x = torch.randn((2 * new, 12, 64), generator=gen(83), device=DEV).half()
    want = check_attention(cache, batch, lens, x[:, :8])
    batch.kv_len[1] = 161
    out = torch.zeros_like(x[:, :8])
    cache.attention(batch, x[:, :8], out=out)
    with pytest.raises(nb.NexusError, match="page table"):
        cache.status()
    assert torch.equal(out[:new].double(), want[:new]) and not out[new:].any()
    before = cache.k_codes.clone()
    cache.append(batch, x[:, 8:10], x[:, 10:])
    with pytest.raises(nb.NexusError, match="page table"):
        cache.status()
    changed = (cache.k_codes != before).flatten(1).any(-1).nonzero().flatten().tolist()
    assert set(changed) <= set(wide[0, 30:].tolist())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [(8, 8), (4, 4)])
@pytest.mark.parametrize("new", [1, 4, 60, 300])
def test_tokens_of_a_page_beyond_the_pool_are_left_out(backend, nb, new, bits, dtype):
    """One bad page among sound ones: what is left is the sequence without its tokens, in both
    kernels.  The other scores are around -20 and below, so that a token counted with score 0
    would take nearly all of the weight."""
    kv, page, dim = new + 420, 16, 64
    batch, pages, rows = make_batch(nb, [(new, kv)], page)
    cache = nb.PagedKvCache.empty(backend, pages, 2, dim, page, bits)
    fill_random(cache, 70)
    q = (0.5 + torch.rand((rows, 8, dim), generator=gen(71), device=DEV)).to(DTYPES[dtype])
    if bits[0] == 8:
        cache.k_codes.copy_(cache.k_codes % 64)            # every element of a key below -0.02 * 64
    else:
        cache.k_scales[..., 1] = -2.0 - cache.k_scales[..., 1].abs()
    for bad in (0, 9, 25):
        whole = batch.page_table.clone()
        batch.page_table[0, bad] = pages
        out = cache.attention(batch, q)
        with pytest.raises(nb.NexusError, match="page"):
            cache.status()
        batch.page_table.copy_(whole)
        left = torch.cat([whole[:, :bad], whole[:, bad + 1:]], 1)
        ref, spread, reach, floor = R.attention(q, cache, [(new, kv - page)], left)
        assert bool(((out.double() - ref).abs() <= R.tolerance(ref, spread, reach, floor, q.dtype)).all())


def test_append_subnormal_groups(backend, nb):
    """f32 groups whose 8-bit scale is a few subnormal steps: its rounding takes quotients beyond
    127, which are held as 127 (largest magnitudes 64 .. 17000 steps of 2^-149)."""
    top = torch.arange(64, 17001, 7, device=DEV)
    rows = top.numel()
    batch, pages, n = make_batch(nb, [(rows, rows)], 64)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 64, (8, 8))
    steps = (torch.rand((rows, 2, 64), generator=gen(72), device=DEV) * 2 - 1) * top[:, None, None]
    steps = steps.round().to(torch.int32)
    steps[:, 0, 5], steps[:, 1, 7] = top.int(), -top.int()
    x = torch.where(steps < 0, steps.abs() | -2 ** 31, steps).view(torch.float32)  # steps of 2^-149 are the bits
    cache.append(batch, x, x)
    k, v = cache.read(batch, n)
    cache.status()
    want = R.held(*R.quantise(x, 8), 8).float()
    assert torch.equal(k, want) and torch.equal(v, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bits_v", [8, 4])
@pytest.mark.parametrize("new", [1, 4, 80, 300])
@pytest.mark.parametrize("first,then", [(1e-30, 1e25), (1e25, 1e-30), (1e-30, 1.0), (1.0, 1e30), (0.0, 1e-30)])
def test_values_far_apart_in_one_sequence(backend, nb, first, then, new, bits_v, dtype):
    """The magnitude of the first tiles' values says nothing about the later ones'."""
    lens = [(new, new + 600), (new, new + 700)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, bits_v))
    fill_random(cache, 73)
    for b in range(2):
        ids = batch.page_table[b].long()
        cache.v_scales[ids[:20]] *= first
        cache.v_scales[ids[20:-(-lens[b][1] // 16)]] *= then
    q = torch.randn((rows, 8, 64), generator=gen(74), device=DEV).to(DTYPES[dtype])
    out = cache.attention(batch, q)
    cache.status()
    parts = R.attention(q, cache, lens, batch.page_table)
    tol = R.tolerance(*parts, q.dtype) - 1e-30 + 2.0 ** -149  # relative to the values, however small they are
    assert bool(((out.double() - parts[0]).abs() <= tol).all())


@pytest.mark.parametrize("kv", [20000, 100000])
@pytest.mark.parametrize("new", [1, 60])
def test_f32_keeps_many_small_weights(backend, nb, new, kv):
    """Every sixteenth key leads by 21 nats, so that each part of the context has such keys: the others are
    below what one f16 holds beside them.  In half of the dimensions the leading values are zero, so that
    the small ones are all there is.

    Two f16 of a weight lose at most 2^-35 of the leading one for each key: e^21 2^-35 of the small ones'
    sum.  Besides that: scores and exp2 to 2^-18 of 21 nats (1e-4 of the small ones' sum), 2e-6 of the
    whole as over other long contexts."""
    batch, pages, rows = make_batch(nb, [(new, kv)], 64)
    cache = nb.PagedKvCache.empty(backend, pages, 1, 64, 64, (8, 8))
    g = gen(75)
    cache.k_scales.fill_(0.01)
    cache.v_scales.fill_(0.02)
    cache.k_codes.copy_(torch.randint(126, 131, cache.k_codes.shape, generator=g, device=DEV, dtype=torch.uint8))
    cache.v_codes.copy_(torch.randint(192, 256, cache.v_codes.shape, generator=g, device=DEV, dtype=torch.uint8))
    q = torch.ones((rows, 4, 64), device=DEV) + 0.01 * torch.randn((rows, 4, 64), generator=g, device=DEV)
    cache.k_codes[:, 0, ::16] = 128 + 100              # a score of 64 * 1.0 * scale
    cache.v_codes[:, 0, ::16, :32] = 128               # zero
    out = cache.attention(batch, q, scale=21.0 / 64)
    cache.status()
    ref = R.attention(q, cache, [(new, kv)], batch.page_table, scale=21.0 / 64)[0]
    small = float((out[..., :32].double() - ref[..., :32]).norm() / ref[..., :32].norm())
    whole = float((out.double() - ref).norm() / ref.norm())
    assert whole < 2e-6, whole
    assert small < 1e-4 + math.exp(21) * 2.0 ** -35, small


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [(8, 8), (4, 4)])
@pytest.mark.parametrize("new", [1, 4, 60])
@pytest.mark.parametrize("scale,size", [(1e8, 1.0), (1e10, 1.0), (1e20, 1.0), (1e30, 1.0), (1e34, 1.0), (2e38, 2.0 ** -10)])
def test_scores_beyond_the_steps_of_f32(backend, nb, scale, size, new, bits, dtype):
    """Scores so large that a step of f32 is many nats: the key with the largest takes all, the output is
    its value (an f16 weight, 2^-11, or two for f32 queries; the output's rounding)."""
    lens = [(new, 700), (new, 90)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, bits)
    fill_random(cache, 76)
    g = gen(77)
    sign = torch.where(torch.rand(64, generator=g, device=DEV) < 0.5, -1.0, 1.0)
    if bits[0] == 4:
        cache.k_scales[..., 1] = 0.0                    # (the zero alone would give every key a part of the score)
    for b, at in ((0, 333), (1, 20)):
        page, slot = int(batch.page_table[b, at // 16]), at % 16
        cache.k_codes[page, :, slot] = (torch.where(sign > 0, 255, 1) if bits[0] == 8 else
                                        torch.where(sign > 0, 15, 1)[0::2] | torch.where(sign > 0, 240, 16)[1::2]
                                        ).to(torch.uint8)
        cache.k_scales[page, :, slot, 0] *= 2.0
    q = (size * sign * (0.5 + torch.rand((rows, 8, 64), generator=g, device=DEV))).to(DTYPES[dtype])
    out = cache.attention(batch, q, scale=scale)
    cache.status()
    for b, at in ((0, 333), (1, 20)):
        page, slot = int(batch.page_table[b, at // 16]), at % 16
        v, z = R.side(cache.v_codes[page, :, slot], cache.v_scales[page, :, slot], bits[1])
        want = (v + z).repeat_interleave(4, 0).expand(new, 8, 64)
        part = (v.abs() + z.abs()).repeat_interleave(4, 0).expand(new, 8, 64)
        w = 2.0 ** -21 if dtype == "f32" else 2.0 ** -11
        tol = torch.finfo(DTYPES[dtype]).eps / 2 * want.abs() + (w + 2.0 ** -20) * part
        assert bool(((out[b * new:(b + 1) * new].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bits_k", [8, 4])
@pytest.mark.parametrize("new", [1, 4, 60])
@pytest.mark.parametrize("power", [-110, -104, 109, 115, 120])
def test_queries_of_any_magnitude(backend, nb, power, new, bits_k, dtype):
    """Queries times 2^n against keys times 2^-n: the same scores to the last bit, the same output."""
    lens = [(new, 300), (new, 61)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (bits_k, 8))
    fill_random(cache, 78)
    if bits_k == 4:  # (nor of a zero)
        zero = cache.k_scales[..., 1]
        cache.k_scales[..., 1] = torch.where(zero < 0, -1.0, 1.0) * zero.abs().clamp(min=2.0 ** -4)
    q = torch.randn((rows, 8, 64), generator=gen(79), device=DEV).to(DTYPES[dtype])
    q = torch.where(q < 0, -1.0, 1.0).to(q.dtype) * q.abs().clamp(min=2.0 ** -4)  # no bit of it falls below f32's last
    want = check_attention(cache, batch, lens, q)
    cache.k_scales.mul_(2.0 ** -power)
    got = cache.attention(batch, q * 2.0 ** power)
    cache.status()
    assert torch.equal(got.double(), want)


def test_a_fault_is_reported_to_one_of_many_callers(backend, nb):
    """status() from eight threads on streams of their own: each fault is reported once."""
    batch, pages, rows = make_batch(nb, [(1, 40)], 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64)
    q = torch.zeros((1, 4, 64), device=DEV)
    batch.page_table[0, 1] = pages
    streams = [torch.cuda.Stream() for _ in range(8)]
    start, end, told = threading.Barrier(9, timeout=60), threading.Barrier(9, timeout=60), []

    def ask(stream):
        with torch.cuda.stream(stream):
            for _ in range(200):
                start.wait()
                try:
                    cache.status()
                except nb.NexusError as e:
                    told.append(str(e))
                end.wait()
    threads = [threading.Thread(target=ask, args=(s,)) for s in streams]
    for t in threads:
        t.start()
    counts = []
    for _ in range(200):
        cache.attention(batch, q)
        torch.cuda.synchronize()
        before = len(told)
        start.wait()
        end.wait()
        counts.append(len(told) - before)
    for t in threads:
        t.join()
    assert counts == [1] * 200
    assert all("page" in m for m in told)


def test_messages_of_calls_that_fail_at_once(backend, nb):
    """Refused calls on four threads: every message read is one of theirs, whole."""
    batch, pages, rows = make_batch(nb, [(1, 20)], 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64)
    three, one = torch.zeros((1, 3, 64), device=DEV), torch.zeros((1, 4, 64), device=DEV)
    calls = (lambda: cache.attention(batch, three), lambda: cache.attention(batch, one, scale=3e38),
             lambda: cache.append(batch, one, one), lambda: cache.attention(batch, one, out=one.expand(1, 4, 64)[:, :2]))
    known, told, lock = set(), set(), threading.Lock()

    def refused(call):
        with pytest.raises(nb.NexusError) as e:
            call()
        return str(e.value)
    for call in calls:
        known.add(refused(call))

    def repeat(call):
        mine = {refused(call) for _ in range(2000)}
        with lock:
            told.update(mine)
    threads = [threading.Thread(target=repeat, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(known) == 4 and told <= known


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits_v", [8, 4])
@pytest.mark.parametrize("new", [1, 4, 60])
@pytest.mark.parametrize("power", range(10, 24, 2))
def test_scores_of_every_magnitude(backend, nb, power, new, bits_v, dtype):
    """Scores of 2^18 .. 2^31 and values of 2^-20 .. 2^20: where a step of f32 is some powers of two, the
    reference of a row has only those to choose from.  The key with the largest score takes all (the
    next one is half of it below), the output is its value."""
    lens = [(new, 700), (new, 90)]
    batch, pages, rows = make_batch(nb, lens, 16)
    cache = nb.PagedKvCache.empty(backend, pages, 2, 64, 16, (8, bits_v))
    g = gen(84)
    sign = torch.where(torch.rand(64, generator=g, device=DEV) < 0.5, -1.0, 1.0)
    q = (sign * (0.5 + torch.rand((rows, 8, 64), generator=g, device=DEV))).to(DTYPES[dtype])
    w = 2.0 ** -21 if dtype == "f32" else 2.0 ** -11
    for step in range(4):
        for size in (-20, -9, -3, 0, 8, 20) if dtype != "f16" else (-9, -3, 0, 8):
            fill_random(cache, 85)
            cache.v_scales.mul_(2.0 ** size)
            for b, at in ((0, 333), (1, 20)):
                page, slot = int(batch.page_table[b, at // 16]), at % 16
                cache.k_codes[page, :, slot] = torch.where(sign > 0, 255, 1).to(torch.uint8)
                cache.k_scales[page, :, slot, 0] *= 2.0
            out = cache.attention(batch, q, scale=1.19 ** step * 1.41 ** (step % 2) * 2.0 ** power)
            for b, at in ((0, 333), (1, 20)):
                page, slot = int(batch.page_table[b, at // 16]), at % 16
                v, z = R.side(cache.v_codes[page, :, slot], cache.v_scales[page, :, slot], bits_v)
                want = (v + z).repeat_interleave(4, 0).expand(new, 8, 64)
                part = (v.abs() + z.abs()).repeat_interleave(4, 0).expand(new, 8, 64)
                tol = torch.finfo(DTYPES[dtype]).eps / 2 * want.abs() + (w + 2.0 ** -20) * part
                if dtype == "f16":
                    tol += 2.0 ** -25  # half of its last step
                assert bool(((out[b * new:(b + 1) * new].double() - want).abs() <= tol).all()), (step, size)
    cache.status()
