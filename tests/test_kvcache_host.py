"""Quantised paged KV cache, host side (CPU): refusals of the C ABI, workspace sizes, index arithmetic."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
PTR = 0x10000  # never dereferenced: every refusal comes before any device work


def cache(nb, **change):
    f = dict(kv_heads=8, head_dim=128, page_tokens=16, num_pages=64, bits_k=8, bits_v=4, k_codes=PTR, v_codes=PTR,
             k_scales=PTR, v_scales=PTR)
    f.update(change)
    return nb._lib.KvCache(**f)


def batch(nb, **change):
    f = dict(n_seqs=3, max_q=4, max_kv=500, table_stride=40, q_start=PTR, kv_len=PTR, page_table=PTR, stream=None,
             flags=0)
    f.update(change)
    return nb._lib.KvBatch(**f)


def rows(nb, n_heads, **change):
    f = dict(data=PTR, format=nb.BF16, heads=n_heads, rows=12, row_stride=n_heads * 128, head_stride=128)
    f.update(change)
    return nb._lib.KvRows(**f)


def message(nb, rc):
    assert rc == nb._lib.NEXUS_E_INVALID
    return nb._lib.load().nexus_cuda_last_error(None).decode()


def attention(nb, c=None, t=None, q=None, o=None, scale=0.0, window=0, sinks=0, ws=PTR, wsb=1 << 30):
    c, t, q, o = c or cache(nb), t or batch(nb), q or rows(nb, 32), o or rows(nb, 32)
    lib = nb._lib.load()
    return message(nb, lib.nexus_cuda_kv_attention(None, C.byref(c), C.byref(t), C.byref(q), C.byref(o), scale, window,
                                                   sinks, ws, wsb))


BAD_CACHE = [dict(head_dim=96), dict(kv_heads=0), dict(kv_heads=2000), dict(page_tokens=8), dict(page_tokens=24),
             dict(page_tokens=8192), dict(num_pages=0), dict(num_pages=2 ** 31), dict(bits_k=3), dict(bits_v=0),
             dict(k_codes=None), dict(v_scales=None), dict(v_codes=PTR + 8), dict(k_scales=PTR + 4)]
BAD_BATCH = [dict(n_seqs=65536), dict(max_q=2 ** 31), dict(max_kv=2 ** 32 - 1), dict(flags=2), dict(q_start=None),
             dict(kv_len=None), dict(page_table=None), dict(kv_len=PTR + 2), dict(table_stride=0)]
BAD_ROWS = [dict(format=2), dict(heads=0), dict(heads=70000), dict(rows=2 ** 31), dict(data=None), dict(data=PTR + 4),
            dict(row_stride=32 * 128 + 4), dict(head_stride=132), dict(row_stride=2 ** 50)]


def test_sound_arguments_reach_the_backend_check(nb):
    assert "backend is NULL" in attention(nb)
    lib, k = nb._lib.load(), rows(nb, 8)
    for fn in (lib.nexus_cuda_kv_append, lib.nexus_cuda_kv_read):
        assert "backend is NULL" in message(nb, fn(None, C.byref(cache(nb)), C.byref(batch(nb)), C.byref(k), C.byref(k)))
    assert "backend is NULL" in message(nb, lib.nexus_cuda_kv_status(None, None, 0))


@pytest.mark.parametrize("change", BAD_CACHE, ids=str)
def test_bad_cache_is_refused(nb, change):
    c, k, lib = cache(nb, **change), rows(nb, 8), nb._lib.load()
    assert message(nb, lib.nexus_cuda_kv_append(None, C.byref(c), C.byref(batch(nb)), C.byref(k), C.byref(k))) \
        .startswith("kv cache:")
    assert attention(nb, c=c).startswith("kv cache:")


@pytest.mark.parametrize("change", BAD_BATCH, ids=str)
def test_bad_batch_is_refused(nb, change):
    t, k, lib = batch(nb, **change), rows(nb, 8), nb._lib.load()
    assert message(nb, lib.nexus_cuda_kv_read(None, C.byref(cache(nb)), C.byref(t), C.byref(k), C.byref(k))) \
        .startswith("kv batch:")
    assert attention(nb, t=t).startswith("kv batch:")


@pytest.mark.parametrize("change", BAD_ROWS, ids=str)
def test_bad_rows_are_refused(nb, change):
    assert attention(nb, q=rows(nb, 32, **change)).startswith("kv rows:")
    assert attention(nb, o=rows(nb, 32, **change)).startswith("kv rows:")


def test_bad_attention_is_refused(nb):
    assert "multiple" in attention(nb, q=rows(nb, 12), o=rows(nb, 12))
    assert "128 query heads" in attention(nb, c=cache(nb, kv_heads=1), q=rows(nb, 129), o=rows(nb, 129))
    for o in (rows(nb, 24), rows(nb, 32, rows=11), rows(nb, 32, format=nb.F16)):
        assert "out must have" in attention(nb, o=o)
    for o in (rows(nb, 32, head_stride=0), rows(nb, 32, row_stride=0), rows(nb, 32, row_stride=2048),
              rows(nb, 32, head_stride=64)):
        assert "overlap" in attention(nb, o=o)
    for scale in (-1.0, float("nan"), float("inf")):
        assert "scale" in attention(nb, scale=scale)
    assert "window" in attention(nb, window=2 ** 31)
    assert "sinks" in attention(nb, sinks=2 ** 31)
    long = batch(nb, n_seqs=1, max_q=1, max_kv=100000)
    assert "too small" in attention(nb, t=long, ws=None, wsb=0)
    assert "too small" in attention(nb, t=long, wsb=16)
    assert "aligned" in attention(nb, t=long, ws=PTR + 4)
    # heads outermost is a layout like any other
    assert "backend" in attention(nb, o=rows(nb, 32, row_stride=128, head_stride=12 * 128))


def test_bad_copies_are_refused(nb):
    lib, c, t, k = nb._lib.load(), cache(nb), batch(nb), rows(nb, 8)
    assert "NULL" in message(nb, lib.nexus_cuda_kv_append(None, C.byref(c), C.byref(t), C.byref(k), None))
    for other in (rows(nb, 4), rows(nb, 8, rows=5)):
        assert "kv rows" in message(nb, lib.nexus_cuda_kv_append(None, C.byref(c), C.byref(t), C.byref(k),
                                                                 C.byref(other)))
    wide = rows(nb, 8, head_stride=0)
    assert "overlap" in message(nb, lib.nexus_cuda_kv_read(None, C.byref(c), C.byref(t), C.byref(wide), None))
    assert "backend" in message(nb, lib.nexus_cuda_kv_append(None, C.byref(c), C.byref(t), C.byref(wide), C.byref(k)))
    assert "unknown flag" in message(nb, lib.nexus_cuda_kv_status(None, None, 4))


def test_workspace_of_f32_chunks_follows_the_rows(nb):
    """One long chunk among many single tokens: the sums take the rows that are there, not n_seqs * max_q."""
    lib, n = nb._lib.load(), C.c_size_t()
    t = batch(nb, n_seqs=64, max_q=8192, max_kv=9000, table_stride=600)
    q = rows(nb, 32, rows=8192 + 63, format=nb.F32)
    assert lib.nexus_cuda_kv_attention_workspace(C.byref(cache(nb)), C.byref(t), C.byref(q), 0, 0, C.byref(n)) == 0
    assert n.value < (8192 + 63 + 64 * 64) * 32 * 128 * 4 * 2


def test_workspace_follows_sizes_only(nb):
    lib = nb._lib.load()

    def need(t, q, window=0, sinks=0, **kw):
        n = C.c_size_t()
        assert lib.nexus_cuda_kv_attention_workspace(C.byref(cache(nb, **kw)), C.byref(t), C.byref(q), window, sinks,
                                                     C.byref(n)) == 0
        return n.value
    one = batch(nb, n_seqs=1, max_q=1, max_kv=100)
    assert need(one, rows(nb, 32, rows=1)) == 0
    long = batch(nb, n_seqs=1, max_q=1, max_kv=100000)
    full = need(long, rows(nb, 32, rows=1))
    assert 0 < need(long, rows(nb, 32, rows=1), window=2000, sinks=4) < full
    assert full == need(long, rows(nb, 32, rows=1, data=PTR * 2), k_codes=PTR * 2)
    assert need(batch(nb, n_seqs=0), rows(nb, 32, rows=0)) == 0
    t, q = batch(nb), rows(nb, 32)
    assert "bytes" in message(nb, lib.nexus_cuda_kv_attention_workspace(C.byref(cache(nb)), C.byref(t), C.byref(q), 0,
                                                                        0, None))


DRIVER = r"""
#include "kv_plan.h"
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
using namespace nx;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)
int main() {
    // ranges and tiles against the definition of what a query sees
    for (int T : {16, 128}) for (int first = -3; first < 300; first += first < 40 ? 1 : 37)
        for (int n : {1, 2, 5, 100}) for (int window : {0, 1, 2, 15, 16, 17, 100, 1000, 2147483647})
            for (int sinks : {0, 1, 4, 16, 17, 200}) {
                const int last = first + n - 1;
                const KvRange r = kv_range(first, last, (uint32_t)window, (uint32_t)sinks);
                const KvTiles t = kv_tiles(r, T);
                CHECK(t.total <= kv_tiles_bound(n, last < 0 ? 0 : last + 1, window, sinks, T));
                int at = 0;
                for (int tile = 0; tile * T <= last + T; tile++) {
                    bool any = false;
                    for (int j = tile * T; j < tile * T + T; j++) {
                        bool seen = false;
                        for (int i = first < 0 ? 0 : first; i <= last; i++) seen |= kv_visible(j, i, window, sinks);
                        any |= seen;
                        CHECK(seen == kv_needed(r, j, j + 1));
                    }
                    CHECK(any == kv_needed(r, tile * T, tile * T + T));
                    if (any) {
                        CHECK(at < (int)t.total && (int)kv_tile_at(t, at) == tile);
                        at++;
                    }
                }
                CHECK(at == (int)t.total);
            }
    // sequences: whatever the arrays hold, rows stay inside
    KvBatchView bt = {};
    bt.n_rows = 100; bt.max_q = 50; bt.max_kv = 1000; bt.stride = 10;
    const uint32_t v[] = {0, 1, 49, 50, 51, 99, 100, 101, 999, 1000, 1001, 0x7fffffffu, 0x80000000u, 0xffffffffu};
    for (uint32_t a : v) for (uint32_t b : v) for (uint32_t kv : v) for (uint32_t shift : {4u, 12u}) {
        unsigned f = 0;
        const KvSeqView s = kv_seq_view(a, b, kv, bt, shift, &f);
        const bool sound = b >= a && b <= 100 && b - a <= 50 && kv <= 1000 && kv <= (10u << shift);
        CHECK(sound == (f == 0));
        CHECK(sound ? (s.q0 == a && s.nq == b - a && s.kv == kv) : (s.nq == 0 && s.kv == 0));
    }
    // the search ends and stays inside for any contents
    std::srand(1);
    for (int n = 0; n < 40; n++) for (int rep = 0; rep < 50; rep++) {
        uint32_t q[41];
        const bool ordered = rep & 1;
        for (int i = 0; i <= n; i++) q[i] = ordered ? (i ? q[i - 1] + std::rand() % 3 : 0) : std::rand();
        for (uint32_t row = 0; row < 130; row++) {
            const uint32_t b = kv_find_seq(q, n, row);
            CHECK(b <= (uint32_t)n);
            if (ordered && b < (uint32_t)n) CHECK(q[b] <= row && row < q[b + 1]);
            if (ordered && b == (uint32_t)n) CHECK(n == 0 || row >= q[n]);
        }
    }
    // division by the group for every row number the chunk kernel has
    for (uint32_t G = 1; G <= 128; G++) {
        const uint32_t m = kv_div_magic(G);
        for (uint32_t r = 0; r < 70000; r++) CHECK(kv_div(r, m) == r / G);
        for (uint32_t r = 65535u * 256u; r > 65535u * 256u - 70000u; r--) CHECK(kv_div(r, m) == r / G);
    }
    // row tiles cover every (token, head) row once, positions in step
    for (uint32_t G : {1u, 3u, 4u, 5u, 8u, 40u, 128u}) for (uint32_t nq : {0u, 1u, 2u, 33u}) for (uint32_t R : {8u, 16u, 128u}) {
        const KvSeqView s = {7, nq, 20};
        uint32_t rows = 0;
        for (uint32_t rt = 0;; rt++) {
            const KvRowTile t = kv_row_tile(s, G, rt, R, 0xffffffffu);
            if (t.n == 0) break;
            CHECK(t.r0 == rows && t.n <= R);
            CHECK(t.first == 20 - (int)nq + (int)(t.r0 / G) && t.last == 20 - (int)nq + (int)((t.r0 + t.n - 1) / G));
            rows += t.n;
        }
        CHECK(rows == nq * G);
        if (nq * G) CHECK(kv_row_tile(s, G, 0, R, nq * G - 1).n == 0);
    }
    // tile slots: one for each (sequence, row tile), below the bound
    for (int rep = 0; rep < 2000; rep++) {
        const uint32_t G = 1 + std::rand() % 128, n = 1 + std::rand() % 9;
        uint64_t at = 0;
        uint32_t q0 = std::rand() % 50;
        for (uint32_t b = 0; b < n; b++) {
            const uint32_t nq = std::rand() % 3 ? std::rand() % 40 : std::rand() % 4000;
            for (uint32_t rt = 0; (uint64_t)rt * 256 < (uint64_t)nq * G; rt++) {
                const uint64_t slot = kv_tile_slot(q0, G, b, rt, 256);
                CHECK(slot >= at);
                at = slot + 1;
            }
            q0 += nq;
        }
        CHECK(at <= (uint64_t)q0 * G / 256 + n);
    }
    return 0;
}
"""


def test_index_arithmetic(tmp_path):
    src = tmp_path / "driver.cpp"
    src.write_text(DRIVER)
    exe = tmp_path / "driver"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                    f"-I{ROOT / 'nexus_b200' / 'csrc'}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_score_scale_keeps_its_product_in_f32(nb):
    """2.5e38 * log2(e) is beyond f32, 2e38 * log2(e) is not."""
    assert "scale" in attention(nb, scale=2.5e38)
    assert "backend" in attention(nb, scale=2e38)


@pytest.mark.parametrize("scale", [0.0, -0.0, -1.0, 1e-50, float("nan")])
def test_binding_refuses_a_scale_that_is_not_positive(nb, scale):
    """0 asks the C call for its default, so a caller's own 0 must not reach it."""
    c = nb.PagedKvCache.__new__(nb.PagedKvCache)
    with pytest.raises(nb.NexusError, match="scale"):
        c.attention(None, None, scale=scale)
