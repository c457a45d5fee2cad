// kv_plan.h -- index arithmetic of the quantised paged KV cache operators,
// shared by the kernels and by host code (plain C++: the CPU tests compile it).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define NX_HD __host__ __device__ __forceinline__
#else
#define NX_HD inline
#endif

namespace nx {

// What a kernel found wrong in the device-side description of a batch
// (or in a page table) and therefore skipped.
enum KvFault : unsigned {
    KV_FAULT_PAGE = 1,    // page id beyond the pool
    KV_FAULT_START = 2,   // q_start not ascending, or beyond the rows given
    KV_FAULT_LENGTH = 4,  // more new tokens than max_q, or a length beyond max_kv or the page table
    KV_FAULT_WAIT = 8     // a bounded wait gave up
};

struct KvBatchView {
    const uint32_t *q_start, *kv_len, *table;
    uint32_t stride, n_seqs, n_rows, max_q, max_kv;
};

// One sequence of a batch: nq new tokens (rows q0 ..), kv cached tokens with
// the new ones the last of them.  A faulty description gives nq = kv = 0.
struct KvSeqView {
    uint32_t q0, nq, kv;
};

NX_HD KvSeqView kv_seq_view(uint32_t q0, uint32_t q1, uint32_t kv, const KvBatchView &bt, uint32_t shift,
                            unsigned *fault) {
    KvSeqView s = {0u, 0u, 0u};
    if (q1 < q0 || q1 > bt.n_rows) {
        *fault |= KV_FAULT_START;
        return s;
    }
    if (q1 - q0 > bt.max_q || kv > bt.max_kv || (uint64_t)kv > ((uint64_t)bt.stride << shift)) {
        *fault |= KV_FAULT_LENGTH;
        return s;
    }
    s.q0 = q0;
    s.nq = q1 - q0;
    s.kv = kv;
    return s;
}

// The sequence of row `row`: the b with q_start[b] <= row < q_start[b + 1],
// n_seqs for a row behind the last sequence.  Bounded for any contents.
NX_HD uint32_t kv_find_seq(const uint32_t *q_start, uint32_t n_seqs, uint32_t row) {
    uint32_t lo = 0, hi = n_seqs;  // first b with q_start[b + 1] > row
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (q_start[mid + 1] > row) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// The keys a set of consecutive queries reads: tokens [lo, end) and, before
// lo, the first `sinks` tokens.  Query positions are first .. last.
struct KvRange {
    uint32_t lo, end, sinks;
};
NX_HD KvRange kv_range(int first, int last, uint32_t window, uint32_t sinks) {
    KvRange r = {0u, 0u, 0u};
    if (last < 0) return r;
    r.end = (uint32_t)last + 1u;
    if (first < 0) first = 0;
    if (window != 0 && (uint32_t)first + 1u > window) r.lo = (uint32_t)first + 1u - window;
    r.sinks = sinks < r.lo ? sinks : r.lo;
    return r;
}
// Whether any token of [j0, j1) is read.
NX_HD bool kv_needed(const KvRange &r, uint32_t j0, uint32_t j1) {
    return j0 < r.end && (j1 > r.lo || j0 < r.sinks);
}
// Query position i sees key j.
NX_HD bool kv_visible(int j, int i, int window, int sinks) {
    return j <= i && (window == 0 || j > i - window || j < sinks);
}

// The tiles of T tokens that cover a range, in order: the sinks' tiles, then
// those from lo on.
struct KvTiles {
    uint32_t sink_tiles, first, total;
};
NX_HD KvTiles kv_tiles(const KvRange &r, uint32_t T) {
    KvTiles t;
    const uint32_t end = (r.end + T - 1) / T;
    t.first = r.lo / T;
    t.sink_tiles = (r.sinks + T - 1) / T;
    if (t.sink_tiles >= t.first) t.sink_tiles = t.first;
    t.total = t.sink_tiles + (end - t.first);
    return t;
}
NX_HD uint32_t kv_tile_at(const KvTiles &t, uint32_t i) { return i < t.sink_tiles ? i : t.first + (i - t.sink_tiles); }

// r / G by multiplication: exact for r < 2^32 / G with magic = ceil(2^32 / G).
// A row's number is below 2^24 in the chunk kernel (its grid's limit of 65535
// tiles of 256 rows) and G at most 128.
NX_HD uint32_t kv_div_magic(uint32_t G) { return G == 1 ? 0u : (uint32_t)(((1ull << 32) + G - 1) / G); }
NX_HD uint32_t kv_div(uint32_t r, uint32_t magic) {
    return magic == 0 ? r : (uint32_t)(((uint64_t)r * magic) >> 32);
}

// Tile rt of R rows of a sequence's (token, head of the group) rows: n rows
// from r0 on, of the tokens at positions first .. last.  Sequences of more
// than `limit` rows are another kernel's (n = 0).
struct KvRowTile {
    uint32_t r0, n;
    int first, last;
};
NX_HD KvRowTile kv_row_tile(const KvSeqView &s, uint32_t G, uint32_t rt, uint32_t R, uint32_t limit) {
    KvRowTile t = {0u, 0u, -1, -1};
    const uint64_t rows = (uint64_t)s.nq * G, r0 = (uint64_t)rt * R;
    if (rows > limit || r0 >= rows) return t;
    t.r0 = (uint32_t)r0;
    t.n = (uint32_t)(rows - r0 < R ? rows - r0 : R);
    const int pos0 = (int)s.kv - (int)s.nq;
    t.first = pos0 + (int)(t.r0 / G);
    t.last = pos0 + (int)((t.r0 + t.n - 1) / G);
    return t;
}

// A number of its own for row tile rt of every sequence, below rows * G / R +
// n_seqs for a batch of `rows` rows: floor((x + y)) + 1 >= floor(x) + ceil(y), so
// the next sequence's numbers start behind this one's.
NX_HD uint64_t kv_tile_slot(uint32_t q0, uint32_t G, uint32_t b, uint32_t rt, uint32_t R) {
    return (uint64_t)q0 * G / R + b + rt;
}

// An upper bound of kv_tiles().total for nq <= q queries of a sequence of at
// most max_kv tokens.
NX_HD uint32_t kv_tiles_bound(uint32_t q, uint32_t max_kv, uint32_t window, uint32_t sinks, uint32_t T) {
    const uint64_t all = ((uint64_t)max_kv + T - 1) / T;
    if (window == 0) return (uint32_t)all;
    const uint64_t w = ((uint64_t)window + q) / T + 2 + ((uint64_t)sinks + T - 1) / T;
    return (uint32_t)(w < all ? w : all);
}

}  // namespace nx
