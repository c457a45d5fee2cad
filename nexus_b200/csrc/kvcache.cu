// kvcache.cu -- entry points of the quantised paged KV cache: argument checks,
// the split of the work, launches (kernels in kernels_kv*.cu).
//
// Every check that the host can make comes before the first CUDA call and
// before the backend is looked at, so a refused call has no effect.  What only
// the device sees is checked by the kernels, which skip it and leave a bit in
// the backend's fault word (kv_plan.h, KvFault) for nexus_cuda_kv_status.
#include <cuda_runtime.h>
#include <math.h>

#include <mutex>

#include "../../include/nexus_cuda.h"
#include "kernels_kv.h"

using namespace nx;

// Backend accessors implemented in engine.cu.
extern int nexus_backend_stream_device(nexus_cuda_backend *b, cudaStream_t *stream, int *device);
extern int nexus_backend_fail(nexus_cuda_backend *b, int code, const char *msg);
extern unsigned *nexus_backend_kv_fault(nexus_cuda_backend *b);
extern std::mutex &nexus_backend_kv_mutex(nexus_cuda_backend *b);

namespace {

size_t elem_bytes(int fmt) { return fmt == NEXUS_FMT_F32 ? 4 : 2; }
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// nullptr, or what is wrong with it.
const char *check_cache(const nexus_kv_cache *c) {
    if (!c) return "kv cache: cache is NULL";
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return "kv cache: head_dim must be 32, 64 or 128";
    if (c->kv_heads == 0 || c->kv_heads > 1024) return "kv cache: kv_heads must be in [1, 1024]";
    if (c->page_tokens < 16 || c->page_tokens > 4096 || (c->page_tokens & (c->page_tokens - 1)))
        return "kv cache: page_tokens must be a power of two in [16, 4096]";
    if (c->num_pages == 0 || c->num_pages > 0x7fffffffu) return "kv cache: num_pages must be in [1, 2^31)";
    if ((c->bits_k != 8 && c->bits_k != 4) || (c->bits_v != 8 && c->bits_v != 4))
        return "kv cache: bits_k and bits_v must be 8 or 4";
    if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales) return "kv cache: NULL buffer";
    if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || !aligned16(c->k_scales) || !aligned16(c->v_scales))
        return "kv cache: buffers must be 16-byte aligned";
    return nullptr;
}

const char *check_batch(const nexus_kv_batch *t) {
    if (!t) return "kv batch: batch is NULL";
    if (t->n_seqs > 65535) return "kv batch: more than 65535 sequences";
    if (t->max_q > 0x7fffffffu || t->max_kv > 0x7fff0000u) return "kv batch: max_q or max_kv beyond 2^31";
    if (t->flags & ~NEXUS_KV_CALLER_STREAM) return "kv batch: unknown flag";
    if (t->n_seqs == 0) return nullptr;
    if (!t->q_start || !t->kv_len || !t->page_table) return "kv batch: NULL device array";
    if ((reinterpret_cast<uintptr_t>(t->q_start) | reinterpret_cast<uintptr_t>(t->kv_len) |
         reinterpret_cast<uintptr_t>(t->page_table)) & 3u)
        return "kv batch: device arrays must be 4-byte aligned";
    if (t->table_stride == 0) return "kv batch: table_stride is 0";
    return nullptr;
}

const char *check_rows(const nexus_kv_rows *r, uint32_t head_dim, bool written) {
    if (!r) return "kv rows: rows are NULL";
    if (r->format != NEXUS_FMT_F32 && r->format != NEXUS_FMT_F16 && r->format != NEXUS_FMT_BF16)
        return "kv rows: format must be f32, f16 or bf16";
    if (r->heads == 0 || r->heads > 65535) return "kv rows: heads must be in [1, 65535]";
    if (r->rows > 0x7fffffffu) return "kv rows: more than 2^31 rows";
    if (r->rows == 0) return nullptr;
    if (!r->data) return "kv rows: NULL data";
    const size_t e = elem_bytes(r->format);
    if (!aligned16(r->data) || (r->row_stride * e) % 16 || (r->head_stride * e) % 16)
        return "kv rows: data and strides must be 16-byte aligned";
    if (r->row_stride > ((size_t)1 << 40) || r->head_stride > ((size_t)1 << 40)) return "kv rows: stride beyond 2^40";
    if (written) {
        // two heads or rows must not share an element
        const bool row_outer = r->row_stride >= (r->heads - 1) * r->head_stride + head_dim;
        const bool head_outer = r->head_stride >= (r->rows - 1) * r->row_stride + head_dim;
        const bool heads_apart = r->heads == 1 || r->head_stride >= head_dim;
        const bool rows_apart = r->rows == 1 || r->row_stride >= head_dim;
        if (!heads_apart || !rows_apart || !(row_outer || head_outer || r->rows == 1 || r->heads == 1))
            return "kv rows: rows that are written overlap";
    }
    return nullptr;
}

KvCacheView cache_view(const nexus_kv_cache *c) {
    KvCacheView v = {};
    v.codes[0] = static_cast<uint8_t *>(c->k_codes);
    v.codes[1] = static_cast<uint8_t *>(c->v_codes);
    v.scales[0] = c->k_scales;
    v.scales[1] = c->v_scales;
    v.bits[0] = (int)c->bits_k;
    v.bits[1] = (int)c->bits_v;
    v.hkv = c->kv_heads;
    v.num_pages = c->num_pages;
    v.head_dim = (int)c->head_dim;
    while ((1u << v.shift) < c->page_tokens) v.shift++;
    return v;
}
KvBatchView batch_view(const nexus_kv_batch *t, size_t rows) {
    KvBatchView v = {t->q_start, t->kv_len, t->page_table, t->table_stride, t->n_seqs, (uint32_t)rows, t->max_q,
                     t->max_kv};
    return v;
}
KvRows rows_view(const nexus_kv_rows *r) {
    KvRows v = {r->data, r->format, r->row_stride, r->head_stride};
    return v;
}

// The backend's device made current for a call, the caller's restored after it.
struct OnDevice {
    int before = -1;
    cudaError_t err = cudaSuccess;
    explicit OnDevice(int dev) {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        if (before != dev) err = cudaSetDevice(dev);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

int cuda_fail(nexus_cuda_backend *b, cudaError_t e) {
    return nexus_backend_fail(b, NEXUS_E_CUDA, cudaGetErrorString(e));
}

// How a call divides its rows and splits the context.  All of it follows from
// sizes and bounds, so that the workspace query and a captured call agree.
struct Split {
    uint32_t tile_rows, row_tiles, nsplit, tiles_per_split;
    size_t records;  // of the workspace, each D + 2 floats
    size_t bytes;
};
struct AttnPlan {
    uint32_t rows_limit;  // sequences of more rows than this go to the chunk kernel
    bool few, chunk;
    bool cluster;         // the few-row kernel's splits join as clusters
    Split f, c;
    size_t sums;  // chunk kernel's sums of f32 queries
    size_t bytes;
};

void plan_records(Split *s, uint64_t tiles, uint32_t head_dim) {
    if (s->nsplit <= 1) return;
    s->records = (size_t)tiles * s->tile_rows * s->nsplit;
    s->bytes = s->records * (head_dim + 2) * sizeof(float);  // (tile_rows is even: a multiple of 16)
}

const char *attn_plan(const nexus_kv_cache *c, const nexus_kv_batch *t, const nexus_kv_rows *q, uint32_t window,
                      uint32_t sinks, AttnPlan *pl) {
    const uint32_t G = q->heads / c->kv_heads;
    const uint64_t rows = (uint64_t)t->max_q * G;
    *pl = AttnPlan{};
    pl->rows_limit = kKvFewRows;
    if (rows == 0 || t->n_seqs == 0 || q->rows == 0) return nullptr;
    pl->few = G <= kKvFewRows;
    pl->chunk = rows > kKvFewRows;
    const uint64_t pairs = (uint64_t)t->n_seqs * c->kv_heads;
    if (pl->few) {
        const uint32_t most = rows < kKvFewRows ? (uint32_t)rows : kKvFewRows;
        pl->f.tile_rows = most <= 8 ? 8 : 16;
        pl->f.row_tiles = 1;
        const uint32_t tiles = kv_tiles_bound((most + G - 1) / G, t->max_kv, window, sinks, kKvFewTile);
        // CTAs resident at once, by the registers of the variant (kernels_kv_few.cuh).
        const uint64_t slots = kKvSms * (pl->f.tile_rows == 16 ? 2 : q->format == NEXUS_FMT_F32 ? 3 : 4);
        // Parts of 8 to 64 tiles, three CTAs an SM while they are short and at most 32 an
        // SM in all.  Few long sequences, and what would be a little more than one round
        // of CTAs, take one round.  Measured (us): one sequence of 577 tokens 14.3 with 8
        // tiles, 16.4 with 16; of 16000 tokens 24.6 with 27 or 32, 32.8 with 8; of 131071
        // tokens (64/8 heads) 59 in one round of 74 parts, 67 in 128; 64 sequences of 1024
        // to 8192 tokens 117 with 64 tiles, 139 with 256.
        const uint64_t ctas = pairs, all = (uint64_t)tiles * ctas;
        uint64_t per = (all + kKvSms * 3 - 1) / (kKvSms * 3);
        per = per < 8 ? 8 : per > 64 ? 64 : per;
        if (ctas * 2 <= kKvSms && per == 64) per = (all + slots - 1) / slots;
        if (per < (all + kKvSms * 32 - 1) / (kKvSms * 32)) per = (all + kKvSms * 32 - 1) / (kKvSms * 32);
        uint64_t nsplit = tiles ? (tiles + per - 1) / per : 1;
        if (ctas <= slots && ctas * nsplit > slots && ctas * nsplit < 2 * slots) {
            per = (tiles + slots / ctas - 1) / (slots / ctas);
            nsplit = (tiles + per - 1) / per;
        }
        pl->f.tiles_per_split = (uint32_t)per;
        pl->f.nsplit = (uint32_t)nsplit;
        // A cluster's parts wait for one another and hold their SM meanwhile: only where
        // every CTA is resident at once (64 ragged sequences: 154 us so, 117 with the
        // workspace).
        pl->cluster = nsplit <= kKvCluster && ctas * nsplit <= slots;
        if (!pl->cluster) plan_records(&pl->f, ctas, c->head_dim);
    }
    if (pl->chunk) {
        pl->c.tile_rows = kKvChunkRows;
        const uint64_t row_tiles = (rows + kKvChunkRows - 1) / kKvChunkRows;
        const uint32_t toks = t->max_q < kKvChunkRows ? t->max_q : kKvChunkRows;
        const uint32_t tiles = kv_tiles_bound(toks, t->max_kv, window, sinks, kKvChunkTile);
        // One CTA an SM: parts only where the rows leave SMs without work, none shorter
        // than four key tiles.
        const uint64_t ctas = pairs * row_tiles, want = ctas >= kKvSms ? 1 : kKvSms / ctas;
        uint64_t per = (tiles + want - 1) / want;
        if (per < 4) per = 4;
        pl->c.tiles_per_split = (uint32_t)per;
        pl->c.nsplit = tiles ? (uint32_t)((tiles + per - 1) / per) : 1;
        if (row_tiles * pl->c.nsplit > 65535) return "kv attention: too many rows per sequence for one call";
        pl->c.row_tiles = (uint32_t)row_tiles;
        plan_records(&pl->c, ctas, c->head_dim);
        if (q->format == NEXUS_FMT_F32 && per > kKvFlushTiles)
            pl->sums = (size_t)(((uint64_t)q->rows * G / kKvChunkRows + t->n_seqs) * c->kv_heads) * pl->c.nsplit *
                       kKvChunkRows * c->head_dim * sizeof(float);  // (kv_tile_slot)
    }
    pl->bytes = pl->f.bytes + pl->c.bytes + pl->sums;
    return nullptr;
}

const char *check_attention(const nexus_kv_cache *c, const nexus_kv_batch *t, const nexus_kv_rows *q, uint32_t window,
                            uint32_t sinks) {
    if (const char *e = check_cache(c)) return e;
    if (const char *e = check_batch(t)) return e;
    if (const char *e = check_rows(q, c->head_dim, false)) return e;
    if (q->heads % c->kv_heads) return "kv attention: query heads must be a multiple of kv_heads";
    if (q->heads / c->kv_heads > 128) return "kv attention: more than 128 query heads per KV head";
    if (window > 0x7fffffffu || sinks > 0x7fffffffu) return "kv attention: window or sinks beyond 2^31";
    return nullptr;
}

int copy_call(nexus_cuda_backend *b, const nexus_kv_cache *cache, const nexus_kv_batch *batch, const nexus_kv_rows *k,
              const nexus_kv_rows *v, bool append) {
    const char *e = check_cache(cache);
    if (!e) e = check_batch(batch);
    if (!e && append && (!k || !v)) e = "kv append: k or v is NULL";
    if (!e && !k && !v) return NEXUS_OK;
    for (const nexus_kv_rows *r : {k, v}) {
        if (!e && r) e = check_rows(r, cache->head_dim, !append);
        if (!e && r && r->heads != cache->kv_heads) e = "kv rows: heads differ from the cache's kv_heads";
    }
    if (!e && k && v && k->rows != v->rows) e = "kv rows: k and v have different row counts";
    const size_t rows = e ? 0 : (k ? k->rows : v->rows);
    if (!e && !b) e = "kv: backend is NULL";
    if (e) return nexus_backend_fail(b, NEXUS_E_INVALID, e);
    if (rows == 0 || batch->n_seqs == 0) return NEXUS_OK;
    cudaStream_t st = nullptr;
    int dev = 0;
    nexus_backend_stream_device(b, &st, &dev);
    if (batch->flags & NEXUS_KV_CALLER_STREAM) st = static_cast<cudaStream_t>(batch->stream);
    OnDevice on(dev);
    if (on.err != cudaSuccess) return cuda_fail(b, on.err);
    KvCopyParams p = {};
    p.cache = cache_view(cache);
    p.batch = batch_view(batch, rows);
    if (k) p.rows[0] = rows_view(k);
    if (v) p.rows[1] = rows_view(v);
    p.fault = nexus_backend_kv_fault(b);
    const cudaError_t r = append ? launch_kv_append(p, st) : launch_kv_read(p, st);
    return r == cudaSuccess ? NEXUS_OK : cuda_fail(b, r);
}

__global__ void k_kv_take_fault(unsigned *fault) { fault[1] = atomicExch(&fault[0], 0u); }

}  // namespace

extern "C" int nexus_cuda_kv_append(nexus_cuda_backend *b, const nexus_kv_cache *cache, const nexus_kv_batch *batch,
                                    const nexus_kv_rows *k, const nexus_kv_rows *v) {
    return copy_call(b, cache, batch, k, v, true);
}

extern "C" int nexus_cuda_kv_read(nexus_cuda_backend *b, const nexus_kv_cache *cache, const nexus_kv_batch *batch,
                                  const nexus_kv_rows *k, const nexus_kv_rows *v) {
    return copy_call(b, cache, batch, k, v, false);
}

extern "C" int nexus_cuda_kv_attention_workspace(const nexus_kv_cache *cache, const nexus_kv_batch *batch,
                                                 const nexus_kv_rows *q, uint32_t window, uint32_t sinks,
                                                 size_t *bytes) {
    const char *e = check_attention(cache, batch, q, window, sinks);
    if (!e && !bytes) e = "kv attention: bytes is NULL";
    AttnPlan pl;
    if (!e) e = attn_plan(cache, batch, q, window, sinks, &pl);
    if (e) return nexus_backend_fail(nullptr, NEXUS_E_INVALID, e);
    *bytes = pl.bytes;
    return NEXUS_OK;
}

extern "C" int nexus_cuda_kv_attention(nexus_cuda_backend *b, const nexus_kv_cache *cache, const nexus_kv_batch *batch,
                                       const nexus_kv_rows *q, const nexus_kv_rows *out, float scale, uint32_t window,
                                       uint32_t sinks, void *workspace, size_t workspace_bytes) {
    const char *e = check_attention(cache, batch, q, window, sinks);
    if (!e) e = check_rows(out, cache->head_dim, true);
    if (!e && (out->rows != q->rows || out->heads != q->heads || out->format != q->format))
        e = "kv attention: out must have q's rows, heads and format";
    // (the kernels take it times log2(e), which has to stay in f32)
    if (!e && !(scale >= 0.0f && scale <= 2.0e38f)) e = "kv attention: scale must be in [0, 2e38]";
    AttnPlan pl;
    if (!e) e = attn_plan(cache, batch, q, window, sinks, &pl);
    if (!e && pl.bytes && (!workspace || workspace_bytes < pl.bytes)) e = "kv attention: workspace too small";
    if (!e && pl.bytes && !aligned16(workspace)) e = "kv attention: workspace must be 16-byte aligned";
    if (!e && !b) e = "kv: backend is NULL";
    if (e) return nexus_backend_fail(b, NEXUS_E_INVALID, e);
    if (q->rows == 0 || batch->n_seqs == 0 || batch->max_q == 0) return NEXUS_OK;
    cudaStream_t st = nullptr;
    int dev = 0;
    nexus_backend_stream_device(b, &st, &dev);
    if (batch->flags & NEXUS_KV_CALLER_STREAM) st = static_cast<cudaStream_t>(batch->stream);
    OnDevice on(dev);
    if (on.err != cudaSuccess) return cuda_fail(b, on.err);
    KvAttnParams p = {};
    p.cache = cache_view(cache);
    p.batch = batch_view(batch, q->rows);
    p.q = rows_view(q);
    p.out = rows_view(out);
    p.group = (int)(q->heads / cache->kv_heads);
    p.group_magic = kv_div_magic((uint32_t)p.group);
    p.key_scale = 2.0f * frexpf((scale != 0.0f ? scale : 1.0f / sqrtf((float)cache->head_dim)) * 1.4426950408889634f,
                                &p.scale_exp);
    p.scale_exp--;
    p.window = window;
    p.sinks = sinks;
    p.fault = nexus_backend_kv_fault(b);
    p.rows_limit = pl.rows_limit;
    cudaError_t r = cudaSuccess;
    for (int chunk = 1; chunk >= 0; chunk--) {
        if (!(chunk ? pl.chunk : pl.few)) continue;
        const Split &s = chunk ? pl.c : pl.f;
        p.chunk = chunk;
        p.nsplit = s.nsplit;
        p.tiles_per_split = s.tiles_per_split;
        p.tile_rows = s.tile_rows;
        p.row_tiles = s.row_tiles;
        p.cluster = !chunk && pl.cluster;
        uint8_t *ws = static_cast<uint8_t *>(workspace);
        p.part = reinterpret_cast<float *>(ws + (chunk ? pl.f.bytes : 0));
        p.ml = p.part + s.records * cache->head_dim;
        p.sums = reinterpret_cast<float *>(ws + pl.f.bytes + pl.c.bytes);
        if (r == cudaSuccess) r = chunk ? launch_kv_attn_chunk(p, st) : launch_kv_attn_few(p, st);
        if (r == cudaSuccess && p.nsplit > 1 && !p.cluster) r = launch_kv_merge(p, st);
    }
    return r == cudaSuccess ? NEXUS_OK : cuda_fail(b, r);
}

extern "C" int nexus_cuda_kv_status(nexus_cuda_backend *b, void *stream, uint32_t flags) {
    if (flags & ~NEXUS_KV_CALLER_STREAM) return nexus_backend_fail(b, NEXUS_E_INVALID, "kv status: unknown flag");
    if (!b) return nexus_backend_fail(b, NEXUS_E_INVALID, "kv: backend is NULL");
    cudaStream_t st = nullptr;
    int dev = 0;
    nexus_backend_stream_device(b, &st, &dev);
    if (flags & NEXUS_KV_CALLER_STREAM) st = static_cast<cudaStream_t>(stream);
    OnDevice on(dev);
    if (on.err != cudaSuccess) return cuda_fail(b, on.err);
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    cudaError_t r = cudaStreamIsCapturing(st, &cap);
    if (r == cudaSuccess && cap != cudaStreamCaptureStatusNone)
        return nexus_backend_fail(b, NEXUS_E_INVALID, "kv status: the stream is being captured");
    unsigned *fault = nexus_backend_kv_fault(b), bits = 0;
    // (the wait is outside the lock: callers on other streams need not share it)
    if (r == cudaSuccess) r = cudaStreamSynchronize(st);
    if (r == cudaSuccess) {
        // the word that the bits are taken to is the backend's: one caller at a time
        std::lock_guard<std::mutex> lk(nexus_backend_kv_mutex(b));
        k_kv_take_fault<<<1, 1, 0, st>>>(fault);
        r = cudaGetLastError();
        if (r == cudaSuccess) r = cudaMemcpyAsync(&bits, fault + 1, sizeof(bits), cudaMemcpyDeviceToHost, st);
        if (r == cudaSuccess) r = cudaStreamSynchronize(st);
    }
    if (r != cudaSuccess) return cuda_fail(b, r);
    if (bits & KV_FAULT_WAIT)
        return nexus_backend_fail(b, NEXUS_E_TIMEOUT, "kv: a kernel's bounded wait gave up (asynchronous copy or MMA never completed)");
    if (bits & KV_FAULT_START)
        return nexus_backend_fail(b, NEXUS_E_INVALID, "kv: q_start is not ascending or runs beyond the rows; the sequence was skipped");
    if (bits & KV_FAULT_LENGTH)
        return nexus_backend_fail(b, NEXUS_E_INVALID, "kv: a sequence exceeds max_q, max_kv or its page table and was skipped");
    if (bits & KV_FAULT_PAGE)
        return nexus_backend_fail(b, NEXUS_E_INVALID, "kv: a page id is beyond the pool; its tokens were skipped");
    return NEXUS_OK;
}
