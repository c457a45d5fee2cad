// kernels_kv.h -- launch interfaces of the quantised paged KV cache operators.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kv_plan.h"

namespace nx {

// Caller-owned cache of one layer: codes [page][kv head][slot][D * bits / 8],
// scales [page][kv head][slot][1 (8 bits) or 2 (4 bits)].  Index 0: keys, 1: values.
struct KvCacheView {
    uint8_t *codes[2];
    float *scales[2];
    int bits[2];
    uint32_t hkv, num_pages, shift;
    int head_dim;
};

// Rows [row][head][head_dim] with strides in elements; fmt is a NEXUS_FMT_* id.
struct KvRows {
    void *data;
    int fmt;
    size_t row_stride, head_stride;
};

struct KvCopyParams {
    KvCacheView cache;
    KvBatchView batch;
    KvRows rows[2];   // keys, values; data == nullptr: side not wanted (read)
    unsigned *fault;
};
cudaError_t launch_kv_append(const KvCopyParams &p, cudaStream_t st);
cudaError_t launch_kv_read(const KvCopyParams &p, cudaStream_t st);

struct KvAttnParams {
    KvCacheView cache;
    KvBatchView batch;
    KvRows q, out;
    int group;
    uint32_t group_magic;      // ceil(2^32 / group), 0 for a group of one (kv_div)
    // score scale * log2(e) = key_scale 2^scale_exp, key_scale in [1, 2): the first goes on
    // the keys' scales and zeros, so that what a row's scores are multiplied by is a power
    // of two and x = score 2^n exact.  Then x - m is rounded once from the x that the
    // reference m was taken from, and however many nats a step of f32 is at x, the largest
    // key of a row has a weight near one (with the whole factor here, scores beyond 2^31
    // left weights of 0 and infinity).
    float key_scale;
    int scale_exp;
    uint32_t window, sinks;
    unsigned *fault;
    // split over the context
    uint32_t nsplit, tiles_per_split;
    float *part, *ml;          // records of unfinished softmaxes (nsplit > 1): D sums; reference, sum of p
    float *sums;               // chunk kernel, f32 queries: a CTA's output sums
    // sequences of at most rows_limit (token, head) rows per KV head are the
    // few-row kernel's, the others the chunk kernel's
    uint32_t rows_limit;
    uint32_t tile_rows, row_tiles;  // rows of a tile (8, 16; chunk 256), tiles a sequence may have
    int chunk;
    int cluster;               // few-row kernel: the splits of a row tile are a cluster
};

// Rows of one KV head (new tokens x query heads of its group) of a sequence
// that the few-row kernel takes.
constexpr uint32_t kKvFewRows = 16;
constexpr uint32_t kKvChunkRows = 256;   // rows of a chunk-kernel CTA
constexpr uint32_t kKvChunkTile = 128;   // tokens of its key tile
constexpr uint32_t kKvFlushTiles = 2;    // f32 queries: key tiles summed in tensor memory
constexpr uint32_t kKvFewTile = 16;      // tokens of one warp's tile
constexpr uint32_t kKvFewWarps = 4;
constexpr uint32_t kKvSms = 148;
constexpr uint32_t kKvCluster = 8;       // most splits that join as a cluster (the portable size)

cudaError_t launch_kv_attn_few(const KvAttnParams &p, cudaStream_t st);
cudaError_t launch_kv_attn_chunk(const KvAttnParams &p, cudaStream_t st);
cudaError_t launch_kv_merge(const KvAttnParams &p, cudaStream_t st);

}  // namespace nx
