// kernels_kv_merge.cu -- dispatch of the attention kernels by head_dim, and the
// join of their context splits.
//
// Each split left, per row, o = sum p v, a reference m and l = sum p in that
// reference (m is a whole number, so the factors between references are exact
// powers of two).  A block joins one row: D / 8 lanes own eight dims each and
// the groups of lanes take the splits in turn, each a running sum in the
// largest reference so far; the groups' sums are then added in order.  The
// order depends on the number of splits alone.  The chunk kernel leaves many rows
// of few splits: there each group has a row of its own and takes its splits in turn
// (a block a row took 150 us for 65536 rows of two).  Bound by latency: four records
// of a group are loaded at once (one lane waiting for every split in turn took
// most of 229 us for 222 splits of a row).
#include "kernels_kv_few.cuh"

namespace nx {

cudaError_t launch_kv_few_d32(const KvAttnParams &p, cudaStream_t st);
cudaError_t launch_kv_few_d64(const KvAttnParams &p, cudaStream_t st);
cudaError_t launch_kv_few_d128(const KvAttnParams &p, cudaStream_t st);
cudaError_t launch_kv_chunk_d32(const KvAttnParams &p, cudaStream_t st);
cudaError_t launch_kv_chunk_d64(const KvAttnParams &p, cudaStream_t st);
cudaError_t launch_kv_chunk_d128(const KvAttnParams &p, cudaStream_t st);

cudaError_t launch_kv_attn_few(const KvAttnParams &p, cudaStream_t st) {
    switch (p.cache.head_dim) {
    case 32: return launch_kv_few_d32(p, st);
    case 64: return launch_kv_few_d64(p, st);
    case 128: return launch_kv_few_d128(p, st);
    default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_kv_attn_chunk(const KvAttnParams &p, cudaStream_t st) {
    switch (p.cache.head_dim) {
    case 32: return launch_kv_chunk_d32(p, st);
    case 64: return launch_kv_chunk_d64(p, st);
    case 128: return launch_kv_chunk_d128(p, st);
    default: return cudaErrorInvalidValue;
    }
}

constexpr int kMergeThreads = 128;
using kvf::join;

template <int D, bool CHUNK>
__global__ void __launch_bounds__(kMergeThreads) k_kv_merge(KvAttnParams p) {
    constexpr int LANES = D / 8, GROUPS = kMergeThreads / LANES;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, d0 = 8 * lane;
    constexpr int STEP = CHUNK ? 1 : GROUPS;  // splits between a group's
    __shared__ float sm_m[GROUPS], sm_l[GROUPS], sm_v[GROUPS][D];
    pdl_wait();  // (launched while the parts' last CTAs run)
    const uint32_t b = blockIdx.y, h = blockIdx.x / p.row_tiles, rt = blockIdx.x % p.row_tiles,
                   r = CHUNK ? blockIdx.z * GROUPS + group : blockIdx.z;
    unsigned fault = 0;
    const KvSeqView seq = kv_load_seq(p.batch, b, p.cache.shift, &fault);  // reported by the parts
    const uint32_t G = (uint32_t)p.group;
    if (fault || (CHUNK ? (uint64_t)seq.nq * G <= p.rows_limit : (uint64_t)seq.nq * G > p.rows_limit)) return;
    const KvRowTile rows = kv_row_tile(seq, G, rt, p.tile_rows, 0xffffffffu);
    if (r >= rows.n) return;
    const KvRange range = kv_range(rows.first, rows.last, p.window, p.sinks);
    const uint32_t total = kv_tiles(range, CHUNK ? kKvChunkTile : kKvFewTile).total;
    const uint32_t used = (total + p.tiles_per_split - 1) / p.tiles_per_split;
    const uint32_t tile = (b * p.cache.hkv + h) * p.row_tiles + rt;
    const size_t src = kvf::few_record(tile, p.tile_rows, r, p.nsplit, 0);
    float m = -INFINITY, l = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    // four records of a group in flight at once
#pragma unroll 1
    for (uint32_t s0 = CHUNK ? 0 : group; s0 < used; s0 += 4 * STEP) {
        float2 ml[4];
        float v1[4][8];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (s0 + u * STEP >= used) continue;
            const size_t at = src + s0 + u * STEP;
            ml[u] = __ldcg(reinterpret_cast<const float2 *>(p.ml) + at);
            const float4 *part = reinterpret_cast<const float4 *>(p.part + at * D + d0);
            const float4 t0 = __ldcg(part), t1 = __ldcg(part + 1);
            v1[u][0] = t0.x; v1[u][1] = t0.y; v1[u][2] = t0.z; v1[u][3] = t0.w;
            v1[u][4] = t1.x; v1[u][5] = t1.y; v1[u][6] = t1.z; v1[u][7] = t1.w;
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (s0 + u * STEP < used) join(m, l, v, ml[u].x, ml[u].y, v1[u]);
    }
    if constexpr (!CHUNK) {
        if (lane == 0) {
            sm_m[group] = m;
            sm_l[group] = l;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) sm_v[group][d0 + j] = v[j];
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int g = 1; g < GROUPS; g++) {
            float v1[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v1[j] = sm_v[g][d0 + j];
            join(m, l, v, sm_m[g], sm_l[g], v1);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= inv;
    const uint32_t tok = (rows.r0 + r) / G, head = h * G + (rows.r0 + r) % G;
    store8(p.out.data, (size_t)(seq.q0 + tok) * p.out.row_stride + head * p.out.head_stride + d0, p.out.fmt, v);
}

cudaError_t launch_kv_merge(const KvAttnParams &p, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    const uint32_t groups = kMergeThreads / ((uint32_t)p.cache.head_dim / 8);
    cfg.gridDim = dim3(p.cache.hkv * p.row_tiles, p.batch.n_seqs, p.chunk ? p.tile_rows / groups : p.tile_rows);
    cfg.blockDim = dim3(kMergeThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    switch (p.cache.head_dim) {
    case 32: return p.chunk ? cudaLaunchKernelEx(&cfg, k_kv_merge<32, true>, p) : cudaLaunchKernelEx(&cfg, k_kv_merge<32, false>, p);
    case 64: return p.chunk ? cudaLaunchKernelEx(&cfg, k_kv_merge<64, true>, p) : cudaLaunchKernelEx(&cfg, k_kv_merge<64, false>, p);
    case 128: return p.chunk ? cudaLaunchKernelEx(&cfg, k_kv_merge<128, true>, p) : cudaLaunchKernelEx(&cfg, k_kv_merge<128, false>, p);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace nx
