// kernels_kv_merge.cu -- dispatch of the attention kernels by head_dim, and the
// join of their context splits.
//
// Each split left, per row, o = sum p v, a reference m and l = sum p in that
// reference (m is a whole number, so the factors between references are exact
// powers of two).  A block joins one row: D / 8 lanes own eight dims each and
// the groups of lanes take the splits in turn, each a running sum in the
// largest reference so far; the groups' sums are then added in order.  The
// order depends on the number of splits alone.  Bound by latency: two rounds
// of loads a group where a single lane would wait for every split in turn
// (222 splits of one row took most of 229 us so).
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

// The running sum v, l in reference m takes another in reference m1.
__device__ __forceinline__ void join(float &m, float &l, float (&v)[8], float m1, float l1, const float (&v1)[8]) {
    const float top = fmaxf(m, m1);
    const float f = m == top ? 1.0f : kvf::pow2_diff(m, top), f1 = m1 == top ? 1.0f : kvf::pow2_diff(m1, top);
    m = top;
    l = fmaf(l1, f1, l * f);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = fmaf(v1[j], f1, v[j] * f);
}

template <int D>
__global__ void __launch_bounds__(kMergeThreads) k_kv_merge(KvAttnParams p) {
    constexpr int RS = D + 2, LANES = D / 8, GROUPS = kMergeThreads / LANES;
    __shared__ float sm_m[GROUPS], sm_l[GROUPS], sm_v[GROUPS][D];
    const uint32_t b = blockIdx.y, h = blockIdx.x / p.row_tiles, rt = blockIdx.x % p.row_tiles, r = blockIdx.z;
    unsigned fault = 0;
    const KvSeqView seq = kv_load_seq(p.batch, b, p.cache.shift, &fault);  // reported by the parts
    const uint32_t G = (uint32_t)p.group;
    if (fault || (p.chunk ? (uint64_t)seq.nq * G <= p.rows_limit : (uint64_t)seq.nq * G > p.rows_limit)) return;
    const KvRowTile rows = kv_row_tile(seq, G, rt, p.tile_rows, 0xffffffffu);
    if (r >= rows.n) return;
    const KvRange range = kv_range(rows.first, rows.last, p.window, p.sinks);
    const uint32_t total = kv_tiles(range, p.chunk ? kKvChunkTile : kKvFewTile).total;
    const uint32_t used = (total + p.tiles_per_split - 1) / p.tiles_per_split;
    const uint32_t tile = (b * p.cache.hkv + h) * p.row_tiles + rt;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, d0 = 8 * lane;
    const float *src = p.part + kvf::few_record(tile, p.tile_rows, r, p.nsplit, 0) * RS;
    float m = -INFINITY, l = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (uint32_t s = group; s < used; s += GROUPS) {
        const float *part = src + (size_t)s * RS;
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part + D));
        float v1[8];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float2 t = __ldcg(reinterpret_cast<const float2 *>(part + d0 + j));
            v1[j] = t.x;
            v1[j + 1] = t.y;
        }
        join(m, l, v, ml.x, ml.y, v1);
    }
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
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= inv;
    const uint32_t tok = (rows.r0 + r) / G, head = h * G + (rows.r0 + r) % G;
    store8(p.out.data, (size_t)(seq.q0 + tok) * p.out.row_stride + head * p.out.head_stride + d0, p.out.fmt, v);
}

cudaError_t launch_kv_merge(const KvAttnParams &p, cudaStream_t st) {
    const dim3 grid(p.cache.hkv * p.row_tiles, p.batch.n_seqs, p.tile_rows);
    switch (p.cache.head_dim) {
    case 32: k_kv_merge<32><<<grid, kMergeThreads, 0, st>>>(p); break;
    case 64: k_kv_merge<64><<<grid, kMergeThreads, 0, st>>>(p); break;
    case 128: k_kv_merge<128><<<grid, kMergeThreads, 0, st>>>(p); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace nx
