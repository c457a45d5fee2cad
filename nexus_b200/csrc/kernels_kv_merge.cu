// kernels_kv_merge.cu -- dispatch of the few-row attention by head_dim, and the
// join of its context splits.
//
// Each split left, per row, o = sum p v, m and l = sum p in its own reference
// m (a whole number, so the factors between references are exact powers of
// two); the parts are added in split order.
#include "kernels_kv_few.cuh"

namespace nx {

cudaError_t launch_kv_few_d32(const KvAttnParams &p, cudaStream_t st);
cudaError_t launch_kv_few_d64(const KvAttnParams &p, cudaStream_t st);
cudaError_t launch_kv_few_d128(const KvAttnParams &p, cudaStream_t st);

cudaError_t launch_kv_attn_few(const KvAttnParams &p, cudaStream_t st) {
    switch (p.cache.head_dim) {
    case 32: return launch_kv_few_d32(p, st);
    case 64: return launch_kv_few_d64(p, st);
    case 128: return launch_kv_few_d128(p, st);
    default: return cudaErrorInvalidValue;
    }
}

template <int D>
__global__ void __launch_bounds__(128) k_kv_merge_few(KvAttnParams p) {
    constexpr int RS = D + 2;
    const uint32_t b = blockIdx.y, h = blockIdx.x / p.row_tiles, rt = blockIdx.x % p.row_tiles;
    unsigned fault = 0;
    const KvSeqView seq = kv_load_seq(p.batch, b, p.cache.shift, &fault);  // reported by the parts
    const uint32_t G = (uint32_t)p.group;
    const KvRowTile rows = kv_row_tile(seq, G, rt, p.tile_rows, p.rows_limit);
    if (fault || rows.n == 0) return;
    const KvRange range = kv_range(rows.first, rows.last, p.window, p.sinks);
    const uint32_t total = kv_tiles(range, kKvFewTile).total;
    const uint32_t used = (total + p.tiles_per_split - 1) / p.tiles_per_split;
    const uint32_t pair = (b * p.cache.hkv + h) * p.row_tiles + rt;
    for (uint32_t i = threadIdx.x; i < rows.n * (D / 8); i += blockDim.x) {
        const uint32_t r = i / (D / 8), d0 = (i % (D / 8)) * 8;
        const float *src = p.part + kvf::few_record(pair, p.tile_rows, r, p.nsplit, 0) * RS;
        float top = -INFINITY;
        for (uint32_t s = 0; s < used; s++) top = fmaxf(top, src[(size_t)s * RS + D]);
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0}, lsum = 0.0f;
        for (uint32_t s = 0; s < used; s++) {
            const float *part = src + (size_t)s * RS;
            const float f = part[D] == top ? 1.0f : kvf::pow2_diff(part[D], top);
            lsum = fmaf(part[D + 1], f, lsum);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = fmaf(part[d0 + j], f, v[j]);
        }
        const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= inv;
        const uint32_t tok = (rows.r0 + r) / G, head = h * G + (rows.r0 + r) % G;
        store8(p.out.data, (size_t)(seq.q0 + tok) * p.out.row_stride + head * p.out.head_stride + d0, p.out.fmt, v);
    }
}

cudaError_t launch_kv_merge_few(const KvAttnParams &p, cudaStream_t st) {
    const dim3 grid(p.cache.hkv * p.row_tiles, p.batch.n_seqs);
    switch (p.cache.head_dim) {
    case 32: k_kv_merge_few<32><<<grid, 128, 0, st>>>(p); break;
    case 64: k_kv_merge_few<64><<<grid, 128, 0, st>>>(p); break;
    case 128: k_kv_merge_few<128><<<grid, 128, 0, st>>>(p); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace nx
