// kernels_kv.cu -- writing new tokens into a quantised paged KV cache, and
// reading them back.
//
// One group is the D elements of one (token, KV head) of keys or values:
//   8 bits: scale = fl(max|x| / 127),  code = rne(x / scale) + 128
//   4 bits: scale = fl((max - min) / 15), zero = fl(min + 8 * scale),
//           code = rne((x - zero) / scale) + 8, clamped to 0..15
// with rne the nearest integer, ties to even, of the exact quotient: the
// quotient by a reciprocal in f32 is off by less than 1e-4 of a code, so only
// quotients that near a tie are taken again in f64.  A group that holds a NaN
// or an infinity (or spans more than f32) gets a NaN scale and reads back as
// NaN throughout, which keeps it from passing as a number.
#include <cuda_runtime.h>

#include "kv_math.cuh"

namespace nx {

constexpr int kKvCopyThreads = 256;

// A thread holds eight elements of a group; D / 8 lanes share one.
template <int D>
__device__ __forceinline__ bool kv_copy_place(const KvCopyParams &p, uint32_t &row, uint32_t &head, int &sub,
                                              int64_t &slot) {
    constexpr int LANES = D / 8;
    const uint64_t gid = (uint64_t)blockIdx.x * kKvCopyThreads + threadIdx.x;
    const uint64_t item = gid / LANES;
    sub = (int)(gid % LANES);
    row = (uint32_t)(item / p.cache.hkv);
    head = (uint32_t)(item % p.cache.hkv);
    slot = -1;
    if (row >= p.batch.n_rows) return false;
    const uint32_t b = kv_find_seq(p.batch.q_start, p.batch.n_seqs, row);
    if (b >= p.batch.n_seqs) return false;
    unsigned fault = 0;
    const KvSeqView s = kv_load_seq(p.batch, b, p.cache.shift, &fault);
    if (fault || row < s.q0 || row - s.q0 >= s.nq) return false;  // kv_check_batch reports it
    const int pos = (int)s.kv - (int)s.nq + (int)(row - s.q0);
    if (pos < 0) return true;  // padding before the sequence: no slot
    const uint32_t page = __ldg(p.batch.table + (size_t)b * p.batch.stride + ((uint32_t)pos >> p.cache.shift));
    if (page >= p.cache.num_pages) {
        if (sub == 0) kv_report(p.fault, KV_FAULT_PAGE);
        return false;
    }
    slot = (int64_t)((((size_t)page * p.cache.hkv + head) << p.cache.shift) +
                     ((uint32_t)pos & ((1u << p.cache.shift) - 1u)));
    return true;
}

// The first block looks every sequence over: a row can belong to a faulty one
// without its own thread seeing that.
__device__ __forceinline__ void kv_check_batch(const KvCopyParams &p) {
    if (blockIdx.x != 0) return;
    unsigned fault = 0;
    for (uint32_t b = threadIdx.x; b < p.batch.n_seqs; b += kKvCopyThreads)
        kv_load_seq(p.batch, b, p.cache.shift, &fault);
    kv_report(p.fault, fault);
}

template <int D>
__device__ __forceinline__ void kv_quantise_group(const float (&x)[8], int bits, uint8_t *codes, float *scales,
                                                  int64_t slot, int sub, unsigned lanes) {
    constexpr int LANES = D / 8;
    // magnitudes compare as integers; a NaN or infinity is the largest
    unsigned top = 0;
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        top = max(top, __shfl_xor_sync(lanes, top, o));
        lo = fminf(lo, __shfl_xor_sync(lanes, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(lanes, hi, o));
    }
    float scale, zero;
    int low, high, mid;
    if (bits == 8) {
        scale = __fdiv_rn(__uint_as_float(top), 127.0f);
        zero = 0.0f;
        low = -127;
        high = 127;
        mid = 128;
    } else {
        scale = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
        zero = __fadd_rn(lo, 8.0f * scale);
        low = -8;
        high = 7;
        mid = 8;
    }
    const bool finite = top < 0x7f800000u && scale <= 3.4028235e38f;
    int c[8];
    if (!finite || scale == 0.0f) {
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = mid;
        if (!finite) scale = zero = kv_nan();
    } else {
        const bool tiny = scale < 1e-30f;  // the reciprocal would leave f32
        const float inv = tiny ? 0.0f : __fdividef(1.0f, scale);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float q = __fsub_rn(x[i], zero) * inv;
            float r = rintf(q);
            if (tiny || fabsf(q - r) > 0.4999f)
                r = (float)rint(((double)x[i] - (double)zero) / (double)scale);
            c[i] = min(high, max(low, (int)r)) + mid;
        }
    }
    if (bits == 8) {
        uint2 w;
        w.x = (uint32_t)c[0] | ((uint32_t)c[1] << 8) | ((uint32_t)c[2] << 16) | ((uint32_t)c[3] << 24);
        w.y = (uint32_t)c[4] | ((uint32_t)c[5] << 8) | ((uint32_t)c[6] << 16) | ((uint32_t)c[7] << 24);
        *reinterpret_cast<uint2 *>(codes + (size_t)slot * D + sub * 8) = w;
        if (sub == 0) scales[slot] = scale;
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) w |= (uint32_t)c[i] << (4 * i);
        *reinterpret_cast<uint32_t *>(codes + (size_t)slot * (D / 2) + sub * 4) = w;
        if (sub == 0) *reinterpret_cast<float2 *>(scales + 2 * slot) = make_float2(scale, zero);
    }
}

template <int D>
__global__ void __launch_bounds__(kKvCopyThreads) k_kv_append(KvCopyParams p) {
    constexpr int LANES = D / 8;
    kv_check_batch(p);
    uint32_t row, head;
    int sub;
    int64_t slot;
    // the lanes of a group agree on everything but `sub`
    if (!kv_copy_place<D>(p, row, head, sub, slot) || slot < 0) return;
    const int lane = threadIdx.x & 31;
    const unsigned lanes = ((1u << LANES) - 1u) << (lane & ~(LANES - 1));
    float x[2][8];
#pragma unroll
    for (int s = 0; s < 2; s++)
        load8(p.rows[s].data, (size_t)row * p.rows[s].row_stride + head * p.rows[s].head_stride + sub * 8,
              p.rows[s].fmt, x[s]);
#pragma unroll
    for (int s = 0; s < 2; s++)
        kv_quantise_group<D>(x[s], p.cache.bits[s], p.cache.codes[s], p.cache.scales[s], slot, sub, lanes);
}

template <int D>
__global__ void __launch_bounds__(kKvCopyThreads) k_kv_read(KvCopyParams p) {
    kv_check_batch(p);
    uint32_t row, head;
    int sub;
    int64_t slot;
    if (!kv_copy_place<D>(p, row, head, sub, slot)) return;
#pragma unroll
    for (int s = 0; s < 2; s++) {
        if (!p.rows[s].data) continue;
        float v[8];
        if (slot < 0) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0.0f;
        } else if (p.cache.bits[s] == 8) {
            const uint2 w = *reinterpret_cast<const uint2 *>(p.cache.codes[s] + (size_t)slot * D + sub * 8);
            const float scale = p.cache.scales[s][slot];
#pragma unroll
            for (int i = 0; i < 8; i++)
                v[i] = __fmul_rn((float)((int)(((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xffu) - 128), scale);
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(p.cache.codes[s] + (size_t)slot * (D / 2) + sub * 4);
            const float2 sz = *reinterpret_cast<const float2 *>(p.cache.scales[s] + 2 * slot);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __fmaf_rn(sz.x, (float)((int)((w >> (4 * i)) & 0xfu) - 8), sz.y);
        }
        store8(p.rows[s].data, (size_t)row * p.rows[s].row_stride + head * p.rows[s].head_stride + sub * 8,
               p.rows[s].fmt, v);
    }
}

template <bool APPEND>
static cudaError_t launch_kv_copy(const KvCopyParams &p, cudaStream_t st) {
    const uint64_t threads = (uint64_t)p.batch.n_rows * p.cache.hkv * (uint64_t)(p.cache.head_dim / 8);
    const uint64_t blocks = (threads + kKvCopyThreads - 1) / kKvCopyThreads;
    if (blocks == 0) return cudaSuccess;
    if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
    const dim3 g((unsigned)blocks), t(kKvCopyThreads);
    switch (p.cache.head_dim) {
    case 32:
        if (APPEND) k_kv_append<32><<<g, t, 0, st>>>(p);
        else k_kv_read<32><<<g, t, 0, st>>>(p);
        break;
    case 64:
        if (APPEND) k_kv_append<64><<<g, t, 0, st>>>(p);
        else k_kv_read<64><<<g, t, 0, st>>>(p);
        break;
    case 128:
        if (APPEND) k_kv_append<128><<<g, t, 0, st>>>(p);
        else k_kv_read<128><<<g, t, 0, st>>>(p);
        break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_kv_append(const KvCopyParams &p, cudaStream_t st) { return launch_kv_copy<true>(p, st); }
cudaError_t launch_kv_read(const KvCopyParams &p, cudaStream_t st) { return launch_kv_copy<false>(p, st); }

}  // namespace nx
