// kernels_kv.cu -- writing new tokens into a quantised paged KV cache, and
// reading them back.
//
// One group is the D elements of one (token, KV head) of keys or values:
//   8 bits: scale = fl(max|x| / 127),  code = rne(x / scale) + 128, the integer held
//           in -127..127 (a subnormal scale can be rounded down by a third)
//   4 bits: scale = fl((max - min) / 15), zero = fl(min + 8 * scale),
//           code = rne((x - zero) / scale) + 8, clamped to 0..15
// with rne the nearest integer, ties to even, of the exact quotient: the
// quotient by a reciprocal in f32 is off by less than 1e-4 of a code, so only
// quotients that near a tie are looked at again, by their remainder.  A group that holds a NaN
// or an infinity (or spans more than f32) gets a NaN scale and reads back as
// NaN throughout, which keeps it from passing as a number.
#include <cuda_runtime.h>

#include "kv_math.cuh"

namespace nx {

constexpr int kKvCopyThreads = 256;

// A thread holds eight elements of a group; D / 8 lanes share one, and a block has
// consecutive rows of one head, whose slots lie next to each other in a page.
template <int D>
struct KvPlace {
    static constexpr int LANES = D / 8, ROWS = kKvCopyThreads / LANES;
    uint32_t row, head;
    int sub;
    int64_t slot;  // -1: padding before the sequence
    bool there;    // the row exists
    __device__ __forceinline__ explicit KvPlace(const KvCopyParams &p) {
        row = blockIdx.x * ROWS + threadIdx.x / LANES;
        head = blockIdx.y;
        sub = threadIdx.x % LANES;
        slot = -1;
        there = row < p.batch.n_rows;
    }
    __device__ __forceinline__ size_t element(const KvRows &r) const {
        return (size_t)row * r.row_stride + (size_t)head * r.head_stride + sub * 8;
    }
    // Finds the row's slot; false where there is nothing to do.
    __device__ __forceinline__ bool find(const KvCopyParams &p) {
        if (!there) return false;
        const uint32_t b = kv_find_seq(p.batch.q_start, p.batch.n_seqs, row);
        if (b >= p.batch.n_seqs) return false;
        unsigned fault = 0;
        const KvSeqView s = kv_load_seq(p.batch, b, p.cache.shift, &fault);
        if (fault || row < s.q0 || row - s.q0 >= s.nq) return false;  // kv_check_batch reports it
        const int pos = (int)s.kv - (int)s.nq + (int)(row - s.q0);
        if (pos < 0) return true;
        const uint32_t page = __ldg(p.batch.table + (size_t)b * p.batch.stride + ((uint32_t)pos >> p.cache.shift));
        if (page >= p.cache.num_pages) {
            if (sub == 0) kv_report(p.fault, KV_FAULT_PAGE);
            return false;
        }
        slot = (int64_t)((((size_t)page * p.cache.hkv + head) << p.cache.shift) +
                         ((uint32_t)pos & ((1u << p.cache.shift) - 1u)));
        return true;
    }
};

// The first block looks every sequence over: a row can belong to a faulty one
// without its own thread seeing that.
__device__ __forceinline__ void kv_check_batch(const KvCopyParams &p) {
    if (blockIdx.x != 0 || blockIdx.y != 0) return;
    unsigned fault = 0;
    for (uint32_t b = threadIdx.x; b < p.batch.n_seqs; b += kKvCopyThreads)
        kv_load_seq(p.batch, b, p.cache.shift, &fault);
    kv_report(p.fault, fault);
}

// One side of a group.  Bound by instructions unless they are few (all checks
// element by element, rint and integer conversions: 130 us for 32194 tokens of
// eight heads, whose bytes take 31): the nearest integer is taken by adding and
// subtracting 1.5 * 2^23, whose low byte is the code, and what is rare is looked
// for once a thread: a quotient near a tie, a value that is not a number.
template <int D, int BITS>
__device__ __forceinline__ void kv_quantise_group(float (&x)[8], uint8_t *codes, float *scales, int64_t slot, int sub,
                                                  unsigned lanes) {
    constexpr int LANES = D / 8;
    constexpr float kRound = 12582912.0f;
    float lo = x[0], hi = x[0], odd = 0.0f;  // odd: NaN where some x is not finite
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (BITS == 8) hi = fmaxf(hi, fabsf(x[i]));
        else {
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
        }
        odd = fmaf(x[i], 0.0f, odd);
    }
    if constexpr (BITS == 8) hi = fabsf(hi);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        if constexpr (BITS == 4) lo = fminf(lo, __shfl_xor_sync(lanes, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(lanes, hi, o));
        odd += __shfl_xor_sync(lanes, odd, o);
    }
    float scale, zero = 0.0f;
    if constexpr (BITS == 8) {
        scale = __fdiv_rn(hi, 127.0f);
    } else {
        scale = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
        zero = __fadd_rn(lo, 8.0f * scale);
    }
    constexpr float low = BITS == 8 ? -127.0f : -8.0f, high = BITS == 8 ? 127.0f : 7.0f;
    const bool finite = odd == 0.0f && scale <= 3.4028235e38f;
    uint32_t t[8];  // 1.5 * 2^23 + code
    if (!finite || scale == 0.0f) {
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = __float_as_uint(kRound);
        if (!finite) scale = zero = kv_nan();
    } else {
        float step = scale, mid = zero;
        if (scale < 1e-30f) {
            // so that the reciprocal stays in f32: by 2^96, exactly (elements that span so
            // little are as small themselves)
            constexpr float kUp96 = 7.9228163e28f;
            step *= kUp96;
            mid *= kUp96;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] *= kUp96;
                // a subnormal scale can be rounded down by up to a third: quotients beyond 127
                // (4-bit ones are clamped below, whatever the scale)
                if constexpr (BITS == 8) x[i] = fminf(fmaxf(x[i], low * step), high * step);
            }
        }
        const float inv = __fdividef(1.0f, step);
        float far = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float q = (BITS == 8 ? x[i] : __fsub_rn(x[i], mid)) * inv;
            if constexpr (BITS == 4) q = fminf(fmaxf(q, low), high);  // (a rounded zero can shift the range)
            const float r = __fadd_rn(q, kRound);
            far = fmaxf(far, fabsf(q - __fsub_rn(r, kRound)));
            t[i] = __float_as_uint(r);
        }
        if (far > 0.4999f) {
            // Near a tie (common: coarse inputs meet ties exactly) the remainder decides, in
            // f32 without an error: d + e = x - zero by two-sum, d - code * scale is a
            // multiple of scale's last place below scale, and its difference to scale / 2
            // one of two neighbours.
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float code = __fsub_rn(__uint_as_float(t[i]), kRound);
                float d = x[i], e = 0.0f;
                if constexpr (BITS == 4) {
                    d = __fsub_rn(x[i], mid);
                    const float bb = __fsub_rn(d, x[i]);
                    e = __fadd_rn(__fsub_rn(x[i], __fsub_rn(d, bb)), -__fadd_rn(mid, bb));
                }
                const float left = __fmaf_rn(-code, step, d), side = left < 0.0f ? -1.0f : 1.0f;
                const float over = __fadd_rn(__fsub_rn(fabsf(left), 0.5f * step), side * e);
                const bool odd_code = t[i] & 1u;
                float c = code;
                if (over > 0.0f || (over == 0.0f && odd_code)) c = __fadd_rn(code, side);
                t[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(c, low), high), kRound));
            }
        }
    }
    if constexpr (BITS == 8) {
        uint2 w;
        w.x = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410) ^ 0x80808080u;
        w.y = __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410) ^ 0x80808080u;
        *reinterpret_cast<uint2 *>(codes + (size_t)slot * D + sub * 8) = w;
        if (sub == 0) scales[slot] = scale;
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) w |= (t[i] & 0xfu) << (4 * i);
        *reinterpret_cast<uint32_t *>(codes + (size_t)slot * (D / 2) + sub * 4) = w ^ 0x88888888u;
        if (sub == 0) *reinterpret_cast<float2 *>(scales + 2 * slot) = make_float2(scale, zero);
    }
}

template <int D>
__global__ void __launch_bounds__(kKvCopyThreads, 5) k_kv_append(KvCopyParams p) {
    constexpr int LANES = D / 8;
    KvPlace<D> at(p);
    // the elements are on their way while the slot is looked up
    float x[2][8];
#pragma unroll
    for (int s = 0; s < 2; s++)
        if (at.there) load8(p.rows[s].data, at.element(p.rows[s]), p.rows[s].fmt, x[s]);
    kv_check_batch(p);
    // (the lanes of a group agree on everything but `sub`)
    if (!at.find(p) || at.slot < 0) return;
    const int lane = threadIdx.x & 31;
    const unsigned lanes = ((1u << LANES) - 1u) << (lane & ~(LANES - 1));
#pragma unroll
    for (int s = 0; s < 2; s++) {
        if (p.cache.bits[s] == 8)
            kv_quantise_group<D, 8>(x[s], p.cache.codes[s], p.cache.scales[s], at.slot, at.sub, lanes);
        else
            kv_quantise_group<D, 4>(x[s], p.cache.codes[s], p.cache.scales[s], at.slot, at.sub, lanes);
    }
}

template <int D>
__global__ void __launch_bounds__(kKvCopyThreads) k_kv_read(KvCopyParams p) {
    kv_check_batch(p);
    KvPlace<D> at(p);
    if (!at.find(p)) return;
    const int64_t slot = at.slot;
    const int sub = at.sub;
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
                // 2^23 + code as f32 bits, less 2^23 + 128
                v[i] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(i < 4 ? w.x : w.y, 0x4b000000u, 0x7540 | (i & 3))), 8388736.0f), scale);
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(p.cache.codes[s] + (size_t)slot * (D / 2) + sub * 4);
            const float2 sz = *reinterpret_cast<const float2 *>(p.cache.scales[s] + 2 * slot);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __fmaf_rn(sz.x, __fsub_rn(__uint_as_float(((w >> (4 * i)) & 0xfu) | 0x4b000000u), 8388616.0f), sz.y);
        }
        store8(p.rows[s].data, at.element(p.rows[s]), p.rows[s].fmt, v);
    }
}

template <bool APPEND>
static cudaError_t launch_kv_copy(const KvCopyParams &p, cudaStream_t st) {
    const uint32_t rows = kKvCopyThreads / ((uint32_t)p.cache.head_dim / 8);
    const dim3 g((p.batch.n_rows + rows - 1) / rows, p.cache.hkv), t(kKvCopyThreads);
    if (g.x == 0) return cudaSuccess;
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
