// kv_math.cuh -- device helpers of the quantised paged KV cache kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels_kv.h"

namespace nx {

constexpr int kFmtF32 = 0, kFmtF16 = 1, kFmtBf16 = 28;  // NEXUS_FMT_*

__device__ __forceinline__ float kv_nan() { return __int_as_float(0x7fffffff); }

// Eight f16 or bf16 elements of 16 bytes.
__device__ __forceinline__ void unpack16(const uint4 &a, int fmt, float (&v)[8]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (fmt == kFmtBf16) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
// Eight consecutive elements (16-byte aligned) as f32.
__device__ __forceinline__ void load8(const void *base, size_t elem, int fmt, float (&v)[8]) {
    if (fmt == kFmtF32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + elem);
        const float4 a = __ldg(p), b = __ldg(p + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        unpack16(__ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + elem)), fmt, v);
    }
}
__device__ __forceinline__ uint32_t pack16(float a, float b, int fmt) {
    if (fmt == kFmtBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void store8(void *base, size_t elem, int fmt, const float (&v)[8]) {
    if (fmt == kFmtF32) {
        float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(base) + elem);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + elem) =
            make_uint4(pack16(v[0], v[1], fmt), pack16(v[2], v[3], fmt), pack16(v[4], v[5], fmt),
                       pack16(v[6], v[7], fmt));
    }
}

// ---- code unpacking: exact small integers as f16 pairs ----
// (w & mask) | 1024: two f16 values 1024 + field
__device__ __forceinline__ uint32_t kv_field(uint32_t w, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(0x64006400u));
    return r;
}
__device__ __forceinline__ uint32_t kv_hsub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t kv_hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// four 8-bit codes of a word -> (c0, c1), (c2, c3) with c = code - 128
__device__ __forceinline__ void unpack_u8(uint32_t w, uint32_t &p01, uint32_t &p23) {
    uint32_t a, b;
    asm("prmt.b32 %0, %1, 0x64646464, 0x4140;" : "=r"(a) : "r"(w));
    asm("prmt.b32 %0, %1, 0x64646464, 0x4342;" : "=r"(b) : "r"(w));
    p01 = kv_hsub2(a, 0x64806480u);  // 1152
    p23 = kv_hsub2(b, 0x64806480u);
}
// eight 4-bit codes of a word -> (c0, c4), (c1, c5), (c2, c6), (c3, c7) with c = code - 8.
// Fields at bit 4 read as 1024 + 16 code: (1024 + 16 code) / 16 - 72 = code - 8, exact.
__device__ __forceinline__ void unpack_u4(uint32_t w, uint32_t (&p)[4]) {
    const uint32_t s = w >> 8;
    p[0] = kv_hsub2(kv_field(w, 0x000f000fu), 0x64086408u);               // 1032
    p[1] = kv_hfma2(kv_field(w, 0x00f000f0u), 0x2c002c00u, 0xd480d480u);  // * 1/16 - 72
    p[2] = kv_hsub2(kv_field(s, 0x000f000fu), 0x64086408u);
    p[3] = kv_hfma2(kv_field(s, 0x00f000f0u), 0x2c002c00u, 0xd480d480u);
}

// The same codes as they stand, in the low bits of f16 (code * 2^-24): pairs (0, 1),
// (2, 3) of a word of 8-bit codes; (0, 4), 16 * (1, 5), (2, 6), 16 * (3, 7) of 4-bit ones
__device__ __forceinline__ void raw_u8(uint32_t w, uint32_t &p01, uint32_t &p23) {
    asm("prmt.b32 %0, %1, 0, 0x4140;" : "=r"(p01) : "r"(w));
    asm("prmt.b32 %0, %1, 0, 0x4342;" : "=r"(p23) : "r"(w));
}
__device__ __forceinline__ void raw_u4(uint32_t w, uint32_t (&p)[4]) {
    const uint32_t s = w >> 8;
    p[0] = w & 0x000f000fu;
    p[1] = w & 0x00f000f0u;
    p[2] = s & 0x000f000fu;
    p[3] = s & 0x00f000f0u;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- packed pairs of f32 (two results an instruction) ----
typedef unsigned long long f2;
__device__ __forceinline__ f2 pk(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void upk(f2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ float4 lds4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ f2 lds2(uint32_t a) {
    f2 v;
    asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ float lds1(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void sts1(uint32_t a, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }
__device__ __forceinline__ void sts4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ float max4(float4 v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
// the first n of 32 bits, any n
__device__ __forceinline__ uint32_t first_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// 2^e: the largest power of f32 above its range, 0 below it.
__device__ __forceinline__ float pow2i(int e) {
    return __int_as_float(e >= -126 ? (127 + min(e, 127)) << 23 : e >= -149 ? 1 << (149 + e) : 0);
}
// The exponent of a row's largest magnitude, by which a row is brought to one magnitude
// whatever its type: to [2^7, 2^8), where queries have 22 significant bits in f16 hi + lo,
// or to [2^14, 2^15), where codes are met as they stand, 2^-24 each (rows below 2^-112
// stay smaller than that, and their scores with any finite key are below 2^26).  What the
// scores are multiplied by, 2^(scale_exp + row_exp) or so, is held at 2^127: scores of keys
// near one are then beyond 2^111.
__device__ __forceinline__ int row_exp(float amax) {
    return min(127, max(-112, (int)((__float_as_uint(amax) >> 23) & 0xffu) - 127));
}

__device__ __forceinline__ void kv_report(unsigned *fault, unsigned bits) {
    if (bits) atomicOr(fault, bits);
}

__device__ __forceinline__ KvSeqView kv_load_seq(const KvBatchView &bt, uint32_t b, uint32_t shift, unsigned *fault) {
    return kv_seq_view(__ldg(bt.q_start + b), __ldg(bt.q_start + b + 1), __ldg(bt.kv_len + b), bt, shift, fault);
}

}  // namespace nx
