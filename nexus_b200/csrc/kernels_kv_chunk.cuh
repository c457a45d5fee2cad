// kernels_kv_chunk.cuh -- attention of a chunk of new tokens over the quantised
// paged KV cache, on the 5th-generation tensor cores.
//
// The mathematics is that of kernels_kv_few.cuh with one reference a row:
//   x_rj = c_r (sk_j (q_r . kc_j) + zk_j sum(q_r)),  p = 2^(x - ref_r)
//   o_r  = ( sum_j (p sv_j) vc_j + sum_j p zv_j ) / sum_j p
// kc, vc integer codes around zero (exact in f16), q as f16 (hi + lo for f32
// queries), the weights p sv rounded to f16 (hi + lo for f32).  ref is a whole
// number chosen so that the largest p * max(sv, |zv|) of the row lies between
// 2^kUp-1 and 2^15; it moves only when a weight would pass 2^15, and then by
// an exact power of two (p alone is kept below 2^60 where values are zero, and
// the values' scales are brought near one first, as there).
//
// Bound: the tensor pipe (4 D flops a visible pair) and, next to it, the
// shared-memory bandwidth that feeds it.  One CTA an SM, 256 rows (row r: token
// r / G, head r % G) in two tiles of 128, keys in tiles of 128 tokens:
//   warps 0-3, 4-7  softmax of row tile 0, 1 (a thread owns a row)
//   warps 8-11      unpack the codes of a key tile into f16 operands in shared
//                   memory (128-byte swizzle), loads one tile ahead in registers
//   warp 12         tcgen05.mma issue: S = Q K^T (128 x 128 x D) and O += P V
// S and O of both tiles fill tensor memory; P overwrites S in place.  While the
// softmax of one tile runs, the tensor pipe works for the other.  Keys come in
// by registers rather than TMA because they must be unpacked on the way.
// Every wait is bounded (as in kernels_gemm.cuh).
#pragma once
#include <type_traits>

#include "kernels_kv_few.cuh"
#include "tcgen05.cuh"

namespace nx {
namespace kvc {
using namespace tc;
using kvf::f16x2;
using kvf::f16x2_back;
using kvf::lg2;
using kvf::pow2_diff;

constexpr int kRows = kKvChunkRows;     // rows of a CTA: two tiles of 128
constexpr int kTok = kKvChunkTile;      // tokens of a key tile
// Four warpgroups; registers move from the copying and issuing ones to the
// softmax (the sum stays at the launch's 512 x 128)
constexpr int kThreads = 16 * 32;
constexpr int kRegsSoftmax = 160, kRegsProducer = 128, kRegsIssue = 64;
static_assert(2 * kRegsSoftmax + kRegsProducer + kRegsIssue <= 4 * 128, "more registers than the block has");
constexpr int kBlk = 128 * 128;         // 128 rows x 64 f16, swizzled
constexpr float kUp = 7.0f;             // a new reference puts the largest weight at 2^6 .. 2^7
constexpr float kMaxWeight = 32768.0f;  // and it is moved when a weight passes 2^15
constexpr float kMaxProb = 60.0f;       // log2 of the largest p where values are zero
constexpr int kScaleSlots = 4;

struct alignas(16) ScaleSlot {
    float sk[kTok], zk[kTok], sv[kTok], zv[kTok], lv[kTok];  // lv = log2 max(sv, |zv|)
    float zmax[4];                                           // largest |zv| per producer warp
    float unit;                                              // what sv and zv were divided by
};

template <int D, bool SPLIT>
struct Smem {
    static constexpr int DB = (D + 63) / 64;
    static constexpr int NQ = SPLIT ? 2 : 1;
    static constexpr int Q_SUB = DB * kBlk * NQ;
    static constexpr int KV = DB * kBlk;
    static constexpr int STAGES = SPLIT && D == 128 ? 1 : 2;
    static constexpr int K0 = 2 * Q_SUB, V0 = K0 + STAGES * KV, SC = V0 + STAGES * KV;
    static constexpr int NEED = SC + kScaleSlots * (int)sizeof(ScaleSlot) + 1024;
    // at least 120 KB: one CTA an SM, since each takes all of tensor memory
    static constexpr int TOTAL = NEED > 120 * 1024 ? NEED : 120 * 1024;
};

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

// 32 columns of the warp's lanes, complete on return.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
// 16 columns: started, and waited for (with every load started before).
__device__ __forceinline__ void tmem_ld16_start(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
// Eight columns, complete on return.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ uint32_t hmul2u(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Operand descriptor, 128-byte swizzle (bits 61-63 = 2), version 1.  K-major:
// 8-row groups 1024 bytes apart (SBO), LBO unused.  MN-major: 64-element blocks
// LBO apart, 8-row (K) groups SBO = 1024 apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)((lbo >> 4) & 0x3fffu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// D f32, A and B f16, M = 128; `mn_b`: B is MN-major
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool mn_b) {
    return (1u << 4) | (mn_b ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// Bounded mbarrier wait; false once this CTA has given up.
__device__ __forceinline__ bool wait_or_fault(unsigned long long *bar, unsigned parity, volatile int *abort_flag,
                                              unsigned *fault) {
    unsigned n = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++n & 255u) == 0) {
            if (*abort_flag) return false;
            if (n > kSpin) {
                *abort_flag = 1;
                atomicOr(fault, KV_FAULT_WAIT);
                return false;
            }
        }
    }
    return true;
}

template <int N>
__device__ __forceinline__ void regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int D, int BK, int BV, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) k_kv_attn_chunk(KvAttnParams p) {
    using S = Smem<D, SPLIT>;
    constexpr int ST = S::STAGES;
    constexpr int RK = D * BK / 8, RV = D * BV / 8;  // code bytes of a token
    constexpr uint32_t kSCol = 0, kOCol = 256;       // per row tile: + 128, + D
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    ScaleSlot *slots = reinterpret_cast<ScaleSlot *>(smem + S::SC);
    __shared__ unsigned long long kfull[2], kempty[2], vfull[2], vempty[2], scfull[kScaleSlots], sfull[2], pready[2],
        qfull, odone;
    __shared__ uint32_t tmem_base_s;
    __shared__ volatile int abort_s;
    __shared__ float row_x[kRows], row_sum[kRows];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = blockIdx.y % p.nsplit, h = blockIdx.x, b = blockIdx.z;
    const uint32_t rt = p.row_tiles - 1 - blockIdx.y / p.nsplit;  // the longest rows first
    unsigned fault = 0;
    const KvSeqView seq = kv_load_seq(p.batch, b, p.cache.shift, &fault);
    if (fault) {
        if (threadIdx.x == 0) kv_report(p.fault, fault);
        return;
    }
    const uint32_t G = (uint32_t)p.group;
    if ((uint64_t)seq.nq * G <= p.rows_limit) return;  // the few-row kernel's
    const KvRowTile rows = kv_row_tile(seq, G, rt, kRows, 0xffffffffu);
    if (rows.n == 0) return;
    const int pos0 = (int)seq.kv - (int)seq.nq;
    const KvRange range = kv_range(rows.first, rows.last, p.window, p.sinks);
    const KvTiles tiles = kv_tiles(range, kTok);
    const uint32_t t_begin = split * p.tiles_per_split, t_end = min(tiles.total, t_begin + p.tiles_per_split);
    if (p.nsplit > 1 && t_begin >= t_end) return;  // the merge knows how many parts there are
    const uint32_t n = t_begin < t_end ? t_end - t_begin : 0;
    // the two row tiles: positions and what they read
    const uint32_t n0 = min(rows.n, 128u), n1 = rows.n - n0;
    const int last0 = pos0 + (int)((rows.r0 + n0 - 1) / G), first1 = pos0 + (int)((rows.r0 + n0) / G);
    const KvRange range0 = kv_range(rows.first, last0, p.window, p.sinks);
    const KvRange range1 = n1 ? kv_range(first1, rows.last, p.window, p.sinks) : KvRange{0u, 0u, 0u};
    auto tile_token = [&](uint32_t i) { return kv_tile_at(tiles, t_begin + i) * kTok; };
    auto active = [&](int sub, uint32_t i) {
        const uint32_t j0 = tile_token(i);
        return kv_needed(sub ? range1 : range0, j0, j0 + kTok);
    };

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&kfull[i], 4);
            mbar_init(&kempty[i], 1);
            mbar_init(&vfull[i], 4);
            mbar_init(&vempty[i], 1);
            mbar_init(&sfull[i], 1);
            mbar_init(&pready[i], 4);
        }
        for (int i = 0; i < kScaleSlots; i++) mbar_init(&scfull[i], 4);
        mbar_init(&qfull, 8);
        mbar_init(&odone, 1);
        abort_s = 0;
        mbar_init_fence();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base_s))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;

    if (warp < 8) {
        // ================= softmax: a thread owns a row =================
        regs_inc<kRegsSoftmax>();
        const int sub = warp >> 2, wq = warp & 3;
        const uint32_t t_lane = (uint32_t)(32 * wq) << 16;
        {
            // this warp's 32 query rows to shared memory, D / 8 lanes a row
            constexpr int LPR = D / 8, RPP = 32 / LPR;
            uint8_t *qs = smem + sub * S::Q_SUB;
#pragma unroll 2
            for (int pass = 0; pass < LPR; pass++) {
                const int rr = 32 * wq + pass * RPP + lane / LPR, cl = lane % LPR;
                const uint32_t in_tile = (uint32_t)(sub * 128 + rr), r = rows.r0 + in_tile;
                float q[8];
                if (in_tile < rows.n) {
                    load8(p.q.data, (size_t)(seq.q0 + r / G) * p.q.row_stride + (h * G + r % G) * p.q.head_stride + cl * 8,
                          p.q.fmt, q);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) q[i] = 0.0f;
                }
                float amax = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(q[i]));
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const float sc = row_scale(amax);
                // elements in the order the codes of a word unpack to
                constexpr int o8[8] = {0, 1, 2, 3, 4, 5, 6, 7}, o4[8] = {0, 4, 1, 5, 2, 6, 3, 7};
                uint32_t hi[4], lo[4];
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v0 = q[BK == 8 ? o8[2 * i] : o4[2 * i]] * sc;
                    const float v1 = q[BK == 8 ? o8[2 * i + 1] : o4[2 * i + 1]] * sc;
                    hi[i] = f16x2(v0, v1);
                    const float2 back = f16x2_back(hi[i]);
                    sum += back.x + back.y;
                    if constexpr (SPLIT) {
                        lo[i] = f16x2(v0 - back.x, v1 - back.y);
                        const float2 lb = f16x2_back(lo[i]);
                        sum += lb.x + lb.y;
                    }
                }
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                uint8_t *dst = qs + (cl >> 3) * kBlk + rr * 128 + (((cl & 7) ^ (rr & 7)) << 4);
                *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (SPLIT)
                    *reinterpret_cast<uint4 *>(dst + S::DB * kBlk) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                if (cl == 0) {
                    row_x[sub * 128 + rr] = p.scale_log2 / sc;
                    row_sum[sub * 128 + rr] = sum;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&qfull);
        }
        const uint32_t in_tile = (uint32_t)(sub * 128 + 32 * wq + lane), r = rows.r0 + in_tile;
        const bool valid = in_tile < rows.n;
        const int pos = valid ? pos0 + (int)(r / G) : -1;
        const float xs = row_x[in_tile], qsum = row_sum[in_tile];
        const f2 xs2 = pk(xs, xs), qsum2 = pk(qsum, qsum);
        const int first = sub ? first1 : rows.first, last = sub ? rows.last : last0;
        // rows that see nothing start with a reference of their own: they never ask for one
        float ref = pos >= 0 ? -INFINITY : 0.0f;
        float unit = 1.0f;
        f2 l2 = pk(0.0f, 0.0f), z2 = l2;  // sums of p and p zv, even and odd columns apart
        const uint32_t scol = tmem + t_lane + kSCol + 128 * sub, ocol = tmem + t_lane + kOCol + D * sub;
        unsigned cnt = 0;
        bool ok = true;
        for (uint32_t i = 0; i < n; i++) {
            if (!active(sub, i)) continue;
            const int j0 = (int)tile_token(i);
            const ScaleSlot *sl = slots + (i % kScaleSlots);
            ok = wait_or_fault(&scfull[i % kScaleSlots], (i / kScaleSlots) & 1, &abort_s, p.fault) &&
                 wait_or_fault(&sfull[sub], cnt & 1, &abort_s, p.fault);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const bool whole = j0 + kTok - 1 <= first &&
                               (p.window == 0 || j0 > last - (int)p.window || j0 + kTok <= (int)p.sinks);
            // visible keys of this row within the tile: [lo, hi) and [0, sink)
            const int hi = pos - j0 + 1, lo = p.window ? max(0, pos - (int)p.window + 1) - j0 : -1;
            const int sink = (int)min(p.sinks, 0x3fffffffu) - j0;
            unit = sl->unit;
            const float zm = fmaxf(fmaxf(sl->zmax[0], sl->zmax[1]), fmaxf(sl->zmax[2], sl->zmax[3]));
            const float plim = BV == 8 ? 9.2e18f : 1.2e30f / fmaxf(zm, 1.3e11f);  // 2^63, 2^100 / |zv|

            // scores of columns c0 .. c0 + 3 in base 2, before the row's factor
            auto scores4 = [&](const uint32_t *s, int c0, f2 &x01, f2 &x23) {
                const float4 sk = *reinterpret_cast<const float4 *>(sl->sk + c0);
                x01 = mul2(pk(__uint_as_float(s[0]), __uint_as_float(s[1])), pk(sk.x, sk.y));
                x23 = mul2(pk(__uint_as_float(s[2]), __uint_as_float(s[3])), pk(sk.z, sk.w));
                if constexpr (BK == 4) {
                    const float4 zk = *reinterpret_cast<const float4 *>(sl->zk + c0);
                    x01 = fma2(pk(zk.x, zk.y), qsum2, x01);
                    x23 = fma2(pk(zk.z, zk.w), qsum2, x23);
                }
            };
            auto seen = [&](int c) { return (c < hi && c >= lo) || (c < sink && c < hi); };
            // A reference for all that has been summed and columns 16 c0 .. of this
            // tile; what has been summed follows: l, z, the output, and the weights
            // of this tile already written.
            auto new_reference = [&](int c0) {
                float mx = -INFINITY, my = -INFINITY;
#pragma unroll 1
                for (int c = c0; c < 8; c++) {
                    uint32_t s[16];
                    tmem_ld16_start(scol + 16 * c, s);
                    tmem_ld16_wait(s);
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const int col = 16 * c + j;
                        f2 x[2];
                        scores4(s + j, col, x[0], x[1]);
                        const float4 lv = *reinterpret_cast<const float4 *>(sl->lv + col);
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            float e0, e1;
                            upk(mul2(x[t], xs2), e0, e1);
                            if (!whole) {
                                e0 = seen(col + 2 * t) ? e0 : -INFINITY;
                                e1 = seen(col + 2 * t + 1) ? e1 : -INFINITY;
                            }
                            mx = fmaxf(mx, fmaxf(e0, e1));
                            my = fmaxf(my, fmaxf(e0 + (t ? lv.z : lv.x), e1 + (t ? lv.w : lv.y)));
                        }
                    }
                }
                const float next = fmaxf(ref, fmaxf(ceilf(my) - kUp, ceilf(mx) - kMaxProb));
                const float f = next == ref ? 1.0f : pow2_diff(ref, next);
                ref = next;
                l2 = mul2(l2, pk(f, f));
                z2 = mul2(z2, pk(f, f));
                if (!__any_sync(0xffffffffu, f != 1.0f)) return;
                if (cnt > 0) {
                    // the products so far are complete: S of this tile was issued after them
#pragma unroll 1
                    for (int c = 0; c < D / 16; c++) {
                        uint32_t o[16];
                        tmem_ld16_start(ocol + 16 * c, o);
                        tmem_ld16_wait(o);
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                        tmem_st16(ocol + 16 * c, o);
                    }
                }
                tmem_wait_st();
                const uint32_t fh = f16x2(f, f);
#pragma unroll 1
                for (int c = 0; c < c0 * S::NQ; c++) {
                    uint32_t w[8];
                    tmem_ld8(scol + 8 * c, w);
#pragma unroll
                    for (int j = 0; j < 8; j++) w[j] = hmul2u(w[j], fh);
                    tmem_st8(scol + 8 * c, w);
                }
            };
            // The weights of 16 columns (those of `cur`, while the loads of the next
            // into `nxt` run) against the current reference, over the scores in place.
            auto weigh16 = [&](auto masked, int c, uint32_t(&cur)[16], uint32_t(&nxt)[16]) {
                constexpr bool MASK = decltype(masked)::value;
                tmem_ld16_wait(cur);
                if (c < 7) tmem_ld16_start(scol + 16 * (c + 1), nxt);
                uint32_t ph[8];
                [[maybe_unused]] uint32_t pl[8];
                f2 l_c, z_c;
                for (bool again = false;; again = true) {
                    const float rf = ref == -INFINITY ? 0.0f : ref;
                    const f2 nref = pk(-rf, -rf);
                    float pmax = 0.0f, wmax = 0.0f;
                    l_c = z_c = pk(0.0f, 0.0f);
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const int col = 16 * c + j;
                        f2 x[2];
                        scores4(cur + j, col, x[0], x[1]);
                        const float4 sv = *reinterpret_cast<const float4 *>(sl->sv + col);
                        [[maybe_unused]] float4 zv;
                        if constexpr (BV == 4) zv = *reinterpret_cast<const float4 *>(sl->zv + col);
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            float e0, e1;
                            upk(fma2(x[t], xs2, nref), e0, e1);
                            float sv0 = t ? sv.z : sv.x, sv1 = t ? sv.w : sv.y;
                            bool b0 = true, b1 = true;
                            if constexpr (MASK) {
                                b0 = seen(col + 2 * t);
                                b1 = seen(col + 2 * t + 1);
                                e0 = b0 ? e0 : -INFINITY;
                                e1 = b1 ? e1 : -INFINITY;
                                sv0 = b0 ? sv0 : 0.0f;
                                sv1 = b1 ? sv1 : 0.0f;
                            }
                            const float p0 = ex2(e0), p1 = ex2(e1);
                            const f2 pp = pk(p0, p1);
                            l_c = add2(l_c, pp);
                            pmax = fmaxf(pmax, fmaxf(p0, p1));
                            if constexpr (BV == 4) {
                                float z0 = t ? zv.z : zv.x, z1 = t ? zv.w : zv.y;
                                if constexpr (MASK) {
                                    z0 = b0 ? z0 : 0.0f;
                                    z1 = b1 ? z1 : 0.0f;
                                }
                                z_c = fma2(pp, pk(z0, z1), z_c);
                            }
                            float w0, w1;
                            upk(mul2(pp, pk(sv0, sv1)), w0, w1);
                            wmax = fmaxf(wmax, fmaxf(w0, w1));
                            const uint32_t hw = f16x2(w0, w1);
                            ph[j / 2 + t] = hw;
                            if constexpr (SPLIT) {
                                const float2 back = f16x2_back(hw);
                                pl[j / 2 + t] = f16x2(w0 - back.x, w1 - back.y);
                            }
                        }
                    }
                    const bool over = ref == -INFINITY || wmax > kMaxWeight || pmax > plim;
                    if (again || !__any_sync(0xffffffffu, over)) break;
                    new_reference(c);
                }
                l2 = add2(l2, l_c);
                z2 = add2(z2, z_c);
                tmem_st8(scol + 8 * S::NQ * c, ph);
                if constexpr (SPLIT) tmem_st8(scol + 8 * S::NQ * c + 8, pl);
            };
            uint32_t sa[16], sb[16];
            tmem_ld16_start(scol, sa);
            auto tile = [&](auto masked) {
#pragma unroll 1
                for (int c = 0; c < 8; c += 2) {
                    weigh16(masked, c, sa, sb);
                    weigh16(masked, c + 1, sb, sa);
                }
            };
            if (whole) tile(std::false_type{});
            else tile(std::true_type{});
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pready[sub]);
            cnt++;
        }
        // ---- output ----
        if (ok) ok = wait_or_fault(&odone, 0, &abort_s, p.fault);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
            tc_fence_after();
            float l, z, odd;
            upk(l2, l, odd);
            l += odd;
            upk(z2, z, odd);
            z += odd;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const uint32_t tile_id = (b * p.cache.hkv + h) * p.row_tiles + rt;
            float *rec = p.nsplit > 1 ? p.part + kvf::few_record(tile_id, kRows, in_tile, p.nsplit, split) * (D + 2)
                                      : nullptr;
            const size_t at = (size_t)(seq.q0 + r / G) * p.out.row_stride + (h * G + r % G) * p.out.head_stride;
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                float o[32];
                if (cnt > 0) {
                    tmem_ld32(ocol + 32 * c, o);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++) o[j] = 0.0f;
                }
                if (valid) {
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        // positions of elements 0..7 within a unit of value codes
                        constexpr int i8[8] = {0, 1, 2, 3, 4, 5, 6, 7}, i4[8] = {0, 2, 4, 6, 1, 3, 5, 7};
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) v[e] = (o[8 * u + (BV == 8 ? i8[e] : i4[e])] + z) * unit;
                        if (rec) {
#pragma unroll
                            for (int e = 0; e < 8; e += 2)
                                *reinterpret_cast<float2 *>(rec + 32 * c + 8 * u + e) = make_float2(v[e], v[e + 1]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; e++) v[e] *= inv;
                            store8(p.out.data, at + 32 * c + 8 * u, p.out.fmt, v);
                        }
                    }
                }
            }
            if (rec && valid) *reinterpret_cast<float2 *>(rec + D) = make_float2(l == 0.0f ? -INFINITY : ref, l);
        }
    } else if (warp < 12) {
        // ================= producers: codes to f16 operands =================
        regs_dec<kRegsProducer>();
        const int pt = threadIdx.x - 256;
        constexpr int CK = RK / 16, CV = RV / 16;  // 16-byte chunks of a token = chunks of a thread
        const uint32_t *table = p.batch.table + (size_t)b * p.batch.stride;
        const uint32_t mask = (1u << p.cache.shift) - 1u;
        // lane l < 8: the page of run l (16 tokens) of tile i; ~0: nothing to read there
        auto run_pages = [&](uint32_t i) -> uint32_t {
            if (i >= n || lane >= kTok / 16) return ~0u;
            const uint32_t j = tile_token(i) + 16 * lane;
            if (!kv_needed(range, j, j + 16)) return ~0u;
            const uint32_t page = __ldg(table + (j >> p.cache.shift));
            if (page < p.cache.num_pages) return page;
            fault = KV_FAULT_PAGE;
            return ~0u;
        };
        auto slot_of = [&](uint32_t page, uint32_t j) {
            return (((size_t)page * p.cache.hkv + h) << p.cache.shift) + (j & mask);
        };
        uint4 kr[CK], vr[CV];
        float rs[4];
        auto load_codes = [&](uint4 *dst, int chunks, const uint8_t *codes, int row_bytes, uint32_t pages, uint32_t i) {
            const uint32_t j0 = tile_token(i);
#pragma unroll
            for (int it = 0; it < chunks; it++) {
                const uint32_t id = it * 128 + pt, row = id / chunks, col = id % chunks;
                const uint32_t page = __shfl_sync(0xffffffffu, pages, row >> 4);
                dst[it] = make_uint4(0u, 0u, 0u, 0u);
                if (page != ~0u)
                    dst[it] = ld_stream(reinterpret_cast<const uint4 *>(codes + slot_of(page, j0 + row) * row_bytes + col * 16));
            }
        };
        auto load_scales = [&](uint32_t pages, uint32_t i) {
            const uint32_t j = tile_token(i) + pt;
            const uint32_t page = __shfl_sync(0xffffffffu, pages, pt >> 4);
            rs[0] = rs[1] = rs[2] = rs[3] = 0.0f;
            if (page != ~0u && kv_needed(range, j, j + 1)) {
                const size_t slot = slot_of(page, j);
                if constexpr (BK == 8) {
                    rs[0] = __ldg(p.cache.scales[0] + slot);
                } else {
                    const float2 v = __ldg(reinterpret_cast<const float2 *>(p.cache.scales[0]) + slot);
                    rs[0] = v.x;
                    rs[1] = v.y;
                }
                if constexpr (BV == 8) {
                    rs[2] = __ldg(p.cache.scales[1] + slot);
                } else {
                    const float2 v = __ldg(reinterpret_cast<const float2 *>(p.cache.scales[1]) + slot);
                    rs[2] = v.x;
                    rs[3] = v.y;
                }
            }
        };
        auto unpack8 = [](const uint4 &v, uint8_t *base, int row, int col) {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            uint4 o[2];
            uint32_t *ow = reinterpret_cast<uint32_t *>(o);
#pragma unroll
            for (int k = 0; k < 4; k++) unpack_u8(w[k], ow[2 * k], ow[2 * k + 1]);
            // lanes of the second 64 dims write their odd chunk first: no two of a
            // quarter warp in one bank
            const int odd = (col >> 2) & 1;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int ch = 2 * col + (k ^ odd);
                const uint4 val = (k ^ odd) ? o[1] : o[0];
                *reinterpret_cast<uint4 *>(base + (ch >> 3) * kBlk + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) = val;
            }
        };
        auto unpack4 = [](const uint4 &v, uint8_t *base, int row, int col) {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t u[4];
                unpack_u4(w[k], u);
                const int ch = 4 * col + k;
                *reinterpret_cast<uint4 *>(base + (ch >> 3) * kBlk + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) =
                    make_uint4(u[0], u[1], u[2], u[3]);
            }
        };
        // power of two on the values' scales and zeros (0: none of them seen so far
        // but zero), the same in all four warps, and its reciprocal
        float lift = 0.0f, unit = 1.0f;
        uint32_t cur = run_pages(0);
        if (n > 0) {
            load_codes(kr, CK, p.cache.codes[0], RK, cur, 0);
            load_scales(cur, 0);
        }
        bool ok = true;
        for (uint32_t i = 0; i < n; i++) {
            const uint32_t st = i % ST, ph = (i / ST) & 1;
            load_codes(vr, CV, p.cache.codes[1], RV, cur, i);
            const uint32_t nxt = run_pages(i + 1);
            ok = __all_sync(0xffffffffu, wait_or_fault(&kempty[st], ph ^ 1, &abort_s, p.fault));
            if (!ok) break;
            uint8_t *kb = smem + S::K0 + st * S::KV;
#pragma unroll
            for (int it = 0; it < CK; it++) {
                const int id = it * 128 + pt;
                if constexpr (BK == 8) unpack8(kr[it], kb, id / CK, id % CK);
                else unpack4(kr[it], kb, id / CK, id % CK);
            }
            ScaleSlot *sl = slots + (i % kScaleSlots);
            if (lift == 0.0f) {
                // every warp looks at the whole tile: no wait between warps
                float mag = 0.0f;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t j = tile_token(i) + 32 * q + lane;
                    const uint32_t page = __shfl_sync(0xffffffffu, cur, (32 * q + lane) >> 4);
                    if (page == ~0u || !kv_needed(range, j, j + 1)) continue;
                    if constexpr (BV == 8) {
                        mag = fmaxf(mag, __ldg(p.cache.scales[1] + slot_of(page, j)));
                    } else {
                        const float2 v = __ldg(reinterpret_cast<const float2 *>(p.cache.scales[1]) + slot_of(page, j));
                        mag = fmaxf(mag, fmaxf(v.x, fabsf(v.y)));
                    }
                }
                mag = warp_max(mag);
                if (mag > 0.0f) {
                    lift = __int_as_float((127 + kvf::near_one(mag)) << 23);
                    unit = __int_as_float((127 - kvf::near_one(mag)) << 23);
                }
            }
            rs[2] *= lift;
            rs[3] *= lift;
            sl->sk[pt] = rs[0];
            sl->sv[pt] = rs[2];
            sl->lv[pt] = lg2(fmaxf(rs[2], fabsf(rs[3])));
            if constexpr (BK == 4) sl->zk[pt] = rs[1];
            if constexpr (BV == 4) sl->zv[pt] = rs[3];
            const float zm = BV == 4 ? warp_max(fabsf(rs[3])) : 0.0f;
            if (lane == 0) sl->zmax[warp - 8] = zm;
            if (pt == 0) sl->unit = unit;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&scfull[i % kScaleSlots]);
                mbar_arrive(&kfull[st]);
            }
            if (i + 1 < n) {
                load_codes(kr, CK, p.cache.codes[0], RK, nxt, i + 1);
                load_scales(nxt, i + 1);
            }
            ok = __all_sync(0xffffffffu, wait_or_fault(&vempty[st], ph ^ 1, &abort_s, p.fault));
            if (!ok) break;
            uint8_t *vb = smem + S::V0 + st * S::KV;
#pragma unroll
            for (int it = 0; it < CV; it++) {
                const int id = it * 128 + pt;
                if constexpr (BV == 8) unpack8(vr[it], vb, id / CV, id % CV);
                else unpack4(vr[it], vb, id / CV, id % CV);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&vfull[st]);
            cur = nxt;
        }
        if (fault) kv_report(p.fault, fault);
    } else if (regs_dec<kRegsIssue>(); warp == 12) {
        // ================= MMA issue (whole warp, elected lane) =================
        constexpr uint32_t id_s = idesc_f16(kTok, false), id_o = idesc_f16(D, true);
        const uint32_t q0 = smem_u32(smem), k0 = smem_u32(smem + S::K0), v0 = smem_u32(smem + S::V0);
        unsigned pc[2] = {0, 0};  // products of P done so far, per row tile
        bool ok = true;
        auto wait = [&](unsigned long long *bar, unsigned parity) {
            ok = __all_sync(0xffffffffu, wait_or_fault(bar, parity, &abort_s, p.fault));
            if (ok) tc_fence_after();
            return ok;
        };
        auto mma_s = [&](int sub, uint32_t st) {
#pragma unroll 1
            for (int part = 0; part < S::NQ; part++)
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++) {
                    const uint32_t off = (ks >> 2) * kBlk + (ks & 3) * 32;
                    umma_f16_w(tmem + kSCol + 128 * sub, desc_sw128(q0 + sub * S::Q_SUB + part * S::DB * kBlk + off, 16),
                               desc_sw128(k0 + st * S::KV + off, 16), id_s, part + ks != 0);
                }
            umma_commit_w(&sfull[sub]);
        };
        auto mma_o = [&](int sub, uint32_t st) {
#pragma unroll (SPLIT ? 2 : 8)
            for (int ks = 0; ks < kTok / 16; ks++) {  // (two products a step for f32 queries)
                const uint64_t bd = desc_sw128(v0 + st * S::KV + ks * 2048, kBlk);
                const uint32_t a = tmem + kSCol + 128 * sub + (SPLIT ? 16 * ks : 8 * ks);
                umma_f16_ts_w(tmem + kOCol + D * sub, a, bd, id_o, pc[sub] != 0 || ks != 0);
                if constexpr (SPLIT) umma_f16_ts_w(tmem + kOCol + D * sub, a + 8, bd, id_o, 1);
            }
        };
        if (n > 0 && wait(&qfull, 0) && wait(&kfull[0], 0)) {
            for (int sub = 0; sub < 2; sub++)
                if (active(sub, 0)) mma_s(sub, 0);
            umma_commit_w(&kempty[0]);
            for (uint32_t i = 0; i < n && ok; i++) {
                const uint32_t st = i % ST, st1 = (i + 1) % ST;
                if (!wait(&vfull[st], (i / ST) & 1)) break;
                bool have_next = false;
                for (int sub = 0; sub < 2 && ok; sub++) {
                    if (active(sub, i)) {
                        if (!wait(&pready[sub], pc[sub] & 1)) break;
                        mma_o(sub, st);
                        pc[sub]++;
                    }
                    if (sub == 1) umma_commit_w(&vempty[st]);
                    if (i + 1 < n) {
                        if (!have_next && !wait(&kfull[st1], ((i + 1) / ST) & 1)) break;
                        have_next = true;
                        if (active(sub, i + 1)) mma_s(sub, st1);
                    }
                }
                if (i + 1 < n && ok) umma_commit_w(&kempty[st1]);
            }
        }
        // every MMA issued has completed before tensor memory is read or freed
        umma_commit_w(&odone);
        if (lane == 0) {
            unsigned k = 0;
            while (!mbar_try_wait(&odone, 0) && ++k < kSpin) {
            }
        }
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int D, int BK, int BV, bool SPLIT>
cudaError_t launch_chunk_t(const KvAttnParams &p, cudaStream_t st) {
    auto *fn = k_kv_attn_chunk<D, BK, BV, SPLIT>;
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D, SPLIT>::TOTAL);
    if (e != cudaSuccess) return e;
    fn<<<dim3(p.cache.hkv, p.row_tiles * p.nsplit, p.batch.n_seqs), kThreads, Smem<D, SPLIT>::TOTAL, st>>>(p);
    return cudaGetLastError();
}

template <int D>
cudaError_t launch_chunk_dim(const KvAttnParams &p, cudaStream_t st) {
    const int bk = p.cache.bits[0], bv = p.cache.bits[1];
    const bool split = p.q.fmt == kFmtF32;
    if (bk == 8) {
        if (bv == 8) return split ? launch_chunk_t<D, 8, 8, true>(p, st) : launch_chunk_t<D, 8, 8, false>(p, st);
        return split ? launch_chunk_t<D, 8, 4, true>(p, st) : launch_chunk_t<D, 8, 4, false>(p, st);
    }
    if (bv == 8) return split ? launch_chunk_t<D, 4, 8, true>(p, st) : launch_chunk_t<D, 4, 8, false>(p, st);
    return split ? launch_chunk_t<D, 4, 4, true>(p, st) : launch_chunk_t<D, 4, 4, false>(p, st);
}

}  // namespace kvc
}  // namespace nx
