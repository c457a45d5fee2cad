// kernels_kv_chunk.cuh -- attention of a chunk of new tokens over the quantised
// paged KV cache, on the 5th-generation tensor cores.
//
// The mathematics is that of kernels_kv_few.cuh with one reference a row:
//   x_rj = c_r (sk_j (q_r . kc_j) + zk_j sum(q_r)),  p = 2^(x - ref_r)
//   o_r  = ( sum_j (p sv_j) vc_j + sum_j p zv_j ) / sum_j p
// kc, vc integer codes around zero (exact in f16), q as f16 (hi + lo for f32
// queries), the weights p sv rounded to f16 (hi + lo for f32; why, there).  ref is a whole
// number chosen so that the largest p * max(sv, |zv|) of the row lies between
// 2^(kUp-1) (kUpSplit for f32 queries) and f16's end; it moves only when a weight
// would pass that, and then by an exact power of two (p alone is kept below 2^96
// where values are zero, and the values' scales are lifted first, as there).
//
// Bound: the tensor pipe (4 D flops a visible pair) and, next to it, the
// shared-memory bandwidth that feeds it.  One CTA an SM, 256 rows (row r: token
// r / G, head r % G) in two tiles of 128, keys in tiles of 128 tokens:
//   warps 0-3, 4-7  softmax of row tile 0, 1.  Tensor memory is read in the
//                   16x256b shape: a thread has four rows and a quarter of the
//                   columns, so that it needs a quarter of the tokens' scales (a
//                   thread a row, each scale read by all 32 lanes, spent 2048
//                   cycles a tile of the shared-memory pipe on them), and the
//                   packed weights of two neighbouring columns are the 16x128b
//                   store's element
//   warps 8-9, 10-11  unpack the key and the value codes of a tile into f16
//                   operands in shared memory (128-byte swizzle); the next tile's
//                   codes are on their way in registers meanwhile
//   warp 12         tcgen05.mma issue: S = Q K^T (128 x 128 x D) and O += P V
// S and O of both tiles fill tensor memory; P overwrites S in place.  While the
// softmax of one tile runs, the tensor pipe works for the other.  Keys come in
// by registers rather than TMA because they must be unpacked on the way.
// The tensor cores round each sum toward zero, an error that grows with the number
// of products summed in place (4.5e-5 of the output after 40000 tokens).  For f32
// queries the output is therefore taken out of tensor memory every kFlush tiles
// and added, correctly rounded, to sums in the caller's workspace (8e-7 to 9e-7 of the
// output at 1000 to 131000 tokens; what is left is the two tiles' own sums).
// Every wait is bounded (as in kernels_gemm.cuh).
// Measured (32/8 heads, D = 128, 8 bits, device time): bf16 4096-token prompt 238 us (578
// TFLOP/s), 2048 tokens behind 14336 744 us (693 TFLOP/s; 0.41 of the measured bf16
// peak), 256 behind 16128 126 us; f32 2048-token prompt 143 us (241 TFLOP/s, each product
// twice).  In the bf16 prompt the tensor pipe is active in 28% of the cycles and 43% of the
// issue slots are used, with 0.6 warps ready a scheduler: a row tile's softmax (dependent
// latencies of its four warps) and its products follow one another, and only the other row
// tile's fill the gap.
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
constexpr int kRegsLaunch = 128, kRegsSoftmax = 160, kRegsProducer = 120, kRegsIssue = 72;
static_assert(2 * kRegsSoftmax + kRegsProducer + kRegsIssue <= 4 * kRegsLaunch && kThreads * kRegsLaunch <= 65536, "more registers than the block has");
constexpr int kBlk = 128 * 128;         // 128 rows x 64 f16, swizzled
// A new reference puts the largest weight at 2^(kUp-1) .. 2^kUp, as low as 16 bits of output
// allow: the lower, the less often it moves.  f16 ends at 2^-25, so that a weight is off
// by up to 2^-28 of the largest besides its own rounding, which 2^17 keys that all lie there
// make half a step of an f16 output.  f32 queries: 2^-35, 4e-6 of the leading value
// for 2^17 such keys (a 2048-token prompt took 136 us at 4, 140 at 10, 142 at 11, 152 at 12,
// where the sums of weights near the largest already reach f16's end).
constexpr float kUp = 4.0f, kUpSplit = 11.0f;
constexpr float kMaxWeight = kvf::kMostF16;  // and it is moved when a weight would leave f16
constexpr float kMaxProb = kvf::kMaxProb;  // log2 of the largest p where values are zero
// Scores beyond this are taken relative to the largest when a reference is chosen: base + t
// then, with t the reference wanted as seen from base, rounded once.  Where that leaves the
// largest weight more than 2^room above the one wanted, the next number up: for steps of up
// to 2^5 (scores of 2^29) the weight stays within f16 whatever the values, beyond that for
// values within 2^15 of the first tile's.
constexpr float kLargeScore = 4194304.0f;
__device__ __forceinline__ float reference(float base, float t, float room) {
    const float m = __fadd_rn(base, t);
    return t - __fsub_rn(m, base) > room ? __fadd_ru(base, t) : m;
}
constexpr int kScaleSlots = 4;
constexpr int kFlush = kKvFlushTiles;

// What the softmax needs of a key tile, by token; byte offsets in shared memory.
struct Slot {
    static constexpr int SK = 0, ZK = 512, SV = 1024, ZV = 1536;  // (the keys' times key_scale)
    static constexpr int LV = 2048;            // log2 max(sv, |zv|)
    static constexpr int SMAX = 2560, ZMAX = 2576;  // largest sv, |zv| of each quarter of the tokens
    static constexpr int UNIT = 2592;          // what sv and zv were divided by
    static constexpr int BAD = 2596;           // bit r: tokens 16 r .. of the tile have no page (nobody sees them)
    static constexpr int BYTES = 2608;
};

template <int D, bool SPLIT>
struct Smem {
    static constexpr int DB = (D + 63) / 64;
    static constexpr int NQ = SPLIT ? 2 : 1;
    static constexpr int Q_SUB = DB * kBlk * NQ;
    static constexpr int KV = DB * kBlk;
    static constexpr int STAGES = SPLIT && D == 128 ? 1 : 2;
    static constexpr int K0 = 2 * Q_SUB, V0 = K0 + STAGES * KV, SC = V0 + STAGES * KV;
    static constexpr int NEED = SC + kScaleSlots * Slot::BYTES + 1024;
    // at least 120 KB: one CTA an SM, since each takes all of tensor memory
    static constexpr int TOTAL = NEED > 120 * 1024 ? NEED : 120 * 1024;
};

// Tensor memory, 32 lanes of a warp as rows g, g + 8 (first half) and g + 16,
// g + 24 (second), g = lane / 4, c = lane % 4.  Loads are complete after
// tmem_wait; `r` is tied to it so that nothing reads it before.
//
// 32 columns of one half: r[4 k + i] is row g + 8 (i / 2), column 8 k + 2 c + i % 2.
__device__ __forceinline__ void tmem_ld_16x256_x4(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_16x256_x4(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
// Eight columns of one half: r[2 k + i] is row g + 8 i, column 4 k + c.
__device__ __forceinline__ void tmem_ld_16x128_x2(uint32_t taddr, uint32_t (&r)[4]) {
    asm volatile("tcgen05.ld.sync.aligned.16x128b.x2.b32 {%0,%1,%2,%3}, [%4];\n tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_16x128_x2(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
// The stores and sums of the common path, left out where `on` (the same in all
// lanes) is zero, without a branch.
__device__ __forceinline__ void tmem_st_16x128_x4_if(unsigned on, uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %9, 0;\n"
        " @p tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n}\n" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(on)
        : "memory");
}
__device__ __forceinline__ void add2_if(unsigned on, f2 &a, f2 b) {
    asm("{\n .reg .pred p;\n setp.ne.u32 p, %2, 0;\n @p add.rn.f32x2 %0, %0, %1;\n}\n" : "+l"(a) : "l"(b), "r"(on));
}
// A lane a row: 32 columns, complete on return.
__device__ __forceinline__ void tmem_ld_rows32(uint32_t taddr, float (&v)[32]) {
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

// The 16-byte chunks of a tile's codes over two producer warps: CPR a row, N a
// thread, LC lanes a row, PER chunks of a lane in a row, ROWS rows between them.
template <int D, int BITS>
struct Chunks {
    static constexpr int CPR = D * BITS / 128, N = 2 * CPR;
    static constexpr int LC = CPR < (BITS == 8 ? 4 : 2) ? CPR : (BITS == 8 ? 4 : 2);
    static constexpr int PER = CPR / LC, RPW = 32 / LC, ROWS = 2 * RPW;
    __device__ static __forceinline__ uint32_t row(int it, int warp, int lane) {
        return (it / PER) * ROWS + warp * RPW + lane / LC;
    }
    __device__ static __forceinline__ uint32_t col(int it, int lane) { return (it % PER) * LC + lane % LC; }
};

// The warpgroup's registers a thread from the launch's 128 to N (each form of the
// instruction goes one way only).
template <int N>
__device__ __forceinline__ void set_regs() {
    if constexpr (N > kRegsLaunch) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    if constexpr (N < kRegsLaunch) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int D, int BK, int BV, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) k_kv_attn_chunk(KvAttnParams p) {
    using S = Smem<D, SPLIT>;
    constexpr int ST = S::STAGES;
    constexpr uint32_t kSCol = 0, kOCol = 256;       // per row tile: + 128, + D
    extern __shared__ uint8_t smem_raw[];
    // operand blocks start on 1024 bytes (the swizzle goes by address)
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    __shared__ unsigned long long kfull[2], kempty[2], vfull[2], vempty[2], scfull[kScaleSlots], sfull[2], pready[2],
        qfull, odone;
    __shared__ uint32_t tmem_base_s;
    __shared__ volatile int abort_s;
    __shared__ float row_x[kRows], row_sum[kRows], row_ref[kRows];

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
            mbar_init(&kfull[i], 2);
            mbar_init(&kempty[i], 1);
            mbar_init(&vfull[i], 2);
            mbar_init(&vempty[i], 1);
            mbar_init(&sfull[i], 1);
            mbar_init(&pready[i], 4);
        }
        for (int i = 0; i < kScaleSlots; i++) mbar_init(&scfull[i], 2);
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
        // ================= softmax: a thread has four rows, a quarter of the columns =================
        set_regs<kRegsSoftmax>();
        const int sub = warp >> 2, wq = warp & 3;
        const uint32_t t_lane = (uint32_t)(32 * wq) << 16;
        {
            // This warp's 32 query rows to shared memory, D / 8 lanes a row: first as they
            // are, every copy in flight at once, each lane's 16 bytes where its f16 will
            // stand (f32: the two halves where hi and lo will), then converted in place.
            // Rolled loops: the code is cold in every CTA, and fetching eight passes
            // unrolled took 8 us.
            constexpr int LPR = D / 8, RPP = 32 / LPR;
            const int cl = lane % LPR;
            const uint32_t qs = sbase + sub * S::Q_SUB + (cl >> 3) * kBlk;
            auto place = [&](int rr) { return qs + rr * 128 + (((cl & 7) ^ (rr & 7)) << 4); };
#pragma unroll 1
            for (int pass = 0; pass < LPR; pass++) {
                const int rr = 32 * wq + pass * RPP + lane / LPR;
                const uint32_t r = rows.r0 + min((uint32_t)(sub * 128 + rr), rows.n - 1), tok = kv_div(r, p.group_magic);
                const size_t at = (size_t)(seq.q0 + tok) * p.q.row_stride + (h * G + r - tok * G) * p.q.head_stride + cl * 8;
                if constexpr (SPLIT) {
                    kvf::cp_async16(place(rr), static_cast<const float *>(p.q.data) + at);
                    kvf::cp_async16(place(rr) + S::DB * kBlk, static_cast<const float *>(p.q.data) + at + 4);
                } else {
                    kvf::cp_async16(place(rr), static_cast<const uint16_t *>(p.q.data) + at);
                }
            }
            kvf::cp_commit();
            kvf::cp_wait<0>();
#pragma unroll 1
            for (int pass = 0; pass < LPR; pass++) {
                const int rr = 32 * wq + pass * RPP + lane / LPR;
                const uint32_t dst = place(rr);
                const float4 raw = lds4(dst);
                float q[8];
                if constexpr (SPLIT) {
                    const float4 raw1 = lds4(dst + S::DB * kBlk);
                    q[0] = raw.x; q[1] = raw.y; q[2] = raw.z; q[3] = raw.w;
                    q[4] = raw1.x; q[5] = raw1.y; q[6] = raw1.z; q[7] = raw1.w;
                } else {
                    unpack16(make_uint4(__float_as_uint(raw.x), __float_as_uint(raw.y), __float_as_uint(raw.z),
                                        __float_as_uint(raw.w)),
                             p.q.fmt, q);
                }
                if ((uint32_t)(sub * 128 + rr) >= rows.n) {
#pragma unroll
                    for (int i = 0; i < 8; i++) q[i] = 0.0f;
                }
                float amax = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(q[i]));
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const int e_row = row_exp(amax);
                const float sc = pow2i(7 - e_row);
                // elements in the order the codes of a word unpack to
                constexpr int o8[8] = {0, 1, 2, 3, 4, 5, 6, 7}, o4[8] = {0, 4, 1, 5, 2, 6, 3, 7};
                uint32_t hi[4];
                [[maybe_unused]] uint32_t lo[4];
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
                sts4(dst, hi[0], hi[1], hi[2], hi[3]);
                if constexpr (SPLIT) sts4(dst + S::DB * kBlk, lo[0], lo[1], lo[2], lo[3]);
                if (cl == 0) {
                    row_x[sub * 128 + rr] = pow2i(p.scale_exp + e_row - 7);
                    row_sum[sub * 128 + rr] = sum;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&qfull);
        }
        // this thread's rows: k = 0..3 is row 32 wq + g + 8 k of the tile
        const int g = lane >> 2, c = lane & 3;
        const int base_row = sub * 128 + 32 * wq;
        int pos[4];
        f2 xs2[4], qsum2[4], l2[4], z2[4];
        float ref[4];
        f2 nref2[4];  // minus the reference (0 while there is none), twice
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t in_tile = (uint32_t)(base_row + g + 8 * k);
            pos[k] = in_tile < rows.n ? pos0 + (int)kv_div(rows.r0 + in_tile, p.group_magic) : -1;
            xs2[k] = pk(row_x[in_tile], row_x[in_tile]);
            qsum2[k] = pk(row_sum[in_tile], row_sum[in_tile]);
            // rows that see nothing start with a reference of their own: they never ask for one
            ref[k] = pos[k] >= 0 ? -INFINITY : 0.0f;
            nref2[k] = pk(0.0f, 0.0f);
            l2[k] = z2[k] = pk(0.0f, 0.0f);  // sums of p and p zv of this thread's columns
        }
        // f32 queries: this thread's sums in the workspace (32 lanes of one element next to
        // each other), what they are to be multiplied by to be in the references' terms,
        // and whether there are any
        [[maybe_unused]] float *sums = nullptr;
        [[maybe_unused]] float sum_f[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        [[maybe_unused]] bool summed = false;
        if constexpr (SPLIT)
            sums = p.sums + (((size_t)kv_tile_slot(seq.q0, G, b, rt, kRows) * p.cache.hkv + h) * p.nsplit + split) * (kRows * D) +
                   warp * (32 * D) + lane;
        bool unset = true;  // some reference may not be set yet
        float unit = 1.0f;
        const int first = sub ? first1 : rows.first, last = sub ? rows.last : last0;
        const uint32_t scol = tmem + t_lane + kSCol + 128 * sub, ocol = tmem + t_lane + kOCol + D * sub;
        constexpr uint32_t kHalf = 16u << 16;  // the second half of the warp's lanes
        unsigned cnt = 0;
        bool ok = true;
        // The output in tensor memory (complete) and the sums: to_sums, into the sums;
        // otherwise their total back into tensor memory.
        [[maybe_unused]] auto flush = [&](bool to_sums) {
#pragma unroll 1
            for (int q = 0; q < D / 32; q++) {
#pragma unroll
                for (int hh = 0; hh < 2; hh++) {
                    uint32_t o[16];
                    float *at = sums + (q * 2 + hh) * 512;
                    tmem_ld_16x256_x4(ocol + hh * kHalf + 32 * q, o);
                    tmem_wait(o);
                    if (summed) {
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            o[j] = __float_as_uint(fmaf(__ldcg(at + 32 * j), sum_f[2 * hh + (j >> 1 & 1)], __uint_as_float(o[j])));
                    }
                    if (to_sums) {
#pragma unroll
                        for (int j = 0; j < 16; j++) __stcg(at + 32 * j, __uint_as_float(o[j]));
                    } else {
                        tmem_st_16x256_x4(ocol + hh * kHalf + 32 * q, o);
                    }
                }
            }
            if (!to_sums) tmem_wait_st();
            summed = true;
#pragma unroll
            for (int k = 0; k < 4; k++) sum_f[k] = 1.0f;
        };
        for (uint32_t i = 0; i < n; i++) {
            if (!active(sub, i)) continue;
            const int j0 = (int)tile_token(i);
            const uint32_t sl = sbase + S::SC + (i % kScaleSlots) * Slot::BYTES;
            ok = wait_or_fault(&scfull[i % kScaleSlots], (i / kScaleSlots) & 1, &abort_s, p.fault) &&
                 wait_or_fault(&sfull[sub], cnt & 1, &abort_s, p.fault);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            if constexpr (SPLIT) {
                if (cnt > 0 && cnt % kFlush == 0) flush(true);  // (the products before S have completed)
            }
            const uint32_t bad = __float_as_uint(lds1(sl + Slot::BAD));
            const bool whole = bad == 0 && j0 + kTok - 1 <= first &&
                               (p.window == 0 || j0 > last - (int)p.window || j0 + kTok <= (int)p.sinks);
            unit = lds1(sl + Slot::UNIT);
            const float svmax = max4(lds4(sl + Slot::SMAX));
            // largest sum of p over four columns of a row: 2^99 (each of them at kMaxProb,
            // twice over), and 2^100 / |zv|
            const float plim = BV == 8 ? 6.4e29f : 1.27e30f / fmaxf(max4(lds4(sl + Slot::ZMAX)), 2.0f);
            const float fast_lim = fminf(plim, kMaxWeight / svmax);  // sums of p up to this keep every weight in f16
            const uint32_t slc = sl + 8 * c;  // this thread's columns: 8 k + 2 c and the next

            // bit 8 t + e: row k sees column c0 + 8 t + 2 c + e
            auto seen = [&](int k, int c0) {
                const int hi = pos[k] - j0 + 1, lo = p.window ? max(0, pos[k] - (int)p.window + 1) - j0 : -1;
                const int sink = min((int)min(p.sinks, 0x3fffffffu) - j0, hi);
                const uint32_t gone = (bad >> (c0 >> 4) & 1 ? 0xffffu : 0u) | (bad >> (c0 >> 4) & 2 ? 0xffff0000u : 0u);
                return (((first_bits(hi - c0) & ~first_bits(lo - c0)) | first_bits(sink - c0)) & ~gone) >> (2 * c);
            };
            // the score of two columns in base 2, before the row's factor
            auto score = [&](const uint32_t *s, f2 sk, [[maybe_unused]] f2 zk, int k) {
                f2 x = mul2(pk(__uint_as_float(s[0]), __uint_as_float(s[1])), sk);
                if constexpr (BK == 4) x = fma2(zk, qsum2[k], x);
                return x;
            };
            // References for all that has been summed and columns 32 q0 .. of this tile;
            // what has been summed follows: l, z, the output, and the weights of this
            // tile already written.
            auto new_reference = [&](int q0) {
                float mx[4], my[4], base[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                // (a second time, relative to the largest score, where that is a large one)
#pragma unroll 1
                for (int pass = 0; pass < 2; pass++) {
#pragma unroll
                    for (int k = 0; k < 4; k++) mx[k] = my[k] = -INFINITY;
#pragma unroll 1
                    for (int q = q0; q < 4; q++) {
#pragma unroll
                        for (int hh = 0; hh < 2; hh++) {
                            uint32_t s[16];
                            tmem_ld_16x256_x4(scol + hh * kHalf + 32 * q, s);
                            tmem_wait(s);
#pragma unroll
                            for (int kk = 0; kk < 2; kk++) {
                                const int k = 2 * hh + kk;
                                const uint32_t bits = whole ? ~0u : seen(k, 32 * q);
#pragma unroll
                                for (int t = 0; t < 4; t++) {
                                    const uint32_t at = slc + 4 * (32 * q + 8 * t);
                                    const f2 lv = lds2(at + Slot::LV);
                                    float e0, e1, v0, v1;
                                    upk(mul2(score(s + 4 * t + 2 * kk, lds2(at + Slot::SK), BK == 4 ? lds2(at + Slot::ZK) : 0, k),
                                             xs2[k]),
                                        e0, e1);
                                    upk(lv, v0, v1);
                                    e0 = bits >> (8 * t) & 1 ? e0 - base[k] : -INFINITY;
                                    e1 = bits >> (8 * t + 1) & 1 ? e1 - base[k] : -INFINITY;
                                    mx[k] = fmaxf(mx[k], fmaxf(e0, e1));
                                    my[k] = fmaxf(my[k], fmaxf(e0 + v0, e1 + v1));
                                }
                            }
                        }
                    }
                    bool large = false;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
#pragma unroll
                        for (int o = 1; o < 4; o <<= 1) {
                            mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], o));
                            my[k] = fmaxf(my[k], __shfl_xor_sync(0xffffffffu, my[k], o));
                        }
                        large |= fabsf(mx[k]) > kLargeScore && fabsf(mx[k]) < INFINITY;
                    }
                    if (pass || !__any_sync(0xffffffffu, large)) break;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (fabsf(mx[k]) > kLargeScore && fabsf(mx[k]) < INFINITY) base[k] = mx[k];
                }
                float f[4];
                bool moved = false;
                unset = false;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float want = fmaxf(ceilf(my[k]) - (SPLIT ? kUpSplit : kUp), ceilf(mx[k]) - kMaxProb);
                    const float next = fmaxf(ref[k], reference(base[k], want, SPLIT ? 4.0f : 11.0f));
                    f[k] = 1.0f;
                    if (next != ref[k]) {
                        const kvf::Pow2 fl(ref[k], next);
                        f[k] = pow2_diff(ref[k], next);
                        l2[k] = mul2(mul2(l2[k], pk(fl.h, fl.h)), pk(fl.g, fl.g));
                    }
                    ref[k] = next;
                    nref2[k] = next == -INFINITY ? pk(0.0f, 0.0f) : pk(-next, -next);
                    unset |= next == -INFINITY;
                    moved |= f[k] != 1.0f;
                    if constexpr (SPLIT) sum_f[k] *= f[k];
                    z2[k] = mul2(z2[k], pk(f[k], f[k]));
                }
                if (!__any_sync(0xffffffffu, moved)) return;
                if (cnt > 0) {
                    // the products so far are complete: S of this tile was issued after them
#pragma unroll 1
                    for (int q = 0; q < D / 32; q++) {
#pragma unroll
                        for (int hh = 0; hh < 2; hh++) {
                            uint32_t o[16];
                            tmem_ld_16x256_x4(ocol + hh * kHalf + 32 * q, o);
                            tmem_wait(o);
#pragma unroll
                            for (int j = 0; j < 16; j++)
                                o[j] = __float_as_uint(__uint_as_float(o[j]) * f[2 * hh + (j >> 1 & 1)]);
                            tmem_st_16x256_x4(ocol + hh * kHalf + 32 * q, o);
                        }
                    }
                }
                tmem_wait_st();
#pragma unroll 1
                for (int q = 0; q < 2 * q0 * S::NQ; q++) {
#pragma unroll
                    for (int hh = 0; hh < 2; hh++) {
                        uint32_t w[4];
                        tmem_ld_16x128_x2(scol + hh * kHalf + 8 * q, w);
                        const uint32_t f0 = f16x2(f[2 * hh], f[2 * hh]), f1 = f16x2(f[2 * hh + 1], f[2 * hh + 1]);
                        tmem_st_16x128_x2(scol + hh * kHalf + 8 * q, hmul2u(w[0], f0), hmul2u(w[1], f1), hmul2u(w[2], f0),
                                          hmul2u(w[3], f1));
                    }
                }
            };
            // The weights of columns 32 q .. + 31 against the references, and their sums.
            // Returns the largest of the sums of p (of four columns each).
            auto weigh = [&](auto masked, int q, const uint32_t(&cur)[2][16], uint32_t(&ph)[2][8], uint32_t(&pl)[2][8],
                             f2(&l_c)[4], f2(&z_c)[4]) -> float {
                constexpr bool MASK = decltype(masked)::value;
                uint32_t bits[4];
#pragma unroll
                for (int k = 0; k < 4; k++) bits[k] = MASK ? seen(k, 32 * q) : ~0u;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const uint32_t at = slc + 4 * (32 * q + 8 * t);
                    const f2 sk = lds2(at + Slot::SK), sv = lds2(at + Slot::SV);
                    [[maybe_unused]] f2 zk, zv;
                    if constexpr (BK == 4) zk = lds2(at + Slot::ZK);
                    else zk = sk;
                    if constexpr (BV == 4) zv = lds2(at + Slot::ZV);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float e0, e1;
                        upk(fma2(score(cur[k >> 1] + 4 * t + 2 * (k & 1), sk, zk, k), xs2[k], nref2[k]), e0, e1);
                        if constexpr (MASK) {
                            e0 = bits[k] >> (8 * t) & 1 ? e0 : -INFINITY;
                            e1 = bits[k] >> (8 * t + 1) & 1 ? e1 : -INFINITY;
                        }
                        const f2 pp = pk(ex2(e0), ex2(e1));
                        l_c[k] = t ? add2(l_c[k], pp) : pp;
                        if constexpr (BV == 4) z_c[k] = t ? fma2(pp, zv, z_c[k]) : mul2(pp, zv);
                        float w0, w1;
                        upk(mul2(pp, sv), w0, w1);
                        const uint32_t hw = f16x2(w0, w1);
                        ph[k >> 1][2 * t + (k & 1)] = hw;
                        if constexpr (SPLIT) {
                            const float2 back = f16x2_back(hw);
                            pl[k >> 1][2 * t + (k & 1)] = f16x2(w0 - back.x, w1 - back.y);
                        }
                    }
                }
                float sum[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float a, b;
                    upk(l_c[k], a, b);
                    sum[k] = fmaxf(a, b);
                }
                return fmaxf(fmaxf(sum[0], sum[1]), fmaxf(sum[2], sum[3]));
            };
            // Writes the weights over the scores and adds the sums, where `on`.
            auto keep = [&](unsigned on, int q, const uint32_t(&ph)[2][8], const uint32_t(&pl)[2][8], const f2(&l_c)[4],
                            const f2(&z_c)[4]) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    add2_if(on, l2[k], l_c[k]);
                    if constexpr (BV == 4) add2_if(on, z2[k], z_c[k]);
                }
#pragma unroll
                for (int hh = 0; hh < 2; hh++) {
                    if constexpr (SPLIT) {
                        // 16 tokens: eight columns of hi, eight of lo
                        uint32_t w[2][8];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            w[0][e] = ph[hh][e];
                            w[0][4 + e] = pl[hh][e];
                            w[1][e] = ph[hh][4 + e];
                            w[1][4 + e] = pl[hh][4 + e];
                        }
                        tmem_st_16x128_x4_if(on, scol + hh * kHalf + 32 * q, w[0]);
                        tmem_st_16x128_x4_if(on, scol + hh * kHalf + 32 * q + 16, w[1]);
                    } else {
                        tmem_st_16x128_x4_if(on, scol + hh * kHalf + 16 * q, ph[hh]);
                    }
                }
            };
            // A quarter of the tile at a time, rolled: the code of a tile has to stay in the
            // instruction caches (four quarters unrolled, with the next one's loads ahead,
            // was slower: 470 against 378 us a round of CTAs at 16384 tokens, and the more
            // so the further the SMs are apart in their tiles).
            auto quarter = [&](auto masked, auto tried, int q, unsigned on) -> unsigned {
                uint32_t s[2][16], ph[2][8];
                [[maybe_unused]] uint32_t pl[2][8];
                f2 l_c[4];
                [[maybe_unused]] f2 z_c[4];
                tmem_ld_16x256_x4(scol + 32 * q, s[0]);
                tmem_ld_16x256_x4(scol + kHalf + 32 * q, s[1]);
                tmem_wait(s[0]);
                tmem_wait(s[1]);
                const float most = weigh(masked, q, s, ph, pl, l_c, z_c);
                if constexpr (decltype(tried)::value) on &= __any_sync(0xffffffffu, most > fast_lim) ? 0u : 1u;
                keep(on, q, ph, pl, l_c, z_c);
                return on;
            };
            // The old references are tried first; a weight is at most a sum of p times the
            // largest scale, and from the first quarter where that says nothing on, the
            // second loop takes over with new ones.
            auto tile = [&](auto masked) {
                int q = 0;
                if (!__any_sync(0xffffffffu, unset)) {
                    unsigned on = 1;
#pragma unroll 1
                    for (int u = 0; u < 4; u++) {
                        on = quarter(masked, std::true_type{}, u, on);
                        q += (int)on;
                    }
                }
                if (q < 4) {
                    new_reference(q);
#pragma unroll 1
                    for (; q < 4; q++) quarter(masked, std::false_type{}, q, 1u);
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
        // the row sums to shared memory, for the lane that writes the row
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float lt, zt, odd;
            upk(l2[k], lt, odd);
            lt += odd;
            upk(z2[k], zt, odd);
            zt += odd;
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                lt += __shfl_xor_sync(0xffffffffu, lt, o);
                zt += __shfl_xor_sync(0xffffffffu, zt, o);
            }
            if (c == 0) {
                row_x[base_row + g + 8 * k] = lt;
                row_sum[base_row + g + 8 * k] = zt;
                row_ref[base_row + g + 8 * k] = ref[k];
            }
        }
        __syncwarp();
        pdl_launch_dependents();
        // ---- output ----
        if (ok) ok = wait_or_fault(&odone, 0, &abort_s, p.fault);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
            tc_fence_after();
            if constexpr (SPLIT) {
                if (summed) flush(false);
            }
            const uint32_t in_tile = (uint32_t)(base_row + lane);
            const bool valid = in_tile < rows.n;
            const float l = row_x[in_tile], z = row_sum[in_tile];
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const bool split_part = p.nsplit > 1;
            // Rows go through the warp's quarter of its Q tile (every product has completed),
            // 16-byte chunks XORed with the row, so that a row leaves in whole lines: in the
            // output's type, or the f32 sums of a part, half of the dims at a time where
            // the quarter holds no more.
            constexpr int ES = SPLIT ? 4 : 2, STAGE = S::Q_SUB / 4, DP = 32 * D * 4 > STAGE ? D / 2 : D;
            static_assert(32 * D * ES <= STAGE && 32 * DP * 4 <= STAGE, "a warp's rows fit its quarter of Q");
            const uint32_t stage = sbase + sub * S::Q_SUB + wq * STAGE;
            const uint32_t rec0 = ((b * p.cache.hkv + h) * p.row_tiles + rt) * kRows;
            auto record = [&](uint32_t row) { return ((size_t)rec0 + row) * p.nsplit + split; };
            const int wide = split_part ? 4 : ES, pass_dims = split_part ? DP : D;
            const int cpr = pass_dims * wide / 16, swz = min(cpr, 8) - 1;  // chunks of a staged row
#pragma unroll 1
            for (int p0 = 0; p0 < D; p0 += pass_dims) {
                __syncwarp();
#pragma unroll 1
                for (int d0 = p0; d0 < p0 + pass_dims; d0 += 32) {
                    float o[32];
                    if (cnt > 0) {
                        tmem_ld_rows32(ocol + d0, o);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j++) o[j] = 0.0f;
                    }
                    const uint32_t row = stage + lane * pass_dims * wide;
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        // positions of elements 0..7 within a unit of value codes
                        constexpr int i8[8] = {0, 1, 2, 3, 4, 5, 6, 7}, i4[8] = {0, 2, 4, 6, 1, 3, 5, 7};
                        // (unit / l by itself may be below f32's normal numbers)
                        const float f = split_part ? 1.0f : inv;
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) v[e] = (o[8 * u + (BV == 8 ? i8[e] : i4[e])] + z) * f * unit;
                        const int ch = (d0 - p0 + 8 * u) * wide / 16;
                        if (SPLIT || split_part) {
                            sts4(row + ((ch ^ (lane & swz)) << 4), __float_as_uint(v[0]), __float_as_uint(v[1]),
                                 __float_as_uint(v[2]), __float_as_uint(v[3]));
                            sts4(row + (((ch + 1) ^ (lane & swz)) << 4), __float_as_uint(v[4]), __float_as_uint(v[5]),
                                 __float_as_uint(v[6]), __float_as_uint(v[7]));
                        } else {
                            sts4(row + ((ch ^ (lane & swz)) << 4), pack16(v[0], v[1], p.out.fmt), pack16(v[2], v[3], p.out.fmt),
                                 pack16(v[4], v[5], p.out.fmt), pack16(v[6], v[7], p.out.fmt));
                        }
                    }
                }
                __syncwarp();
#pragma unroll 4
                for (int id = lane; id < 32 * cpr; id += 32) {
                    const int rr = id / cpr, ch = id % cpr;  // (cpr is a power of two)
                    const float4 v = lds4(stage + rr * (pass_dims * wide) + ((ch ^ (rr & swz)) << 4));
                    const uint32_t tile_row = (uint32_t)(base_row + rr), gr = rows.r0 + tile_row;
                    if (tile_row >= rows.n) continue;
                    if (split_part) {
                        *reinterpret_cast<float4 *>(p.part + record(tile_row) * D + p0 + ch * 4) = v;
                    } else {
                        const uint32_t tok = kv_div(gr, p.group_magic);
                        *reinterpret_cast<float4 *>(static_cast<uint8_t *>(p.out.data) +
                                                    ((size_t)(seq.q0 + tok) * p.out.row_stride +
                                                     (h * G + gr - tok * G) * p.out.head_stride) * ES + ch * 16) = v;
                    }
                }
            }
            if (split_part && valid)
                reinterpret_cast<float2 *>(p.ml)[record(in_tile)] = make_float2(l == 0.0f ? -INFINITY : row_ref[in_tile], l);
        }
    } else if (warp < 12) {
        // ================= producers: codes to f16 operands =================
        set_regs<kRegsProducer>();
        const bool keys = warp < 10;
        const int pw = warp & 1;
        const uint32_t *table = p.batch.table + (size_t)b * p.batch.stride;
        const uint32_t mask = (1u << p.cache.shift) - 1u;
        // Lane l < 8: the page of run l (16 tokens) of tile i, ~0 where nothing of it is
        // read (a table's own ~0 is taken for the one before, as far beyond any pool).
        // Loaded two tiles ahead; looked at by page_ok.
        auto load_pages = [&](uint32_t i) -> uint32_t {
            if (i >= n || lane >= kTok / 16) return ~0u;
            const uint32_t j = tile_token(i) + 16 * lane;
            return kv_needed(range, j, j + 16) ? min(__ldg(table + (j >> p.cache.shift)), ~1u) : ~0u;
        };
        bool no_page = false;  // lane l < 8: run l of the tile is read and has no page in the pool
        auto page_ok = [&](uint32_t page) -> uint32_t {
            no_page = page >= p.cache.num_pages && page != ~0u;
            if (no_page) fault = KV_FAULT_PAGE;
            return page < p.cache.num_pages ? page : ~0u;
        };
        auto slot_of = [&](uint32_t page, uint32_t j) {
            return (((size_t)page * p.cache.hkv + h) << p.cache.shift) + (j & mask);
        };
        // A thread's chunks of 16 bytes: LC lanes a row, so that the eight lanes of
        // a store phase write eight different 16-byte columns of the swizzled rows
        // Lane l < 8 finds run l; runs without a page read page 0 (nobody sees them), so
        // that no load waits for a branch.
        auto load_codes = [&](auto bits_c, uint4 *dst, const uint8_t *codes, uint32_t pages, uint32_t i) {
            using C = Chunks<D, decltype(bits_c)::value>;
            const uint64_t run = reinterpret_cast<uint64_t>(codes) +
                                 slot_of(pages == ~0u ? 0u : pages, tile_token(i) + 16 * lane) * (C::CPR * 16);
            uint64_t from = 0;
#pragma unroll
            for (int it = 0; it < C::N; it++) {
                const uint32_t row = C::row(it, pw, lane), col = C::col(it, lane);
                if (it % C::PER == 0) from = __shfl_sync(0xffffffffu, run, row >> 4) + (row & 15) * (C::CPR * 16);
                dst[it] = ld_stream(reinterpret_cast<const uint4 *>(from + col * 16));
            }
        };
        auto store_codes = [&](auto bits_c, const uint4 *src, uint32_t base) {
            constexpr int BITS = decltype(bits_c)::value;
            using C = Chunks<D, BITS>;
            const uint32_t row0 = C::row(0, pw, lane), at = base + row0 * 128;
            const uint32_t c16 = ((uint32_t)(lane % C::LC) * (BITS == 8 ? 2 : 4) ^ (row0 & 7)) << 4;
#pragma unroll
            for (int it = 0; it < C::N; it++) {
                const uint32_t w[4] = {src[it].x, src[it].y, src[it].z, src[it].w};
                const uint32_t dst = at + (it % C::PER) * kBlk + (it / C::PER) * C::ROWS * 128;
                if constexpr (BITS == 8) {
                    uint32_t u[8];
#pragma unroll
                    for (int k = 0; k < 4; k++) unpack_u8(w[k], u[2 * k], u[2 * k + 1]);
                    sts4(dst + c16, u[0], u[1], u[2], u[3]);
                    sts4(dst + (c16 ^ 16u), u[4], u[5], u[6], u[7]);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t u[4];
                        unpack_u4(w[k], u);
                        sts4(dst + (c16 ^ (16u * k)), u[0], u[1], u[2], u[3]);
                    }
                }
            }
        };
        bool ok = true;
        uint32_t next = load_pages(0);
        if (keys) {
            const std::integral_constant<int, BK> kbits{};
            // Scales and zeros of tokens pt and pt + 64: key, value
            const int pt = 32 * pw + lane;
            uint4 kr[Chunks<D, BK>::N];
            float rs[2][4];
            auto load_scales = [&](uint32_t pages, uint32_t i) {
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const uint32_t j = tile_token(i) + pt + 64 * t;
                    const uint32_t page = __shfl_sync(0xffffffffu, pages, (pt + 64 * t) >> 4);
                    rs[t][0] = rs[t][1] = rs[t][2] = rs[t][3] = 0.0f;
                    if (page == ~0u || !kv_needed(range, j, j + 1)) continue;
                    const size_t slot = slot_of(page, j);
                    if constexpr (BK == 8) {
                        rs[t][0] = __ldg(p.cache.scales[0] + slot);
                    } else {
                        const float2 v = __ldg(reinterpret_cast<const float2 *>(p.cache.scales[0]) + slot);
                        rs[t][0] = v.x;
                        rs[t][1] = v.y;
                    }
                    if constexpr (BV == 8) {
                        rs[t][2] = __ldg(p.cache.scales[1] + slot);
                    } else {
                        const float2 v = __ldg(reinterpret_cast<const float2 *>(p.cache.scales[1]) + slot);
                        rs[t][2] = v.x;
                        rs[t][3] = v.y;
                    }
                }
            };
            // power of two on the values' scales and zeros (0: none of them seen so far
            // but zero), the same in both warps, and its reciprocal
            float lift = 0.0f, unit = 1.0f;
            uint32_t cur = page_ok(next);
            if (n > 0) {
                load_codes(kbits, kr, p.cache.codes[0], cur, 0);
                load_scales(cur, 0);
            }
            next = load_pages(1);
            for (uint32_t i = 0; i < n; i++) {
                const uint32_t st = i % ST, ph = (i / ST) & 1;
                ok = __all_sync(0xffffffffu, wait_or_fault(&kempty[st], ph ^ 1, &abort_s, p.fault));
                if (!ok) break;
                store_codes(kbits, kr, sbase + S::K0 + st * S::KV);
                const uint32_t sl = sbase + S::SC + (i % kScaleSlots) * Slot::BYTES;
                if (lift == 0.0f) {
                    // both warps look at the whole tile: no wait between them
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
                        lift = __int_as_float((127 + kvf::value_lift(mag)) << 23);
                        unit = __int_as_float((127 - kvf::value_lift(mag)) << 23);
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const uint32_t at = sl + 4 * (pt + 64 * t);
                    float sv = rs[t][2] * lift, zv = rs[t][3] * lift;
                    if (!(fabsf(sv) <= 3.4e38f && fabsf(zv) <= 3.4e38f)) {
                        // not a number: the score says so to the rows that see the token,
                        // the others multiply its value by zero
                        rs[t][0] = kv_nan();
                        sv = zv = 0.0f;
                    }
                    sts1(at + Slot::SK, rs[t][0] * p.key_scale);
                    sts1(at + Slot::SV, sv);
                    sts1(at + Slot::LV, lg2(fmaxf(sv, fabsf(zv))));
                    if constexpr (BK == 4) sts1(at + Slot::ZK, rs[t][1] * p.key_scale);
                    if constexpr (BV == 4) sts1(at + Slot::ZV, zv);
                    const float sm = warp_max(sv), zm = BV == 4 ? warp_max(fabsf(zv)) : 0.0f;
                    if (lane == 0) {
                        sts1(sl + Slot::SMAX + 4 * (pw + 2 * t), sm);
                        sts1(sl + Slot::ZMAX + 4 * (pw + 2 * t), zm);
                    }
                }
                if (pt == 0) sts1(sl + Slot::UNIT, unit);
                if (pw == 0) {
                    const uint32_t bad = __ballot_sync(0xffffffffu, no_page);
                    if (lane == 0) sts1(sl + Slot::BAD, __uint_as_float(bad));
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&scfull[i % kScaleSlots]);
                    mbar_arrive(&kfull[st]);
                }
                cur = page_ok(next);
                if (i + 1 < n) {
                    load_codes(kbits, kr, p.cache.codes[0], cur, i + 1);
                    load_scales(cur, i + 1);
                }
                next = load_pages(i + 2);
            }
            if (fault) kv_report(p.fault, fault);
        } else {
            const std::integral_constant<int, BV> vbits{};
            uint4 vr[Chunks<D, BV>::N];
            if (n > 0) load_codes(vbits, vr, p.cache.codes[1], page_ok(next), 0);
            next = load_pages(1);
            for (uint32_t i = 0; i < n; i++) {
                const uint32_t st = i % ST, ph = (i / ST) & 1;
                ok = __all_sync(0xffffffffu, wait_or_fault(&vempty[st], ph ^ 1, &abort_s, p.fault));
                if (!ok) break;
                store_codes(vbits, vr, sbase + S::V0 + st * S::KV);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&vfull[st]);
                const uint32_t cur = page_ok(next);
                if (i + 1 < n) load_codes(vbits, vr, p.cache.codes[1], cur, i + 1);
                next = load_pages(i + 2);
            }
        }
    } else if (set_regs<kRegsIssue>(); warp == 12) {
        // ================= MMA issue (whole warp, elected lane) =================
        // One warp for both row tiles, in turn: each tile's products run while the
        // other's softmax does (with a warp each, the two fell into step and the
        // tensor pipe waited: 2048 tokens behind 14336 took 1020 against 979 us).  The products run in
        // the order of issue: P V reads P before the next S is written over it.
        constexpr uint32_t id_s = idesc_f16(kTok, false), id_o = idesc_f16(D, true);
        const uint32_t q0 = sbase, k0 = sbase + S::K0, v0 = sbase + S::V0;
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
                umma_f16_ts_w(tmem + kOCol + D * sub, a, bd, id_o, (SPLIT ? pc[sub] % kFlush : pc[sub]) != 0 || ks != 0);
                if constexpr (SPLIT) umma_f16_ts_w(tmem + kOCol + D * sub, a + 8, bd, id_o, 1);
            }
        };
        // (also without a key tile: the outputs are staged where the queries are being converted)
        if (wait(&qfull, 0) && n > 0 && wait(&kfull[0], 0)) {
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
