// kernels_kv_few.cuh -- attention of a few query rows (a decode token, a short
// draft window) over the quantised paged KV cache.
//
// For one (sequence, KV head) the rows are the new tokens x the G query heads
// of the group (row r: token r / G, head r % G of the group), in tiles of 8 or
// 16.  With key j = zk_j + sk_j * kc_j (kc integer codes around zero, zk = 0 for
// 8 bits) and likewise values:
//   x_rj = c_r * (sk_j * (q_r . kc_j) + zk_j * sum(q_r)),  p = 2^(x - m_r)
//   o_r  = ( sum_j (p sv_j) vc_j + sum_j p zv_j ) / sum_j p
// so the two products run on exact small integers in f16 and everything that
// is not an integer stays in f32.  The rounded factors are q (22 bits as f16
// hi + lo for f32 queries, 11 bits otherwise: bf16 and f16 are exact) and the
// weight p sv (f16; hi + lo for f32 queries).  One f16 a weight is what the tensor cores
// multiply at full rate: each is off by 2^-12 at most, either way, which leaves outputs of
// 16 bits as far from the 64-bit ones as f32 weights do (1.7e-3 in bf16, 2.1e-4 in f16,
// of either).  The reference m is a whole
// number that puts the largest p * max(sv, |zv|) of the row at 2^9 .. 2^10 when
// it is set and is set anew when that passes 2^15: rescaling is by exact powers
// of two, and whatever the scale of the values the weights stay in f16's range
// with their 11 bits down to 2^-23 of the largest.  Where the values are zero
// only p bounds m (2^96 at most, and 2^31 of those stay in f32).  p makes up for
// the magnitude of the values, which later tiles may change at will: over 2^86
// down and 2^100 up from those of the first tile that is not all zero, which a
// power of two brings near one (value_lift).
//
// Bound: HBM, the visible codes and scales once (264 bytes a token and head at
// D = 128 and 8 bits, 144 at 4).  Layout:
//  - S^T = K Q^T and O^T = V^T P^T on mma.sync.m16n8k16 (M = 16 tokens or 16
//    dims, N = 8 rows): the rows of a decode step fill half of one N = 8 tile,
//    where the 128-row tcgen05 tile would be empty but for 4 of 128, and both
//    operands are unpacked in registers, which tcgen05 could not read.
//  - A warp owns 16-token tiles (one page holds a tile whole); their codes and
//    scales come by cp.async into a ring of three slots of its own, so two tiles a
//    warp are in flight and no barrier is in the loop.
//  - The context is split over CTAs.  Up to eight parts, where every CTA of the call
//    is resident at once, are a cluster, which joins them through distributed shared
//    memory (parts beyond a sequence's end leave at once); otherwise they go to the
//    workspace and k_kv_merge joins them.  Either way in order.
// Measured (device time): 64 sequences of 1024 to 8192 tokens, 32/8 heads: bf16 115 us at
// 4 bits (3.0 TB/s; 65% of the issue slots, for the unpacking and a tile's chain), 123 us
// at 8 bits (5.1 TB/s), f32 152 us at 8 bits (4.1 TB/s); 16 sequences of 1000 to 6000
// tokens with four new ones each, 8 bits, bf16: 56 us; one of 131071 tokens, 64/8 heads,
// f16, 8 bits: 58 us with its join (4.7 TB/s).
#pragma once
#include <type_traits>

#include "kv_math.cuh"

namespace nx {
namespace kvf {

constexpr int kWarps = kKvFewWarps;
constexpr int kStages = 3;
// Four CTAs an SM (16 warps) for 16-bit queries of up to 8 rows: the loop is a chain
// of short latencies, and the warps are what hides them
constexpr float kUp = 10.0f;         // log2 of the largest weight under a new reference
constexpr float kLimit = 32768.0f;   // largest weight any reference stays for
constexpr float kMostF16 = 65504.0f;
constexpr float kMaxProb = 96.0f;    // log2 of the largest p
// f32 queries: what the second f16 of a weight is multiplied by (at most half a step of the
// first, 2^3 for one of 2^15, so that it stays in f16).  A weight is then off by 2^-36 at
// most where it is small, 2^-45 of the largest (by itself f16 ends at 2^-25).
constexpr float kLoUp = 2048.0f;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_if(bool on, uint32_t dst, const void *src) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %2, 0;\n @p cp.async.cg.shared.global [%0], [%1], 16;\n}\n" ::"r"(dst),
                 "l"(src), "r"((uint32_t)on)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 f16x2_back(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^(a - b) exactly, for whole a <= b, either possibly -inf (0 then); 0 below f32's
// normal range.  For sums of weights, which a factor below that leaves nothing of
// (2^15 times their number, against 2^9 at least for the key that moved the reference).
__device__ __forceinline__ float pow2_diff(float a, float b) {
    const float d = a - b;
    return d >= -126.0f ? __int_as_float((127 + (int)d) << 23) : 0.0f;
}
// The same for sums of p: those of keys whose values are small are as large against the
// others' as their scores say, however far the references are apart (p lies between 2^-126
// and 2^96): a factor in two halves, each a normal number.
struct Pow2 {
    float h, g;
    __device__ __forceinline__ Pow2(float a, float b) {
        const float d = a - b;
        const int e = d >= -252.0f ? (int)d : -252;
        h = __int_as_float((127 + e / 2) << 23);
        g = d >= -252.0f ? __int_as_float((127 + e - e / 2) << 23) : 0.0f;
    }
    __device__ __forceinline__ float times(float v) const { return v * h * g; }
};

// O += V^T P^T of one tile.  The tensor cores round each sum toward zero, an error
// that grows with the number of tiles summed in place (2.2e-5 of the output after
// 40000 tokens); for f32 queries a tile is summed alone and added correctly rounded.
// Their weights' second halves come times 2^11 (kLoUp).
template <int NS>
__device__ __forceinline__ void add_tile(float (&o)[4], const uint32_t (&a)[4], const uint32_t (&p)[NS][2]) {
    if constexpr (NS == 1) {
        mma16816(o, a, p[0]);
    } else {
        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma16816(t, a, p[1]);
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] *= 1.0f / kLoUp;
        mma16816(t, a, p[0]);
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] += t[i];
    }
}

template <int D, int BK, int BV>
struct Tile {
    static constexpr int RK = D * BK / 8, RV = D * BV / 8;       // code bytes of a token
    static constexpr int K = 16 * RK, V = 16 * RV;               // code bytes of a tile
    static constexpr int KS = BK == 8 ? 64 : 128, VS = BV == 8 ? 64 : 128;
    static constexpr int BYTES = K + V + KS + VS;
    static constexpr int SMEM = kWarps * kStages * BYTES;
};
// 16-byte chunks of a 128-byte row are stored XORed with the row, so that the
// fragment loads of a quarter warp fall into different banks
template <int RB>
__device__ __forceinline__ int k_swz(int row) {
    return RB == 128 ? 4 * (row & 1) : 0;
}
template <int RB>
__device__ __forceinline__ int v_swz(int row) {
    return RB == 128 ? 2 * ((row >> 1) & 3) : RB == 64 ? (row >> 1) & 3 : 0;
}

template <int N>
__device__ __forceinline__ void lds_words(const uint8_t *p, uint32_t (&w)[N], int at) {
    if constexpr (N % 4 == 0) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        w[at] = v.x;
        w[at + 1] = v.y;
        w[at + 2] = v.z;
        w[at + 3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x;
        w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

// log2 of what scales and zeros are multiplied by when the largest of the first tile that is
// not all zero is `mag`: to 2^0 .. 2^9, but up by no more than 2^24, so that later values up
// to 2^104 stay in f32.
__device__ __forceinline__ int value_lift(float mag) {
    const int e = (int)((__float_as_uint(mag) >> 23) & 0xffu) - 127;
    return e > 8 ? 8 - e : min(24, max(0, -e));
}
// ---- distributed shared memory of a cluster ----
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ float cluster_ld(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
// The running sum v, l in reference m takes another in reference m1.
__device__ __forceinline__ void join(float &m, float &l, float (&v)[8], float m1, float l1, const float (&v1)[8]) {
    const float top = fmaxf(m, m1);
    const float f = m == top ? 1.0f : pow2_diff(m, top), f1 = m1 == top ? 1.0f : pow2_diff(m1, top);
    const float low = fminf(m, m1);
    if (low < top - 126.0f && low != -INFINITY) l = Pow2(m, top).times(l) + Pow2(m1, top).times(l1);
    else l = fmaf(l1, f1, l * f);
    m = top;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = fmaf(v1[j], f1, v[j] * f);
}
// Record of row r of a (sequence, KV head) pair and split s.
__host__ __device__ inline size_t few_record(uint32_t pair, uint32_t rows, uint32_t r, uint32_t nsplit, uint32_t s) {
    return ((size_t)pair * rows + r) * nsplit + s;
}

template <int D, int BK, int BV, int NR, bool SPLIT>
__global__ void __launch_bounds__(kWarps * 32, NR == 1 ? (SPLIT ? 3 : 4) : 2) k_kv_attn_few(KvAttnParams p) {
    using T = Tile<D, BK, BV>;
    constexpr int KW = D * BK / 128;       // 32-bit words of a key row per thread
    constexpr int UNITS = D / 32;          // units of eight consecutive elements of a row per thread
    constexpr int KSTEPS = D / 16;
    constexpr int MT = D / 16;             // 16-dim tiles of the output
    constexpr int NS = SPLIT ? 2 : 1;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    constexpr uint32_t R = 8 * NR;
    const uint32_t split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    unsigned fault = 0;
    const KvSeqView seq = kv_load_seq(p.batch, b, p.cache.shift, &fault);
    if (fault) {
        if (threadIdx.x == 0) kv_report(p.fault, fault);
        return;
    }
    const uint32_t G = (uint32_t)p.group;
    const KvRowTile rows = kv_row_tile(seq, G, 0, R, p.rows_limit);
    if (rows.n == 0) return;
    const int pos0 = (int)seq.kv - (int)seq.nq;
    const KvRange range = kv_range(rows.first, rows.last, p.window, p.sinks);
    const KvTiles tiles = kv_tiles(range, kKvFewTile);
    const uint32_t t_begin = split * p.tiles_per_split;
    const uint32_t t_end = min(tiles.total, t_begin + p.tiles_per_split);
    // (whoever joins the parts knows how many there are)
    if (p.nsplit > 1 && t_begin >= t_end && (split > 0 || !p.cluster)) return;

    // ---- copies: lane L of a batch of 32 tiles holds the page of tile L ----
    const uint32_t n_mine = t_begin + warp < t_end ? (t_end - t_begin - warp + kWarps - 1) / kWarps : 0;
    const uint32_t *table = p.batch.table + (size_t)b * p.batch.stride;
    auto tile_token = [&](uint32_t k) { return kv_tile_at(tiles, t_begin + warp + k * kWarps) * kKvFewTile; };
    auto load_page = [&](uint32_t k) -> uint32_t {
        if (k >= n_mine) return 0u;
        return __ldg(table + (tile_token(k) >> p.cache.shift));
    };
    uint32_t page_cur = load_page(lane), page_next = load_page(32 + lane);
    uint8_t *ring = smem + warp * kStages * T::BYTES;
    const uint32_t ring_s = smem_u32(ring);
    unsigned bad = 0;  // bit k & 31: tile k has no valid page
    auto issue = [&](uint32_t k) {
        if (k < n_mine) {
            if ((k & 31u) == 0 && k > 0) {
                page_cur = page_next;
                page_next = load_page(k + 32 + lane);
            }
            uint32_t page = __shfl_sync(0xffffffffu, page_cur, k & 31u);
            bad &= ~(1u << (k & 31u));
            if (page >= p.cache.num_pages) {
                // (page 0 is read in its place, and nothing made of it)
                bad |= 1u << (k & 31u);
                fault = KV_FAULT_PAGE;
                page = 0;
            }
            const size_t slot = (((size_t)page * p.cache.hkv + h) << p.cache.shift) +
                                (tile_token(k) & ((1u << p.cache.shift) - 1u));
            const uint32_t dst = ring_s + (k % kStages) * T::BYTES;
            const uint8_t *ks = p.cache.codes[0] + slot * T::RK + lane * 16, *vs = p.cache.codes[1] + slot * T::RV + lane * 16;
#pragma unroll
            for (int i = 0; i < (T::K / 16 + 31) / 32; i++) {
                const int ch = i * 32 + lane, row = ch / (T::RK / 16), col = ch % (T::RK / 16);
                cp_async16_if(T::K / 16 >= 32 || ch < T::K / 16, dst + row * T::RK + ((col ^ k_swz<T::RK>(row)) * 16),
                              ks + i * 512);
            }
#pragma unroll
            for (int i = 0; i < (T::V / 16 + 31) / 32; i++) {
                const int ch = i * 32 + lane, row = ch / (T::RV / 16), col = ch % (T::RV / 16);
                cp_async16_if(T::V / 16 >= 32 || ch < T::V / 16, dst + T::K + row * T::RV + ((col ^ v_swz<T::RV>(row)) * 16),
                              vs + i * 512);
            }
            // scales: lanes 0-15 of the keys', 16-31 of the values'
            const int sl = lane & 15;
            const uint8_t *ss = lane < 16 ? reinterpret_cast<const uint8_t *>(p.cache.scales[0]) + slot * (T::KS / 16)
                                          : reinterpret_cast<const uint8_t *>(p.cache.scales[1]) + slot * (T::VS / 16);
            cp_async16_if(sl < (lane < 16 ? T::KS : T::VS) / 16, dst + T::K + T::V + (lane < 16 ? 0 : T::KS) + sl * 16,
                          ss + sl * 16);
        }
        cp_commit();
    };
#pragma unroll
    for (int k = 0; k < kStages - 1; k++) issue(k);

    // ---- queries: row g (+ 8) as the B operand, in the order of the code words ----
    // 16-bit queries meet the codes as they stand: a code in the low bits of an f16 is
    // code * 2^-24, exact, and a 4-bit one four bits up 16 times that, which those
    // elements of the query make up for.  The codes are then not around zero, and the
    // products cancel against zero - mid * scale, which costs f32 a few units in the
    // last place of the score (too many for f32 queries, whose codes are centred).
    constexpr bool RAW = !SPLIT;
    // Of the 2^24, 2^5 go on the keys' scales and 2^19 on the row's factor: neither leaves f32
    // before the scores of centred codes would (keys of 2^114, queries times scale of 2^122).
    constexpr int kNorm = RAW ? 14 : 7;
    constexpr float kRawUp = 16777216.0f, kKeyUp = RAW ? 32.0f : 1.0f;
    const float key_factor = p.key_scale * kKeyUp;
    uint32_t qf[NR][NS][KSTEPS][2];
    f2 x_scale[NR], x_sum[NR];  // of this thread's columns, rows 2c and 2c + 1
    int x_pos[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
        const uint32_t r = rows.r0 + 8 * nr + g, tok = r / G, head = h * G + r % G;
        const bool used = (uint32_t)(8 * nr + g) < rows.n;
        float q[UNITS][8];
        float amax = 0.0f;
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            // first element of the unit: 8-bit rows come in 16-byte chunks c and c + 4
            // (two units each; 8 bytes at D = 32), 4-bit rows in chunks of up to 16 bytes
            int e;
            if constexpr (BK == 8) e = D == 32 ? 8 * c : (u >> 1) * 64 + c * 16 + (u & 1) * 8;
            else e = c * (D / 4) + 8 * u;
            if (used) {
                load8(p.q.data, (size_t)(seq.q0 + tok) * p.q.row_stride + head * p.q.head_stride + e, p.q.fmt, q[u]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) q[u][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(q[u][i]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e_row = row_exp(amax);
        const float sc = pow2i(kNorm - e_row);
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            // element pairs of a k step: (0,1)(2,3) then (4,5)(6,7) of 8-bit words,
            // (0,4)(1,5) then (2,6)(3,7) of a 4-bit word
            constexpr int o8[8] = {0, 1, 2, 3, 4, 5, 6, 7}, o4[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float up = RAW && BK == 4 && (i & 1) ? 16.0f : 1.0f;
                const float v0 = q[u][BK == 8 ? o8[2 * i] : o4[2 * i]] * (sc / up);
                const float v1 = q[u][BK == 8 ? o8[2 * i + 1] : o4[2 * i + 1]] * (sc / up);
                const uint32_t hi = f16x2(v0, v1);
                const float2 back = f16x2_back(hi);
                qf[nr][0][2 * u + (i >> 1)][i & 1] = hi;
                sum += (back.x + back.y) * up;
                if constexpr (SPLIT) {
                    const uint32_t lo = f16x2(v0 - back.x, v1 - back.y);
                    const float2 lb = f16x2_back(lo);
                    qf[nr][NS - 1][2 * u + (i >> 1)][i & 1] = lo;
                    sum += lb.x + lb.y;
                }
            }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if constexpr (RAW) sum *= kKeyUp / kRawUp;  // (the sum in the scores' units)
        const float xs = pow2i(p.scale_exp + e_row - kNorm + (RAW ? 24 - 5 : 0));
        const int pos = used ? pos0 + (int)tok : -1;
        float xe[2], se[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            xe[e] = __shfl_sync(0xffffffffu, xs, (2 * c + e) * 4);
            se[e] = __shfl_sync(0xffffffffu, sum, (2 * c + e) * 4);
            x_pos[nr][e] = __shfl_sync(0xffffffffu, pos, (2 * c + e) * 4);
        }
        x_scale[nr] = pk(xe[0], xe[1]);
        x_sum[nr] = pk(se[0], se[1]);
    }

    float o[NR][MT][4], m[NR][2];
    f2 l[NR], z[NR], nm[NR];  // nm: minus the reference, 0 while there is none
    bool unset = false;       // some reference is not set yet
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[nr][j][i] = 0.0f;
        l[nr] = z[nr] = nm[nr] = pk(0.0f, 0.0f);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            // rows that see nothing start with a reference of their own: they never ask for one
            m[nr][e] = x_pos[nr][e] >= 0 ? -INFINITY : 0.0f;
            unset |= m[nr][e] == -INFINITY;
        }
    }
    unset = __any_sync(0xffffffffu, unset);

    // power of two on the values' scales and zeros (0: none of them seen so far but
    // zero) and its reciprocal
    float lift = 0.0f, unit = 1.0f;
    for (uint32_t k = 0; k < n_mine; k++) {
        cp_wait<kStages - 2>();
        __syncwarp();
        const uint8_t *st = ring + (k % kStages) * T::BYTES;
        const int j0 = (int)tile_token(k);
        if (!((bad >> (k & 31u)) & 1u)) {
            // ---- S^T = K Q^T ----
            uint32_t kw[2][KW];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int row = g + 8 * t;
                const uint8_t *kr = st + row * T::RK;
                if constexpr (T::RK == 128) {
                    lds_words<KW>(kr + ((c ^ k_swz<128>(row)) * 16), kw[t], 0);
                    lds_words<KW>(kr + (((c + 4) ^ k_swz<128>(row)) * 16), kw[t], 4);
                } else {
                    lds_words<KW>(kr + c * (T::RK / 4), kw[t], 0);
                }
            }
            float s[NR][4];
#pragma unroll
            for (int nr = 0; nr < NR; nr++) s[nr][0] = s[nr][1] = s[nr][2] = s[nr][3] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ks += BK == 8 ? 1 : 2) {
                if constexpr (BK == 8) {
                    uint32_t a[4];
                    if constexpr (RAW) {
                        raw_u8(kw[0][ks], a[0], a[2]);
                        raw_u8(kw[1][ks], a[1], a[3]);
                    } else {
                        unpack_u8(kw[0][ks], a[0], a[2]);
                        unpack_u8(kw[1][ks], a[1], a[3]);
                    }
#pragma unroll
                    for (int nr = 0; nr < NR; nr++)
#pragma unroll
                        for (int n = 0; n < NS; n++) mma16816(s[nr], a, qf[nr][n][ks]);
                } else {
                    uint32_t u0[4], u1[4];
                    if constexpr (RAW) {
                        raw_u4(kw[0][ks >> 1], u0);
                        raw_u4(kw[1][ks >> 1], u1);
                    } else {
                        unpack_u4(kw[0][ks >> 1], u0);
                        unpack_u4(kw[1][ks >> 1], u1);
                    }
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const uint32_t a[4] = {u0[2 * half], u1[2 * half], u0[2 * half + 1], u1[2 * half + 1]};
#pragma unroll
                        for (int nr = 0; nr < NR; nr++)
#pragma unroll
                            for (int n = 0; n < NS; n++) mma16816(s[nr], a, qf[nr][n][ks + half]);
                    }
                }
            }
            // ---- scales of tokens j0 + g and j0 + g + 8 ----
            float sk[2], zk[2], sv[2], zv[2];
            const float *kscale = reinterpret_cast<const float *>(st + T::K + T::V);
            const float *vscale = reinterpret_cast<const float *>(st + T::K + T::V + T::KS);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int i = g + 8 * t;
                sk[t] = BK == 8 ? kscale[i] : kscale[2 * i];
                zk[t] = BK == 8 ? 0.0f : kscale[2 * i + 1];
                sv[t] = BV == 8 ? vscale[i] : vscale[2 * i];
                zv[t] = BV == 8 ? 0.0f : vscale[2 * i + 1];
                sk[t] *= key_factor;
                if constexpr (BK == 4) zk[t] *= p.key_scale;
                if constexpr (RAW) zk[t] = fmaf((BK == 8 ? -128.0f : -8.0f) / kKeyUp, sk[t], zk[t]);
            }
            if (lift == 0.0f) {
                float mag = 0.0f;
#pragma unroll
                for (int t = 0; t < 2; t++)
                    if (kv_needed(range, j0 + g + 8 * t, j0 + g + 8 * t + 1))
                        mag = fmaxf(mag, fmaxf(sv[t], fabsf(zv[t])));
                mag = warp_max(mag);
                if (mag > 0.0f) {
                    lift = __int_as_float((127 + value_lift(mag)) << 23);
                    unit = __int_as_float((127 - value_lift(mag)) << 23);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; t++) {
                sv[t] *= lift;
                if constexpr (BV == 4) zv[t] *= lift;
            }
            // every token of the tile seen by every row?
            const bool whole = j0 + (int)kKvFewTile - 1 <= rows.first &&
                               (p.window == 0 || j0 > rows.last - (int)p.window ||
                                j0 + (int)kKvFewTile <= (int)p.sinks);
            // score of token half t and this thread's two rows, before the row's factor
            auto score = [&](int nr, int t) {
                const f2 v = mul2(pk(s[nr][2 * t], s[nr][2 * t + 1]), pk(sk[t], sk[t]));
                return RAW || BK == 4 ? fma2(pk(zk[t], zk[t]), x_sum[nr], v) : v;
            };
            uint32_t pf[NR][NS][2];
            // Weights against the references, first the old ones: true where they hold.
            auto weigh = [&](auto masked, float limit) -> bool {
                constexpr bool MASK = decltype(masked)::value;
                f2 pp[NR][2], ww[NR][2];
                float top = 0.0f;
#pragma unroll
                for (int nr = 0; nr < NR; nr++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        float e0, e1;
                        upk(fma2(score(nr, t), x_scale[nr], nm[nr]), e0, e1);
                        float v0 = sv[t], v1 = sv[t];
                        if constexpr (MASK) {
                            // (a hidden token's values may be anything)
                            if (!kv_visible(j0 + g + 8 * t, x_pos[nr][0], (int)p.window, (int)p.sinks)) {
                                e0 = -INFINITY;
                                v0 = 0.0f;
                            }
                            if (!kv_visible(j0 + g + 8 * t, x_pos[nr][1], (int)p.window, (int)p.sinks)) {
                                e1 = -INFINITY;
                                v1 = 0.0f;
                            }
                        }
                        const float p0 = ex2(e0), p1 = ex2(e1);
                        pp[nr][t] = pk(p0, p1);
                        ww[nr][t] = mul2(pp[nr][t], pk(v0, v1));
                        float w0, w1;
                        upk(ww[nr][t], w0, w1);
                        // a weight above 2^15, or p above 2^96
                        top = fmaxf(fmaxf(top, fmaxf(w0, w1)), fmaxf(p0, p1) * 4.1359031e-25f);
                    }
                if (__any_sync(0xffffffffu, top > limit)) return false;
#pragma unroll
                for (int nr = 0; nr < NR; nr++) {
                    l[nr] = add2(l[nr], add2(pp[nr][0], pp[nr][1]));
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        float w0, w1;
                        upk(ww[nr][t], w0, w1);
                        if constexpr (BV == 4) {
                            float p0, p1;
                            upk(pp[nr][t], p0, p1);
                            const bool h0 = MASK && p0 == 0.0f, h1 = MASK && p1 == 0.0f;
                            z[nr] = fma2(pp[nr][t], pk(h0 ? 0.0f : zv[t], h1 ? 0.0f : zv[t]), z[nr]);
                        }
                        const uint32_t hi = f16x2(w0, w1);
                        pf[nr][0][t] = transpose8x8(hi);
                        if constexpr (SPLIT) {
                            const float2 back = f16x2_back(hi);
                            pf[nr][NS - 1][t] = transpose8x8(f16x2((w0 - back.x) * kLoUp, (w1 - back.y) * kLoUp));
                        }
                    }
                }
                return true;
            };
            // References that hold for this tile, or (higher) the whole numbers after the present
            // ones; the sums so far follow.
            auto new_reference = [&](bool higher) {
                unset = false;
#pragma unroll
                for (int nr = 0; nr < NR; nr++) {
                    float x[2][2];
#pragma unroll
                    for (int t = 0; t < 2; t++) upk(mul2(score(nr, t), x_scale[nr]), x[t][0], x[t][1]);
                    float cm[2], ch[2], cg[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float mx = -INFINITY, my = -INFINITY;
#pragma unroll
                        for (int t = 0; t < 2; t++)
                            if (whole || kv_visible(j0 + g + 8 * t, x_pos[nr][e], (int)p.window, (int)p.sinks)) {
                                mx = fmaxf(mx, x[t][e]);
                                my = fmaxf(my, x[t][e] + lg2(BV == 8 ? sv[t] : fmaxf(sv[t], fabsf(zv[t]))));
                            }
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) {
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
                            my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, w));
                        }
                        const float m1 = higher ? __fadd_ru(m[nr][e], 1.0f)
                                                : fmaxf(m[nr][e], fmaxf(ceilf(mx) - kMaxProb, ceilf(my) - kUp));
                        cm[e] = ch[e] = cg[e] = 1.0f;
                        if (m1 != m[nr][e]) {
                            const Pow2 f(m[nr][e], m1);
                            cm[e] = pow2_diff(m[nr][e], m1);
                            ch[e] = f.h;
                            cg[e] = f.g;
                        }
                        m[nr][e] = m1;
                        unset |= m1 == -INFINITY;
                    }
                    nm[nr] = pk(m[nr][0] == -INFINITY ? 0.0f : -m[nr][0], m[nr][1] == -INFINITY ? 0.0f : -m[nr][1]);
                    l[nr] = mul2(mul2(l[nr], pk(ch[0], ch[1])), pk(cg[0], cg[1]));
                    z[nr] = mul2(z[nr], pk(cm[0], cm[1]));
#pragma unroll
                    for (int j = 0; j < MT; j++)
#pragma unroll
                        for (int i = 0; i < 4; i++) o[nr][j][i] *= cm[i & 1];
                }
                unset = __any_sync(0xffffffffu, unset);
            };
            // After new references weights are at most 2^kUp, but where a step of f32 at x is
            // several powers of two (scores of 2^25 and more) those are up to two steps off:
            // then the next ones.  (Weights of infinite scales or scores stay as they are.)
            bool renew = unset;
            float limit = kLimit;
            int tries = 0;
            while (true) {
                if (renew) {
                    new_reference(tries > 0);
                    limit = ++tries < 4 ? kMostF16 : INFINITY;
                }
                if (whole ? weigh(std::false_type{}, limit) : weigh(std::true_type{}, limit)) break;
                renew = true;
            }
            // ---- O^T += V^T P^T: tokens 2c, 2c + 1, 2c + 8, 2c + 9, dims g * D/8 .. ----
            constexpr int VW = T::RV / 32;  // words per token (0: two bytes)
            const uint8_t *vr = st + T::K;
            auto v_at = [&](int i) {
                const int row = 2 * c + (i & 1) + 8 * (i >> 1);
                const int byte = g * (T::RV / 8);
                return vr + row * T::RV + ((((byte >> 4) ^ v_swz<T::RV>(row)) << 4) | (byte & 15));
            };
            if constexpr (VW > 0) {
                uint32_t vw[4][VW];
#pragma unroll
                for (int i = 0; i < 4; i++) lds_words<VW>(v_at(i), vw[i], 0);
#pragma unroll
                for (int w = 0; w < VW; w++) {
                    if constexpr (BV == 8) {
                        // interleave the bytes of tokens (0, 1) and (2, 3), then unpack pairs
                        uint32_t a01, a23, b01, b23;
                        asm("prmt.b32 %0, %1, %2, 0x5140;" : "=r"(a01) : "r"(vw[0][w]), "r"(vw[1][w]));
                        asm("prmt.b32 %0, %1, %2, 0x7362;" : "=r"(a23) : "r"(vw[0][w]), "r"(vw[1][w]));
                        asm("prmt.b32 %0, %1, %2, 0x5140;" : "=r"(b01) : "r"(vw[2][w]), "r"(vw[3][w]));
                        asm("prmt.b32 %0, %1, %2, 0x7362;" : "=r"(b23) : "r"(vw[2][w]), "r"(vw[3][w]));
                        uint32_t a[4], a2[4];
                        unpack_u8(a01, a[0], a[1]);
                        unpack_u8(b01, a[2], a[3]);
                        unpack_u8(a23, a2[0], a2[1]);
                        unpack_u8(b23, a2[2], a2[3]);
#pragma unroll
                        for (int nr = 0; nr < NR; nr++) {
                            add_tile<NS>(o[nr][2 * w], a, pf[nr]);
                            add_tile<NS>(o[nr][2 * w + 1], a2, pf[nr]);
                        }
                    } else {
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            uint32_t a01, b01;
                            if (half == 0) {
                                asm("prmt.b32 %0, %1, %2, 0x5410;" : "=r"(a01) : "r"(vw[0][w]), "r"(vw[1][w]));
                                asm("prmt.b32 %0, %1, %2, 0x5410;" : "=r"(b01) : "r"(vw[2][w]), "r"(vw[3][w]));
                            } else {
                                asm("prmt.b32 %0, %1, %2, 0x7632;" : "=r"(a01) : "r"(vw[0][w]), "r"(vw[1][w]));
                                asm("prmt.b32 %0, %1, %2, 0x7632;" : "=r"(b01) : "r"(vw[2][w]), "r"(vw[3][w]));
                            }
                            uint32_t ua[4], ub[4];
                            unpack_u4(a01, ua);
                            unpack_u4(b01, ub);
                            const uint32_t a[4] = {ua[0], ua[1], ub[0], ub[1]}, a2[4] = {ua[2], ua[3], ub[2], ub[3]};
#pragma unroll
                            for (int nr = 0; nr < NR; nr++) {
                                add_tile<NS>(o[nr][4 * w + 2 * half], a, pf[nr]);
                                add_tile<NS>(o[nr][4 * w + 2 * half + 1], a2, pf[nr]);
                            }
                        }
                    }
                }
            } else {
                // D = 32 at 4 bits: two bytes a token
                uint32_t u[2];
#pragma unroll
                for (int i = 0; i < 2; i++)
                    u[i] = (uint32_t) * reinterpret_cast<const uint16_t *>(v_at(2 * i)) |
                           ((uint32_t) * reinterpret_cast<const uint16_t *>(v_at(2 * i + 1)) << 16);
                uint32_t ua[4], ub[4];
                unpack_u4(u[0], ua);
                unpack_u4(u[1], ub);
                const uint32_t a[4] = {ua[0], ua[1], ub[0], ub[1]}, a2[4] = {ua[2], ua[3], ub[2], ub[3]};
#pragma unroll
                for (int nr = 0; nr < NR; nr++) {
                    add_tile<NS>(o[nr][0], a, pf[nr]);
                    add_tile<NS>(o[nr][1], a2, pf[nr]);
                }
            }
        }
        __syncwarp();  // every lane has read the slot that the next copy reuses
        issue(k + kStages - 1);
    }
    cp_wait<0>();
    if (fault && lane == 0) kv_report(p.fault, fault);

    pdl_launch_dependents();
    // ---- join the warps: records of (row, dim) in the first one's reference ----
    __syncthreads();
    constexpr int RS = D + 2;
    float *rec = reinterpret_cast<float *>(smem);  // [warp][8 NR rows][D + 2]
#pragma unroll
    for (int nr = 0; nr < NR; nr++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float lt, zt, other;
            upk(l[nr], e ? other : lt, e ? lt : other);
            upk(z[nr], e ? other : zt, e ? zt : other);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
                lt += __shfl_xor_sync(0xffffffffu, lt, w);
                zt += __shfl_xor_sync(0xffffffffu, zt, w);
            }
            float *r = rec + (warp * 8 * NR + 8 * nr + 2 * c + e) * RS;
#pragma unroll
            for (int j = 0; j < MT; j++) {
                r[g * (D / 8) + 2 * j] = (o[nr][j][e] + zt) * unit;
                r[g * (D / 8) + 2 * j + 1] = (o[nr][j][2 + e] + zt) * unit;
            }
            if (g == 0) {
                r[D] = m[nr][e];
                r[D + 1] = lt;
            }
        }
    __syncthreads();
    const uint32_t pair = b * p.cache.hkv + h;
    float *mine = rec + kWarps * 8 * NR * RS;  // this part's records, for the cluster
    auto finish = [&](uint32_t r, uint32_t d0, float l_all, float(&v)[8]) {
        const float inv = l_all == 0.0f ? 0.0f : 1.0f / l_all;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= inv;
        const uint32_t tok = (rows.r0 + r) / G, head = h * G + (rows.r0 + r) % G;
        store8(p.out.data, (size_t)(seq.q0 + tok) * p.out.row_stride + head * p.out.head_stride + d0, p.out.fmt, v);
    };
    for (uint32_t i = threadIdx.x; i < rows.n * (D / 8); i += kWarps * 32) {
        const uint32_t r = i / (D / 8), d0 = (i % (D / 8)) * 8;
        float top = -INFINITY, l_all = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float *src = rec + (w * 8 * NR + r) * RS;
            float v1[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v1[j] = src[d0 + j];
            join(top, l_all, v, src[D], src[D + 1], v1);
        }
        if (p.nsplit > 1) {
            const size_t at = few_record(pair, R, r, p.nsplit, split);
            float *dst = p.cluster ? mine + r * RS : p.part + at * D;
            float *ml = p.cluster ? mine + r * RS + D : p.ml + at * 2;
#pragma unroll
            for (int j = 0; j < 8; j += 2) *reinterpret_cast<float2 *>(dst + d0 + j) = make_float2(v[j], v[j + 1]);
            if (d0 == 0) *reinterpret_cast<float2 *>(ml) = make_float2(top, l_all);
        } else {
            finish(r, d0, l_all, v);
        }
    }
    if (p.cluster && p.nsplit > 1) {
        const uint32_t used = max(1u, (tiles.total + p.tiles_per_split - 1) / p.tiles_per_split);
        __syncwarp();
        cluster_sync();
        for (uint32_t i = split * (kWarps * 32) + threadIdx.x; i < rows.n * (D / 8); i += used * (kWarps * 32)) {
            const uint32_t r = i / (D / 8), d0 = (i % (D / 8)) * 8;
            float top = -INFINITY, l_all = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            for (uint32_t s = 0; s < used; s++) {
                const uint32_t src = cluster_addr(smem_u32(mine + r * RS), s);
                float v1[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v1[j] = cluster_ld(src + 4 * (d0 + j));
                join(top, l_all, v, cluster_ld(src + 4 * D), cluster_ld(src + 4 * D + 4), v1);
            }
            finish(r, d0, l_all, v);
        }
        __syncwarp();
        cluster_sync();  // nobody leaves while its records are read
    }
}

template <int D, int BK, int BV, int NR, bool SPLIT>
cudaError_t launch_few_t(const KvAttnParams &p, cudaStream_t st) {
    using T = Tile<D, BK, BV>;
    constexpr int JOIN = (kWarps + 1) * 8 * NR * (D + 2) * 4;
    constexpr int SMEM = T::SMEM > JOIN ? T::SMEM : JOIN;
    auto *fn = k_kv_attn_few<D, BK, BV, NR, SPLIT>;
    if (SMEM > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.nsplit, p.cache.hkv, p.batch.n_seqs);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {p.nsplit, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = p.cluster && p.nsplit > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, fn, p);
}

template <int D, int BK, int BV>
cudaError_t launch_few_bits(const KvAttnParams &p, cudaStream_t st) {
    const bool split = p.q.fmt == kFmtF32;
    if (p.tile_rows == 8)
        return split ? launch_few_t<D, BK, BV, 1, true>(p, st) : launch_few_t<D, BK, BV, 1, false>(p, st);
    return split ? launch_few_t<D, BK, BV, 2, true>(p, st) : launch_few_t<D, BK, BV, 2, false>(p, st);
}

template <int D>
cudaError_t launch_few_dim(const KvAttnParams &p, cudaStream_t st) {
    const int bk = p.cache.bits[0], bv = p.cache.bits[1];
    if (bk == 8) return bv == 8 ? launch_few_bits<D, 8, 8>(p, st) : launch_few_bits<D, 8, 4>(p, st);
    return bv == 8 ? launch_few_bits<D, 4, 8>(p, st) : launch_few_bits<D, 4, 4>(p, st);
}

}  // namespace kvf
}  // namespace nx
