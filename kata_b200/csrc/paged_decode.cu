// Attention of the newest tokens over a paged KV cache, split over the cache's length and joined (kata_paged_decode, include/kata_paged.h).
//   o_r = sum_j p_rj v_j / sum_j p_rj, p_rj = exp(q_r . k_j - m_r), j over the slots row r sees; row r = t * group + j of a KV head's 16-row block.
// With weights: w[kv head][j] += sum_r p_rj / l_r, which needs the joined (m, l); the fp32 scores are kept and a second, small kernel forms the sums.
//
// Bound by HBM (4096 bytes of K+V per slot at fp16 with 4 heads of 256, each read once), so the work split is that of the contiguous decode kernel:
// the tiles (16 or 32 slots of one KV head, 16 KiB of K+V) of all (sequence, KV head) segments form one list, cut into one contiguous range per SM, the
// ranges' partial rows joined by the last CTA of a segment (at most 8 of them) or by a combine grid. Inside a CTA four rings of a score warp and two value warps take
// the tiles in turn; a producer warp refills the rings' stages with TMA. What pages change:
//  - A tile is made of 16-slot groups, and a group never crosses a page (pages are powers of two from 16 slots on). The tensor map is a rank-5 view of
//    the pool, {128-byte column block, 16 rows, column blocks, 16-row groups, KV heads}: the group is a coordinate, so one instruction
//    brings the 16 or 32 slots of a tile wherever their page lies, in the same shared-memory order ([group][column block][16 rows][128 bytes], swizzled) for
//    every page size. Pages of 16 slots under 32-slot tiles take two instructions.
//  - The producer reads the page number of a tile three tiles before it needs it, the score warp that of its int8 scales six tiles before: neither waits for a table look-up.
//  - Groups behind the last slot repeat the last page (their table entry may not exist); such slots are masked, and their V rows zeroed in shared
//    memory, so whatever lies there (NaN included) has no part in the result.
// Head layouts: head_dim 256 or 128, up to 16 query heads per KV head; tokens beyond 16 / group run as further passes.
//
// Precision: fp16 products, fp32 sums. The exponent carries an offset (kPShift) so that p lies high in fp16's range: it cancels in p / l and keeps
// small p out of the subnormals. p is rounded to fp16 before P.V as in the contiguous kernel (relative error 2^-11 at most, what the bf16 or fp16
// output is rounded by anyway); FINE (fp32 outputs) carries it in two fp16 terms and takes int8 codes without the 1152 bias whose subtraction would cost
// some ten bits.
#include <algorithm>

#include "attn_tile.cuh"
#include "paged_internal.cuh"

namespace kata {
namespace {

using namespace ptx;

constexpr int kRings = 4, kWarps = 3 * kRings + 1, kThreads = kWarps * 32, kMaxStages = 8;

template <int HD, bool K8, bool FINE> struct PGeo {
    static constexpr int kRowBytes = HD * (K8 ? 1 : 2), kNB = kRowBytes / 128;           // bytes and 128-byte column blocks of a head row
    static constexpr int kNK = (HD == 256 && !K8) ? 1 : 2, kTile = 16 * kNK;             // 16-slot groups and slots per tile
    static constexpr int kGroupBytes = 16 * kRowBytes, kHalfBytes = kNK * kGroupBytes;   // K (or V) of one group, of one tile
    static constexpr int kStageBytes = 2 * kHalfBytes, kStages = kStageBytes == 16384 ? 3 : 6;
    static constexpr int kMergeStride = HD + 8;                                          // floats per row of the cross-ring merge buffer
    static constexpr int kRingBytes = kStages * kStageBytes;
    static constexpr int kQStride = HD * 2 + 16;
    static constexpr int kPStride = 32 * kNK + 16, kPTerm = 16 * kPStride, kPBytes = kPTerm * (FINE ? 2 : 1) + 64;   // a P slot: one or two fp16 blocks, 16 rescale factors
    static constexpr int kPShift = K8 ? 5 : 15;                                          // p is carried as 2^kPShift * p (int8: p times a scale up to 516 has to stay below 65504)
    static constexpr int kOffBars = 16 * kQStride, kOffQsum = kOffBars + 704, kOffMl = kOffQsum + 64, kOffPair = kOffMl + 512, kOffStages = kOffPair + kRings * 2 * kPBytes;
    static constexpr int kSmem = kOffStages + 1024 + kRings * kRingBytes;
    static_assert(16 * kMergeStride * 4 <= kRingBytes && kSmem <= 232448, "shared memory");
};
constexpr int kOffEBars = kRings * kMaxStages * 8, kOffPBars = 2 * kOffEBars;   // inside the barrier block: 'full', 'empty', then per ring two 'P full' and two 'P empty'
static_assert(kOffPBars + kRings * 32 <= 704, "barrier block");

struct PagedPlan {
    int32_t n, T, group, kv_heads, n_ctas, q_tiles, r_tiles, cps;   // as in the contiguous kernel: CTA c owns tiles [c*q + min(c,r), ..), or (cps > 0) a share of one segment
    int32_t tok_stride, tok0, page_shift, width, groups_per_box, merge_in_kernel;
    int64_t layer_row0;
    int32_t seq[KATA_PAGED_MAX_BATCH];
    int32_t kend[KATA_PAGED_MAX_BATCH];            // slots the last token of this pass sees (may be 0)
    int32_t tile_start[KATA_PAGED_MAX_BATCH + 1];
};
static_assert(sizeof(PagedPlan) + 2 * sizeof(CUtensorMap) + 128 <= 4096, "kernel parameters");

__host__ __device__ __forceinline__ int plan_ntiles(const PagedPlan& p, int b) { return (p.tile_start[b + 1] - p.tile_start[b]) / p.kv_heads; }
__host__ __device__ __forceinline__ int plan_first_tile(const PagedPlan& p, int c) {
    if (p.cps) { const int seg = c / p.cps, j = c - seg * p.cps, nt = plan_ntiles(p, 0); return seg * nt + (int)((int64_t)nt * j / p.cps); }
    return c * p.q_tiles + (c < p.r_tiles ? c : p.r_tiles);
}
__host__ __device__ __forceinline__ int plan_cta_of_tile(const PagedPlan& p, int tile) {
    if (p.cps) { const int nt = plan_ntiles(p, 0), seg = tile / nt, lt = tile - seg * nt; return seg * p.cps + (int)(((int64_t)(lt + 1) * p.cps + nt - 1) / nt) - 1; }
    const int big = p.r_tiles * (p.q_tiles + 1);
    return tile < big ? tile / (p.q_tiles + 1) : p.r_tiles + (tile - big) / p.q_tiles;
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const void* tmap, int x, int r, int c, int g, int h, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(r), "r"(c), "r"(g), "r"(h), "r"(bar) : "memory");
}

// Score warp, one tile: s[nt][e] = q_row . k of n-tile nt (8 slots: key0 + 8*nt + 2*t4 + e; elements 2, 3: row g + 8), scaled (int8) and masked.
template <int HD, bool K8, bool FINE>
__device__ __forceinline__ void paged_scores(const uint32_t q_sm, const uint32_t k_sm, const int key0, const int lim0, const int lim1, const float (&ks)[2 * PGeo<HD, K8, FINE>::kNK][2], const float (&qs)[2],
                                             const int lane, float (&s)[2 * PGeo<HD, K8, FINE>::kNK][4]) {
    using G = PGeo<HD, K8, FINE>; constexpr int NK = G::kNK, NT = 2 * NK;
    const int t4 = lane & 3; const uint32_t rx = lane & 7, q1 = (lane >> 3) & 1;
    const uint32_t qa = q_sm + (lane & 15) * G::kQStride + (lane >> 4) * 16, ka = k_sm + (rx + ((lane >> 4) << 3)) * 128;
    const uint32_t ko[4] = {((0 + q1) ^ rx) << 4, ((2 + q1) ^ rx) << 4, ((4 + q1) ^ rx) << 4, ((6 + q1) ^ rx) << 4};
    float s2[NT][4];   // a second accumulator chain per n-tile
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) { s[nt][e] = 0.0f; s2[nt][e] = 0.0f; }
    if (!K8) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk += 2) {
            uint32_t a0, a1, a2, a3, c0, c1, c2, c3;
            ldsm_x4(qa + kk * 32, a0, a1, a2, a3); ldsm_x4(qa + kk * 32 + 32, c0, c1, c2, c3);
#pragma unroll
            for (int sb = 0; sb < NK; sb++) {
                uint32_t b0, b1, b2, b3, d0, d1, d2, d3; const uint32_t kb = ka + sb * G::kGroupBytes + (kk >> 2) * 2048;
                ldsm_x4(kb + ko[kk & 3], b0, b1, b2, b3); ldsm_x4(kb + ko[(kk & 3) + 1], d0, d1, d2, d3);
                mma16816(s[2 * sb], a0, a1, a2, a3, b0, b1); mma16816(s[2 * sb + 1], a0, a1, a2, a3, b2, b3);
                mma16816(s2[2 * sb], c0, c1, c2, c3, d0, d1); mma16816(s2[2 * sb + 1], c0, c1, c2, c3, d2, d3);
            }
        }
    } else {
#pragma unroll
        for (int k2 = 0; k2 < HD / 32; k2++) {   // a 16-byte chunk is a 16-dim block
            uint32_t a0, a1, a2, a3, c0, c1, c2, c3;
            ldsm_x4(qa + (2 * k2) * 32, a0, a1, a2, a3); ldsm_x4(qa + (2 * k2 + 1) * 32, c0, c1, c2, c3);
#pragma unroll
            for (int sb = 0; sb < NK; sb++) {
                uint32_t r0, r1, r2, r3;
                ldsm_x4(ka + sb * G::kGroupBytes + (k2 >> 2) * 2048 + ko[k2 & 3], r0, r1, r2, r3);
                r0 ^= 0x80808080u; r1 ^= 0x80808080u; r2 ^= 0x80808080u; r3 ^= 0x80808080u;
                auto dq = [](uint32_t x, uint32_t sel) { return FINE ? deq2(x, sel) : deq2_biased(x, sel); };
                mma16816(s[2 * sb], a0, a1, a2, a3, dq(r0, 0x4140u), dq(r0, 0x4342u)); mma16816(s[2 * sb + 1], a0, a1, a2, a3, dq(r2, 0x4140u), dq(r2, 0x4342u));
                mma16816(s2[2 * sb], c0, c1, c2, c3, dq(r1, 0x4140u), dq(r1, 0x4342u)); mma16816(s2[2 * sb + 1], c0, c1, c2, c3, dq(r3, 0x4140u), dq(r3, 0x4342u));
            }
        }
    }
    const float b0 = (K8 && !FINE) ? kI8Bias * qs[0] : 0.0f, b1 = (K8 && !FINE) ? kI8Bias * qs[1] : 0.0f;   // biased codes: the scores were formed against code + 1152
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float x = s[nt][e] + s2[nt][e], y = s[nt][2 + e] + s2[nt][2 + e];
            if (K8) { x = (x - b0) * ks[nt][e]; y = (y - b1) * ks[nt][e]; }
            const int key = key0 + nt * 8 + 2 * t4 + e;   // masked by select: what lies there may be anything
            s[nt][e] = key < lim0 ? x : -INFINITY; s[nt][2 + e] = key < lim1 ? y : -INFINITY;
        }
}

// Online softmax of a tile's scores: pr = 2^shift * exp(s - m), the state and the rescale factors of rows g and g + 8 brought up to date.
template <int NT, int SHIFT>
__device__ __forceinline__ void paged_softmax(const float (&s)[NT][4], ScoreState& st, float (&pr)[NT][4], float& al0, float& al1) {
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) { mx0 = fmaxf(mx0, fmaxf(s[nt][0], s[nt][1])); mx1 = fmaxf(mx1, fmaxf(s[nt][2], s[nt][3])); }
    mx0 *= kLog2e; mx1 *= kLog2e;
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    const float mn0 = fmaxf(st.m0, mx0), mn1 = fmaxf(st.m1, mx1);
    al0 = (mn0 == -INFINITY) ? 1.0f : ex2(st.m0 - mn0); al1 = (mn1 == -INFINITY) ? 1.0f : ex2(st.m1 - mn1);
    const float sub0 = (mn0 == -INFINITY) ? 0.0f : mn0 - SHIFT, sub1 = (mn1 == -INFINITY) ? 0.0f : mn1 - SHIFT;
    st.m0 = mn0; st.m1 = mn1;
    float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        pr[nt][0] = ex2(fmaf(s[nt][0], kLog2e, -sub0)); pr[nt][1] = ex2(fmaf(s[nt][1], kLog2e, -sub0));
        pr[nt][2] = ex2(fmaf(s[nt][2], kLog2e, -sub1)); pr[nt][3] = ex2(fmaf(s[nt][3], kLog2e, -sub1));
        sum0 += pr[nt][0] + pr[nt][1]; sum1 += pr[nt][2] + pr[nt][3];
    }
    st.l0 = st.l0 * al0 + sum0; st.l1 = st.l1 * al1 + sum1;
}

template <int HD, bool K8, bool FINE>
__device__ __forceinline__ void paged_publish(const uint32_t p_sm, float* alpha, const float (&pr)[2 * PGeo<HD, K8, FINE>::kNK][4], const float al0, const float al1, const int lane) {
    using G = PGeo<HD, K8, FINE>; const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int nt = 0; nt < 2 * G::kNK; nt++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float x = pr[nt][2 * h], y = pr[nt][2 * h + 1]; const uint32_t at = p_sm + (g + 8 * h) * G::kPStride + (8 * nt + 2 * t4) * 2, hi = pack_h2(x, y);
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(hi) : "memory");
            if (FINE) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + G::kPTerm), "r"(pack_h2(x - f.x, y - f.y)) : "memory");
            }
        }
    if (t4 == 0) { alpha[g] = al0; alpha[g + 8] = al1; }
}

// Value warp, one tile: O = O * alpha + P V on half vh of the head dims.
template <int HD, bool K8, bool FINE>
__device__ __forceinline__ void paged_values(const uint32_t v_sm, const uint32_t p_sm, const float* alpha, ValueStateT<HD / 16>& st, const int lane, const int vh) {
    using G = PGeo<HD, K8, FINE>; constexpr int NK = G::kNK, NJ = HD / 16;
    const int g = lane >> 2; const float al0 = alpha[g], al1 = alpha[g + 8];
    uint32_t pa[NK][4], pl[NK][4];
#pragma unroll
    for (int sb = 0; sb < NK; sb++) {
        const uint32_t at = p_sm + (lane & 15) * G::kPStride + sb * 32 + (lane >> 4) * 16;
        ldsm_x4(at, pa[sb][0], pa[sb][1], pa[sb][2], pa[sb][3]);
        if (FINE) ldsm_x4(at + G::kPTerm, pl[sb][0], pl[sb][1], pl[sb][2], pl[sb][3]);
    }
    if (__any_sync(0xffffffffu, al0 != 1.0f || al1 != 1.0f)) {
#pragma unroll
        for (int j = 0; j < NJ; j++) { st.o[j][0] *= al0; st.o[j][1] *= al0; st.o[j][2] *= al1; st.o[j][3] *= al1; }
    }
    if (K8 && !FINE) {   // sums of the rounded P: the bias term of the biased codes
        float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
        for (int sb = 0; sb < NK; sb++) {
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&pa[sb][0])), f1 = __half22float2(*reinterpret_cast<const __half2*>(&pa[sb][1]));
            const float2 f2 = __half22float2(*reinterpret_cast<const __half2*>(&pa[sb][2])), f3 = __half22float2(*reinterpret_cast<const __half2*>(&pa[sb][3]));
            a0 += (f0.x + f0.y) + (f2.x + f2.y); a1 += (f1.x + f1.y) + (f3.x + f3.y);
        }
        st.ps0 = st.ps0 * al0 + a0; st.ps1 = st.ps1 * al1 + a1;
    }
    const uint32_t rx = lane & 7, ud = lane >> 4;
    constexpr int kC0 = HD * (K8 ? 1 : 2) / 2 / 16;   // first 16-byte chunk of the second half of a head row
    const uint32_t va = v_sm + (rx + ((lane >> 3) & 1) * 8) * 128 + (uint32_t)(vh * (kC0 >> 3)) * 2048, cb = (uint32_t)vh * (kC0 & 7);   // 128-wide int8 heads: the halves share a column block
    const uint32_t vo[4] = {((cb + 0 + ud) ^ rx) << 4, ((cb + 2 + ud) ^ rx) << 4, ((cb + 4 + ud) ^ rx) << 4, ((cb + 6 + ud) ^ rx) << 4};
    auto mma = [&](float (&c)[4], int sb, uint32_t b0, uint32_t b1) {
        mma16816(c, pa[sb][0], pa[sb][1], pa[sb][2], pa[sb][3], b0, b1);
        if (FINE) mma16816(c, pl[sb][0], pl[sb][1], pl[sb][2], pl[sb][3], b0, b1);
    };
    if (!K8) {
#pragma unroll
        for (int j2 = 0; j2 < NJ / 2; j2++)
#pragma unroll
            for (int sb = 0; sb < NK; sb++) {
                uint32_t b0, b1, b2, b3; ldsm_x4_t(va + sb * G::kGroupBytes + (j2 >> 2) * 2048 + vo[j2 & 3], b0, b1, b2, b3);
                mma(st.o[2 * j2], sb, b0, b1); mma(st.o[2 * j2 + 1], sb, b2, b3);
            }
    } else {
#pragma unroll
        for (int j2 = 0; j2 < NJ / 4; j2++)
#pragma unroll
            for (int sb = 0; sb < NK; sb++) {
                uint32_t r0, r1, r2, r3; ldsm_x4_t(va + sb * G::kGroupBytes + vo[j2], r0, r1, r2, r3);
                r0 ^= 0x80808080u; r1 ^= 0x80808080u; r2 ^= 0x80808080u; r3 ^= 0x80808080u;
                auto dq = [](uint32_t x, uint32_t sel) { return FINE ? deq2(x, sel) : deq2_biased(x, sel); };
                mma(st.o[4 * j2 + 0], sb, dq(r0, 0x4240u), dq(r1, 0x4240u)); mma(st.o[4 * j2 + 1], sb, dq(r0, 0x4341u), dq(r1, 0x4341u));
                mma(st.o[4 * j2 + 2], sb, dq(r2, 0x4240u), dq(r3, 0x4240u)); mma(st.o[4 * j2 + 3], sb, dq(r2, 0x4341u), dq(r3, 0x4341u));
            }
    }
}

struct PagedOut { const float* gate; void* out; int32_t kind; float* fin_ml; };   // fin_ml: joined (m, l) per (segment, row), with weights only

// Final value of row r of a segment, dims d and d + 1: normalised, gated, stored. A row that saw no slot has l = 0 and gets zeros.
template <int HD> __device__ __forceinline__ void paged_emit(const PagedPlan& p, const PagedOut& o, int b, int kvh, int r, int d, float M, float L, float A0, float A1) {
    const int t = r / p.group, head = kvh * p.group + (r - t * p.group);
    const int64_t oi = (((int64_t)b * p.tok_stride + p.tok0 + t) * (p.kv_heads * p.group) + head) * HD + d;
    float y0 = A0 / L, y1 = A1 / L;
    if (o.gate) { const float2 gt = *reinterpret_cast<const float2*>(o.gate + oi); y0 *= sigmoid_fast(gt.x); y1 *= sigmoid_fast(gt.y); }
    if (L == 0.0f) { y0 = 0.0f; y1 = 0.0f; }
    store_act2(o.out, oi, y0, y1, o.kind);
    if (o.fin_ml && d == 0) *reinterpret_cast<float2*>(o.fin_ml + ((int64_t)(b * p.kv_heads + kvh) * 16 + r) * 2) = make_float2(M, L);
}

template <int HD, bool K8, bool FINE>
__global__ void __launch_bounds__(kThreads, 1) paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedPlan p,
                                                                   const int32_t* __restrict__ tables, const __half* __restrict__ q16, const PagedOut o, const __half* __restrict__ ksc, const __half* __restrict__ vsc,
                                                                   float* scores, float* scratch_o, float* scratch_ml, int32_t* counters, int32_t* err) {
    using G = PGeo<HD, K8, FINE>; constexpr int kStages = G::kStages, kTile = G::kTile, NK = G::kNK, NT = 2 * NK;
    if (threadIdx.x == 0) { prefetch_tmap(&tm_k); prefetch_tmap(&tm_v); }
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, ring = w & 3, h = w >> 2, g = lane >> 2, t4 = lane & 3;   // h = 0 score warp, 1 and 2 value warps, 3 producer
    const uint32_t sm_base = smem_u32(smem), bars = sm_base + G::kOffBars + ring * kMaxStages * 8, ebars = bars + kOffEBars;
    const uint32_t stage_off = ((sm_base + G::kOffStages + 1023u) & ~1023u) - sm_base, ring_stage0 = sm_base + stage_off + ring * G::kRingBytes;
    const uint32_t pfull = sm_base + G::kOffBars + kOffPBars + ring * 16, pempty = pfull + kRings * 16;
    const int p_off = G::kOffPair + ring * 2 * G::kPBytes;
    float* sm_ml = reinterpret_cast<float*>(smem + G::kOffMl);
    __shared__ int s_flag;

    if (h == 0 && lane == 0) { for (int s = 0; s < kStages; s++) { mbar_init(bars + s * 8, 1); mbar_init(ebars + s * 8, 3); } for (int s = 0; s < 2; s++) { mbar_init(pfull + s * 8, 1); mbar_init(pempty + s * 8, 2); } }
    fence_mbar_init();
    __syncthreads();
    pdl_wait(); pdl_launch_dependents();   // the set-up above overlapped the previous kernel's tail; nothing it wrote is read before this

    const int kvh_n = p.kv_heads, rows = p.group * p.T, srow = rows <= 8 ? 8 : 16, mask = (1 << p.page_shift) - 1;
    int tile = plan_first_tile(p, blockIdx.x); const int tile_end = plan_first_tile(p, blockIdx.x + 1);
    int b = 0; uint32_t it = 0; bool dead = false;   // it: tiles this ring has consumed so far

    while (tile < tile_end) {
        while (p.tile_start[b + 1] <= tile) b++;
        const int nt = plan_ntiles(p, b), kvh = (tile - p.tile_start[b]) / nt, lt0 = (tile - p.tile_start[b]) - kvh * nt;
        const int seg_first = p.tile_start[b] + kvh * nt, seg_end = seg_first + nt, my_end = min(tile_end, seg_end), n_here = my_end - tile;
        const int kend = p.kend[b], last = max(kend - 1, 0);
        const int32_t* table = tables + (int64_t)p.seq[b] * p.width;
        const int n_mine = n_here > ring ? (n_here - ring + kRings - 1) / kRings : 0;   // this ring's tiles: lt0 + ring, lt0 + ring + 4, ...
        const uint32_t it_seg = it;
        ScoreState ss; ValueStateT<HD / 16> vst; vst.clear();
        const int r0t = g / p.group, r1t = (g + 8) / p.group;
        const int lim0 = g < rows ? kend - p.T + 1 + r0t : 0, lim1 = g + 8 < rows ? kend - p.T + 1 + r1t : 0;   // rows g and g + 8 see slots below these (never, when 0 or less)

        // ---- producer: lane r serves ring r; page numbers are read three tiles ahead
        int32_t pgA[2], pgB[2], pgC[2];
        auto slot_of = [&](int i, int x) { return (lt0 + lane + i * kRings) * kTile + x * 16 * p.groups_per_box; };
        auto load_pages = [&](int i, int32_t (&pg)[2]) {
            pg[0] = __ldcg(table + (min(slot_of(i, 0), last) >> p.page_shift));
            pg[1] = p.groups_per_box < NK ? __ldcg(table + (min(slot_of(i, 1), last) >> p.page_shift)) : 0;
        };
        const int nm = n_here > lane ? (n_here - lane + kRings - 1) / kRings : 0;
        auto produce = [&](int i_from, int i_to) {
            for (int i = i_from; i < min(i_to, nm); i++) {
                const uint32_t cur = it + (uint32_t)i, sx = cur % kStages;
                const uint32_t bar = sm_base + G::kOffBars + lane * kMaxStages * 8 + sx * 8, dst = sm_base + stage_off + lane * G::kRingBytes + sx * G::kStageBytes;
                const int32_t pg[2] = {pgA[0], pgA[1]};
                pgA[0] = pgB[0]; pgA[1] = pgB[1]; pgB[0] = pgC[0]; pgB[1] = pgC[1];
                if (i + 3 < nm) load_pages(i + 3, pgC);
                if (i >= kStages && !dead && !mbar_wait_bounded(bar + kOffEBars, ((cur / kStages) - 1u) & 1u, err)) { dead = true; atomicExch(err, 3); }
                mbar_arrive_expect_tx(bar, (uint32_t)G::kStageBytes);
#pragma unroll
                for (int x = 0; x < NK; x++) {
                    if (x && p.groups_per_box == NK) break;
                    const int grp = (int)((p.layer_row0 + ((int64_t)pg[x] << p.page_shift) + (slot_of(i, x) & mask)) >> 4);
                    tma_load_5d(dst + x * G::kGroupBytes, &tm_k, 0, 0, 0, grp, kvh, bar); tma_load_5d(dst + G::kHalfBytes + x * G::kGroupBytes, &tm_v, 0, 0, 0, grp, kvh, bar);
                }
            }
        };
        if (h == 3 && lane < kRings) {   // every stage is free here
            if (nm > 0) load_pages(0, pgA);
            if (nm > 1) load_pages(1, pgB);
            if (nm > 2) load_pages(2, pgC);
            produce(0, kStages);
        }
        // ---- int8 scales: lane j of the score warp fetches those of the tile's slot j, three tiles ahead, its page number three tiles before that
        auto scale_slot = [&](int i) { return min((lt0 + ring + i * kRings) * kTile + (lane & (kTile - 1)), last); };
        auto load_page1 = [&](int i) { return __ldcg(table + (scale_slot(i) >> p.page_shift)); };
        auto load_scales = [&](int i, int32_t pg, uint32_t& ks, uint32_t& vs) {
            const int64_t at = (((int64_t)pg << p.page_shift) + (scale_slot(i) & mask)) * kvh_n + kvh;   // ksc, vsc: this layer's planes
            ks = __ldcg(reinterpret_cast<const unsigned short*>(ksc) + at); vs = __ldcg(reinterpret_cast<const unsigned short*>(vsc) + at);
        };
        uint32_t kA = 0, kB = 0, kC = 0, vA = 0, vB = 0, vC = 0; int32_t gD = 0, gE = 0, gF = 0;
        if (K8 && h == 0 && n_mine > 0) {   // tiles past the end repeat the last slot: harmless, and the loads need no guards
            const int32_t g0 = load_page1(0), g1 = load_page1(1), g2 = load_page1(2); gD = load_page1(3); gE = load_page1(4); gF = load_page1(5);
            load_scales(0, g0, kA, vA); load_scales(1, g1, kB, vB); load_scales(2, g2, kC, vC);
        }
        // ---- the 16-row query block (rows t * group + j, zero behind the last)
        for (int ch = tid; ch < 16 * (HD / 8); ch += kThreads) {
            const int r = ch / (HD / 8), c16 = ch % (HD / 8); uint4 v = make_uint4(0, 0, 0, 0);
            if (r < rows) { const int t = r / p.group, j = r - t * p.group; v = *reinterpret_cast<const uint4*>(q16 + (((int64_t)b * p.tok_stride + p.tok0 + t) * (kvh_n * p.group) + kvh * p.group + j) * HD + c16 * 8); }
            stage_q_chunk<K8>(smem + r * G::kQStride, c16, v);
        }
        __syncthreads();
        if (K8 && !FINE) {   // row sums of the query block, for the bias of the codes
            for (int r = w; r < 16; r += kWarps) {
                float a = 0.0f;
                for (int c = lane; c < HD / 8; c += 32) {
                    const uint4 v = *reinterpret_cast<const uint4*>(smem + r * G::kQStride + c * 16); const __half2* hp = reinterpret_cast<const __half2*>(&v);
#pragma unroll
                    for (int e = 0; e < 4; e++) { const float2 f = __half22float2(hp[e]); a += f.x + f.y; }
                }
#pragma unroll
                for (int off = 16; off >= 1; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
                if (lane == 0) reinterpret_cast<float*>(smem + G::kOffQsum)[r] = a;
            }
            __syncthreads();
        }
        const float qs[2] = {(K8 && !FINE) ? reinterpret_cast<const float*>(smem + G::kOffQsum)[g] : 0.0f, (K8 && !FINE) ? reinterpret_cast<const float*>(smem + G::kOffQsum)[g + 8] : 0.0f};

        if (h == 3) {
            if (lane < kRings) { produce(kStages, 1 << 30); it += (uint32_t)nm; }   // 'it' of producer lane r counts ring r's tiles
            __syncwarp();
        } else if (h == 0) {
            for (int i = 0; i < n_mine; i++) {
                const uint32_t cur = it_seg + (uint32_t)i, stg = cur % kStages, par = (cur / kStages) & 1u, slot = cur & 1u;
                const int key0 = (lt0 + ring + i * kRings) * kTile;
                const uint32_t k_cur = kA, v_cur = vA; kA = kB; kB = kC; vA = vB; vB = vC;
                if (K8 && i + 3 < n_mine) { const int32_t pg = gD; gD = gE; gE = gF; gF = load_page1(i + 6); load_scales(i + 3, pg, kC, vC); }
                // a wait that runs out is recorded once; afterwards waits are skipped, the control flow and every arrival stay as they are
                if (!dead && !mbar_wait_bounded(bars + stg * 8, par, err)) { dead = true; atomicExch(err, 1); }
                float ks[NT][2], vs[NT][2];
#pragma unroll
                for (int q = 0; q < 4 * NK; q++) {
                    const int src = 8 * (q >> 1) + 2 * t4 + (q & 1);
                    ks[q >> 1][q & 1] = K8 ? __half2float(__ushort_as_half((unsigned short)__shfl_sync(0xffffffffu, k_cur, src))) : 1.0f;
                    vs[q >> 1][q & 1] = K8 ? __half2float(__ushort_as_half((unsigned short)__shfl_sync(0xffffffffu, v_cur, src))) : 1.0f;
                }
                float s[NT][4], pr[NT][4], al0, al1;
                paged_scores<HD, K8, FINE>(sm_base, ring_stage0 + stg * G::kStageBytes, key0, lim0, lim1, ks, qs, lane, s);
                __syncwarp();
                if (lane == 0) mbar_arrive(ebars + stg * 8);   // K of this stage is no longer needed
                paged_softmax<NT, G::kPShift>(s, ss, pr, al0, al1);
                if (scores) {   // [tile of the list][slot][8 or 16 rows]: full 32-byte sectors
                    float* st = scores + ((int64_t)(tile + ring + i * kRings) * kTile + 2 * t4) * srow + g;
#pragma unroll
                    for (int nt8 = 0; nt8 < NT; nt8++)
#pragma unroll
                        for (int e = 0; e < 2; e++) { st[(8 * nt8 + e) * srow] = s[nt8][e]; if (srow == 16) st[(8 * nt8 + e) * 16 + 8] = s[nt8][2 + e]; }
                }
                if (K8) {
#pragma unroll
                    for (int q = 0; q < NT; q++) { pr[q][0] *= vs[q][0]; pr[q][1] *= vs[q][1]; pr[q][2] *= vs[q][0]; pr[q][3] *= vs[q][1]; }
                }
                if (cur >= 2 && !dead && !mbar_wait_bounded(pempty + slot * 8, ((cur >> 1) - 1u) & 1u, err)) { dead = true; atomicExch(err, 4); }
                paged_publish<HD, K8, FINE>(sm_base + p_off + slot * G::kPBytes, reinterpret_cast<float*>(smem + p_off + (slot + 1) * G::kPBytes - 64), pr, al0, al1, lane);
                __syncwarp();
                if (lane == 0) mbar_arrive(pfull + slot * 8);
            }
            ss.l0 += __shfl_xor_sync(0xffffffffu, ss.l0, 1); ss.l0 += __shfl_xor_sync(0xffffffffu, ss.l0, 2);
            ss.l1 += __shfl_xor_sync(0xffffffffu, ss.l1, 1); ss.l1 += __shfl_xor_sync(0xffffffffu, ss.l1, 2);
            if (t4 == 0) { sm_ml[(ring * 16 + g) * 2] = ss.m0; sm_ml[(ring * 16 + g) * 2 + 1] = ss.l0; sm_ml[(ring * 16 + g + 8) * 2] = ss.m1; sm_ml[(ring * 16 + g + 8) * 2 + 1] = ss.l1; }
        } else {
            const int vh = h - 1;
            for (int i = 0; i < n_mine; i++) {
                const uint32_t cur = it_seg + (uint32_t)i, stg = cur % kStages, par = (cur / kStages) & 1u, slot = cur & 1u;
                const uint32_t vt = ring_stage0 + stg * G::kStageBytes + G::kHalfBytes;
                const int key0 = (lt0 + ring + i * kRings) * kTile;
                if (!dead && !mbar_wait_bounded(bars + stg * 8, par, err)) { dead = true; atomicExch(err, 1); }
                if (!K8 && key0 + kTile > kend) {   // the V rows behind the last slot become zeros (0 x NaN is not 0; int8 codes are finite whatever they are)
                    const int nk = max(0, kend - key0);
                    constexpr int kHC = G::kRowBytes / 32;   // 16-byte chunks of half a head row
                    for (int idx = lane; idx < (kTile - nk) * kHC; idx += 32) {
                        const int r = nk + idx / kHC, c = vh * kHC + idx % kHC;
                        *reinterpret_cast<uint4*>(smem + (vt - sm_base) + (r >> 4) * G::kGroupBytes + (c >> 3) * 2048 + (r & 15) * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();   // generic writes to a stage that TMA fills again
                    __syncwarp();
                }
                if (!dead && !mbar_wait_bounded(pfull + slot * 8, (cur >> 1) & 1u, err)) { dead = true; atomicExch(err, 5); }
                paged_values<HD, K8, FINE>(vt, sm_base + p_off + slot * G::kPBytes, reinterpret_cast<const float*>(smem + p_off + (slot + 1) * G::kPBytes - 64), vst, lane, vh);
                __syncwarp();
                if (lane == 0) { mbar_arrive(pempty + slot * 8); mbar_arrive(ebars + stg * 8); }
            }
            if (K8 && !FINE) vst.finish_bias(kI8Bias);
        }
        if (h != 3) it = it_seg + (uint32_t)n_mine;

        // ---- join the four rings (every tile issued has been waited for: no copy is in flight)
        __syncthreads();
        if (h == 1 || h == 2) {
            float* mo = reinterpret_cast<float*>(smem + stage_off + ring * G::kRingBytes);
#pragma unroll
            for (int j = 0; j < HD / 16; j++)
#pragma unroll
                for (int c = 0; c < 2; c++) { const int d = (h - 1) * (HD / 2) + dim_of<K8>(j, c, t4); mo[g * G::kMergeStride + d] = vst.o[j][c]; mo[(g + 8) * G::kMergeStride + d] = vst.o[j][2 + c]; }
        }
        __syncthreads();
        constexpr int kTpr = HD / 2, kRowPar = 384 / kTpr;   // threads per row (two dims each), rows at a time over the twelve ring warps
        const int seg = b * kvh_n + kvh, c_first = plan_cta_of_tile(p, seg_first), n_contrib = plan_cta_of_tile(p, seg_end - 1) - c_first + 1;
        const int d0 = 2 * (tid % kTpr), rsel = h < 3 ? tid / kTpr : rows; const bool whole = n_contrib == 1;
        float* slot_o = scratch_o + (int64_t)(blockIdx.x + seg) * (16 * HD); float* slot_ml = scratch_ml + (int64_t)(blockIdx.x + seg) * 32;   // (CTA, segment) pairs have CTA + segment of their own
        for (int r = rsel; r < rows; r += kRowPar) {
            float M = -INFINITY, L = 0.0f, A0 = 0.0f, A1 = 0.0f;
#pragma unroll
            for (int ww = 0; ww < kRings; ww++) M = fmaxf(M, sm_ml[(ww * 16 + r) * 2]);
#pragma unroll
            for (int ww = 0; ww < kRings; ww++) {
                const float mm = sm_ml[(ww * 16 + r) * 2], wt = (mm == -INFINITY) ? 0.0f : ex2(mm - M);
                const float* src = reinterpret_cast<const float*>(smem + stage_off + ww * G::kRingBytes) + r * G::kMergeStride + d0;
                L += sm_ml[(ww * 16 + r) * 2 + 1] * wt;
                if (wt != 0.0f) { A0 += src[0] * wt; A1 += src[1] * wt; }
            }
            if (whole) paged_emit<HD>(p, o, b, kvh, r, d0, M, L, A0, A1);
            else { *reinterpret_cast<float2*>(slot_o + r * HD + d0) = make_float2(A0, A1); if (d0 == 0) { slot_ml[r * 2] = M; slot_ml[r * 2 + 1] = L; } }
        }
        if (!whole && p.merge_in_kernel) {   // the last of (at most 8) contributors joins everybody's partial rows
            __threadfence();
            __syncthreads();
            if (tid == 0) { const int old = atomicAdd(&counters[seg], 1); s_flag = (old == n_contrib - 1); }
            __syncthreads();
            if (s_flag) {
                __threadfence();
                for (int r = rsel; r < rows; r += kRowPar) {
                    float M = -INFINITY, L = 0.0f, A0 = 0.0f, A1 = 0.0f;
                    for (int c = 0; c < n_contrib; c++) M = fmaxf(M, __ldcg(scratch_ml + (int64_t)(c_first + c + seg) * 32 + r * 2));
#pragma unroll 4
                    for (int c = 0; c < n_contrib; c++) {
                        const int64_t sl = c_first + c + seg; const float mm = __ldcg(scratch_ml + sl * 32 + r * 2), wt = (mm == -INFINITY) ? 0.0f : ex2(mm - M);
                        const float2 oo = __ldcg(reinterpret_cast<const float2*>(scratch_o + sl * (16 * HD) + r * HD + d0));
                        L += __ldcg(scratch_ml + sl * 32 + r * 2 + 1) * wt; A0 += oo.x * wt; A1 += oo.y * wt;
                    }
                    paged_emit<HD>(p, o, b, kvh, r, d0, M, L, A0, A1);
                }
                if (tid == 0) counters[seg] = 0;   // ready for the next call
            }
        }
        fence_proxy_async();   // the merge buffers lie in the stages that the next segment's TMA writes
        __syncthreads();
        tile = my_end;
    }
}

// Joins the partial rows of segments cut between more than 8 CTAs: one CTA per (row, segment), 1024 / HD groups of HD threads folding contributors
// q, q + groups, ... with a maximum of their own, up to twelve of them requested at once, then the groups through shared memory.
template <int HD>
__global__ void __launch_bounds__(1024) paged_combine_kernel(const __grid_constant__ PagedPlan p, const PagedOut o, const float* __restrict__ scratch_o, const float* __restrict__ scratch_ml) {
    constexpr int kQ = 1024 / HD, kU = 48 / kQ;
    __shared__ float s_acc[kQ][HD], s_M[kQ], s_L[kQ];
    const int r = blockIdx.x, seg = blockIdx.y, b = seg / p.kv_heads, kvh = seg - b * p.kv_heads, d = threadIdx.x % HD, q = threadIdx.x / HD;
    const int nt = plan_ntiles(p, b), first = p.tile_start[b] + kvh * nt, c_first = plan_cta_of_tile(p, first), n_c = plan_cta_of_tile(p, first + nt - 1) - c_first + 1;
    pdl_wait(); pdl_launch_dependents();
    if (n_c == 1) return;   // written by its only contributor
    const float* ml = scratch_ml + (int64_t)(c_first + seg) * 32 + r * 2; const float* po = scratch_o + (int64_t)(c_first + seg) * (16 * HD) + r * HD + d;
    float M = -INFINITY, L = 0.0f, A = 0.0f;
    for (int c0 = q; c0 < n_c; c0 += 48) {
        float mm[kU], ll[kU], oo[kU], Mn = M;
#pragma unroll
        for (int u = 0; u < kU; u++) {
            const int c = c0 + kQ * u; const bool ok = c < n_c;
            mm[u] = ok ? __ldcg(ml + c * 32) : -INFINITY; ll[u] = ok ? __ldcg(ml + c * 32 + 1) : 0.0f; oo[u] = ok ? __ldcg(po + (int64_t)c * (16 * HD)) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kU; u++) Mn = fmaxf(Mn, mm[u]);
        const float keep = (M == -INFINITY) ? 0.0f : ex2(M - Mn);
        A *= keep; L *= keep; M = Mn;
#pragma unroll
        for (int u = 0; u < kU; u++) { const float wt = (mm[u] == -INFINITY) ? 0.0f : ex2(mm[u] - Mn); A = fmaf(oo[u], wt, A); L = fmaf(ll[u], wt, L); }
    }
    s_acc[q][d] = A;
    if (d == 0) { s_M[q] = M; s_L[q] = L; }
    __syncthreads();
    if (q || (d & 1)) return;
    M = -INFINITY; L = 0.0f; float A0 = 0.0f, A1 = 0.0f;
#pragma unroll
    for (int u = 0; u < kQ; u++) M = fmaxf(M, s_M[u]);
#pragma unroll
    for (int u = 0; u < kQ; u++) { const float wt = (s_M[u] == -INFINITY) ? 0.0f : ex2(s_M[u] - M); A0 = fmaf(s_acc[u][d], wt, A0); A1 = fmaf(s_acc[u][d + 1], wt, A1); L = fmaf(s_L[u], wt, L); }
    paged_emit<HD>(p, o, b, kvh, r, d, M, L, A0, A1);
}

// weight[kv head][slot] += sum over the rows of 2^(s * log2 e - m + shift) / l: the slot's final probabilities, from the scores the decode kernel
// kept and the joined (m, l). A thread per (slot, KV head) in the order of the tile list: 32 (or 64) contiguous bytes per thread, nothing shared, no atomics.
__global__ void __launch_bounds__(256) paged_weight_kernel(const __grid_constant__ PagedPlan p, const int32_t* __restrict__ tables, const float* __restrict__ scores, const float* __restrict__ fin_ml,
                                                           float* __restrict__ weight /* the layer's plane [page][kv head][slot] */, const int tile_shift, const float shift) {
    pdl_wait(); pdl_launch_dependents();
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; const int tile = (int)(idx >> tile_shift);
    if (tile >= p.tile_start[p.n]) return;
    int lo = 0, hi = p.n - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (p.tile_start[mid] <= tile) lo = mid; else hi = mid - 1; }
    const int b = lo, nt = plan_ntiles(p, b), kvh = (tile - p.tile_start[b]) / nt, slot = ((tile - p.tile_start[b] - kvh * nt) << tile_shift) + (int)(idx & ((1 << tile_shift) - 1));
    if (slot >= p.kend[b]) return;
    const int rows = p.group * p.T, srow = rows <= 8 ? 8 : 16;
    const float4* s4 = reinterpret_cast<const float4*>(scores + idx * srow); const float2* ml = reinterpret_cast<const float2*>(fin_ml) + (int64_t)(b * p.kv_heads + kvh) * 16;
    float sum = 0.0f;
    for (int r4 = 0; r4 < rows; r4 += 4) {
        const float4 v = __ldcg(s4 + (r4 >> 2)); const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (r4 + e >= rows) break;
            const float2 m = __ldcg(ml + r4 + e);
            if (x[e] != -INFINITY) sum += ex2(fmaf(x[e], kLog2e, shift - m.x)) / m.y;   // a masked slot adds nothing (its row may have no maximum at all)
        }
    }
    const int page = __ldcg(tables + (int64_t)p.seq[b] * p.width + (slot >> p.page_shift));
    weight[(((int64_t)page * p.kv_heads + kvh) << p.page_shift) + (slot & ((1 << p.page_shift) - 1))] += sum;
}

// The work split (host only): tiles, ranges and where the partial rows are joined. p.n, p.kv_heads and p.kend are set.
int split_paged_tiles(PagedPlan& p, int tile_keys, int sm_count) {
    int total = 0; bool same = true;
    for (int i = 0; i < p.n; i++) {
        p.tile_start[i] = total; total += p.kv_heads * std::max(1, (p.kend[i] + tile_keys - 1) / tile_keys);   // a sequence without keys has one (masked) tile: its rows are written
        same = same && (i == 0 || total - p.tile_start[i] == p.tile_start[1]);
    }
    for (int i = p.n; i <= KATA_PAGED_MAX_BATCH; i++) p.tile_start[i] = total;
    p.cps = 0; p.n_ctas = std::max(1, std::min(sm_count, total)); p.q_tiles = total / p.n_ctas; p.r_tiles = total % p.n_ctas;
    // equal segments that divide nearly all SMs get CTAs of their own: none then pays for crossing into a second segment (4 to 5 us in the contiguous kernel)
    const int n_seg = p.n * p.kv_heads, nt = plan_ntiles(p, 0), cps = n_seg <= sm_count ? std::min(sm_count / n_seg, nt) : 0;
    if (same && cps >= 1 && (cps == nt || cps * n_seg * 100 >= sm_count * 97)) { p.cps = cps; p.n_ctas = cps * n_seg; }
    int most = 1;
    for (int i = 0; i < p.n; i++) for (int kv = 0; kv < p.kv_heads; kv++) { const int n = plan_ntiles(p, i), f = p.tile_start[i] + kv * n; most = std::max(most, plan_cta_of_tile(p, f + n - 1) - plan_cta_of_tile(p, f) + 1); }
    p.merge_in_kernel = most <= 8;   // few contributors: the last one joins them (no second kernel); many: one SM would pull them all, a grid does it in one round trip
    return most;
}

}  // namespace

int paged_tile_keys(const PagedCtx& c) { return (c.cfg.head_dim == 256 && !c.int8()) ? 16 : 32; }
// (CTA + segment) slots of partial rows
size_t paged_part_floats(const PagedCtx& c) { return (size_t)(c.sm_count + KATA_PAGED_MAX_BATCH * c.cfg.kv_heads) * 16 * c.cfg.head_dim; }
size_t paged_part_ml_floats(const PagedCtx& c) { return (size_t)(c.sm_count + KATA_PAGED_MAX_BATCH * c.cfg.kv_heads) * 32; }

#define KATA_PAGED_KERNELS(X) X(256, false, false) X(256, false, true) X(256, true, false) X(256, true, true) X(128, false, false) X(128, false, true) X(128, true, false) X(128, true, true)

cudaError_t configure_paged_decode(const PagedCtx& c) {   // shared-memory opt-in, per device
    cudaError_t e = cudaSuccess;
#define X(HD, K8, FINE) if (e == cudaSuccess && c.cfg.head_dim == HD && c.int8() == K8) e = cudaFuncSetAttribute(paged_decode_kernel<HD, K8, FINE>, cudaFuncAttributeMaxDynamicSharedMemorySize, PGeo<HD, K8, FINE>::kSmem);
    KATA_PAGED_KERNELS(X)
#undef X
    return e;
}

cudaError_t launch_paged_decode(PagedCtx& c, int layer, int n, const int32_t* seq, const int32_t* n_slots, int T, const __half* q16, const float* gate, void* out, int out_dtype, bool accumulate, cudaStream_t s) {
    const int per_pass = std::max(1, 16 / c.group), tile_keys = paged_tile_keys(c), hd = c.cfg.head_dim; const bool fine = out_dtype == KATA_ACT_F32;
    for (int t0 = 0; t0 < T; t0 += per_pass) {   // each pass is independent: all rows are in the cache, token t of the call sees slots below n_slots - T + 1 + t
        PagedPlan p{}; p.n = n; p.T = std::min(per_pass, T - t0); p.group = c.group; p.kv_heads = c.cfg.kv_heads; p.tok_stride = T; p.tok0 = t0;
        p.page_shift = c.page_shift; p.width = c.width; p.groups_per_box = c.box_groups; p.layer_row0 = (int64_t)layer * c.rows_per_layer;
        for (int i = 0; i < n; i++) { p.seq[i] = seq[i]; p.kend[i] = std::max(0, n_slots[i] - T + t0 + p.T); }
        split_paged_tiles(p, tile_keys, c.sm_count);
        // a pass's limits are kend - p.T + 1 + t: where kend was raised to 0 they are 0 or less, as they should be
        const PagedOut o{gate, out, out_dtype, accumulate ? c.fin_ml : nullptr}; float* scores = accumulate ? c.scores : nullptr;
        if (accumulate && p.tile_start[n] > c.score_tiles) return cudaErrorInvalidValue;   // cannot be: the pool bounds the tiles
        cudaError_t e = cudaErrorInvalidValue;
#define X(HD, K8, FINE) if (hd == HD && c.int8() == K8 && fine == FINE) e = launch_pdl(paged_decode_kernel<HD, K8, FINE>, dim3(p.n_ctas), dim3(kThreads), PGeo<HD, K8, FINE>::kSmem, s, c.tm_k, c.tm_v, p, (const int32_t*)c.d_table, q16, o, \
            (const __half*)c.layer_plane(KATA_PAGED_K_SCALE, layer), (const __half*)c.layer_plane(KATA_PAGED_V_SCALE, layer), scores, c.part_o, c.part_ml, c.counters, c.d_err);
        KATA_PAGED_KERNELS(X)
#undef X
        if (e != cudaSuccess) return e;
        c.launches++;
        if (!p.merge_in_kernel) {
            const dim3 grid(c.group * p.T, n * c.cfg.kv_heads);
            e = hd == 256 ? launch_pdl(paged_combine_kernel<256>, grid, dim3(1024), 0, s, p, o, (const float*)c.part_o, (const float*)c.part_ml) : launch_pdl(paged_combine_kernel<128>, grid, dim3(1024), 0, s, p, o, (const float*)c.part_o, (const float*)c.part_ml);
            if (e != cudaSuccess) return e;
            c.launches++;
        }
        if (accumulate) {
            const int64_t keys = (int64_t)p.tile_start[n] * tile_keys;
            e = launch_pdl(paged_weight_kernel, dim3((unsigned)((keys + 255) / 256)), dim3(256), 0, s, p, (const int32_t*)c.d_table, (const float*)c.scores, (const float*)c.fin_ml, (float*)c.layer_plane(KATA_PAGED_WEIGHT, layer),
                           tile_keys == 16 ? 4 : 5, c.int8() ? (float)PGeo<256, true, false>::kPShift : (float)PGeo<256, false, false>::kPShift);
            if (e != cudaSuccess) return e;
            c.launches++;
        }
    }
    return cudaGetLastError();
}

}  // namespace kata

extern "C" int kata_paged_decode_plan(int32_t n, const int32_t* n_keys, int32_t kv_heads, int32_t tile_keys, int32_t sm_count, int32_t* first_tile, int32_t first_tile_cap, int32_t* max_contrib) {
    using namespace kata;
    if (n < 1 || n > KATA_PAGED_MAX_BATCH || !n_keys || kv_heads < 1 || kv_heads > KATA_PAGED_MAX_KV_HEADS || (tile_keys != 16 && tile_keys != 32) || sm_count < 1 || !first_tile || !max_contrib) return -1;
    PagedPlan p{}; p.n = n; p.kv_heads = kv_heads;
    for (int i = 0; i < n; i++) { if (n_keys[i] < 0 || n_keys[i] > KATA_PAGED_MAX_SLOTS) return -1; p.kend[i] = n_keys[i]; }
    *max_contrib = split_paged_tiles(p, tile_keys, sm_count);
    if (p.n_ctas + 1 > first_tile_cap) return -1;
    for (int cta = 0; cta <= p.n_ctas; cta++) first_tile[cta] = plan_first_tile(p, cta);
    for (int cta = 0; cta < p.n_ctas; cta++) for (int t = first_tile[cta]; t < first_tile[cta + 1]; t++) if (plan_cta_of_tile(p, t) != cta) return -2;   // the two maps disagree
    return p.n_ctas;
}
