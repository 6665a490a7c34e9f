// Attention of the newest tokens over a paged KV cache, split over the cache's length and joined (kata_paged_decode, include/kata_paged.h).
//   o_r = sum_j p_rj v_j / sum_j p_rj, p_rj = exp(q_r . k_j - m_r), j over the slots row r sees; row r = t * group + j of a KV head's 16-row block.
// With weights: w[kv head][j] += sum_r p_rj / l_r, which needs the joined (m, l); the fp32 scores are kept and a second, small kernel forms the sums.
//
// Bound by HBM (4096 bytes of K+V per slot at fp16 with 4 heads of 256, each read once), so the work split is that of the contiguous decode kernel:
// the tiles (16, 32 or 64 slots of one KV head, 16 KiB of K+V) of all (sequence, KV head) segments form one list, cut into one contiguous range per SM, the
// ranges' partial rows joined by the last CTA of a segment (at most 8 of them) or by a combine grid. Inside a CTA four rings of a score warp and two value warps take
// the tiles in turn; producer warps refill the rings' stages with TMA. The three kinds of warps pass from one segment into the next on their own (mbarriers for what they hand over, named barriers
// within a kind): the producers and the score warps work on the next segment while the value warps add the rings up and write the rows. With all of them stopping at a segment's end, 32 int8
// sequences of 300 to 32K slots took 202 us in short loops (182 so; in long ones the clock falls under the power limit: 191 to 216, by the GPU), 256 fp16 sequences of 200 slots 68 us (62). What pages change:
//  - A tile is made of 16-slot groups, and a group never crosses a page (pages are powers of two from 16 slots on). The tensor map is a rank-5 view of
//    the pool, {128-byte column block, 16 rows, column blocks, 16-row groups, KV heads}: the group is a coordinate, so one instruction
//    brings the 16 or 32 slots of a tile wherever their page lies, in the same shared-memory order ([group][column block][16 rows][128 bytes], swizzled) for
//    every page size. Pages of 16 slots under 32-slot tiles take two instructions.
//  - The producer reads the page number of a tile three tiles before it needs it. In the int8 mode a ring has a producer warp
//    of its own, whose lanes fetch the slots' K and V scales as well, three tiles ahead, and leave them in shared memory: the score warp waited when it had the loads (359 us for 32 sequences of 300 to
//    32K slots, 228 with a producer per ring, all else as it was then), and so it did with one warp for the four rings' scales (352 us).
//  - Groups behind the last slot repeat the last page (their table entry may not exist); such slots are masked, and their V rows zeroed in shared
//    memory, so whatever lies there (NaN included) has no part in the result. Nor has the row of a later token in an earlier one's.
// Head layouts: head_dim 256 or 128, up to 16 query heads per KV head; tokens beyond 16 / group run as further passes.
//
// The matrix instructions take the keys (and the head dims of V) as their 16 rows and the query rows as their 8 columns: S^T = K Q^T, O^T = V^T P^T. One token of up to 8 heads
// per KV head then costs half the instructions, softmax and registers of a 16-row block (NR = 1 against NR = 2 column tiles); the query's fragments stay in registers
// for the whole segment. With the query rows as the 16 rows instead, 32 sequences of 300 to 32K int8 slots took 280 us (228 at that time).
//
// Precision: fp16 products, fp32 sums. The exponent carries an offset (kPShift) so that p lies high in fp16's range: it cancels in p / l and keeps
// small p out of the subnormals. p goes into P.V in two fp16 terms (about 22 bits; int8 caches with 16-bit outputs: one term, 2^-11 relative, below bf16's own step: the second
// costs 32 ragged sequences 201 us instead of 191, with two tokens 264 instead of 244, and 18 of 15,000 slots with heads of 128 106 instead of 102), for int8 caches times the slot's V scale in units of
// a power of two above the largest V scale of the tile: O and alpha carry the units from tile to tile, so small values keep as many bits as large ones (with the bare scale, whose products sank into fp16's subnormals, outputs
// were off by 1e-5 at V scales of 1e-3 and by 1 % at 1e-6). What is lost lies below 2^-40 of the row's heaviest p times the tile's largest scale. int8 codes are taken
// without the 1152 bias of the contiguous kernel (whose subtraction costs some ten bits), and a tile's P.V is formed in fresh accumulators and added to O with a rounded fma (the matrix
// unit truncates its sums: over hundreds of tiles that showed as 3e-6 in fp32 outputs).
#include <algorithm>

#include "attn_tile.cuh"
#include "paged_internal.cuh"

namespace kata {
namespace {

using namespace ptx;

constexpr int kRings = 4, kMaxStages = 6;

// The barrier block: per ring and stage 'full' and 'empty', per ring two 'P full' and two 'P empty', then two 'sums full' and two 'sums empty'.
constexpr int kOffEBars = kRings * kMaxStages * 8, kOffPBars = 2 * kOffEBars, kOffSBars = kOffPBars + kRings * 32, kBarBytes = kOffSBars + 128;

template <int HD, bool K8, int NR> struct PGeo {   // NR: column tiles of 8 query rows
    static constexpr int kThreads = (3 * kRings + (K8 ? kRings : 1)) * 32;               // fp16: one producer warp, lane r for ring r (in step: 121 us for 37 sequences of 5,200 slots, 127 with one per ring, 140 with one whose lanes drift apart); int8: one per ring
    static constexpr int kRowBytes = HD * (K8 ? 1 : 2);                                  // bytes of a head row
    static constexpr int kNK = (HD == 256 && !K8) ? 1 : (HD == 128 && K8 && NR == 1) ? 4 : 2, kTile = 16 * kNK;   // 16-slot groups and slots per tile: 16 KiB of K and V; 8 KiB for int8 rows of 128 under two column tiles (shared memory has no room for their P). 18 sequences of 15,000 such rows x 8 heads: 95 us, 106 with 8 KiB tiles
    static constexpr int kGroupBytes = 16 * kRowBytes, kHalfBytes = kNK * kGroupBytes;   // K (or V) of one group, of one tile
    static constexpr int kStageBytes = 2 * kHalfBytes, kStages = kStageBytes == 16384 ? 3 : 6;
    static constexpr int kRingBytes = kStages * kStageBytes;
    static constexpr int kQStride = HD * 2 + 16, kQBytes = NR * 8 * kQStride;                // the query block: fp16 rows, 16 bytes of padding
    static constexpr int kPStride = 32 * kNK + 16, kPTerm = NR * 8 * kPStride, kPBytes = 2 * kPTerm + 64;   // a P slot: two fp16 blocks (heads and remainders), 16 rescale factors
    static constexpr int kPShift = 15;                                                   // p is carried as 2^kPShift * p (int8: times a scale below 1)
    static constexpr int kAcc = HD / 32 * NR * 4, kRedBytes = 2 * kAcc * 128;            // accumulators per value-warp lane; the block in which the rings add them up
    // (m, l) of every ring's rows, of their join, and (int8) what a ring's rows of O are multiplied by when they are joined.
    // NR = 1: a block of its own, and two slots for the rings' (m, l): the score warps go on into the next segment. NR = 2: no room, it lies where the P slots are and the score warps wait.
    static constexpr int kSums = NR == 1 ? 2 : 1;
    static constexpr int kOffBars = kQBytes, kOffMl = kOffBars + kBarBytes, kOffPair = kOffMl + kSums * (512 + (K8 ? 256 : 0)) + 128, kOffRed = kOffPair + (NR == 1 ? kRings * 2 * kPBytes : 0);
    static constexpr int kOffScale = NR == 1 ? kOffRed + kRedBytes : kOffPair + (kRings * 2 * kPBytes > kRedBytes ? kRings * 2 * kPBytes : kRedBytes), kOffStages = kOffScale + (K8 ? kRings * kStages * kTile * 4 : 0);   // scales: [ring][stage][slot] K and V packed
    static constexpr int kSmem = kOffStages + 1024 + kRings * kRingBytes;
    static_assert(kSmem <= 232448, "shared memory");
};
constexpr int kMaxCtas = 192;
struct PagedPlan {
    int32_t two_terms;                                              // P in two fp16 terms (fp32 outputs; always where it is free)
    int32_t n, T, group, kv_heads, n_ctas;
    int32_t tok_stride, tok0, page_shift, width, groups_per_box, merge_in_kernel;
    int64_t layer_row0;
    int32_t cut[kMaxCtas + 1];                     // CTA c has the tiles [cut[c], cut[c + 1])
    int32_t seq[KATA_PAGED_MAX_BATCH];
    int32_t kend[KATA_PAGED_MAX_BATCH];            // slots the last token of this pass sees (may be 0)
    int32_t tile_start[KATA_PAGED_MAX_BATCH + 1];  // first tile of a sequence; its tiles are those of KV head 0, of head 1, ...
};
static_assert(sizeof(PagedPlan) + 2 * sizeof(CUtensorMap) + 128 <= 32764, "kernel parameters");

__host__ __device__ __forceinline__ int plan_ntiles(const PagedPlan& p, int b) { return (p.tile_start[b + 1] - p.tile_start[b]) / p.kv_heads; }
// The first and the last CTA of a segment, from CTA c that has some of it.
__host__ __device__ __forceinline__ int plan_first_cta(const PagedPlan& p, int c, int seg_first) { while (p.cut[c] > seg_first) c--; return c; }
__host__ __device__ __forceinline__ int plan_last_cta(const PagedPlan& p, int c, int seg_end) { while (p.cut[c + 1] < seg_end) c++; return c; }
__host__ __device__ __forceinline__ int plan_cta_of(const PagedPlan& p, int tile) {   // the CTA that has a tile
    int lo = 0, hi = p.n_ctas - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (p.cut[mid] <= tile) lo = mid; else hi = mid - 1; }
    return lo;
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const void* tmap, int x, int r, int c, int g, int h, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(r), "r"(c), "r"(g), "r"(h), "r"(bar) : "memory");
}

__device__ __forceinline__ void stsm_x4_t(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
__device__ __forceinline__ void stsm_x2_t(uint32_t addr, uint32_t r0, uint32_t r1) {
    asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1,%2};" ::"r"(addr), "r"(r0), "r"(r1) : "memory");
}

// Fragments (m16n8k16, g = lane / 4, t4 = lane % 4). S^T: elements 0, 1 = slot g, query rows 2 * t4 and the next; elements 2, 3 = slot g + 8. O^T: the same with head dims for slots.
// int8 codes lie four dims (K) or two dims of two slots (V) to a register: their dims are taken in the order 4*t4 + {0, 1}, 4*t4 + {2, 3} (K: the staged
// query columns are permuted alike) and 2*g, 2*g + 1 (V).

// The query's fragments of k-steps kk, kk + 1 for column tile nr
__device__ __forceinline__ void q_frags(const uint32_t q_sm, const int stride, const int nr, const int kk, const int lane, uint32_t (&f0)[2], uint32_t (&f1)[2]) {
    ldsm_x4(q_sm + (nr * 8 + (lane & 7)) * stride + (2 * kk + (lane >> 3)) * 16, f0[0], f0[1], f1[0], f1[1]);
}

// Score warp, one tile: s[sb][nr] = the fragment of 16-slot group sb and column tile nr, scaled (int8). qf: the query's fragments (NR = 1).
template <int HD, bool K8, int NR>
__device__ __forceinline__ void paged_scores(const uint32_t q_sm, const uint32_t k_sm, const uint32_t (&qf)[HD / 16][2], const float (&ks)[PGeo<HD, K8, NR>::kNK][2], const int lane, float (&s)[PGeo<HD, K8, NR>::kNK][NR][4]) {
    using G = PGeo<HD, K8, NR>; constexpr int NK = G::kNK;
    const uint32_t rx = lane & 7, hi = lane >> 4, ka = k_sm + (rx + ((lane >> 3) & 1) * 8) * 128;   // lanes 0-15: slots 0-15 at one chunk, lanes 16-31: at the next
    const uint32_t ko[4] = {((0 + hi) ^ rx) << 4, ((2 + hi) ^ rx) << 4, ((4 + hi) ^ rx) << 4, ((6 + hi) ^ rx) << 4};
    float s2[NK][NR][4];   // a second accumulator chain
#pragma unroll
    for (int sb = 0; sb < NK; sb++)
#pragma unroll
        for (int nr = 0; nr < NR; nr++)
#pragma unroll
            for (int e = 0; e < 4; e++) { s[sb][nr][e] = 0.0f; s2[sb][nr][e] = 0.0f; }
#pragma unroll
    for (int kk = 0; kk < HD / 16; kk += 2) {   // two k-steps of 16 dims
        uint32_t b[2][NR][2];
        if (NR == 1) { b[0][0][0] = qf[kk][0]; b[0][0][1] = qf[kk][1]; b[1][0][0] = qf[kk + 1][0]; b[1][0][1] = qf[kk + 1][1]; }
        else {
#pragma unroll
            for (int nr = 0; nr < NR; nr++) q_frags(q_sm, G::kQStride, nr, kk, lane, b[0][nr], b[1][nr]);
        }
#pragma unroll
        for (int sb = 0; sb < NK; sb++) {
            const uint32_t kb = ka + sb * G::kGroupBytes;
            uint32_t a[2][4];
            if (!K8) {   // a k-step is two 16-byte chunks
                ldsm_x4(kb + (kk >> 2) * 2048 + ko[kk & 3], a[0][0], a[0][1], a[0][2], a[0][3]); ldsm_x4(kb + (kk >> 2) * 2048 + ko[(kk & 3) + 1], a[1][0], a[1][1], a[1][2], a[1][3]);
            } else {     // a k-step is one chunk of 16 codes
                uint32_t r[4]; ldsm_x4(kb + (kk >> 3) * 2048 + ko[(kk >> 1) & 3], r[0], r[1], r[2], r[3]);
#pragma unroll
                for (int x = 0; x < 4; x++) { r[x] ^= 0x80808080u; a[x >> 1][x & 1] = deq2(r[x], 0x4140u); a[x >> 1][2 + (x & 1)] = deq2(r[x], 0x4342u); }
            }
#pragma unroll
            for (int nr = 0; nr < NR; nr++) { mma16816(s[sb][nr], a[0][0], a[0][1], a[0][2], a[0][3], b[0][nr][0], b[0][nr][1]); mma16816(s2[sb][nr], a[1][0], a[1][1], a[1][2], a[1][3], b[1][nr][0], b[1][nr][1]); }
        }
    }
#pragma unroll
    for (int sb = 0; sb < NK; sb++)
#pragma unroll
        for (int nr = 0; nr < NR; nr++)
#pragma unroll
            for (int e = 0; e < 4; e++) { s[sb][nr][e] += s2[sb][nr][e]; if (K8) s[sb][nr][e] *= ks[sb][e >> 1]; }
}

// Online softmax state of query rows nr * 8 + 2 * t4 + {0, 1}: maximum (log2 units) and this lane's share of the sum
template <int NR> struct RowsState { float m[NR][2], l[NR][2]; };

// pr = 2^SHIFT * 2^(s - m) in place of s; the state and the rescale factors brought up to date. LOG2: s is in log2 units already, so that no score passes the maximum (s - (m - SHIFT) may round up to 16, where P's
// scale below 1 keeps it within fp16). Else the product with log2 e is fused with the subtraction; above kRoundedMax it and the rounded maximum can be whole units apart, P would leave fp16's range, and it is rounded too.
constexpr float kRoundedMax = 0x1p22f;
template <int NK, int NR, int SHIFT, bool LOG2>
__device__ __forceinline__ void paged_softmax(float (&s)[NK][NR][4], RowsState<NR>& st, float (&al)[NR][2]) {
#pragma unroll
    for (int nr = 0; nr < NR; nr++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float mx = -INFINITY;
#pragma unroll
            for (int sb = 0; sb < NK; sb++) mx = fmaxf(mx, fmaxf(s[sb][nr][e], s[sb][nr][2 + e]));
            if (!LOG2) mx *= kLog2e;
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4)); mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8)); mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = fmaxf(st.m[nr][e], mx), sub = (mn == -INFINITY) ? 0.0f : mn - SHIFT;
            al[nr][e] = (mn == -INFINITY) ? 1.0f : ex2(st.m[nr][e] - mn); st.m[nr][e] = mn;
            float sum = 0.0f, scale = kLog2e, add = -sub;
            if (!LOG2 && fabsf(mn) > kRoundedMax && fabsf(mn) < INFINITY) {
#pragma unroll
                for (int sb = 0; sb < NK; sb++) { s[sb][nr][e] = __fmul_rn(s[sb][nr][e], kLog2e) - mn; s[sb][nr][2 + e] = __fmul_rn(s[sb][nr][2 + e], kLog2e) - mn; }
                scale = 1.0f; add = SHIFT;
            }
#pragma unroll
            for (int sb = 0; sb < NK; sb++) {
                s[sb][nr][e] = ex2(LOG2 ? s[sb][nr][e] - sub : fmaf(s[sb][nr][e], scale, add)); s[sb][nr][2 + e] = ex2(LOG2 ? s[sb][nr][2 + e] - sub : fmaf(s[sb][nr][2 + e], scale, add));
                sum += s[sb][nr][e] + s[sb][nr][2 + e];
            }
            st.l[nr][e] = st.l[nr][e] * al[nr][e] + sum;
        }
}

// P goes to shared memory as [query row][slot] fp16, heads and (two terms) remainders; the rescale factors behind it.
template <int HD, bool K8, int NR>
__device__ __forceinline__ void paged_publish(const uint32_t p_sm, float* alpha, const float (&pr)[PGeo<HD, K8, NR>::kNK][NR][4], const float (&al)[NR][2], const int two_terms, const int lane) {
    using G = PGeo<HD, K8, NR>; constexpr int NK = G::kNK;
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
        uint32_t hi[2 * NK], lo[2 * NK];   // 8-slot blocks
#pragma unroll
        for (int x = 0; x < 2 * NK; x++) {
            const float u = pr[x >> 1][nr][2 * (x & 1)], v = pr[x >> 1][nr][2 * (x & 1) + 1];
            hi[x] = pack_h2(u, v);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[x]));
            lo[x] = pack_h2(u - f.x, v - f.y);
        }
        const uint32_t at = p_sm + (nr * 8 + (lane & 7)) * G::kPStride + ((lane >> 3) & (NK == 1 ? 1 : 3)) * 16;
        if constexpr (NK > 1) {
#pragma unroll
            for (int x = 0; x < 2 * NK; x += 4) { stsm_x4_t(at + x * 16, hi[x], hi[x + 1], hi[x + 2], hi[x + 3]); if (two_terms) stsm_x4_t(at + x * 16 + G::kPTerm, lo[x], lo[x + 1], lo[x + 2], lo[x + 3]); }
        } else { stsm_x2_t(at, hi[0], hi[1]); if (two_terms) stsm_x2_t(at + G::kPTerm, lo[0], lo[1]); }
        if (lane < 4) *reinterpret_cast<float2*>(alpha + nr * 8 + 2 * lane) = make_float2(al[nr][0], al[nr][1]);
    }
}

// Value warp, one tile: O^T = O^T * alpha + V^T P^T on half vh of the head dims (HD / 32 tiles of 16 dims).
template <int HD, int NR> struct ValueAcc {
    float o[HD / 32][NR][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < HD / 32; j++)
#pragma unroll
            for (int nr = 0; nr < NR; nr++) { o[j][nr][0] = o[j][nr][1] = o[j][nr][2] = o[j][nr][3] = 0.0f; }
    }
};
template <int HD, bool K8, int NR, bool TWO>
__device__ __forceinline__ void paged_values(const uint32_t v_sm, const uint32_t p_sm, const float* alpha, ValueAcc<HD, NR>& st, const int lane, const int vh) {
    using G = PGeo<HD, K8, NR>; constexpr int NK = G::kNK;
    float2 al[NR]; uint32_t ph[NR][2 * NK], pl[NR][2 * NK];
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
        al[nr] = *reinterpret_cast<const float2*>(alpha + nr * 8 + 2 * (lane & 3));
        const uint32_t at = p_sm + (nr * 8 + (lane & 7)) * G::kPStride + ((lane >> 3) & (NK == 1 ? 1 : 3)) * 16;
        auto load = [&](uint32_t a, uint32_t (&x)[2 * NK]) {
            if constexpr (NK > 1) {
#pragma unroll
                for (int y = 0; y < 2 * NK; y += 4) ldsm_x4(a + y * 16, x[y], x[y + 1], x[y + 2], x[y + 3]);
            }
            else asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(a));
        };
        load(at, ph[nr]);
        if (TWO) load(at + G::kPTerm, pl[nr]);
    }
    const uint32_t rx = lane & 7, q1 = (lane >> 3) & 1, q2 = lane >> 4;
    constexpr int kC0 = HD * (K8 ? 1 : 2) / 2 / 16;   // first 16-byte chunk of the second half of a head row
    const uint32_t cb = (uint32_t)vh * (kC0 & 7);     // 128-wide int8 heads: the halves share a column block
    auto step = [&](int j, int sb, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, float (&c)[NR][4]) {
#pragma unroll
        for (int nr = 0; nr < NR; nr++) { mma16816(c[nr], a0, a1, a2, a3, ph[nr][2 * sb], ph[nr][2 * sb + 1]); if (TWO) mma16816(c[nr], a0, a1, a2, a3, pl[nr][2 * sb], pl[nr][2 * sb + 1]); }
    };
    auto add = [&](int j, const float (&c)[NR][4]) {
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
            st.o[j][nr][0] = fmaf(st.o[j][nr][0], al[nr].x, c[nr][0]); st.o[j][nr][1] = fmaf(st.o[j][nr][1], al[nr].y, c[nr][1]);
            st.o[j][nr][2] = fmaf(st.o[j][nr][2], al[nr].x, c[nr][2]); st.o[j][nr][3] = fmaf(st.o[j][nr][3], al[nr].y, c[nr][3]);
        }
    };
    if (!K8) {   // a tile of 16 dims is two chunks: lanes 0-7 slots 0-7 at the first, 8-15 at the second, 16-31 slots 8-15
        const uint32_t va = v_sm + (rx + q2 * 8) * 128 + (uint32_t)(vh * (kC0 >> 3)) * 2048;
        const uint32_t vo[4] = {((0 + q1) ^ rx) << 4, ((2 + q1) ^ rx) << 4, ((4 + q1) ^ rx) << 4, ((6 + q1) ^ rx) << 4};
#pragma unroll
        for (int j = 0; j < HD / 32; j++) {
            float c[NR][4] = {};
#pragma unroll
            for (int sb = 0; sb < NK; sb++) {
                uint32_t a0, a1, a2, a3; ldsm_x4_t(va + sb * G::kGroupBytes + (j >> 2) * 2048 + vo[j & 3], a0, a1, a2, a3);
                step(j, sb, a0, a1, a2, a3, c);
            }
            add(j, c);
        }
    } else {     // a tile of 16 dims is one chunk: lanes 0-15 slots 0-15 at one chunk, lanes 16-31 at the next
        const uint32_t va = v_sm + (rx + q1 * 8) * 128 + (uint32_t)(vh * (kC0 >> 3)) * 2048;
        const uint32_t vo[4] = {((cb + 0 + q2) ^ rx) << 4, ((cb + 2 + q2) ^ rx) << 4, ((cb + 4 + q2) ^ rx) << 4, ((cb + 6 + q2) ^ rx) << 4};
#pragma unroll
        for (int j = 0; j < HD / 32; j += 2) {
            float c0[NR][4] = {}, c1[NR][4] = {};
#pragma unroll
            for (int sb = 0; sb < NK; sb++) {
                uint32_t r0, r1, r2, r3; ldsm_x4_t(va + sb * G::kGroupBytes + vo[j >> 1], r0, r1, r2, r3);   // r0, r1: slots 0-7, 8-15 of one chunk; r2, r3: of the next
                r0 ^= 0x80808080u; r1 ^= 0x80808080u; r2 ^= 0x80808080u; r3 ^= 0x80808080u;
                step(j, sb, deq2(r0, 0x4240u), deq2(r0, 0x4341u), deq2(r1, 0x4240u), deq2(r1, 0x4341u), c0);
                step(j + 1, sb, deq2(r2, 0x4240u), deq2(r2, 0x4341u), deq2(r3, 0x4240u), deq2(r3, 0x4341u), c1);
            }
            add(j, c0); add(j + 1, c1);
        }
    }
}

// Value warp, the last tiles of an fp16 segment, half vh of the head dims: slots [0, part) are seen by every token of the pass, [part, nk) by some, the others by none. The rows that no token sees become zeros
// (0 x NaN is not 0; int8 codes are finite whatever they are). In those that some see, infinities and NaN become zeros, and what comes of them (the two terms of P make NaN of either) goes into the
// rows of O that see them: bit 16 * y + x of the result says that dim 8 * x + g of column 8 * (y >> 1) + 2 * t4 + (y & 1) is NaN. all_see: as in the kernel, less the tile's first slot. The caller
// puts them in once it is through with its tiles: in the loop the registers are missing (one sequence of 32K slots 30.9 us instead of 29.6).
template <int HD, int NR>
__device__ __forceinline__ uint64_t clean_v_rows(uint8_t* v, int part, int nk, int all_see, int group, int lane, int vh) {
    using G = PGeo<HD, false, NR>; constexpr int kHC = HD / 16;   // 16-byte chunks of half a head row
    auto chunk = [&](int r, int c) { c += vh * kHC; return v + (r >> 4) * G::kGroupBytes + (c >> 3) * 2048 + (r & 15) * 128 + (((c & 7) ^ (r & 7)) << 4); };
    auto odd = [](uint32_t h) { return (h & 0x7c00u) == 0x7c00u; };
#pragma unroll 1
    for (int i = lane; i < (G::kTile - nk) * kHC; i += 32) *reinterpret_cast<uint4*>(chunk(nk + i / kHC, i % kHC)) = make_uint4(0, 0, 0, 0);
    bool any = false;
    uint64_t bad = 0;
#pragma unroll 1
    for (int i = lane; i < (nk - part) * kHC; i += 32) {
        const uint4 x = *reinterpret_cast<const uint4*>(chunk(part + i / kHC, i % kHC));
        any = any || odd(x.x) || odd(x.x >> 16) || odd(x.y) || odd(x.y >> 16) || odd(x.z) || odd(x.z >> 16) || odd(x.w) || odd(x.w >> 16);
    }
    if (__any_sync(0xffffffffu, any)) {
#pragma unroll 1
        for (int r = part; r < nk; r++) {
            uint64_t dims = 0;
#pragma unroll 1
            for (int x = 0; x < kHC; x++) dims |= (uint64_t)odd(*reinterpret_cast<const unsigned short*>(chunk(r, x) + 2 * (lane >> 2))) << x;
#pragma unroll 1
            for (int y = 0; y < 2 * NR; y++) if (r < all_see + ((y >> 1) * 8 + 2 * (lane & 3) + (y & 1)) / group) bad |= dims << (16 * y);   // token t sees slots below all_see + t
        }
        __syncwarp();
#pragma unroll 1
        for (int i = lane; i < (nk - part) * kHC * 8; i += 32) {
            unsigned short* h = reinterpret_cast<unsigned short*>(chunk(part + i / (kHC * 8), i / 8 % kHC)) + i % 8;
            if (odd(*h)) *h = 0;
        }
    }
    fence_proxy_async();   // generic writes to a stage that TMA fills again
    __syncwarp();
    return bad;
}

struct PagedOut { const float* gate; void* out; int32_t kind; float* fin_ml; };   // fin_ml: joined (m, 1 / l) per (segment, row), with weights only

// Final value of row r of a segment, dims d and d + 1: normalised, gated, stored. A row that saw no slot has L = 0 and gets zeros.
template <int HD> __device__ __forceinline__ int64_t paged_out_at(const PagedPlan& p, int b, int kvh, int r, int d) {
    const int t = r / p.group;
    return (((int64_t)b * p.tok_stride + p.tok0 + t) * (p.kv_heads * p.group) + kvh * p.group + r - t * p.group) * HD + d;
}
__device__ __forceinline__ float2 paged_gate(const PagedOut& o, int64_t at) { return o.gate ? __ldcg(reinterpret_cast<const float2*>(o.gate + at)) : make_float2(0.0f, 0.0f); }
__device__ __forceinline__ void paged_emit(const PagedPlan& p, const PagedOut& o, int b, int kvh, int r, int d, int64_t at, float2 gate, float M, float L, float A0, float A1) {
    const float inv = L == 0.0f ? 0.0f : 1.0f / L; float2 y = make_float2(L == 0.0f ? 0.0f : A0 * inv, L == 0.0f ? 0.0f : A1 * inv);
    if (o.gate) { y.x *= sigmoid_fast(gate.x); y.y *= sigmoid_fast(gate.y); }
    store_act2(o.out, at, y.x, y.y, o.kind);
    if (o.fin_ml && d == 0) *reinterpret_cast<float2*>(o.fin_ml + ((int64_t)(b * p.kv_heads + kvh) * 16 + r) * 2) = make_float2(M, 1.0f / L);   // for the weights
}

template <int HD, bool K8, int NR>   // NR: column tiles of 8 query rows
__global__ void __launch_bounds__(PGeo<HD, K8, NR>::kThreads, 1) paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedPlan p,
                                                                   const int32_t* __restrict__ tables, const __half* __restrict__ q16, const PagedOut o, const __half* __restrict__ ksc, const __half* __restrict__ vsc,
                                                                   float* scores, float* scratch_o, float* scratch_ml, int32_t* counters, int32_t* err) {
    using G = PGeo<HD, K8, NR>; constexpr int kStages = G::kStages, kTile = G::kTile, NK = G::kNK;
    if (threadIdx.x == 0) { prefetch_tmap(&tm_k); prefetch_tmap(&tm_v); }
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, h = w >> 2, ring = (h == 3 && !K8) ? lane & 3 : w & 3, g = lane >> 2, t4 = lane & 3;   // h = 0 score warp, 1 and 2 value warps, 3 producer
    const bool issues = h == 3 && (K8 ? lane == 0 : lane < kRings);
    const uint32_t sm_base = smem_u32(smem), bars = sm_base + G::kOffBars + ring * kMaxStages * 8, ebars = bars + kOffEBars;
    const uint32_t stage_off = ((sm_base + G::kOffStages + 1023u) & ~1023u) - sm_base, ring_stage0 = sm_base + stage_off + ring * G::kRingBytes;
    const uint32_t pfull = sm_base + G::kOffBars + kOffPBars + ring * 16, pempty = pfull + kRings * 16;
    const int p_off = G::kOffPair + ring * 2 * G::kPBytes;
    float* sm_ml = reinterpret_cast<float*>(smem + G::kOffMl); float* joined_ml = sm_ml + G::kSums * kRings * 32; float* red = reinterpret_cast<float*>(smem + G::kOffRed);
    __shared__ int s_flag;
    const uint32_t sfull = sm_base + G::kOffBars + kOffSBars, sempty = sfull + 16;
    auto score_sync = []() { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    auto value_sync = []() { asm volatile("bar.sync 2, 256;" ::: "memory"); };

    if (h == 0 && lane == 0) { for (int s = 0; s < kStages; s++) { mbar_init(bars + s * 8, 1); mbar_init(ebars + s * 8, 3); } for (int s = 0; s < 2; s++) { mbar_init(pfull + s * 8, 1); mbar_init(pempty + s * 8, 2); } }
    if (tid == 0) { for (int s = 0; s < G::kSums; s++) { mbar_init(sfull + s * 8, kRings); mbar_init(sempty + s * 8, 2 * kRings); } }
    fence_mbar_init();
    __syncthreads();
    pdl_wait(); pdl_launch_dependents();   // the set-up above overlapped the previous kernel's tail; nothing it wrote is read before this

    const int kvh_n = p.kv_heads, rows = p.group * p.T, srow = NR * 8, mask = (1 << p.page_shift) - 1;
    int tile = p.cut[blockIdx.x]; const int tile_end = p.cut[blockIdx.x + 1];
    int b = 0; uint32_t it = 0, n_segs = 0; bool dead = false;   // it: tiles this ring has worked on so far; n_segs: segments
    // The three kinds of warps go from segment to segment on their own; barriers in shared memory hold them together.

    if (h == 3) {
        if (tile >= tile_end) return;
        // ---- producer: brings in the ring's tiles, refilling a stage as soon as its three warps have released it; page numbers are read three tiles
        // ahead. int8: lane j also fetches the K and V scale of slot j, three tiles ahead (under load a request takes as long as all that is in flight before it), the page number of
        // that three tiles earlier still, and stores it before the tile's copy is issued. Unrolled by three so that every load has registers of its own. What the first three tiles of the next
        // segment need is requested during this one (148 int8 sequences of 3,600 slots, four segments per CTA: 203 us without).
        constexpr int SL = K8 ? kTile / 32 : 1;   // scales per lane: slots lane, lane + 32
        struct Seg { int kvh, lt0, n_here, n_mine, last; const int32_t* table; };
        auto segment = [&](int first) {
            while (p.tile_start[b + 1] <= first) b++;
            const int nt = plan_ntiles(p, b), kvh = (first - p.tile_start[b]) / nt, lt0 = first - p.tile_start[b] - kvh * nt, n_here = min(tile_end - first, nt - lt0);
            return Seg{kvh, lt0, n_here, n_here > ring ? (n_here - ring + kRings - 1) / kRings : 0, max(p.kend[b] - 1, 0), tables + (int64_t)p.seq[b] * p.width};
        };
        auto first_slot = [&](const Seg& g, int i) { return (g.lt0 + ring + i * kRings) * kTile; };
        auto load_pages = [&](const Seg& g, int i, int32_t (&x)[NK]) {   // of every box
#pragma unroll
            for (int y = 0; y < NK; y++) if (!(y & (p.groups_per_box - 1))) x[y] = __ldcg(g.table + (min(first_slot(g, i) + 16 * y, g.last) >> p.page_shift));
        };
        auto scale_slot = [&](const Seg& g, int i, int x) { return min(first_slot(g, i) + 32 * x + lane, g.last); };   // slots behind the last repeat it: finite scales, and probabilities 0
        auto scale_pages = [&](const Seg& g, int i, int32_t (&page)[SL]) {
#pragma unroll
            for (int x = 0; x < SL; x++) page[x] = __ldcg(g.table + (scale_slot(g, i, x) >> p.page_shift));
        };
        auto load_scales = [&](const Seg& g, int i, const int32_t (&page)[SL], unsigned short (&sc)[SL][2]) {
#pragma unroll
            for (int x = 0; x < SL; x++) {
                const int64_t at = (((int64_t)page[x] << p.page_shift) + (scale_slot(g, i, x) & mask)) * kvh_n + g.kvh;   // ksc, vsc: this layer's planes
                sc[x][0] = __ldcg(reinterpret_cast<const unsigned short*>(ksc) + at); sc[x][1] = __ldcg(reinterpret_cast<const unsigned short*>(vsc) + at);
            }
        };
        uint32_t issued = 0;
        Seg sg = segment(tile), next = sg; int32_t pg[3][NK], npg[3][NK], spg[3][SL], nspg[3][SL]; unsigned short sc8[3][SL][2], nsc8[3][SL][2];
        if (issues) { load_pages(sg, 0, pg[0]); load_pages(sg, 1, pg[1]); load_pages(sg, 2, pg[2]); }
        if (K8) {
#pragma unroll
            for (int j = 0; j < 3; j++) scale_pages(sg, j, spg[j]);
#pragma unroll
            for (int j = 0; j < 3; j++) { load_scales(sg, j, spg[j], sc8[j]); scale_pages(sg, j + 3, spg[j]); }
        }
        while (true) {
            tile += sg.n_here;
            const bool more = tile < tile_end;
            if (more) {
                next = segment(tile);
                if (issues) { load_pages(next, 0, npg[0]); load_pages(next, 1, npg[1]); load_pages(next, 2, npg[2]); }
                if (K8) { scale_pages(next, 0, nspg[0]); scale_pages(next, 1, nspg[1]); scale_pages(next, 2, nspg[2]); }
            }
            const int n_steps = K8 ? sg.n_mine : (sg.n_here + kRings - 1) / kRings;   // the same for all lanes: they stay in step
            auto next_scales = [&]() {
#pragma unroll
                for (int j = 0; j < 3; j++) { load_scales(next, j, nspg[j], nsc8[j]); scale_pages(next, j + 3, nspg[j]); }
            };
            if (K8 && more && n_steps <= 3) next_scales();
            for (int i0 = 0; i0 < n_steps; i0 += 3) {
                if (K8 && more && i0 == 3) next_scales();
#pragma unroll
                for (int j = 0; j < 3; j++) {
                    const int i = i0 + j;
                    if (i >= n_steps) break;
                    bool has = issues && i < sg.n_mine;
                    const uint32_t cur = it + (uint32_t)i, sx = cur % kStages, bar = bars + sx * 8, dst = ring_stage0 + sx * G::kStageBytes;
                    if (has && !dead && !mbar_wait_bounded(ebars + sx * 8, ((cur / kStages) + 1u) & 1u, err)) { dead = true; atomicExch(err, 3); }   // the first time round the wait is for the phase before the first: over at once
                    has = has && !dead;   // after a wait that ran out no further copy is asked for
                    __syncwarp();
                    if (K8) {
#pragma unroll
                        for (int x = 0; x < SL; x++) reinterpret_cast<uint32_t*>(smem + G::kOffScale)[(ring * kStages + sx) * kTile + 32 * x + lane] = (uint32_t)sc8[j][x][0] | (uint32_t)sc8[j][x][1] << 16;
                        __syncwarp();   // the arrival below publishes them
                    }
                    if (has) {
                        mbar_arrive_expect_tx(bar, (uint32_t)G::kStageBytes); issued = cur + 1;
#pragma unroll
                        for (int x = 0; x < NK; x++) {
                            if (x & (p.groups_per_box - 1)) continue;
                            const int grp = (int)((p.layer_row0 + ((int64_t)pg[j][x] << p.page_shift) + ((first_slot(sg, i) + 16 * x) & mask)) >> 4);
                            tma_load_5d(dst + x * G::kGroupBytes, &tm_k, 0, 0, 0, grp, sg.kvh, bar); tma_load_5d(dst + G::kHalfBytes + x * G::kGroupBytes, &tm_v, 0, 0, 0, grp, sg.kvh, bar);
                        }
                        load_pages(sg, i + 3, pg[j]);   // behind the ring's last tile: the last page again
                    }
                    if (K8) { load_scales(sg, i + 3, spg[j], sc8[j]); scale_pages(sg, i + 6, spg[j]); }
                }
            }
            __syncwarp();
            if (!more) break;
            it += (uint32_t)sg.n_mine; sg = next;
#pragma unroll
            for (int j = 0; j < 3; j++) {
#pragma unroll
                for (int x = 0; x < NK; x++) pg[j][x] = npg[j][x];
#pragma unroll
                for (int x = 0; x < SL; x++) if (K8) { spg[j][x] = nspg[j][x]; sc8[j][x][0] = nsc8[j][x][0]; sc8[j][x][1] = nsc8[j][x][1]; }
            }
        }
        if (issues && *reinterpret_cast<volatile int32_t*>(err) != 0)   // somewhere a wait ran out: its warps no longer wait for copies, so the copies under way are waited for here (within the same limit)
            for (uint32_t c = issued > (uint32_t)kStages ? issued - kStages : 0; c < issued; c++) mbar_wait_bounded(bars + c % kStages * 8, (c / kStages) & 1u);
        return;
    }

    while (tile < tile_end) {
        while (p.tile_start[b + 1] <= tile) b++;
        const int nt = plan_ntiles(p, b), kvh = (tile - p.tile_start[b]) / nt, lt0 = (tile - p.tile_start[b]) - kvh * nt;
        const int seg_first = tile - lt0, seg_end = seg_first + nt, my_end = min(tile_end, seg_end), n_here = my_end - tile;
        const int kend = p.kend[b];
        const int n_mine = n_here > ring ? (n_here - ring + kRings - 1) / kRings : 0;   // this ring's tiles: lt0 + ring, lt0 + ring + 4, ...
        const uint32_t it_seg = it, sums = n_segs % G::kSums, sums_par = (n_segs / G::kSums) & 1u;
        float* ml_seg = sm_ml + sums * kRings * 32; float* factor = joined_ml + 32 + sums * kRings * 16;
        const int all_see = kend - p.T + 1;   // slots below this are seen by every row (columns that hold no query too: nobody reads what they get)

        if (h == 0) {
            // ---- score warps. The query block first: rows t * group + j, zero behind the last; int8: columns permuted inside each 16-dim block
            constexpr int kQLoads = NR * 8 * (HD / 8) / 128; uint4 qv[kQLoads];
#pragma unroll
            for (int x = 0; x < kQLoads; x++) {
                const int ch = tid + x * 128, r = ch / (HD / 8), c16 = ch % (HD / 8), t = r / p.group, j = r - t * p.group;
                qv[x] = r < rows ? *reinterpret_cast<const uint4*>(q16 + (((int64_t)b * p.tok_stride + p.tok0 + t) * (kvh_n * p.group) + kvh * p.group + j) * HD + c16 * 8) : make_uint4(0, 0, 0, 0);
            }
            score_sync();   // the block before has been read
#pragma unroll
            for (int x = 0; x < kQLoads; x++) { const int ch = tid + x * 128; stage_q_chunk<K8>(smem + ch / (HD / 8) * G::kQStride, ch % (HD / 8), qv[x]); }
            score_sync();
            if (!dead && !mbar_wait_bounded(sempty + sums * 8, sums_par ^ 1u, err)) { dead = true; atomicExch(err, 6); }   // the sums of kSums segments ago have been read
            RowsState<NR> ss; int lim[NR][2], o_unit = 127; uint32_t qf[HD / 16][2], spoilt = 0;   // o_unit: O is carried in units of 2^(o_unit - 127) (int8)
#pragma unroll
            for (int nr = 0; nr < NR; nr++)
#pragma unroll
                for (int e = 0; e < 2; e++) { const int r = nr * 8 + 2 * t4 + e; ss.m[nr][e] = -INFINITY; ss.l[nr][e] = 0.0f; lim[nr][e] = r < rows ? kend - p.T + 1 + r / p.group : 0; }   // the row sees slots below this (none, when 0 or less)
            if (NR == 1) {
#pragma unroll
                for (int kk = 0; kk < HD / 16; kk += 2) q_frags(sm_base, G::kQStride, 0, kk, lane, qf[kk], qf[kk + 1]);
            }
            for (int i = 0; i < n_mine; i++) {
                const uint32_t cur = it_seg + (uint32_t)i, stg = cur % kStages, par = (cur / kStages) & 1u, slot = cur & 1u;
                const int key0 = (lt0 + ring + i * kRings) * kTile;
                // a wait that runs out is recorded once; afterwards waits are skipped, the control flow and every arrival stay as they are
                if (!dead && !mbar_wait_bounded(bars + stg * 8, par, err)) { dead = true; atomicExch(err, 1); }
                uint32_t sc[NK][2]; float ks[NK][2];   // K scale in the low half, V scale in the high half, of slots 16 * sb + g and 8 further
#pragma unroll
                for (int sb = 0; sb < NK; sb++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        if (K8) sc[sb][e] = *reinterpret_cast<const uint32_t*>(smem + G::kOffScale + (ring * kStages + stg) * kTile * 4 + (16 * sb + 8 * e + g) * 4);
                        ks[sb][e] = K8 ? __half2float(__ushort_as_half((unsigned short)sc[sb][e])) * kLog2e : 1.0f;   // int8: scores in log2 units
                    }
                float s[NK][NR][4], al[NR][2];
                paged_scores<HD, K8, NR>(sm_base, ring_stage0 + stg * G::kStageBytes, qf, ks, lane, s);
                __syncwarp();
                if (lane == 0) mbar_arrive(ebars + stg * 8);   // K and the scales (in registers by now) of this stage are no longer needed
                if (key0 + kTile > all_see) {   // masked by select: what lies behind the last slot may be anything
                    if (K8) {   // a V scale of infinity or NaN: 0 x that is not 0. The rows that see it become NaN when the rings are joined
#pragma unroll
                        for (int sb = 0; sb < NK; sb++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const int slot_no = key0 + 16 * sb + 8 * e + g;
                                if (slot_no < all_see || (sc[sb][e] & 0x7c000000u) != 0x7c000000u) continue;
                                sc[sb][e] &= 0xffffu;
#pragma unroll
                                for (int x = 0; x < 2 * NR; x++) if (slot_no < lim[x >> 1][x & 1]) spoilt |= 1u << x;
                            }
                    }
#pragma unroll
                    for (int sb = 0; sb < NK; sb++)
#pragma unroll
                        for (int nr = 0; nr < NR; nr++)
#pragma unroll
                            for (int e = 0; e < 4; e++) if (key0 + 16 * sb + 8 * (e >> 1) + g >= lim[nr][e & 1]) s[sb][nr][e] = -INFINITY;
                }
                if (scores) {   // [tile of the list][slot][8 or 16 rows]: full 32-byte sectors
                    float* st = scores + ((int64_t)(tile + ring + i * kRings) * kTile + g) * srow + 2 * t4;
#pragma unroll
                    for (int sb = 0; sb < NK; sb++)
#pragma unroll
                        for (int nr = 0; nr < NR; nr++)
#pragma unroll
                            for (int e = 0; e < 2; e++) *reinterpret_cast<float2*>(st + (16 * sb + 8 * e) * srow + nr * 8) = make_float2(s[sb][nr][2 * e], s[sb][nr][2 * e + 1]);
                }
                paged_softmax<NK, NR, G::kPShift, K8>(s, ss, al);
                if (K8) {   // P holds p times the V scale in units of 2^(exponent of the tile's largest + 1), so that it fills fp16's range whatever the size of the values; O follows from tile to tile by alpha
                    float vs[NK][2], top = 0.0f;
#pragma unroll
                    for (int sb = 0; sb < NK; sb++)
#pragma unroll
                        for (int e = 0; e < 2; e++) { vs[sb][e] = __half2float(__ushort_as_half((unsigned short)(sc[sb][e] >> 16))); top = fmaxf(top, fabsf(vs[sb][e])); }
                    const int unit = min(max((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23), 103), 143) + 1;   // biased; 2^-24 is the smallest scale, infinity counts as 2^16
                    const float inv = __uint_as_float((uint32_t)(254 - unit) << 23), turn = __uint_as_float((uint32_t)(127 + o_unit - unit) << 23);
                    o_unit = unit;
#pragma unroll
                    for (int nr = 0; nr < NR; nr++) { al[nr][0] *= turn; al[nr][1] *= turn; }
#pragma unroll
                    for (int sb = 0; sb < NK; sb++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
#pragma unroll
                            for (int nr = 0; nr < NR; nr++) s[sb][nr][e] *= vs[sb][e >> 1] * inv;
                        }
                }
                if (cur >= 2 && !dead && !mbar_wait_bounded(pempty + slot * 8, ((cur >> 1) - 1u) & 1u, err)) { dead = true; atomicExch(err, 4); }
                paged_publish<HD, K8, NR>(sm_base + p_off + slot * G::kPBytes, reinterpret_cast<float*>(smem + p_off + (slot + 1) * G::kPBytes - 64), s, al, p.two_terms, lane);
                __syncwarp();
                if (lane == 0) mbar_arrive(pfull + slot * 8);
            }
#pragma unroll
            for (int nr = 0; nr < NR; nr++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float l = ss.l[nr][e];
                    l += __shfl_xor_sync(0xffffffffu, l, 4); l += __shfl_xor_sync(0xffffffffu, l, 8); l += __shfl_xor_sync(0xffffffffu, l, 16);
                    if (g == 0) *reinterpret_cast<float2*>(ml_seg + (ring * 16 + nr * 8 + 2 * t4 + e) * 2) = make_float2(ss.m[nr][e], l);
                    if (K8 && g == 0) factor[ring * 16 + nr * 8 + 2 * t4 + e] = __uint_as_float((uint32_t)o_unit << 23);
                }
            __syncwarp();
            if (K8 && spoilt) {
#pragma unroll 1
                for (int x = 0; x < 2 * NR; x++) if (spoilt >> x & 1u) factor[ring * 16 + (x >> 1) * 8 + 2 * t4 + (x & 1)] = NAN;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(sfull + sums * 8);
        } else {
            const int vh = h - 1; ValueAcc<HD, NR> vst; vst.clear(); uint64_t bad = 0;
            for (int i = 0; i < n_mine; i++) {
                const uint32_t cur = it_seg + (uint32_t)i, stg = cur % kStages, par = (cur / kStages) & 1u, slot = cur & 1u;
                const uint32_t vt = ring_stage0 + stg * G::kStageBytes + G::kHalfBytes;
                const int key0 = (lt0 + ring + i * kRings) * kTile;
                if (!dead && !mbar_wait_bounded(bars + stg * 8, par, err)) { dead = true; atomicExch(err, 1); }
                if (!K8 && key0 + kTile > all_see) bad |= clean_v_rows<HD, NR>(smem + (vt - sm_base), max(0, all_see - key0), max(0, min(kend - key0, kTile)), all_see - key0, p.group, lane, vh);   // at most the ring's last tile
                if (!dead && !mbar_wait_bounded(pfull + slot * 8, (cur >> 1) & 1u, err)) { dead = true; atomicExch(err, 5); }
                const float* alpha = reinterpret_cast<const float*>(smem + p_off + (slot + 1) * G::kPBytes - 64);
                if (!K8 || p.two_terms) paged_values<HD, K8, NR, true>(vt, sm_base + p_off + slot * G::kPBytes, alpha, vst, lane, vh); else paged_values<HD, K8, NR, false>(vt, sm_base + p_off + slot * G::kPBytes, alpha, vst, lane, vh);
                __syncwarp();
                if (lane == 0) { mbar_arrive(pempty + slot * 8); mbar_arrive(ebars + stg * 8); }
            }
            // ---- join the four rings: ring 3 leaves its rows of O^T, scaled to the joint maximum, where the P slots were, ring 2 adds its own, ring 1, ring 0. The same lane holds the same
            // dims and rows in every ring, and the order is fixed. The producers are in the next segment meanwhile.
            if (!K8 && bad != 0) {
#pragma unroll
                for (int x = 0; x < HD / 16; x++)
#pragma unroll
                    for (int y = 0; y < 2 * NR; y++) if (bad >> (16 * y + x) & 1u) vst.o[x >> 1][y >> 1][2 * (x & 1) + (y & 1)] = NAN;
            }
            if (!dead && !mbar_wait_bounded(sfull + sums * 8, sums_par, err)) { dead = true; atomicExch(err, 7); }   // the rings' (m, l) are there
            value_sync();   // the segment before has left the block (NR = 2: and P is read)
#pragma unroll
            for (int nr = 0; nr < NR; nr++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = nr * 8 + 2 * t4 + e; float mx = -INFINITY, l = 0.0f, mine = 0.0f;
#pragma unroll
                    for (int ww = 0; ww < kRings; ww++) mx = fmaxf(mx, ml_seg[(ww * 16 + r) * 2]);
#pragma unroll
                    for (int ww = 0; ww < kRings; ww++) {
                        const float mm = ml_seg[(ww * 16 + r) * 2], wt = mm == -INFINITY ? 0.0f : ex2(mm - mx);
                        l += ml_seg[(ww * 16 + r) * 2 + 1] * wt;
                        if (ww == ring) mine = wt;
                    }
                    if (K8 && mine != 0.0f) mine *= factor[ring * 16 + r];
                    if (ring == 0 && vh == 0 && g == 0) *reinterpret_cast<float2*>(joined_ml + r * 2) = make_float2(mx, l);
#pragma unroll
                    for (int j = 0; j < HD / 32; j++) { vst.o[j][nr][e] = mine == 0.0f ? 0.0f : vst.o[j][nr][e] * mine; vst.o[j][nr][2 + e] = mine == 0.0f ? 0.0f : vst.o[j][nr][2 + e] * mine; }
                }
            float* mine = red + vh * G::kAcc * 32 + lane;   // [half][accumulator][lane]
#pragma unroll 1
            for (int from = kRings - 1; from >= 0; from--) {
                if (ring == from) {
#pragma unroll
                    for (int j = 0; j < HD / 32; j++)
#pragma unroll
                        for (int nr = 0; nr < NR; nr++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                float* at = mine + ((j * NR + nr) * 4 + e) * 32;
                                *at = (from == kRings - 1 ? 0.0f : *at) + vst.o[j][nr][e];
                            }
                }
                if (from) asm volatile("bar.sync %0, 128;" ::"r"(3 + vh) : "memory");   // the four value warps of this half
            }
            value_sync();   // the CTA's rows are there
            // ---- final rows, or a partial
            const int seg = b * kvh_n + kvh;
            const bool whole = n_here == nt;
            constexpr int kTpr = HD / 2, kRowPar = 256 / kTpr;   // threads per row (two dims each), rows at a time
            const int vtid = tid - 128, d0 = 2 * (vtid % kTpr), dx = d0 & 15;
            const float* from = red + ((d0 / (HD / 2)) * G::kAcc + (d0 % (HD / 2)) / 16 * NR * 4 + (K8 ? 0 : dx >> 3) * 2) * 32 + (K8 ? dx >> 1 : dx & 7) * 4;   // of d0; d0 + 1 lies two accumulators (int8) or four lanes further
            constexpr int kIters = NR * 8 / kRowPar; const int r0 = vtid / kTpr;
            if (whole) {
                float2 gate[kIters];   // requested together
#pragma unroll
                for (int x = 0; x < kIters; x++) if (r0 + x * kRowPar < rows) gate[x] = paged_gate(o, paged_out_at<HD>(p, b, kvh, r0 + x * kRowPar, d0));
#pragma unroll
                for (int x = 0; x < kIters; x++) {
                    const int r = r0 + x * kRowPar; const float* at = from + ((r >> 3) * 4 + (r & 1)) * 32 + ((r & 7) >> 1);
                    if (r < rows) paged_emit(p, o, b, kvh, r, d0, paged_out_at<HD>(p, b, kvh, r, d0), gate[x], joined_ml[r * 2], joined_ml[r * 2 + 1], at[0], at[K8 ? 64 : 4]);
                }
            } else {   // (CTA, segment) pairs have CTA + segment of their own
                const int64_t sl = blockIdx.x + seg;
                for (int r = r0; r < rows; r += kRowPar) {
                    const float* at = from + ((r >> 3) * 4 + (r & 1)) * 32 + ((r & 7) >> 1);
                    *reinterpret_cast<float2*>(scratch_o + sl * (16 * HD) + r * HD + d0) = make_float2(at[0], at[K8 ? 64 : 4]);
                    if (d0 == 0) *reinterpret_cast<float2*>(scratch_ml + sl * 32 + r * 2) = make_float2(joined_ml[r * 2], joined_ml[r * 2 + 1]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(sempty + sums * 8);
            if (p.merge_in_kernel && !whole) {   // the last of (at most 8) contributors joins everybody's partial rows
                const int c_first = plan_first_cta(p, blockIdx.x, seg_first), n_contrib = plan_last_cta(p, blockIdx.x, seg_end) - c_first + 1;
                __threadfence();
                value_sync();
                if (vtid == 0) { const int old = atomicAdd(&counters[seg], 1); s_flag = (old == n_contrib - 1); if (s_flag) counters[seg] = 0; }   // zero again for the next call
                value_sync();
                if (s_flag) {
                    __threadfence();
                    for (int r = r0; r < rows; r += kRowPar) {
                        const int64_t sl = c_first + seg, at = paged_out_at<HD>(p, b, kvh, r, d0); const float2 gate = paged_gate(o, at);
                        float2 ml[8], oo[8]; float M = -INFINITY, L = 0.0f, A0 = 0.0f, A1 = 0.0f;
#pragma unroll
                        for (int c = 0; c < 8; c++) {
                            ml[c] = c < n_contrib ? __ldcg(reinterpret_cast<const float2*>(scratch_ml + (sl + c) * 32 + r * 2)) : make_float2(-INFINITY, 0.0f);
                            oo[c] = c < n_contrib ? __ldcg(reinterpret_cast<const float2*>(scratch_o + (sl + c) * (16 * HD) + r * HD + d0)) : make_float2(0.0f, 0.0f);
                        }
#pragma unroll
                        for (int c = 0; c < 8; c++) M = fmaxf(M, ml[c].x);
#pragma unroll
                        for (int c = 0; c < 8; c++) { const float wt = ml[c].x == -INFINITY ? 0.0f : ex2(ml[c].x - M); L += ml[c].y * wt; A0 += oo[c].x * wt; A1 += oo[c].y * wt; }
                        paged_emit(p, o, b, kvh, r, d0, at, gate, M, L, A0, A1);
                    }
                }
            }
        }
        it += (uint32_t)n_mine; n_segs++;
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
    const int nt = plan_ntiles(p, b), seg_first = p.tile_start[b] + kvh * nt, c_first = plan_cta_of(p, seg_first), n_c = plan_cta_of(p, seg_first + nt - 1) - c_first + 1;
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
    const int64_t at = paged_out_at<HD>(p, b, kvh, r, d);
    paged_emit(p, o, b, kvh, r, d, at, paged_gate(o, at), M, L, A0, A1);
}

// weight[kv head][slot] += sum over the rows of 2^(s * log2 e - m + shift) / l (int8: s is in log2 units): the slot's final probabilities, from the scores the decode kernel
// kept and the joined (m, 1 / l). A thread per (slot, KV head) in the order of the tile list: 32 (or 64) contiguous bytes per thread, nothing shared, no atomics. All of a thread's requests are
// under way before the first is used (107K slots x 4 heads: 7.9 us, 10.3 with a loop over the rows).
template <int ROWS>   // 8 or 16 stored rows
__global__ void __launch_bounds__(256) paged_weight_kernel(const __grid_constant__ PagedPlan p, const int32_t* __restrict__ tables, const float* __restrict__ scores, const float* __restrict__ fin_ml,
                                                           float* __restrict__ weight /* the layer's plane [page][kv head][slot] */, const int tile_shift, const float shift, const bool log2) {
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; const int tile = (int)(idx >> tile_shift);
    int lo = 0, hi = p.n - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (p.tile_start[mid] <= tile) lo = mid; else hi = mid - 1; }
    const int b = lo, nt = plan_ntiles(p, b), kvh = (tile - p.tile_start[b]) / nt, slot = ((tile - p.tile_start[b] - kvh * nt) << tile_shift) + (int)(idx & ((1 << tile_shift) - 1));
    pdl_wait(); pdl_launch_dependents();
    if (tile >= p.tile_start[p.n] || slot >= p.kend[b]) return;
    const int page = __ldcg(tables + (int64_t)p.seq[b] * p.width + (slot >> p.page_shift)), rows = p.group * p.T;
    const float4* s4 = reinterpret_cast<const float4*>(scores + idx * ROWS); const float4* ml4 = reinterpret_cast<const float4*>(fin_ml) + (int64_t)(b * p.kv_heads + kvh) * 8;
    float4 v[ROWS / 4], ml[ROWS / 2];
#pragma unroll
    for (int i = 0; i < ROWS / 4; i++) v[i] = __ldcg(s4 + i);
#pragma unroll
    for (int i = 0; i < ROWS / 2; i++) if (2 * i < rows) ml[i] = __ldcg(ml4 + i);   // of two rows; of an odd last row's neighbour too, unused
    float* at = weight + (((int64_t)page * p.kv_heads + kvh) << p.page_shift) + (slot & ((1 << p.page_shift) - 1));
    const float before = *at; float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const float x = r % 4 == 0 ? v[r / 4].x : r % 4 == 1 ? v[r / 4].y : r % 4 == 2 ? v[r / 4].z : v[r / 4].w, m = r & 1 ? ml[r / 2].z : ml[r / 2].x, inv = r & 1 ? ml[r / 2].w : ml[r / 2].y;
        if (r < rows && x != -INFINITY) sum += ex2(log2 ? x - (m - shift) : fabsf(m) > kRoundedMax ? (__fmul_rn(x, kLog2e) - m) + shift : fmaf(x, kLog2e, shift - m)) * inv;   // as the decode kernel formed it (log2: int8); a masked slot adds nothing (its row may have no maximum at all)
    }
    *at = before + sum;
}

// The work split (host only): tiles, ranges and where the partial rows are joined. p.n, p.kv_heads and p.kend are set.
int split_paged_tiles(PagedPlan& p, int tile_keys, int sm_count) {
    sm_count = std::min(sm_count, kMaxCtas);
    int total = 0; bool same = true;
    for (int i = 0; i < p.n; i++) {
        p.tile_start[i] = total; total += p.kv_heads * std::max(1, (p.kend[i] + tile_keys - 1) / tile_keys);   // a sequence without keys has one (masked) tile: its rows are written
        same = same && (i == 0 || total - p.tile_start[i] == p.tile_start[1]);
    }
    for (int i = p.n; i <= KATA_PAGED_MAX_BATCH; i++) p.tile_start[i] = total;
    // Equal segments that divide nearly all SMs, or whose shares are hardly longer than an even split's, get CTAs of their own: none then pays for a second segment (eight sequences of 300 slots:
    // 128 CTAs of 5 tiles 12.7 us, 148 of 4.1 tiles 16.3 us).
    const int n_seg = p.n * p.kv_heads, nt0 = plan_ntiles(p, 0), cps = n_seg <= sm_count ? std::min(sm_count / n_seg, nt0) : 0;
    constexpr int kPad = 8, kSnap = 4;
    int most = 1;
    if (same && cps >= 1 && (cps * n_seg * 100 >= sm_count * 97 || (nt0 + cps - 1) / cps <= total / sm_count + kPad)) {
        p.n_ctas = cps * n_seg; most = cps;
        for (int c = 0; c < p.n_ctas; c++) p.cut[c] = c / cps * nt0 + (int)((int64_t)nt0 * (c % cps) / cps);
        p.cut[p.n_ctas] = total;
    } else {
        // A segment costs a CTA more than its tiles: its rows are joined and written, the next one's query staged, some 3 us beside 0.37 us a tile. Many short segments would pile up in a few CTAs
        // (32 int8 sequences of 300 to 32K slots, sorted by length, in short loops: 218 us, 182 like this): each counts as kPad tiles more, where the ranges are long enough for that. A cut that falls within kSnap tiles of an
        // end of a segment moves there: less than what the second piece would cost.
        p.n_ctas = std::max(1, std::min(sm_count, total));
        const int pad = total >= (int64_t)sm_count * 4 * kPad ? kPad : 0, snap = pad ? kSnap : 0; const int64_t places = total + (int64_t)n_seg * pad;
        int c = 0; int64_t place = 0, next = 0;   // place: of the segment (its pad, then its tiles); next: of cut c
        for (int i = 0; i < p.n; i++) {
            const int nt = plan_ntiles(p, i);
            for (int kv = 0; kv < p.kv_heads; kv++, place += nt + pad) {
                int cuts_inside = 0;
                while (c < p.n_ctas && next < place + nt + pad) {
                    int in = (int)(next - place) - pad;
                    in = in <= snap ? 0 : in >= nt - snap ? nt : in;
                    p.cut[c] = p.tile_start[i] + kv * nt + in; cuts_inside += in > 0 && in < nt;
                    next = places * ++c / p.n_ctas;
                }
                most = std::max(most, cuts_inside + 1);
            }
        }
        p.cut[p.n_ctas] = total;
    }
    p.merge_in_kernel = most <= 8;   // few contributors: the last one joins them (no second kernel); many: one SM would pull them all, a grid does it in one round trip
    return most;
}

}  // namespace

static int tile_keys_of(const PagedCtx& c, int rows) { return c.cfg.head_dim == 256 ? (c.int8() ? 32 : 16) : (c.int8() && rows <= 8) ? 64 : 32; }   // PGeo::kTile
int64_t paged_score_slots(const PagedCtx& c) { return (int64_t)c.cfg.kv_heads * ((int64_t)c.cfg.n_pages * c.cfg.page_size + 64 * KATA_PAGED_MAX_BATCH); }   // no page is shared, so the pool bounds a launch's slots; each sequence's are rounded up to a tile
// (CTA + segment) slots of partial rows
size_t paged_part_floats(const PagedCtx& c) { return (size_t)(c.sm_count + KATA_PAGED_MAX_BATCH * c.cfg.kv_heads) * 16 * c.cfg.head_dim; }
size_t paged_part_ml_floats(const PagedCtx& c) { return (size_t)(c.sm_count + KATA_PAGED_MAX_BATCH * c.cfg.kv_heads) * 32; }

#define KATA_PAGED_KERNELS(X) X(256, false, 1) X(256, false, 2) X(256, true, 1) X(256, true, 2) X(128, false, 1) X(128, false, 2) X(128, true, 1) X(128, true, 2)

cudaError_t configure_paged_decode(const PagedCtx& c) {   // shared-memory opt-in, per device
    cudaError_t e = cudaSuccess;
#define X(HD, K8, NR) if (e == cudaSuccess && c.cfg.head_dim == HD && c.int8() == K8) e = cudaFuncSetAttribute(paged_decode_kernel<HD, K8, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, PGeo<HD, K8, NR>::kSmem);
    KATA_PAGED_KERNELS(X)
#undef X
    return e;
}

cudaError_t launch_paged_decode(PagedCtx& c, int layer, int n, const int32_t* seq, const int32_t* n_slots, int T, const __half* q16, const float* gate, void* out, int out_dtype, bool accumulate, cudaStream_t s) {
    const int per_pass = std::max(1, 16 / c.group), hd = c.cfg.head_dim;
    for (int t0 = 0; t0 < T; t0 += per_pass) {   // each pass is independent: all rows are in the cache, token t of the call sees slots below n_slots - T + 1 + t
        PagedPlan p{}; p.n = n; p.T = std::min(per_pass, T - t0); p.group = c.group; p.kv_heads = c.cfg.kv_heads; p.tok_stride = T; p.tok0 = t0;
        p.two_terms = !c.int8() || out_dtype == KATA_ACT_F32; p.page_shift = c.page_shift; p.width = c.width; p.groups_per_box = c.box_groups; p.layer_row0 = (int64_t)layer * c.rows_per_layer;
        for (int i = 0; i < n; i++) { p.seq[i] = seq[i]; p.kend[i] = std::max(0, n_slots[i] - T + t0 + p.T); }
        const int tile_keys = tile_keys_of(c, c.group * p.T);
        split_paged_tiles(p, tile_keys, c.sm_count);
        // a pass's limits are kend - p.T + 1 + t: where kend was raised to 0 they are 0 or less, as they should be
        const PagedOut o{gate, out, out_dtype, accumulate ? c.fin_ml : nullptr}; float* scores = accumulate ? c.scores : nullptr;
        if (accumulate && (int64_t)p.tile_start[n] * tile_keys > paged_score_slots(c)) return cudaErrorInvalidValue;   // cannot be: the pool bounds them
        cudaError_t e = cudaErrorInvalidValue;
#define X(HD, K8, NR) if (hd == HD && c.int8() == K8 && (c.group * p.T > 8) == (NR == 2)) e = launch_pdl(paged_decode_kernel<HD, K8, NR>, dim3(p.n_ctas), dim3(PGeo<HD, K8, NR>::kThreads), PGeo<HD, K8, NR>::kSmem, s, c.tm_k, c.tm_v, p, (const int32_t*)c.d_table, q16, o, \
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
            e = launch_pdl(c.group * p.T > 8 ? paged_weight_kernel<16> : paged_weight_kernel<8>, dim3((unsigned)((keys + 255) / 256)), dim3(256), 0, s, p, (const int32_t*)c.d_table, (const float*)c.scores, (const float*)c.fin_ml,
                           (float*)c.layer_plane(KATA_PAGED_WEIGHT, layer), tile_keys == 16 ? 4 : tile_keys == 32 ? 5 : 6, (float)PGeo<256, true, 1>::kPShift, c.int8());
            if (e != cudaSuccess) return e;
            c.launches++;
        }
    }
    return cudaGetLastError();
}

}  // namespace kata

extern "C" int kata_paged_decode_plan(int32_t n, const int32_t* n_keys, int32_t kv_heads, int32_t tile_keys, int32_t sm_count, int32_t* first_tile, int32_t first_tile_cap, int32_t* max_contrib) {
    using namespace kata;
    if (n < 1 || n > KATA_PAGED_MAX_BATCH || !n_keys || kv_heads < 1 || kv_heads > KATA_PAGED_MAX_KV_HEADS || (tile_keys != 16 && tile_keys != 32 && tile_keys != 64) || sm_count < 1 || !first_tile || !max_contrib) return -1;
    PagedPlan p{}; p.n = n; p.kv_heads = kv_heads;
    for (int i = 0; i < n; i++) { if (n_keys[i] < 0 || n_keys[i] > KATA_PAGED_MAX_SLOTS) return -1; p.kend[i] = n_keys[i]; }
    *max_contrib = split_paged_tiles(p, tile_keys, sm_count);
    if (p.n_ctas + 1 > first_tile_cap) return -1;
    for (int cta = 0; cta <= p.n_ctas; cta++) first_tile[cta] = p.cut[cta];
    for (int i = 0, cta = 0; i < n; i++) for (int kv = 0; kv < kv_heads; kv++) for (int lt = 0; lt < plan_ntiles(p, i); lt++) {
        const int nt = plan_ntiles(p, i), first = p.tile_start[i] + kv * nt, t = first + lt;
        while (p.cut[cta + 1] <= t) cta++;
        if (plan_cta_of(p, t) != cta || plan_first_cta(p, cta, first) != plan_cta_of(p, first) || plan_last_cta(p, cta, first + nt) != plan_cta_of(p, first + nt - 1)) return -2;   // the maps disagree
    }
    return p.n_ctas;
}
