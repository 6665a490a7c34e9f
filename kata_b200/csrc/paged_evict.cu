// Eviction from a paged cache by accumulated attention weight (kata_paged_evict): per layer, sequence and KV head the `keep` heaviest slots stay.
//   key(slot) = +inf for protected slots (age < sink or age >= seen - recent), else the weight; order: key descending, then slot ascending.
// Slots kept below `keep` stay where they are; the i-th kept slot at or behind `keep` moves into the i-th free slot below it. Every row that moves is read
// behind `keep` and written below it, so no order of the copies can clobber one, and as few rows move as can.
//
// select, up to 5,120 slots: one CTA per (layer, sequence, KV head) with the slots' keys (weights as order-preserving 32-bit integers) in registers. The keep-th largest bit by bit from
// the top, a count over the block per bit (some 330 clocks), ended early once a count is `keep` (histograms of digits in shared memory were slower: their atomics take a
// clock per lane); then the words of 32 slots get their prefix sums by ballots and shuffles, the movers go to a list in shared memory in order, and every free slot
// takes the mover of its rank.
// select_cluster, above that: eight CTAs with a contiguous eighth of the slots each (one SM needs 12 us for the loads of 32K slots alone). Up to 131,072 slots the keys are in registers, and the
// threshold is found by bounds: a sample of 512 keys gives two values that it hardly lies outside of (three standard deviations), the keys between them go to every CTA through distributed
// shared memory, and each narrows them by counting at interpolated values until a warp can rank the rest (8 x 32K slots to 4,096 with the moves 70 us; narrowed by a second sample and
// searched bit by bit by one warp 75). Where the counts do not confirm the bounds, or too many keys lie between (one value shared
// by many slots), and for longer sequences, whose keys are read again in every pass, a radix select over the cluster's summed histograms finds it. Ranks of free slots and movers come
// from prefix sums per word; the free slots are listed by rank where they lie, and each mover looks its own up.
// move: a warp per 32 destinations, lanes agreeing by ballot on those that receive a row; each row is 16-byte copies of K and V. Bound by HBM: 2 x row bytes per move.
#include <algorithm>
#include <type_traits>

#include <cooperative_groups.h>

#include "paged_internal.cuh"

namespace kata {
namespace {

constexpr int kSelThreads = 512, kSelWarps = kSelThreads / 32;
constexpr int kSelOne = 10 * kSelThreads, kSelMany = 64;   // one CTA per (layer, sequence, KV head) up to so many slots, or (up to 32,768) when there are so many of them: 256 times 8,000 slots took 36 us
                                                           // beside the move so, 180 us as clusters, whose latency then adds up
constexpr int kSelCluster = 8, kCluSlots = kSelCluster * kSelThreads, kCluMax = 8 * kCluSlots;   // slots of a cluster per register of its threads; slots that it, or one CTA, selects from by bounds
constexpr int kSample = kSelThreads, kOwn = 2 * kSelThreads;   // keys in the sample; keys that may lie between the bounds per CTA

struct EvictArgs {
    int keep, sink, recent, width, page_shift, kv_heads, n, layer0;
    int64_t plane_stride;                 // elements of a weight / age plane of one layer
    const int32_t* tables; float* weight; int32_t* age; int32_t* src;
};

__device__ __forceinline__ uint32_t order_key(float w) {   // larger float, larger integer; NaN below everything (1; 0 stands for no slot); -0 = +0
    if (w != w) return 1u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int warp_inclusive(int v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) { const int o = __shfl_up_sync(0xffffffffu, v, off); if (lane >= off) v += o; }
    return v;
}
// c += k >= at, as a compare and a predicated add (the compiler's form of `c += k >= at` takes 8 clocks a key, this 4)
__device__ __forceinline__ void add_if_ge(int& c, uint32_t k, uint32_t at) { asm("{\n .reg .pred p;\n setp.ge.u32 p, %1, %2;\n @p add.s32 %0, %0, 1;\n}" : "+r"(c) : "r"(k), "r"(at)); }

// A value between lo and hi that at least `target` of a warp's keys reach: exactly so many, or it is the target-th largest key itself. All keys are at least lo (or 0: none).
template <int N> __device__ __forceinline__ uint32_t warp_search(const uint32_t (&k)[N], int target, uint32_t lo, uint32_t hi) {
    uint32_t v = lo == hi ? lo : lo & ~(0xffffffffu >> __clz(lo ^ hi));
#pragma unroll 1
    for (int bit = lo == hi ? -1 : 31 - __clz(lo ^ hi); bit >= 0; bit--) {
        const uint32_t at = v | 1u << bit; int c[4] = {};
#pragma unroll
        for (int i = 0; i < N; i++) add_if_ge(c[i & 3], k[i], at);
        const int n = __reduce_add_sync(0xffffffffu, (c[0] + c[1]) + (c[2] + c[3]));
        if (n >= target) v = at;
        if (n == target) break;
    }
    return v;
}
__device__ __forceinline__ uint32_t evict_key(const EvictArgs& a, const int32_t* table, const float* weight, const int32_t* age, int kvh, int j, int newest) {   // of one slot
    const int64_t at = (((int64_t)__ldcg(table + (j >> a.page_shift)) * a.kv_heads + kvh) << a.page_shift) + (j & ((1 << a.page_shift) - 1));
    const int ag = __ldcg(age + at); const float wt = __ldcg(weight + at);
    return (ag < a.sink || ag >= newest) ? 0xFF800000u : order_key(wt);   // 0xFF800000: the key of +inf
}
// the same for N slots of a thread, slot(i) clamped to the last: without branches, so that the requests are under way together, eight slots at a time
template <int N, typename F> __device__ __forceinline__ void evict_keys(const EvictArgs& a, const int32_t* table, const float* weight, const int32_t* age, int kvh, int n_slots, int newest, F slot, uint32_t (&key)[N]) {
    const int in_page = (1 << a.page_shift) - 1;
#pragma unroll
    for (int i = 0; i < N; i++) key[i] = (uint32_t)__ldcg(table + (min(slot(i), n_slots - 1) >> a.page_shift));
#pragma unroll
    for (int i0 = 0; i0 < N; i0 += 8) {
        float wt[8]; int ag[8];
#pragma unroll
        for (int x = 0; x < 8; x++) if (i0 + x < N) {
            const int64_t at = (((int64_t)(int32_t)key[i0 + x] * a.kv_heads + kvh) << a.page_shift) + (min(slot(i0 + x), n_slots - 1) & in_page);
            wt[x] = __ldcg(weight + at); ag[x] = __ldcg(age + at);
        }
#pragma unroll
        for (int x = 0; x < 8; x++) if (i0 + x < N) key[i0 + x] = slot(i0 + x) < n_slots ? ((ag[x] < a.sink || ag[x] >= newest) ? 0xFF800000u : order_key(wt[x])) : 0u;
    }
}
// of a value per warp, the sum over the warps before this one; s: kSelWarps words, not in use
__device__ __forceinline__ int warps_before(int32_t* s, int v) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (lane == 0) s[w] = v;
    __syncthreads();
    return (int)__reduce_add_sync(0xffffffffu, lane < w ? s[lane] : 0);
}

// grid (kv heads, sequences, layers). ITEMS: words of 32 slots per warp; warp w has words w * ITEMS .. and lane i (for more than 32: and i + 32) keeps what concerns word w * ITEMS + i
template <int ITEMS>
__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(const __grid_constant__ PagedBatch b, const __grid_constant__ EvictArgs a) {
    __shared__ uint16_t list[ITEMS * kSelThreads / 2];   // the movers in order: at most half of the slots
    __shared__ int32_t s_n[2][kSelWarps], s_b[kSelWarps], s_c[kSelWarps], s_d[kSelWarps];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, kvh = blockIdx.x, bi = blockIdx.y, l = blockIdx.z, S = b.slot[bi], keep = a.keep;
    pdl_wait(); pdl_launch_dependents();
    int32_t* src = a.src + (((int64_t)l * a.n + bi) * a.kv_heads + kvh) * keep;
    if (S <= keep) { for (int j = tid; j < keep; j += kSelThreads) src[j] = j < S ? j : -1; return; }
    const int j0 = w * ITEMS * 32 + lane;   // slot of item i: j0 + 32 * i
    uint32_t key[ITEMS];
    evict_keys(a, a.tables + (int64_t)b.seq[bi] * a.width, a.weight + (int64_t)(a.layer0 + l) * a.plane_stride, a.age + (int64_t)(a.layer0 + l) * a.plane_stride, kvh, S, b.age[bi] - a.recent, [&](int i) { return j0 + 32 * i; }, key);
    // ---- the keep-th largest key: the largest value that at least `keep` keys reach
    uint32_t prefix = 0; int reach = S;   // keys >= prefix
#pragma unroll 1
    for (int bit = 31; bit >= 0 && reach != keep; bit--) {
        int c[2] = {};
#pragma unroll
        for (int i = 0; i < ITEMS; i++) add_if_ge(c[i & 1], key[i], prefix | 1u << bit);
        int n = __reduce_add_sync(0xffffffffu, c[0] + c[1]);
        if (lane == 0) s_n[bit & 1][w] = n;   // two rows in turn: one barrier per count
        __syncthreads();
        n = __reduce_add_sync(0xffffffffu, lane < kSelWarps ? s_n[bit & 1][lane] : 0);
        if (n >= keep) { prefix |= 1u << bit; reach = n; }
    }
    // ---- every key above prefix is kept; of those equal to it (all of them, when as many as `keep` reach it) the lowest
    constexpr int WL = (ITEMS + 31) / 32;   // words per lane: w * ITEMS + lane and, 32 further, another
    uint32_t gt[WL] = {}, eq[WL] = {};
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const uint32_t g = __ballot_sync(0xffffffffu, key[i] > prefix), e = __ballot_sync(0xffffffffu, key[i] == prefix);
        if (lane == (i & 31)) { gt[i >> 5] = g; eq[i >> 5] = e; }
    }
    // exclusive ranks of the words' counts over the whole block, in word order; s: kSelWarps words; returns the sum over all
    auto ranks = [&](const int (&n)[WL], int (&at)[WL], int32_t* s) {
        int base = 0;
#pragma unroll
        for (int x = 0; x < WL; x++) { const int inc = warp_inclusive(n[x]); at[x] = base + inc - n[x]; base += __shfl_sync(0xffffffffu, inc, 31); }
        const int bef = warps_before(s, base);
#pragma unroll
        for (int x = 0; x < WL; x++) at[x] += bef;
        return (int)__reduce_add_sync(0xffffffffu, lane < kSelWarps ? s[lane] : 0);
    };
    uint32_t kept[WL]; int n[WL], at[WL];
#pragma unroll
    for (int x = 0; x < WL; x++) { kept[x] = gt[x] | eq[x]; n[x] = __popc(eq[x]); }
    if (reach != keep) {   // reach - keep of the keys equal to prefix are too many: the highest slots go
        const int all = ranks(n, at, s_d);
#pragma unroll
        for (int x = 0; x < WL; x++) {
            uint32_t stay = 0, rest = eq[x];
            for (int m = min(all - (reach - keep) - at[x], 32); m > 0 && rest; m--) { stay |= rest & (0u - rest); rest &= rest - 1; }
            kept[x] = gt[x] | stay;
        }
    }
    uint32_t hole[WL], mover[WL]; int h_at[WL];
#pragma unroll
    for (int x = 0; x < WL; x++) {
        const int i = lane + 32 * x, jw = (w * ITEMS + i) * 32; const uint32_t below = i >= ITEMS ? 0u : jw + 32 <= keep ? 0xffffffffu : jw >= keep ? 0u : (1u << (keep - jw)) - 1;   // slots of the word below `keep`
        hole[x] = ~kept[x] & below; mover[x] = kept[x] & ~below;
    }
#pragma unroll
    for (int x = 0; x < WL; x++) n[x] = __popc(hole[x]);
    ranks(n, h_at, s_c);
#pragma unroll
    for (int x = 0; x < WL; x++) n[x] = __popc(mover[x]);
    ranks(n, at, s_b);
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const uint32_t mv = __shfl_sync(0xffffffffu, mover[i >> 5], i & 31); const int m_at = __shfl_sync(0xffffffffu, at[i >> 5], i & 31);
        if ((mv >> lane) & 1u) list[m_at + __popc(mv & ((1u << lane) - 1))] = (uint16_t)(j0 + 32 * i);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const uint32_t hl = __shfl_sync(0xffffffffu, hole[i >> 5], i & 31); const int a_h = __shfl_sync(0xffffffffu, h_at[i >> 5], i & 31), j = j0 + 32 * i;
        if (j < keep) src[j] = ((hl >> lane) & 1u) ? (int)list[a_h + __popc(hl & ((1u << lane) - 1))] : j;
    }
}

// grid (8 * kv heads, sequences, layers), clusters of 8 CTAs; CTA `rank` of a cluster has words [rank * wpc, (rank + 1) * wpc) of 32 slots, warp w of it words w, w + 16, ... ITEMS: keys per thread, at most
// as many words per warp (0: the keys are not kept). Dynamic shared memory: three words per word of slots, then the list of the CTA's free slots (16 bits each)
template <int ITEMS>
__global__ void __launch_bounds__(kSelThreads) paged_select_cluster_kernel(const __grid_constant__ PagedBatch b, const __grid_constant__ EvictArgs a, const int wpc) {
    namespace cg = cooperative_groups; constexpr int CS = kSelCluster;
    extern __shared__ __align__(16) uint32_t dyn[];
    uint32_t* kept = dyn; int32_t* pre_h = reinterpret_cast<int32_t*>(dyn + wpc); int32_t* pre_m = pre_h + wpc; uint16_t* list = reinterpret_cast<uint16_t*>(dyn + 3 * wpc);
    // the keys between the bounds, of every CTA of the cluster; or the four histograms of the radix select
    __shared__ __align__(16) uint32_t pool[ITEMS ? CS * kOwn : 4 * 1024]; int32_t* const hist = reinterpret_cast<int32_t*>(pool);
    __shared__ uint32_t sample[kSample], s_bound[2]; __shared__ int32_t s_cand[CS], s_above[CS], s_eq[CS], s_holes[CS], s_movers[CS], s_sum[3], s_warp[kSelWarps]; __shared__ int s_bin, s_left, s_n;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rank = blockIdx.x % CS, kvh = blockIdx.x / CS, bi = blockIdx.y, l = blockIdx.z, S = b.slot[bi], keep = a.keep, newest = b.age[bi] - a.recent;   // ages from `newest` on are protected
    auto peer = [&](auto* p, int r) { return cg::this_cluster().map_shared_rank(p, r); };
    auto sync_all = [&]() { cg::this_cluster().sync(); };
    if (tid == 0) { s_n = s_left = 0; s_sum[0] = s_sum[1] = s_sum[2] = 0; }
    pdl_wait(); pdl_launch_dependents();
    int32_t* src = a.src + (((int64_t)l * a.n + bi) * a.kv_heads + kvh) * keep;
    if (S <= keep) { for (int j = rank * kSelThreads + tid; j < keep; j += CS * kSelThreads) src[j] = j < S ? j : -1; return; }   // (the whole cluster)
    cg::this_cluster().barrier_arrive();   // waited for before the first access to another CTA's shared memory: it has to have started
    const int32_t* table = a.tables + (int64_t)b.seq[bi] * a.width; const float* weight = a.weight + (int64_t)(a.layer0 + l) * a.plane_stride; const int32_t* age = a.age + (int64_t)(a.layer0 + l) * a.plane_stride;
    const int j0 = rank * wpc * 32, mine = min(max(S - j0, 0), wpc * 32), words = (mine + 31) >> 5;   // slots j0 .. j0 + mine - 1 are this CTA's; item i of a thread: j0 + tid + 512 * i
    constexpr bool REGS = ITEMS > 0;
    uint32_t key[REGS ? ITEMS : 1];
    if (REGS) evict_keys(a, table, weight, age, kvh, S, newest, [&](int i) { return tid + i * kSelThreads < mine ? j0 + tid + i * kSelThreads : S; }, key);
    auto each = [&](auto f) {   // f(key, position among the CTA's slots), a warp's lanes together; key 0 behind the last
        if constexpr (REGS) {
#pragma unroll
            for (int i = 0; i < ITEMS; i++) f(key[i], tid + i * kSelThreads);
        } else for (int q0 = w * 32; q0 < mine; q0 += kSelThreads) f(q0 + lane < mine ? evict_key(a, table, weight, age, kvh, j0 + q0 + lane, newest) : 0u, q0 + lane);
    };
    __syncthreads();
    int turn = 0;
    auto total = [&](int v) {   // over the block; three words taken in turn: one barrier per sum
        v = (int)__reduce_add_sync(0xffffffffu, v);
        if (lane == 0) atomicAdd(&s_sum[turn], v);
        __syncthreads();
        const int t = s_sum[turn]; turn = turn == 2 ? 0 : turn + 1;
        if (tid == 0) s_sum[turn == 2 ? 0 : turn + 1] = 0;   // read by everybody before this barrier, used after the next
        return t;
    };
    auto slot_for = [&](int n) {   // where a thread's n values go in a list counted by s_n
        const int inc = warp_inclusive(n); int at = 0;
        if (lane == 31 && inc) at = atomicAdd(&s_n, inc);
        return __shfl_sync(0xffffffffu, at, 31) + inc - n;
    };
    uint32_t prefix = 0; int left = keep;   // left: how many of the keys equal to prefix (of the keys that match it, on the way) are kept
    bool found = false;
    if constexpr (REGS) {   // ---- the keep-th largest key by bounds
        constexpr int step = kSelThreads * CS / kSample;
        cg::this_cluster().barrier_wait();
        if (tid % step == 0) {   // every CTA's share of the sample, to every CTA
            uint32_t k = 0;
#pragma unroll
            for (int i = 0; i < ITEMS; i++) if (tid / step % ITEMS == i) k = key[i];
            for (int r = 0; r < CS; r++) peer(&sample[0], r)[rank * (kSample / CS) + tid / step] = k;
        }
        sync_all();
        if (w < 2) {   // where the keep-th largest of the S keys hardly lies above (warp 0) or below (warp 1)
            uint32_t k[kSample / 32]; int n_s = 0;
#pragma unroll
            for (int i = 0; i < kSample / 32; i++) { k[i] = sample[i * 32 + lane]; n_s += k[i] != 0u; }
            n_s = __reduce_add_sync(0xffffffffu, n_s);
            const float f = (float)keep / (float)S, mid = f * n_s, dev = 3.0f * sqrtf(n_s * f * (1.0f - f)) + 3.0f; const int t = w == 0 ? (int)(mid - dev) : (int)(mid + dev) + 1;   // rank in the sample
            const uint32_t v = t < 1 ? 0xffffffffu : t > n_s ? 1u : warp_search(k, t, 1u, 0xffffffffu);
            if (lane == 0) s_bound[w] = max(v, 1u);
        }
        __syncthreads();
        const uint32_t hi = s_bound[0], lo = min(s_bound[1], hi); int up = 0, c = 0;
#pragma unroll
        for (int i = 0; i < ITEMS; i++) { up += key[i] > hi; c += key[i] >= lo && key[i] <= hi; }
        int at = slot_for(c);
#pragma unroll
        for (int i = 0; i < ITEMS; i++) if (key[i] >= lo && key[i] <= hi) { if (at < kOwn) pool[rank * kOwn + at] = key[i]; at++; }
        up = total(up);
        for (int q = tid; q < min(s_n, kOwn); q += kSelThreads) {   // to the other CTAs
            const uint32_t k = pool[rank * kOwn + q];
            for (int r = 1; r < CS; r++) peer(&pool[0], (rank + r) % CS)[rank * kOwn + q] = k;
        }
        if (tid < CS) { peer(&s_cand[0], tid)[rank] = s_n; peer(&s_above[0], tid)[rank] = up; }
        sync_all();
        int above = 0, between = 0, most = 0;
#pragma unroll
        for (int r = 0; r < CS; r++) { above += s_above[r]; between += s_cand[r]; most = max(most, s_cand[r]); }
        const int need = keep - above;   // the need-th largest of the keys between
        found = most <= kOwn && need > 0 && need <= between;   // the same in every CTA of the cluster, as all that follows from it
        if (found) {   // in every CTA by itself: n_from >= need of them reach `from`, n_to < need reach `to`; values between are tried, a little to either side of where the counts say that the key should lie (every
            // fourth time halfway), until at most 32 keys are left for a warp to rank, or `from` is the key itself
            constexpr int N = CS * kOwn / kSelThreads;
            uint32_t k[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                int q = tid + i * kSelThreads, r = 0; k[i] = 0u;
                if (q < between) { while (q >= s_cand[r]) q -= s_cand[r++]; k[i] = pool[r * kOwn + q]; }
            }
            uint32_t from = lo, to = min(hi, 0xFF800000u) + 1u; int n_from = between, n_to = 0;   // (0xFF800000: the largest key)
#pragma unroll 1
            for (int step = 0; n_from - n_to > 32 && to - from > 1u; step++) {
                const uint32_t gap = to - from; const int past = n_from - need > need - n_to ? n_from - need - 8 : n_from - need + 8;   // keys to leave behind
                const uint32_t at = from + (step % 4 == 3 ? gap / 2 : min(max((uint32_t)((float)gap * ((float)past / (float)(n_from - n_to))), 1u), gap - 1u));
                int c[4] = {};
#pragma unroll
                for (int i = 0; i < N; i++) if (i * kSelThreads < between) add_if_ge(c[i & 3], k[i], at);
                const int n = total(c[0] + c[1] + c[2] + c[3]);
                if (n >= need) { from = at; n_from = n; } else { to = at; n_to = n; }
            }
            prefix = from; left = need - n_to;   // `from` is one of many equal keys, unless
            if (to - from > 1u) {
#pragma unroll
                for (int i = 0; i < N; i++) if (k[i] >= from && k[i] < to) sample[atomicAdd(&s_left, 1)] = k[i];
                __syncthreads();
                const uint32_t mine_k = lane < n_from - n_to ? sample[lane] : 0u; int above_k = 0;   // every warp ranks them for itself
#pragma unroll
                for (int x = 0; x < 32; x++) above_k += __shfl_sync(0xffffffffu, mine_k, x) > mine_k;
                // the largest key with fewer than `left` above it lies at rank `left`, ties included: the smallest of those
                const uint32_t best = __reduce_min_sync(0xffffffffu, mine_k && above_k < left ? mine_k : 0xffffffffu);
                const int over = __popc(__ballot_sync(0xffffffffu, mine_k > best));
                prefix = best; left -= over;
            }
        }
    }
    if (!REGS) cg::this_cluster().barrier_wait();
    if (!found) {   // ---- or by a radix select: digits of 8 bits, four histograms of 256 bins each, picked by lane (fewer lanes meet)
        for (int i = tid; i < 4 * 1024; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        uint32_t mask = 0;
#pragma unroll 1
        for (int pass = 0; pass < 4; pass++) {
            const int shift = 24 - 8 * pass; int32_t* hp = hist + pass * 1024;
            each([&](uint32_t k, int) { if (k != 0u && (k & mask) == prefix) atomicAdd(&hp[((k >> shift) & 255u) * 4 + (lane & 3)], 1); });
            sync_all();
            int c = 0;   // thread t < 256: bin 255 - t
            if (tid < 256) for (int r = 0; r < CS; r++) { const int4 v = *reinterpret_cast<const int4*>(peer(hp + (255 - tid) * 4, r)); c += v.x + v.y + v.z + v.w; }
            const int inc = warp_inclusive(c), before = warps_before(s_warp, __shfl_sync(0xffffffffu, inc, 31)) + inc - c;   // keys in higher bins
            if (tid < 256 && before < left && before + c >= left) { s_bin = 255 - tid; s_left = left - before; }
            __syncthreads();
            prefix |= (uint32_t)s_bin << shift; mask |= 255u << shift; left = s_left;
            __syncthreads();
        }
    }
    // ---- prefix is the keep-th largest key; of the slots that have it, the `left` lowest are kept
    each([&](uint32_t k, int q) {
        const uint32_t gt = __ballot_sync(0xffffffffu, k > prefix), eq = __ballot_sync(0xffffffffu, k == prefix); const int wd = q >> 5;
        if (lane == 0 && wd < words) { kept[wd] = gt; pre_h[wd] = (int32_t)eq; }
    });
    __syncthreads();
    auto ranks = [&](auto count, int32_t* pre, int32_t* sums) {   // pre[word] = sum of count over the CTA's words before it; sums[rank], in every CTA: over all of them. Thread t has words [t * per, ..)
        const int per = (words + kSelThreads - 1) / kSelThreads, lo = min(tid * per, words), hi = min(lo + per, words);
        int n = 0;
        for (int wd = lo; wd < hi; wd++) n += count(wd);
        const int inc = warp_inclusive(n); int run = warps_before(s_warp, __shfl_sync(0xffffffffu, inc, 31)) + inc - n;
        for (int wd = lo; wd < hi; wd++) { const int c = count(wd); pre[wd] = run; run += c; }
        if (tid == kSelThreads - 1) for (int r = 0; r < CS; r++) peer(sums, r)[rank] = run;
        __syncthreads();   // s_warp is used again
    };
    ranks([&](int wd) { return __popc((uint32_t)pre_h[wd]); }, pre_m, s_eq);
    sync_all();
    int taken = 0;   // slots with the threshold key in the CTAs before
    for (int r = 0; r < rank; r++) taken += s_eq[r];
    auto below = [&](int wd) { const int j = j0 + wd * 32; return j + 32 <= keep ? 0xffffffffu : j >= keep ? 0u : (1u << (keep - j)) - 1; };   // slots of a word below `keep`
    for (int wd = tid; wd < words; wd += kSelThreads) {
        uint32_t eq = (uint32_t)pre_h[wd], take = 0;
        for (int n = min(left - taken - pre_m[wd], 32); n > 0 && eq; n--) { take |= eq & (0u - eq); eq &= eq - 1; }
        kept[wd] |= take;
    }
    __syncthreads();
    ranks([&](int wd) { return __popc(~kept[wd] & below(wd)); }, pre_h, s_holes);
    ranks([&](int wd) { return __popc(kept[wd] & ~below(wd)); }, pre_m, s_movers);
    // ---- slots that stay; free slots into the list, by rank
    for (int q = tid; j0 + q < keep && q < mine; q += kSelThreads) {
        const int wd = q >> 5; const uint32_t bit = 1u << (q & 31), kp = kept[wd];
        if (kp & bit) src[j0 + q] = j0 + q; else list[pre_h[wd] + __popc(~kp & (bit - 1))] = (uint16_t)q;
    }
    sync_all();
    // ---- movers: the free slot of the same rank, wherever in the cluster it lies
    int rk0 = 0;
    for (int r = 0; r < rank; r++) rk0 += s_movers[r];
    for (int q0 = max(keep - j0, 0) + tid; q0 < mine; q0 += 4 * kSelThreads) {   // four at a time: the reads of other CTAs' lists are under way together
        int at[4]; uint32_t to[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int q = q0 + u * kSelThreads, wd = q >> 5; const uint32_t bit = 1u << (q & 31);
            at[u] = -1;
            if (q < mine && (kept[wd] & bit)) {
                int rk = rk0 + pre_m[wd] + __popc(kept[wd] & ~below(wd) & (bit - 1)), r = 0;
                while (r < CS - 1 && rk >= s_holes[r]) rk -= s_holes[r++];
                at[u] = r * wpc * 32; to[u] = peer(list, r)[rk];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++) if (at[u] >= 0) src[at[u] + to[u]] = j0 + q0 + u * kSelThreads;
    }
    sync_all();   // nobody leaves while its shared memory may still be read
}

// grid (ceil(keep / 256), kv heads * sequences, layers) x 256 threads: a warp per 32 destinations. CH: 16-byte chunks of a head row
template <int CH>
__global__ void __launch_bounds__(256) paged_move_kernel(const __grid_constant__ PagedBatch b, const __grid_constant__ EvictArgs a, uint8_t* kp, uint8_t* vp, __half* ksc, __half* vsc, const int64_t rows_per_layer) {
    pdl_wait(); pdl_launch_dependents();
    const int lane = threadIdx.x & 31, j = blockIdx.x * 256 + threadIdx.x, bi = blockIdx.y / a.kv_heads, kvh = blockIdx.y - bi * a.kv_heads, l = blockIdx.z;
    const int32_t* src = a.src + (((int64_t)l * a.n + bi) * a.kv_heads + kvh) * a.keep; const int32_t* table = a.tables + (int64_t)b.seq[bi] * a.width;
    const int from = j < a.keep ? __ldcg(src + j) : -1; const bool moves = from >= 0 && from != j;
    const int64_t row0 = (int64_t)(a.layer0 + l) * rows_per_layer; int64_t rs = 0, rd = 0;
    if (moves) {
        rs = row0 + paged_row(table, from, a.page_shift); rd = row0 + paged_row(table, j, a.page_shift);
        const int m = (1 << a.page_shift) - 1; const int64_t ws = (((rs >> a.page_shift) * a.kv_heads + kvh) << a.page_shift) + (from & m), wd = (((rd >> a.page_shift) * a.kv_heads + kvh) << a.page_shift) + (j & m);
        a.weight[wd] = a.weight[ws]; a.age[wd] = a.age[ws];
        if (ksc) { ksc[rd * a.kv_heads + kvh] = ksc[rs * a.kv_heads + kvh]; vsc[rd * a.kv_heads + kvh] = vsc[rs * a.kv_heads + kvh]; }
    }
    uint32_t todo = __ballot_sync(0xffffffffu, moves);
    // a row pair is 2 * CH chunks (K, then V): a warp copies 64 / (2 * CH) pairs per two chunks a lane, four such steps in flight
    constexpr int kPer = CH >= 32 ? 1 : 32 / CH, kU = 4;   // pairs per step; lane's pair and chunk within a step
    const int sub = lane / (CH >= 32 ? 32 : CH), ch = lane % (CH >= 32 ? 32 : CH);
    while (todo) {
        uint4 kx[kU], vx[kU]; int64_t dst[kU];
#pragma unroll
        for (int u = 0; u < kU; u++) {
            int pick = -1;
#pragma unroll
            for (int x = 0; x < kPer; x++) { const int f = todo ? __ffs(todo) - 1 : -1; if (todo) todo &= todo - 1; if (x == sub) pick = f; }
            const int64_t s = __shfl_sync(0xffffffffu, rs, pick < 0 ? 0 : pick), d = __shfl_sync(0xffffffffu, rd, pick < 0 ? 0 : pick);
            dst[u] = pick < 0 ? -1 : ((d * a.kv_heads + kvh) * CH + ch) * 16;
            if (pick >= 0) { const int64_t at = ((s * a.kv_heads + kvh) * CH + ch) * 16; kx[u] = __ldcs(reinterpret_cast<const uint4*>(kp + at)); vx[u] = __ldcs(reinterpret_cast<const uint4*>(vp + at)); }
        }
#pragma unroll
        for (int u = 0; u < kU; u++) if (dst[u] >= 0) { *reinterpret_cast<uint4*>(kp + dst[u]) = kx[u]; *reinterpret_cast<uint4*>(vp + dst[u]) = vx[u]; }
    }
}


}  // namespace

cudaError_t configure_paged_evict(const PagedCtx&) {   // shared-memory opt-in, per device
    cudaError_t e = cudaFuncSetAttribute(paged_select_cluster_kernel<8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCluMax / 32 / kSelCluster * 76);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_select_cluster_kernel<0>, cudaFuncAttributeMaxDynamicSharedMemorySize, KATA_PAGED_MAX_SLOTS / 32 / kSelCluster * 76);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(paged_select_cluster_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * kCluMax / 32 / kSelCluster * 76);
}

cudaError_t launch_paged_evict(PagedCtx& c, int layer, int n_layers, const PagedBatch& b, int keep, int sink, int recent, int32_t* src, cudaStream_t s) {
    EvictArgs a{}; a.keep = keep; a.sink = sink; a.recent = recent; a.width = c.width; a.page_shift = c.page_shift; a.kv_heads = c.cfg.kv_heads; a.n = b.n; a.layer0 = layer;
    a.plane_stride = c.rows_per_layer * c.cfg.kv_heads; a.tables = c.d_table; a.weight = (float*)c.plane[KATA_PAGED_WEIGHT]; a.age = (int32_t*)c.plane[KATA_PAGED_AGE]; a.src = src;
    int most = 0; for (int i = 0; i < b.n; i++) most = std::max(most, b.slot[i]);
    cudaError_t e;
    const int64_t segments = (int64_t)c.cfg.kv_heads * b.n * n_layers;
    if (most <= kSelOne || (most <= kCluMax && segments >= kSelMany)) {
        const dim3 grid(c.cfg.kv_heads, b.n, n_layers);
#define KATA_SELECT(N) launch_pdl(paged_select_kernel<N>, grid, dim3(kSelThreads), 0, s, b, a)
        const int items = (most + kSelThreads - 1) / kSelThreads;
        static_assert(kCluMax == 64 * kSelThreads, "the largest variant holds what a cluster holds");
        e = items <= 2 ? KATA_SELECT(2) : items <= 10 ? KATA_SELECT(10) : items <= 24 ? KATA_SELECT(24) : KATA_SELECT(64);
#undef KATA_SELECT
    } else {
        const int wpc = ((most + 31) / 32 + kSelCluster - 1) / kSelCluster;
        static_assert(KATA_PAGED_MAX_SLOTS / kSelCluster <= 65536 && kCluSlots % (32 * kSelCluster) == 0, "free slots are listed with 16 bits");
        cudaLaunchConfig_t cfg{}; cfg.gridDim = dim3(kSelCluster * c.cfg.kv_heads, b.n, n_layers); cfg.blockDim = dim3(kSelThreads); cfg.dynamicSmemBytes = (size_t)wpc * 76; cfg.stream = s;
        cudaLaunchAttribute at[2]; at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; at[0].val.programmaticStreamSerializationAllowed = 1;
        at[1].id = cudaLaunchAttributeClusterDimension; at[1].val.clusterDim.x = kSelCluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
        cfg.attrs = at; cfg.numAttrs = 2;
        e = most <= kCluMax ? cudaLaunchKernelEx(&cfg, paged_select_cluster_kernel<8>, b, a, wpc) : most <= 4 * kCluMax ? cudaLaunchKernelEx(&cfg, paged_select_cluster_kernel<32>, b, a, wpc) : cudaLaunchKernelEx(&cfg, paged_select_cluster_kernel<0>, b, a, wpc);
    }
    if (e != cudaSuccess) return e;
    c.launches++;
    if (most <= keep) return cudaGetLastError();   // nothing to move in any sequence
    auto move = [&](auto kernel) {
        return launch_pdl(kernel, dim3((keep + 255) / 256, c.cfg.kv_heads * b.n, n_layers), dim3(256), 0, s, b, a, (uint8_t*)c.plane[KATA_PAGED_K], (uint8_t*)c.plane[KATA_PAGED_V], (__half*)c.plane[KATA_PAGED_K_SCALE], (__half*)c.plane[KATA_PAGED_V_SCALE], c.rows_per_layer);
    };
    const int chunks = c.cfg.head_dim * c.elt / 16;
    e = chunks == 32 ? move(paged_move_kernel<32>) : chunks == 16 ? move(paged_move_kernel<16>) : move(paged_move_kernel<8>);
    if (e != cudaSuccess) return e;
    c.launches++;
    return cudaGetLastError();
}

}  // namespace kata
