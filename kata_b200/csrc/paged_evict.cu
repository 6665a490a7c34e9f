// Eviction from a paged cache by accumulated attention weight (kata_paged_evict): per layer, sequence and KV head the `keep` heaviest slots stay.
//   key(slot) = +inf for protected slots (age < sink or age >= seen - recent), else the weight; order: key descending, then slot ascending.
// Slots kept below `keep` stay where they are; the i-th kept slot at or behind `keep` moves into the i-th free slot below it. Every row that moves is read
// behind `keep` and written below it, so no order of the copies can clobber one, and as few rows move as can.
//
// select: one CTA per (layer, sequence, KV head). Weights as order-preserving 32-bit integers, kept in shared memory when they fit; the keep-th largest by a radix select over digits of
// 11, 11 and 10 bits; then bit masks of the slots (32 per word) with prefix sums per word give every free slot its rank and every rank its mover.
// move: a warp per 32 destinations, lanes agreeing by ballot on those that receive a row; each row is 16-byte copies of K and V. Bound by HBM: 2 x row bytes per move.
#include <algorithm>

#include "paged_internal.cuh"

namespace kata {
namespace {

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32, kBins = 2048;
constexpr int kSelSmemMax = 222 * 1024;

struct EvictArgs {
    int keep, sink, recent, width, page_shift, kv_heads, n, layer0;
    int64_t plane_stride;                 // elements of a weight / age plane of one layer
    const int32_t* tables; float* weight; int32_t* age; int32_t* src;
};

__device__ __forceinline__ uint32_t order_key(float w) {   // larger float, larger integer; NaN below everything; -0 = +0
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// exclusive prefix sums over x[0, n) in place, by the whole block; returns the total to every thread
__device__ int block_exclusive_scan(int32_t* x, int n, int32_t* s_warp) {
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, per = (n + kSelThreads - 1) / kSelThreads, lo = min(tid * per, n), hi = min(lo + per, n);
    int sum = 0;
    for (int i = lo; i < hi; i++) sum += x[i];
    int inc = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) { const int o = __shfl_up_sync(0xffffffffu, inc, off); if (lane >= off) inc += o; }
    if (lane == 31) s_warp[w] = inc;
    __syncthreads();
    if (w == 0) {
        int v = s_warp[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) { const int o = __shfl_up_sync(0xffffffffu, v, off); if (lane >= off) v += o; }
        s_warp[lane] = v;
    }
    __syncthreads();
    int run = inc - sum + (w ? s_warp[w - 1] : 0); const int total = s_warp[kSelWarps - 1];
    for (int i = lo; i < hi; i++) { const int c = x[i]; x[i] = run; run += c; }
    __syncthreads();
    return total;
}

// grid (kv heads, sequences, layers)
__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(const __grid_constant__ PagedBatch b, const __grid_constant__ EvictArgs a, const int words_cap, const int cached) {
    extern __shared__ __align__(16) uint32_t dyn[];
    uint32_t* kept = dyn; int32_t* pre_h = reinterpret_cast<int32_t*>(dyn + words_cap); int32_t* pre_m = pre_h + words_cap; uint32_t* keys = dyn + 3 * words_cap;   // keys: when cached
    __shared__ int32_t hist[kBins]; __shared__ int32_t s_warp[kSelWarps]; __shared__ int s_bin, s_left;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, kvh = blockIdx.x, bi = blockIdx.y, l = blockIdx.z, S = b.slot[bi], seen = b.age[bi], keep = a.keep;
    pdl_wait(); pdl_launch_dependents();
    int32_t* src = a.src + (((int64_t)l * a.n + bi) * a.kv_heads + kvh) * keep;
    if (S <= keep) { for (int j = tid; j < keep; j += kSelThreads) src[j] = j < S ? j : -1; return; }
    const int32_t* table = a.tables + (int64_t)b.seq[bi] * a.width; const float* weight = a.weight + (int64_t)(a.layer0 + l) * a.plane_stride; const int32_t* age = a.age + (int64_t)(a.layer0 + l) * a.plane_stride;
    const int newest = seen - a.recent;   // ages from here on are protected
    auto load_key = [&](int j) {
        const int64_t at = (((int64_t)__ldcg(table + (j >> a.page_shift)) * a.kv_heads + kvh) << a.page_shift) + (j & ((1 << a.page_shift) - 1));
        const int ag = __ldcg(age + at);
        return (ag < a.sink || ag >= newest) ? 0xFF800000u : order_key(__ldcg(weight + at));   // 0xFF800000: the key of +inf
    };
    auto key_of = [&](int j) { return cached ? keys[j] : load_key(j); };
    if (cached) for (int j = tid; j < S; j += kSelThreads) keys[j] = load_key(j);
    // ---- the keep-th largest key
    uint32_t prefix = 0, prefix_mask = 0; int left = keep;   // left: how many of the keys that match the prefix are kept
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int j = tid; j < S; j += kSelThreads) { const uint32_t k = key_of(j); if ((k & prefix_mask) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1); }
        __syncthreads();
        // the bin, from the top, in which the count passes `left`: thread t owns bins 2t and 2t + 1 counted from the top
        const int top0 = hist[kBins - 1 - 2 * tid], top1 = hist[kBins - 2 - 2 * tid]; int inc = top0 + top1;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) { const int o = __shfl_up_sync(0xffffffffu, inc, off); if (lane >= off) inc += o; }
        if (lane == 31) s_warp[w] = inc;
        __syncthreads();
        if (w == 0) {
            int v = s_warp[lane];
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) { const int o = __shfl_up_sync(0xffffffffu, v, off); if (lane >= off) v += o; }
            s_warp[lane] = v;
        }
        __syncthreads();
        const int before = inc - top0 - top1 + (w ? s_warp[w - 1] : 0);   // keys in higher bins than this thread's
        if (before < left && before + top0 >= left) { s_bin = kBins - 1 - 2 * tid; s_left = left - before; }
        else if (before + top0 < left && before + top0 + top1 >= left) { s_bin = kBins - 2 - 2 * tid; s_left = left - before - top0; }
        __syncthreads();
        prefix |= (uint32_t)s_bin << shift; prefix_mask |= ((1u << bits) - 1) << shift; left = s_left;
        __syncthreads();
    }
    // prefix is the keep-th largest key; of the slots that have it, the `left` lowest are kept
    const int words = (S + 31) >> 5;
    for (int wd = w; wd < words; wd += kSelWarps) {
        const int j = wd * 32 + lane; const uint32_t k = j < S ? key_of(j) : 0u;
        const uint32_t gt = __ballot_sync(0xffffffffu, j < S && k > prefix), eq = __ballot_sync(0xffffffffu, j < S && k == prefix);
        if (lane == 0) { kept[wd] = gt; pre_h[wd] = (int32_t)eq; pre_m[wd] = __popc(eq); }
    }
    __syncthreads();
    block_exclusive_scan(pre_m, words, s_warp);
    for (int wd = tid; wd < words; wd += kSelThreads) {
        uint32_t eq = (uint32_t)pre_h[wd], take = 0;
        for (int n = min(left - pre_m[wd], 32); n > 0 && eq; n--) { take |= eq & (0u - eq); eq &= eq - 1; }
        const uint32_t kp = kept[wd] | take; kept[wd] = kp;
        const int j0 = wd * 32; const uint32_t below = j0 + 32 <= keep ? 0xffffffffu : j0 >= keep ? 0u : (1u << (keep - j0)) - 1;   // slots of this word below `keep`
        pre_h[wd] = __popc(~kp & below); pre_m[wd] = __popc(kp & ~below);
    }
    __syncthreads();
    block_exclusive_scan(pre_h, words, s_warp);
    block_exclusive_scan(pre_m, words, s_warp);
    for (int j = tid; j < keep; j += kSelThreads) {
        const int wd = j >> 5; const uint32_t bit = 1u << (j & 31), kp = kept[wd];
        int from = j;
        if (!(kp & bit)) {
            const int r = pre_h[wd] + __popc(~kp & (bit - 1));   // its rank among the free slots: the mover of that rank comes here
            int lo = keep >> 5, hi = words - 1;                  // the last word whose movers start at or before rank r
            while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (pre_m[mid] <= r) lo = mid; else hi = mid - 1; }
            uint32_t mv = kept[lo] & (lo * 32 >= keep ? 0xffffffffu : ~((1u << (keep - lo * 32)) - 1));
            for (int n = r - pre_m[lo]; n > 0; n--) mv &= mv - 1;
            from = lo * 32 + __ffs(mv) - 1;
        }
        src[j] = from;
    }
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

cudaError_t configure_paged_evict(const PagedCtx&) { return cudaFuncSetAttribute(paged_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelSmemMax - kBins * 4 - 1024); }

cudaError_t launch_paged_evict(PagedCtx& c, int layer, int n_layers, const PagedBatch& b, int keep, int sink, int recent, int32_t* src, cudaStream_t s) {
    EvictArgs a{}; a.keep = keep; a.sink = sink; a.recent = recent; a.width = c.width; a.page_shift = c.page_shift; a.kv_heads = c.cfg.kv_heads; a.n = b.n; a.layer0 = layer;
    a.plane_stride = c.rows_per_layer * c.cfg.kv_heads; a.tables = c.d_table; a.weight = (float*)c.plane[KATA_PAGED_WEIGHT]; a.age = (int32_t*)c.plane[KATA_PAGED_AGE]; a.src = src;
    int most = 0; for (int i = 0; i < b.n; i++) most = std::max(most, b.slot[i]);
    const int words = (most + 31) / 32, budget = kSelSmemMax - kBins * 4 - 1024, cached = words * 12 + words * 128 <= budget ? 1 : 0;   // keys of up to some 48,000 slots are kept in shared memory, else read again in every pass
    cudaError_t e = launch_pdl(paged_select_kernel, dim3(c.cfg.kv_heads, b.n, n_layers), dim3(kSelThreads), (size_t)words * (cached ? 140 : 12), s, b, a, words, cached);
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
