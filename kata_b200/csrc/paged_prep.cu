// The kernel that appends to a paged cache (kata_paged_prep): per-head RMSNorm, rotary positions with up to three axes, gate split, the fp16
// prescaled query, and the K and V rows written (or quantised) into their pages; and the copy of contiguous rows into pages (kata_paged_import).
//
// Memory-bound: 57 KB in and 40 KB out per token of the 24 / 4 x 256 layout with fp32 activations. One warp per (head slot, token) row, 8 (or 4) consecutive dims per lane, so that
// every access is a 128-bit one and the rotary pair (i, i + rot_dim / 2) is a fixed distance in lanes apart.
// Angles: a position p turns frequency i by p * theta^(-2i / rot_dim) / 2 pi circles. The fraction of a circle is p * F_i mod 2^64 with F_i the 64-bit
// fixed-point value of one position's turn: one integer product, exact modulo whole turns, so far positions are as accurate as near ones
// (p * 2^-65 circles from the rounding of F_i). sincospif then takes the top 32 bits as a signed fraction.
#include <cmath>
#include <type_traits>

#include "paged_internal.cuh"

namespace kata {

bool make_rot_tab(RotTab& t, int rot_dim, double theta, const int32_t* section, int interleaved) {
    const int n = rot_dim / 2;
    if (rot_dim < 0 || rot_dim % 2 || n > kPagedMaxRot || section[0] < 0 || section[1] < 0 || section[2] < 0 || (int64_t)section[0] + section[1] + section[2] != n) return false;
    if (n && !(theta > 0.0 && std::isfinite(theta))) return false;
    t = RotTab{};
    int count[3] = {0, 0, 0};
    for (int i = 0; i < n; i++) {
        const int a = i % 3;
        t.axis[i] = interleaved ? ((a && i < 3 * section[a]) ? a : 0) : i < section[0] ? 0 : i < section[0] + section[1] ? 1 : 2;
        count[t.axis[i]]++;
        const long double turns = powl((long double)theta, -(long double)i / n) / 6.283185307179586476925286766559L;
        const long double frac = turns - floorl(turns);
        t.freq[i] = (uint64_t)(int64_t)llrintl((frac >= 0.5L ? frac - 1.0L : frac) * 18446744073709551616.0L);   // modulo one turn
    }
    return count[0] == section[0] && count[1] == section[1] && count[2] == section[2];
}

namespace {

struct PrepArgs {
    int T, width, page_shift, heads, kv_heads, rot_half, gated, first_slot;   // first_slot: heads when only K and V are appended, else 0
    float q_scale;
    const int32_t* axis_pos; const int32_t* tables; const RotTab* rot;
    const void* q; const void* k; const void* v; const float* qnorm; const float* knorm;
    __half* q16; float* gate; void* kp; void* vp; __half* ksc; __half* vsc; float* weight; int32_t* age;   // the planes of the layer
};

template <typename T, int N> __device__ __forceinline__ void load_dims(const T* p, float (&v)[N]) {   // N consecutive elements, N * sizeof(T) a multiple of 8 bytes
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) { const float4 f = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i); v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w; }
    } else {
        uint32_t u[N / 2];
        if (N == 8) { const uint4 x = *reinterpret_cast<const uint4*>(p); u[0] = x.x; u[1] = x.y; u[N / 2 - 2] = x.z; u[N / 2 - 1] = x.w; }
        else { const uint2 x = *reinterpret_cast<const uint2*>(p); u[0] = x.x; u[1] = x.y; }
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            float2 f;
            if (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
}
template <int N> __device__ __forceinline__ void store_half(__half* p, const float (&v)[N]) {
    uint32_t u[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; i++) { const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]); u[i] = *reinterpret_cast<const uint32_t*>(&h); }
    if (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[N / 2 - 2], u[N / 2 - 1]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
}
// symmetric int8 codes of a head row (rounded to fp16 first) and its scale: the arithmetic of the contiguous cache's quantiser, bit for bit
template <int N> __device__ __forceinline__ void store_int8(int8_t* p, __half* scale, const float (&x)[N], int lane) {
    float v[N], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) { v[i] = __half2float(__float2half_rn(x[i])); amax = fmaxf(amax, fabsf(v[i])); }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    const __half sc = amax > 0.0f ? __float2half_rn(__fdiv_rn(amax, 127.0f)) : __float2half_rn(1.0f);
    const float inv = __fdiv_rn(1.0f, __half2float(sc));
    uint32_t u[N / 4] = {};
#pragma unroll
    for (int i = 0; i < N; i++) u[i >> 2] |= ((uint32_t)(int)fminf(fmaxf(rintf(__fmul_rn(v[i], inv)), -127.0f), 127.0f) & 0xffu) << (8 * (i & 3));
    if (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[N / 4 - 1]); else *reinterpret_cast<uint32_t*>(p) = u[0];
    if (lane == 0) *scale = sc;
}

// grid (ceil(head slots / 8), T, sequences) x 256 threads: warp w handles one head slot (queries, then keys, then values) of one token
template <typename TIn, int HD, bool K8>
__global__ void __launch_bounds__(256) paged_prep_kernel(const __grid_constant__ PagedBatch b, const __grid_constant__ PrepArgs a) {
    constexpr int N = HD / 32;   // dims per lane
    __shared__ float s_sin[kPagedMaxRot], s_cos[kPagedMaxRot];
    const int tid = threadIdx.x, lane = tid & 31, h = a.first_slot + blockIdx.x * 8 + (tid >> 5), t = blockIdx.y, bi = blockIdx.z;
    uint64_t freq = 0; int axis = 0;
    if (tid < a.rot_half) { freq = a.rot->freq[tid]; axis = a.rot->axis[tid]; }   // written once, at creation: read ahead of the wait
    pdl_wait(); pdl_launch_dependents();
    const int64_t tok = (int64_t)bi * a.T + t;
    const bool live = h < a.heads + 2 * a.kv_heads, is_q = h < a.heads, is_k = !is_q && h < a.heads + a.kv_heads;
    const int hh = is_q ? h : is_k ? h - a.heads : h - a.heads - a.kv_heads;
    float v[N], gt[N], w[N];
    if (live) {
        const TIn* src = is_q ? reinterpret_cast<const TIn*>(a.q) + (tok * a.heads + hh) * (a.gated ? 2 * HD : HD) : reinterpret_cast<const TIn*>(is_k ? a.k : a.v) + (tok * a.kv_heads + hh) * HD;
        load_dims<TIn, N>(src + lane * N, v);
        if (is_q && a.gate) load_dims<TIn, N>(src + HD + lane * N, gt);
        if (is_q || is_k) load_dims<float, N>((is_q ? a.qnorm : a.knorm) + lane * N, w);
    }
    if (tid < a.rot_half) {
        const int pos = a.axis_pos ? __ldg(a.axis_pos + tok * 3 + axis) : b.age[bi] + t;
        const float turn = (float)(int32_t)((freq * (uint64_t)(int64_t)pos) >> 32) * 0x1p-31f;   // in half circles, [-1, 1)
        sincospif(turn, &s_sin[tid], &s_cos[tid]);
    }
    __syncthreads();
    if (!live) return;
    const int slot = b.slot[bi] + t; const int64_t row = paged_row(a.tables + (int64_t)b.seq[bi] * a.width, slot, a.page_shift);
    if (is_q || is_k) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) sum = fmaf(v[i], v[i], sum);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const float r = __fdiv_rn(1.0f, __fsqrt_rn(sum * (1.0f / HD) + kEps));
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = v[i] * r * w[i];
        const int lanes = a.rot_half / N;   // lanes of the first half of the rotated dims
        if (lanes) {
            const bool lo = lane < lanes, hi = !lo && lane < 2 * lanes; const int partner = lo ? lane + lanes : hi ? lane - lanes : lane, f0 = (lo ? lane : hi ? lane - lanes : 0) * N;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float o = __shfl_sync(0xffffffffu, v[i], partner), sn = s_sin[f0 + i], cs = s_cos[f0 + i];
                if (lo) v[i] = v[i] * cs - o * sn; else if (hi) v[i] = o * sn + v[i] * cs;
            }
        }
    }
    if (is_q) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] *= a.q_scale;
        store_half<N>(a.q16 + (tok * a.heads + hh) * HD + lane * N, v);
        if (a.gate) {
            float4* dst = reinterpret_cast<float4*>(a.gate + (tok * a.heads + hh) * HD + lane * N);
#pragma unroll
            for (int i = 0; i < N; i += 4) dst[i / 4] = make_float4(gt[i], gt[i + 1], gt[i + 2], gt[i + 3]);
        }
        return;
    }
    const int64_t at = (row * a.kv_heads + hh) * HD + lane * N;
    if (K8) store_int8<N>(reinterpret_cast<int8_t*>(is_k ? a.kp : a.vp) + at, (is_k ? a.ksc : a.vsc) + row * a.kv_heads + hh, v, lane);
    else store_half<N>(reinterpret_cast<__half*>(is_k ? a.kp : a.vp) + at, v);
    if (is_k && a.weight && lane == 0) {   // a new key has received nothing yet
        const int off = slot & ((1 << a.page_shift) - 1); const int64_t wi = (((row >> a.page_shift) * a.kv_heads + hh) << a.page_shift) + off;
        a.weight[wi] = 0.0f; a.age[wi] = b.age[bi] + t;
    }
}

// one warp per (slot, KV head): K and V head rows and their scales from a contiguous arena [row][4][256] into the slot's page
template <bool K8>
__global__ void __launch_bounds__(128) paged_import_kernel(const int32_t* __restrict__ table, const int page_shift, const int slot0, const int age0, const int64_t src_row, const uint8_t* __restrict__ sk, const uint8_t* __restrict__ sv,
                                                           const __half* __restrict__ sks, const __half* __restrict__ svs, uint8_t* kp, uint8_t* vp, __half* ksc, __half* vsc, float* weight, int32_t* age) {
    constexpr int kBytes = K8 ? 256 : 512;
    const int lane = threadIdx.x & 31, hh = threadIdx.x >> 5, slot = slot0 + blockIdx.x; const int64_t row = paged_row(table, slot, page_shift), sr = src_row + blockIdx.x;
    if (lane * 16 < kBytes) {
        *reinterpret_cast<uint4*>(kp + (row * 4 + hh) * kBytes + lane * 16) = *reinterpret_cast<const uint4*>(sk + (sr * 4 + hh) * kBytes + lane * 16);
        *reinterpret_cast<uint4*>(vp + (row * 4 + hh) * kBytes + lane * 16) = *reinterpret_cast<const uint4*>(sv + (sr * 4 + hh) * kBytes + lane * 16);
    }
    if (lane == 0) {
        if (K8) { ksc[row * 4 + hh] = sks[sr * 4 + hh]; vsc[row * 4 + hh] = svs[sr * 4 + hh]; }
        if (weight) { const int64_t wi = (((row >> page_shift) * 4 + hh) << page_shift) + (slot & ((1 << page_shift) - 1)); weight[wi] = 0.0f; age[wi] = age0 + blockIdx.x; }
    }
}

}  // namespace

cudaError_t launch_paged_prep(PagedCtx& c, int layer, const PagedBatch& b, int T, const int32_t* axis_pos, const void* q, const void* k, const void* v, int act_dtype,
                              const float* qnorm, const float* knorm, __half* q16, float* gate, cudaStream_t s) {
    PrepArgs a{}; a.T = T; a.width = c.width; a.page_shift = c.page_shift; a.heads = c.cfg.heads; a.kv_heads = c.cfg.kv_heads; a.rot_half = c.cfg.rot_dim / 2; a.gated = (c.cfg.flags & KATA_PAGED_GATED) ? 1 : 0;
    a.first_slot = q ? 0 : c.cfg.heads; a.q_scale = (float)(1.0 / std::sqrt((double)c.cfg.head_dim));
    a.axis_pos = axis_pos; a.tables = c.d_table; a.rot = c.d_rot; a.q = q; a.k = k; a.v = v; a.qnorm = qnorm; a.knorm = knorm; a.q16 = q16; a.gate = gate;
    a.kp = c.layer_plane(KATA_PAGED_K, layer); a.vp = c.layer_plane(KATA_PAGED_V, layer); a.ksc = (__half*)c.layer_plane(KATA_PAGED_K_SCALE, layer); a.vsc = (__half*)c.layer_plane(KATA_PAGED_V_SCALE, layer);
    a.weight = (float*)c.layer_plane(KATA_PAGED_WEIGHT, layer); a.age = (int32_t*)c.layer_plane(KATA_PAGED_AGE, layer);
    const dim3 grid((c.cfg.heads + 2 * c.cfg.kv_heads - a.first_slot + 7) / 8, T, b.n), block(256);
    cudaError_t e = cudaErrorInvalidValue;
#define X(KIND, TIN) if (act_dtype == KIND) e = c.cfg.head_dim == 256 ? (c.int8() ? launch_pdl(paged_prep_kernel<TIN, 256, true>, grid, block, 0, s, b, a) : launch_pdl(paged_prep_kernel<TIN, 256, false>, grid, block, 0, s, b, a)) \
                                                                     : (c.int8() ? launch_pdl(paged_prep_kernel<TIN, 128, true>, grid, block, 0, s, b, a) : launch_pdl(paged_prep_kernel<TIN, 128, false>, grid, block, 0, s, b, a));
    X(KATA_ACT_F32, float) X(KATA_ACT_BF16, __nv_bfloat16) X(KATA_ACT_F16, __half)
#undef X
    if (e != cudaSuccess) return e;
    c.launches++;
    return cudaGetLastError();
}

cudaError_t launch_paged_import(PagedCtx& c, int layer, int seq, int slot0, int n_rows, int age0, const Ctx& src, int64_t src_row, cudaStream_t s) {
    const int32_t* table = c.d_table + (int64_t)seq * c.width;
    auto go = [&](auto kernel) {
        kernel<<<n_rows, 128, 0, s>>>(table, c.page_shift, slot0, age0, src_row, (const uint8_t*)src.k_arena, (const uint8_t*)src.v_arena, src.ksc, src.vsc, (uint8_t*)c.layer_plane(KATA_PAGED_K, layer), (uint8_t*)c.layer_plane(KATA_PAGED_V, layer),
                                      (__half*)c.layer_plane(KATA_PAGED_K_SCALE, layer), (__half*)c.layer_plane(KATA_PAGED_V_SCALE, layer), (float*)c.layer_plane(KATA_PAGED_WEIGHT, layer), (int32_t*)c.layer_plane(KATA_PAGED_AGE, layer));
    };
    if (c.int8()) go(paged_import_kernel<true>); else go(paged_import_kernel<false>);
    c.launches++;
    return cudaGetLastError();
}

}  // namespace kata
