// The kernel that appends to a paged cache (kata_paged_prep): per-head RMSNorm, rotary positions with up to three axes, gate split, the fp16
// prescaled query, and the K and V rows written (or quantised) into their pages; and the copy of contiguous rows into pages (kata_paged_import).
//
// Memory-bound: 57 KB in and 40 KB out per token of the 24 / 4 x 256 layout with fp32 activations. One warp per (head slot, token) row, 8 (or 4) consecutive dims per lane, so that
// every access is a 128-bit one and the rotary pair (i, i + rot_dim / 2) is a fixed distance in lanes apart.
// Angles: a position p turns frequency i by p * theta^(-2i / rot_dim) / 2 pi circles. The fraction of a circle is p * F_i mod 2^64 with F_i the 64-bit
// fixed-point value of one position's turn: one integer product, exact modulo whole turns, so far positions are as accurate as near ones
// (p * 2^-65 circles from the rounding of F_i). sincospif then takes the top 32 bits as a signed fraction.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_internal.cuh"

namespace kata {

bool make_rot_tab(RotTab& t, int rot_dim, double theta, const int32_t* section, int interleaved) {
    const int n = rot_dim / 2;
    if (rot_dim < 0 || rot_dim % 2 || n > kPagedMaxRot) return false;
    if (n && !(theta > 0.0 && std::isfinite(theta))) return false;
    t = RotTab{};
    if (!rotary_axes(n, section, interleaved, t.axis)) return false;
    for (int i = 0; i < n; i++) {
        const long double turns = powl((long double)theta, -(long double)i / n) / 6.283185307179586476925286766559L;
        const long double frac = turns - floorl(turns);
        t.freq[i] = (uint64_t)(int64_t)llrintl((frac >= 0.5L ? frac - 1.0L : frac) * 18446744073709551616.0L);   // modulo one turn
    }
    return true;
}

namespace {

struct PrepArgs {
    int T, width, page_shift, heads, kv_heads, rot_half, gated, first_slot;   // first_slot: heads when only K and V are appended, else 0
    float q_scale;
    const int32_t* axis_pos; const int32_t* tables; const RotTab* rot;
    const void* q; const void* k; const void* v; const float* qnorm; const float* knorm;
    __half* q16; float* gate; void* kp; void* vp; __half* ksc; __half* vsc; float* weight; int32_t* age;   // the planes of the layer
};

// N consecutive elements as they lie (8 to 32 bytes), and as fp32
template <typename T, int N> struct Raw { uint32_t u[N * sizeof(T) / 4]; };
template <typename T, int N> __device__ __forceinline__ void load_raw(const T* p, Raw<T, N>& r) {
    constexpr int W = N * sizeof(T) / 4;
    if constexpr (W == 2) { const uint2 x = __ldcs(reinterpret_cast<const uint2*>(p)); r.u[0] = x.x; r.u[1] = x.y; }
    else {
#pragma unroll
        for (int i = 0; i < W; i += 4) { const uint4 x = __ldcs(reinterpret_cast<const uint4*>(p) + i / 4); r.u[i] = x.x; r.u[i + 1] = x.y; r.u[i + 2] = x.z; r.u[i + 3] = x.w; }
    }
}
template <typename T, int N> __device__ __forceinline__ void to_float(const Raw<T, N>& r, float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = __uint_as_float(r.u[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            if constexpr (std::is_same<T, __half>::value) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.u[i])); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
            else { v[2 * i] = __uint_as_float(r.u[i] << 16); v[2 * i + 1] = __uint_as_float(r.u[i] & 0xffff0000u); }   // bf16: the upper half of an fp32
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

// grid (G, T, sequences) x 256 threads: warp w of CTA g handles head slots 8 * g + w, + 8 * G, ... (queries, then keys, then values) of a token, ROWS of them at a time: it requests all their rows (32
// registers as they lie) before it works on the first, since what bounds the kernel is the bytes under way. 8 x 1024 tokens in bf16 (570 MB): 137 us with a row per warp and a CTA per 8 rows, 143 with a
// row ahead, 106 us so (5.4 TB/s); in fp32 (800 MB) 130 us (6.2 TB/s). A persistent form that requests the next token's rows while it works on one took 149 us: its registers spill, and its warps wait for one
// another. Three CTAs per SM (80 registers): with two, the int8 path's own choice, its 8 x 509 tokens took 70 us instead of 57. The CTA forms the token's sines and cosines once, while the
// rows are under way. G = 4 when there are so few tokens that their CTAs fit the GPU at once anyway (one token: 2.7 us, 4.4 with G = 1), else 1.
template <typename TIn, int HD, bool K8>
__global__ void __launch_bounds__(256, 3) paged_prep_kernel(const __grid_constant__ PagedBatch b, const __grid_constant__ PrepArgs a) {
    constexpr int N = HD / 32, ROWS = 64 / (N * (int)sizeof(TIn));   // dims per lane; rows and their gates in 32 registers
    __shared__ float s_sin[kPagedMaxRot], s_cos[kPagedMaxRot];
    const int tid = threadIdx.x, lane = tid & 31, t = blockIdx.y, bi = blockIdx.z, n_slots = a.heads + 2 * a.kv_heads, step = 8 * gridDim.x;
    uint64_t freq = 0; int axis = 0;
    if (tid < a.rot_half) { freq = a.rot->freq[tid]; axis = a.rot->axis[tid]; }   // written once, at creation: read ahead of the wait
    pdl_wait(); pdl_launch_dependents();
    const int64_t tok = (int64_t)bi * a.T + t;
    const int q_row = a.gated ? 2 * HD : HD, n_q = a.heads, n_qk = a.heads + a.kv_heads;
    const TIn* q = reinterpret_cast<const TIn*>(a.q) + tok * n_q * q_row + lane * N;                                           // head h: + h * q_row
    const TIn* k = reinterpret_cast<const TIn*>(a.k) + (tok * a.kv_heads - n_q) * HD + lane * N;                               // head slot h: + h * HD
    const TIn* v = reinterpret_cast<const TIn*>(a.v) + (tok * a.kv_heads - n_qk) * HD + lane * N;
    Raw<TIn, N> row_raw[ROWS], gate_raw[ROWS];
    auto load_rows = [&](int h0) {
#pragma unroll
        for (int x = 0; x < ROWS; x++) {
            const int h = h0 + x * step;
            if (h < n_q) {
                load_raw<TIn, N>(q + h * q_row, row_raw[x]);
                if (a.gate) load_raw<TIn, N>(q + h * q_row + HD, gate_raw[x]);
            } else if (h < n_slots) load_raw<TIn, N>((h < n_qk ? k : v) + h * HD, row_raw[x]);
        }
    };
    int h0 = a.first_slot + 8 * blockIdx.x + (tid >> 5);
    load_rows(h0);
    const int slot = b.slot[bi] + t; const int64_t row = paged_row(a.tables + (int64_t)b.seq[bi] * a.width, slot, a.page_shift);
    if (tid < a.rot_half) {
        const int pos = a.axis_pos ? __ldcg(a.axis_pos + tok * 3 + axis) : b.age[bi] + t;
        const float turn = (float)(int32_t)((freq * (uint64_t)(int64_t)pos) >> 32) * 0x1p-31f;   // in half circles, [-1, 1)
        sincospif(turn, &s_sin[tid], &s_cos[tid]);
    }
    __syncthreads();
    // A lane's factors, the same for every row: x <- x * cs + (its partner's x) * sn, with sn negated for the first of a pair and 1 and 0 for dims that are not rotated
    const int lanes = a.rot_half / N; const bool lo = lane < lanes, hi = !lo && lane < 2 * lanes; const int partner = lo ? lane + lanes : hi ? lane - lanes : lane;
    float cs[N], sn[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int f = (lo ? lane : lane - lanes) * N + i;
        cs[i] = (lo || hi) ? s_cos[f] : 1.0f; sn[i] = lo ? -s_sin[f] : hi ? s_sin[f] : 0.0f;
    }
    __half* q16 = a.q16 + tok * n_q * HD + lane * N; float* gate = a.gate + tok * n_q * HD + lane * N;
    for (; h0 < n_slots; h0 += ROWS * step) {
#pragma unroll
        for (int x = 0; x < ROWS; x++) {
            const int h = h0 + x * step;
            if (h >= n_slots) break;
            float f[N];
            if (h < n_q && a.gate) {
                to_float<TIn, N>(gate_raw[x], f);
#pragma unroll
                for (int i = 0; i < N; i += 4) __stcs(reinterpret_cast<float4*>(gate + h * HD + i), make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]));
            }
            to_float<TIn, N>(row_raw[x], f);
            if (h < n_qk) {
                const float4* ws = reinterpret_cast<const float4*>((h < n_q ? a.qnorm : a.knorm) + lane * N);
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < N; i++) sum = fmaf(f[i], f[i], sum);
#pragma unroll
                for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                const float r = rsqrtf(sum * (1.0f / HD) + kEps) * (h < n_q ? a.q_scale : 1.0f);   // rsqrtf: off by at most two units in the last place
#pragma unroll
                for (int i = 0; i < N; i += 4) { const float4 w = __ldg(ws + i / 4); f[i] *= r * w.x; f[i + 1] *= r * w.y; f[i + 2] *= r * w.z; f[i + 3] *= r * w.w; }
                if (lanes) {
#pragma unroll
                    for (int i = 0; i < N; i++) { const float o = __shfl_sync(0xffffffffu, f[i], partner); f[i] = fmaf(o, sn[i], f[i] * cs[i]); }
                }
                if (h < n_q) { store_half<N>(q16 + h * HD, f); continue; }
            }
            const bool is_k = h < n_qk; const int hh = h - (is_k ? n_q : n_qk); const int64_t at = (row * a.kv_heads + hh) * HD + lane * N;
            if (K8) store_int8<N>(reinterpret_cast<int8_t*>(is_k ? a.kp : a.vp) + at, (is_k ? a.ksc : a.vsc) + row * a.kv_heads + hh, f, lane);
            else store_half<N>(reinterpret_cast<__half*>(is_k ? a.kp : a.vp) + at, f);
            if (is_k && a.weight && lane == 0) {   // a new key has received nothing yet
                const int64_t wi = (((row >> a.page_shift) * a.kv_heads + hh) << a.page_shift) + (slot & ((1 << a.page_shift) - 1));
                a.weight[wi] = 0.0f; a.age[wi] = b.age[bi] + t;
            }
        }
        if (h0 + ROWS * step < n_slots) load_rows(h0 + ROWS * step);
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
    const int rows8 = (c.cfg.heads + 2 * c.cfg.kv_heads - a.first_slot + 7) / 8;
    const dim3 grid((int64_t)T * b.n * std::min(rows8, 4) <= 8 * c.sm_count ? std::min(rows8, 4) : 1, T, b.n), block(256);   // few tokens: as many CTAs as fit the GPU at once
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
