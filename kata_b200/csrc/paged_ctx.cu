// Context object and C ABI of the paged cache (include/kata_paged.h): pools, page tables and their device copy, argument checks.
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <new>

#include "paged_internal.cuh"

struct kata_paged_ctx { kata::PagedCtx c; };

using kata::PagedCtx;

namespace {

int pfail(PagedCtx& c, int code, const char* fmt, ...) {
    char buf[384]; va_list ap; va_start(ap, fmt); vsnprintf(buf, sizeof buf, fmt, ap); va_end(ap);
    try { c.err = buf; } catch (const std::exception&) {}
    return code;
}
int pcuda(PagedCtx& c, cudaError_t e, const char* what) { cudaGetLastError();   // reported here: not again by the next call
    return pfail(c, KATA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e)); }

struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int dev) { cudaGetDevice(&prev); if (prev != dev) cudaSetDevice(dev); else prev = -1; }
    ~DeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};

bool misaligned(std::initializer_list<const void*> ptrs) { for (const void* p : ptrs) if ((uintptr_t)p & 15) return true; return false; }

// layer, batch size and sequence ids; `once`: a sequence may be named only once (calls that write what belongs to it)
int check_batch(PagedCtx& c, int layer, int n_layers, int n, const int32_t* seq, const int32_t* slots, bool once) {
    if (layer < 0 || n_layers < 1 || layer > c.cfg.n_layers - n_layers) return pfail(c, KATA_ERR_RANGE, "layers [%d,%lld) outside [0,%d)", layer, (long long)layer + n_layers, c.cfg.n_layers);
    if (n < 1 || n > KATA_PAGED_MAX_BATCH || !seq || !slots) return pfail(c, KATA_ERR_ARG, "batch of %d sequences (1..%d) needs sequence ids and slots", n, KATA_PAGED_MAX_BATCH);
    if (++c.stamp_now == INT32_MAX) { std::fill(c.stamp.begin(), c.stamp.end(), 0); c.stamp_now = 1; }
    for (int i = 0; i < n; i++) {
        if (seq[i] < 0 || seq[i] >= c.cfg.n_seqs) return pfail(c, KATA_ERR_RANGE, "sequence id %d outside [0,%d)", seq[i], c.cfg.n_seqs);
        if (once && c.stamp[seq[i]] == c.stamp_now) return pfail(c, KATA_ERR_ARG, "sequence %d is named twice in one call that writes to it", seq[i]);
        c.stamp[seq[i]] = c.stamp_now;
    }
    return KATA_OK;
}
int check_slots(PagedCtx& c, int seq, int64_t lo, int64_t hi) {   // slots [lo, hi) are reserved
    if (lo < 0 || hi < lo || hi > c.pages->capacity(seq)) return pfail(c, KATA_ERR_RANGE, "slots [%lld,%lld) of sequence %d: %lld are reserved", (long long)lo, (long long)hi, seq, (long long)c.pages->capacity(seq));
    return KATA_OK;
}
int check_not_shared(PagedCtx& c, int seq, int lo, int n) { return c.pages->shared(seq, lo, n) ? pfail(c, KATA_ERR_MODE, "slots [%d,%d) of sequence %d lie in a page shared with another sequence", lo, lo + n, seq) : KATA_OK; }

int not_capturing(PagedCtx& c, cudaStream_t s, const char* what) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    const cudaError_t e = cudaStreamIsCapturing(s, &st);
    if (e != cudaSuccess) { cudaGetLastError(); return pcuda(c, e, what); }
    return st == cudaStreamCaptureStatusNone ? KATA_OK : pfail(c, KATA_ERR_MODE, "%s changes the page table: not inside a stream capture", what);
}

// brings the device's copy of a sequence's table entries [from, count) up to date; the source is pageable, so it has been read when the call returns
cudaError_t upload_table(PagedCtx& c, int seq, int from, cudaStream_t s) {
    const int n = c.pages->count[seq] - from;
    return n > 0 ? cudaMemcpyAsync(c.d_table + (int64_t)seq * c.width + from, c.pages->row(seq) + from, (size_t)n * 4, cudaMemcpyHostToDevice, s) : cudaSuccess;
}

}  // namespace

extern "C" {

int kata_paged_create(const kata_paged_config* cfg, kata_paged_ctx** out) {
    if (!out) return KATA_ERR_ARG;
    *out = nullptr;
    if (!cfg) return KATA_ERR_ARG;
    const int H = cfg->heads, KVH = cfg->kv_heads, hd = cfg->head_dim;
    if (cfg->n_layers < 1 || cfg->n_seqs < 1 || cfg->n_pages < 1 || cfg->max_slots < 1 || cfg->max_slots > KATA_PAGED_MAX_SLOTS || cfg->page_size < 16 || cfg->page_size > 1024 || (cfg->page_size & (cfg->page_size - 1))) return KATA_ERR_ARG;
    if (KVH < 1 || KVH > KATA_PAGED_MAX_KV_HEADS || H < KVH || H % KVH || H / KVH > KATA_PAGED_MAX_GROUP || (hd != 128 && hd != 256)) return KATA_ERR_ARG;
    if (cfg->kv_mode != KATA_KV_FP16 && cfg->kv_mode != KATA_KV_INT8) return KATA_ERR_MODE;
    if (cfg->rot_dim < 0 || cfg->rot_dim > hd || cfg->rot_dim % 16 || (cfg->flags & ~(KATA_PAGED_GATED | KATA_PAGED_WEIGHTS))) return KATA_ERR_ARG;
    kata::RotTab rot;
    if (!kata::make_rot_tab(rot, cfg->rot_dim, cfg->rope_theta, cfg->section, cfg->interleaved)) return KATA_ERR_ARG;
    const int64_t rows_per_layer = (int64_t)cfg->n_pages * cfg->page_size, rows = rows_per_layer * cfg->n_layers;
    if (rows_per_layer > INT32_MAX || rows / 16 > INT32_MAX) return KATA_ERR_RANGE;
    for (int p = 0; p < KATA_PAGED_PLANES; p++) if ((uintptr_t)cfg->planes[p] & 127) return KATA_ERR_ARG;
    int ndev = 0;
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || cfg->device < 0 || cfg->device >= ndev) { cudaGetLastError(); return KATA_ERR_CUDA; }
    kata_paged_ctx* h = new (std::nothrow) kata_paged_ctx();
    if (!h) return KATA_ERR_NOMEM;
    PagedCtx& c = h->c; c.cfg = *cfg; c.group = H / KVH; c.elt = cfg->kv_mode == KATA_KV_INT8 ? 1 : 2; c.rows_per_layer = rows_per_layer;
    while ((1 << c.page_shift) < cfg->page_size) c.page_shift++;
    const int rc = kata_pages_create(cfg->n_pages, cfg->page_size, cfg->n_seqs, cfg->max_slots, &c.pages);
    if (rc != KATA_OK) { delete h; return rc; }
    try { c.stamp.assign(cfg->n_seqs, 0); } catch (const std::exception&) { kata_pages_destroy(c.pages); delete h; return KATA_ERR_NOMEM; }
    c.width = c.pages->width;
    DeviceGuard guard(cfg->device);
    cudaDeviceGetAttribute(&c.sm_count, cudaDevAttrMultiProcessorCount, cfg->device);
    c.box_groups = ((hd == 128 || c.int8()) && cfg->page_size >= 32) ? 2 : 1;   // tiles of 32 slots and more
    bool ok = true;
    for (int p = 0; p < KATA_PAGED_PLANES && ok; p++) {
        const size_t bytes = (size_t)rows * c.plane_row_bytes(p);
        if (!bytes) continue;
        if (cfg->planes[p]) { c.plane[p] = cfg->planes[p]; continue; }
        ok = cudaMalloc(&c.plane[p], bytes) == cudaSuccess;
        if (ok) { c.owned[p] = true; ok = cudaMemset(c.plane[p], 0, bytes) == cudaSuccess; }
    }
    // the rest in one block (a context in 85 us instead of 126). What has to start at zero lies first (the table's zeros: every entry is a page of the pool at all times)
    size_t size = 0, zeros = 0;
    auto part = [&](size_t bytes) { const size_t at = size; size += (bytes + 255) / 256 * 256; return at; };
    const int per_pass = std::max(1, 16 / c.group) * c.group, score_rows = std::min(per_pass, KATA_MAX_VERIFY * c.group) <= 8 ? 8 : 16;
    const size_t at_table = part((size_t)cfg->n_seqs * c.width * 4), at_counters = part((size_t)KATA_PAGED_MAX_BATCH * KVH * 4), at_err = part(4);
    zeros = size;
    const size_t at_rot = part(sizeof(kata::RotTab)), at_o = part(kata::paged_part_floats(c) * 4), at_ml = part(kata::paged_part_ml_floats(c) * 4);
    const size_t at_scores = part(c.weights() ? (size_t)kata::paged_score_slots(c) * score_rows * 4 : 0), at_fin = part(c.weights() ? (size_t)KATA_PAGED_MAX_BATCH * KVH * 16 * 2 * 4 : 0);
    ok = ok && cudaMalloc(&c.block, size) == cudaSuccess && cudaMemset(c.block, 0, zeros) == cudaSuccess;
    if (ok) {
        uint8_t* base = (uint8_t*)c.block;
        c.d_table = (int32_t*)(base + at_table); c.counters = (int32_t*)(base + at_counters); c.d_err = (int32_t*)(base + at_err); c.d_rot = (kata::RotTab*)(base + at_rot);
        c.part_o = (float*)(base + at_o); c.part_ml = (float*)(base + at_ml);
        if (c.weights()) { c.scores = (float*)(base + at_scores); c.fin_ml = (float*)(base + at_fin); }
    }
    if (!ok) { cudaGetLastError(); kata_paged_destroy(h); return KATA_ERR_NOMEM; }
    if (cudaMemcpy(c.d_rot, &rot, sizeof rot, cudaMemcpyHostToDevice) != cudaSuccess || kata::configure_paged_decode(c) != cudaSuccess || kata::configure_paged_evict(c) != cudaSuccess ||
        !kata::make_paged_tmap(&c.tm_k, c.plane[KATA_PAGED_K], c.elt, rows, KVH, hd, c.box_groups) || !kata::make_paged_tmap(&c.tm_v, c.plane[KATA_PAGED_V], c.elt, rows, KVH, hd, c.box_groups) ||
        cudaDeviceSynchronize() != cudaSuccess) { cudaGetLastError(); kata_paged_destroy(h); return KATA_ERR_CUDA; }
    *out = h;
    return KATA_OK;
}

int kata_paged_destroy(kata_paged_ctx* h) {
    if (!h) return KATA_ERR_ARG;
    PagedCtx& c = h->c; DeviceGuard guard(c.cfg.device);
    for (int p = 0; p < KATA_PAGED_PLANES; p++) if (c.owned[p]) cudaFree(c.plane[p]);
    if (c.block) cudaFree(c.block);
    if (c.pages) kata_pages_destroy(c.pages);
    delete h;
    return KATA_OK;
}

const char* kata_paged_last_error(const kata_paged_ctx* h) { return h ? h->c.err.c_str() : "null context"; }
uint64_t kata_paged_launch_count(const kata_paged_ctx* h) { return h ? h->c.launches : 0; }
const kata_pages* kata_paged_table(const kata_paged_ctx* h) { return h ? h->c.pages : nullptr; }
void* kata_paged_plane_ptr(kata_paged_ctx* h, int32_t layer, int32_t plane) {
    if (!h || layer < 0 || layer >= h->c.cfg.n_layers || plane < 0 || plane >= KATA_PAGED_PLANES) return nullptr;
    return h->c.layer_plane(plane, layer);
}

int kata_paged_check(kata_paged_ctx* h, void* stream) {
    if (!h) return KATA_ERR_ARG;
    PagedCtx& c = h->c; DeviceGuard guard(c.cfg.device);
    cudaError_t e = cudaStreamSynchronize((cudaStream_t)stream); if (e != cudaSuccess) return pcuda(c, e, "synchronize");
    int32_t flag = 0; e = cudaMemcpy(&flag, c.d_err, 4, cudaMemcpyDeviceToHost); if (e != cudaSuccess) return pcuda(c, e, "read error word");
    if (flag) { cudaMemset(c.d_err, 0, 4); return pfail(c, KATA_ERR_DEVICE_WAIT, "a bounded device-side wait ran out (code %d); results of that call are invalid", flag); }
    return KATA_OK;
}

int kata_paged_reserve(kata_paged_ctx* h, int32_t seq, int32_t n_slots, void* stream) {
    if (!h) return KATA_ERR_ARG;
    PagedCtx& c = h->c; DeviceGuard guard(c.cfg.device);
    if (int rc = not_capturing(c, (cudaStream_t)stream, "reserve")) return rc;
    const int before = seq >= 0 && seq < c.cfg.n_seqs ? c.pages->count[seq] : 0;
    const int rc = c.pages->reserve(seq, n_slots);
    if (rc != KATA_OK) return pfail(c, rc, "reserve of %d slots for sequence %d (%d sequences of at most %d slots, %d pages free)", n_slots, seq, c.cfg.n_seqs, c.cfg.max_slots, kata_pages_free_count(c.pages));
    const cudaError_t e = upload_table(c, seq, before, (cudaStream_t)stream);
    if (e != cudaSuccess) { c.pages->trim(seq, before * c.cfg.page_size); return pcuda(c, e, "reserve"); }
    return KATA_OK;
}

int kata_paged_trim(kata_paged_ctx* h, int32_t seq, int32_t n_slots) {
    if (!h) return KATA_ERR_ARG;
    const int rc = h->c.pages->trim(seq, n_slots);
    return rc == KATA_OK ? KATA_OK : pfail(h->c, rc, "trim of sequence %d to %d slots", seq, n_slots);
}

int kata_paged_fork(kata_paged_ctx* h, int32_t src, int32_t dst, int32_t n_slots, void* stream) {
    if (!h) return KATA_ERR_ARG;
    PagedCtx& c = h->c; DeviceGuard guard(c.cfg.device); cudaStream_t s = (cudaStream_t)stream;
    if (c.weights()) return pfail(c, KATA_ERR_MODE, "a context that keeps attention weights cannot share pages");
    if (int rc = not_capturing(c, s, "fork")) return rc;
    int32_t from, to, slots;
    const int rc = c.pages->fork(src, dst, n_slots, from, to, slots);
    if (rc != KATA_OK) return pfail(c, rc, "fork of %d slots of sequence %d to sequence %d (which must hold no pages)", n_slots, src, dst);
    cudaError_t e = cudaSuccess;
    for (int p = 0; p < KATA_PAGED_PLANES && slots && e == cudaSuccess; p++) {
        const size_t rb = c.plane_row_bytes(p), pitch = rb * c.rows_per_layer;
        if (!rb) continue;
        uint8_t* base = (uint8_t*)c.plane[p]; const size_t page = rb * c.cfg.page_size;
        for (int l = 0; l < c.cfg.n_layers && e == cudaSuccess; l++) e = cudaMemcpyAsync(base + l * pitch + to * page, base + l * pitch + from * page, rb * slots, cudaMemcpyDeviceToDevice, s);
    }
    if (e == cudaSuccess) e = upload_table(c, dst, 0, s);
    if (e != cudaSuccess) { c.pages->trim(dst, 0); return pcuda(c, e, "fork"); }
    return KATA_OK;
}

int kata_paged_prep(kata_paged_ctx* h, int32_t layer, int32_t n, const int32_t* seq_ids, const int32_t* slot0, int32_t T, const int32_t* d_axis_pos, const int32_t* age0,
                    const void* d_q, const void* d_k, const void* d_v, int32_t act_dtype, const float* d_qnorm, const float* d_knorm, void* d_q16, float* d_gate, void* stream) {
    if (!h) return KATA_ERR_ARG;
    PagedCtx& c = h->c;
    if (T < 1 || T > KATA_MAX_CHUNK) return pfail(c, KATA_ERR_RANGE, "prep of %d tokens (1..%d)", T, KATA_MAX_CHUNK);
    if (act_dtype != KATA_ACT_F32 && act_dtype != KATA_ACT_BF16 && act_dtype != KATA_ACT_F16) return pfail(c, KATA_ERR_ARG, "unknown activation dtype %d", act_dtype);
    if (!d_k || !d_v || !d_knorm || (d_q && (!d_qnorm || !d_q16))) return pfail(c, KATA_ERR_ARG, "prep needs k, v and knorm, and with a query qnorm and q16");
    if (d_gate && (!d_q || !(c.cfg.flags & KATA_PAGED_GATED))) return pfail(c, KATA_ERR_ARG, "a gate needs query rows of a gated context");
    if (misaligned({d_q, d_k, d_v, d_qnorm, d_knorm, d_q16, d_gate}) || ((uintptr_t)d_axis_pos & 3)) return pfail(c, KATA_ERR_ARG, "prep needs its rows on 16-byte boundaries");
    if (int rc = check_batch(c, layer, 1, n, seq_ids, slot0, true)) return rc;
    kata::PagedBatch b{}; b.n = n;
    for (int i = 0; i < n; i++) {
        if (int rc = check_slots(c, seq_ids[i], slot0[i], (int64_t)slot0[i] + T)) return rc;
        if (int rc = check_not_shared(c, seq_ids[i], slot0[i], T)) return rc;
        b.seq[i] = seq_ids[i]; b.slot[i] = slot0[i]; b.age[i] = age0 ? age0[i] : slot0[i];
        if (b.age[i] < 0 || b.age[i] > INT32_MAX - T) return pfail(c, KATA_ERR_RANGE, "age %d of sequence %d", b.age[i], seq_ids[i]);
    }
    DeviceGuard guard(c.cfg.device);
    const cudaError_t e = kata::launch_paged_prep(c, layer, b, T, d_axis_pos, d_q, d_k, d_v, act_dtype, d_qnorm, d_knorm, (__half*)d_q16, d_gate, (cudaStream_t)stream);
    return e == cudaSuccess ? KATA_OK : pcuda(c, e, "prep launch");
}

int kata_paged_decode(kata_paged_ctx* h, int32_t layer, int32_t n, const int32_t* seq_ids, const int32_t* n_slots, int32_t T, const void* d_q16, const float* d_gate, void* d_out, int32_t out_dtype, int32_t accumulate, void* stream) {
    if (!h) return KATA_ERR_ARG;
    PagedCtx& c = h->c;
    if (T < 1 || T > KATA_MAX_VERIFY) return pfail(c, KATA_ERR_RANGE, "decode takes 1..%d query tokens, not %d", KATA_MAX_VERIFY, T);
    if (!d_q16 || !d_out) return pfail(c, KATA_ERR_ARG, "decode needs q16 and out");
    if (out_dtype != KATA_ACT_F32 && out_dtype != KATA_ACT_BF16 && out_dtype != KATA_ACT_F16) return pfail(c, KATA_ERR_ARG, "unknown output dtype %d", out_dtype);
    if (misaligned({d_q16, d_gate, d_out})) return pfail(c, KATA_ERR_ARG, "decode needs q16, gate and out on 16-byte boundaries");
    if (accumulate && !c.weights()) return pfail(c, KATA_ERR_MODE, "this context keeps no attention weights (KATA_PAGED_WEIGHTS)");
    if (int rc = check_batch(c, layer, 1, n, seq_ids, n_slots, accumulate != 0)) return rc;
    for (int i = 0; i < n; i++) if (int rc = check_slots(c, seq_ids[i], 0, n_slots[i])) return rc;
    DeviceGuard guard(c.cfg.device);
    const cudaError_t e = kata::launch_paged_decode(c, layer, n, seq_ids, n_slots, T, (const __half*)d_q16, d_gate, d_out, out_dtype, accumulate != 0, (cudaStream_t)stream);
    return e == cudaSuccess ? KATA_OK : pcuda(c, e, "decode launch");
}

int kata_paged_evict(kata_paged_ctx* h, int32_t layer, int32_t n_layers, int32_t n, const int32_t* seq_ids, const int32_t* n_slots, const int32_t* seen, int32_t keep, int32_t sink, int32_t recent, int32_t* d_src, void* stream) {
    if (!h) return KATA_ERR_ARG;
    PagedCtx& c = h->c;
    if (!c.weights()) return pfail(c, KATA_ERR_MODE, "this context keeps no attention weights (KATA_PAGED_WEIGHTS)");
    if (keep < 1 || sink < 0 || recent < 0 || (int64_t)sink + recent > keep) return pfail(c, KATA_ERR_RANGE, "keep %d slots, the first %d and the newest %d tokens among them", keep, sink, recent);
    if (keep > c.cfg.max_slots) return pfail(c, KATA_ERR_RANGE, "a budget of %d slots: sequences hold at most %d", keep, c.cfg.max_slots);
    if (!seen || !d_src || ((uintptr_t)d_src & 3)) return pfail(c, KATA_ERR_ARG, "evict needs the tokens seen and src");
    if (int rc = check_batch(c, layer, n_layers, n, seq_ids, n_slots, true)) return rc;
    if (n_layers > 65535 || (int64_t)n * c.cfg.kv_heads > 65535) return pfail(c, KATA_ERR_RANGE, "%d layers in one call", n_layers);
    kata::PagedBatch b{}; b.n = n;
    for (int i = 0; i < n; i++) {
        if (int rc = check_slots(c, seq_ids[i], 0, n_slots[i])) return rc;
        if (seen[i] < 0) return pfail(c, KATA_ERR_RANGE, "sequence %d has seen %d tokens", seq_ids[i], seen[i]);
        b.seq[i] = seq_ids[i]; b.slot[i] = n_slots[i]; b.age[i] = seen[i];
    }
    DeviceGuard guard(c.cfg.device);
    const cudaError_t e = kata::launch_paged_evict(c, layer, n_layers, b, keep, sink, recent, d_src, (cudaStream_t)stream);
    return e == cudaSuccess ? KATA_OK : pcuda(c, e, "evict launch");
}

int kata_paged_import(kata_paged_ctx* h, int32_t layer, int32_t seq, int32_t slot0, int32_t n_rows, int32_t age0, kata_attn_ctx* src, int32_t src_layer, int32_t src_seq, int32_t src_pos, void* stream) {
    if (!h) return KATA_ERR_ARG;
    PagedCtx& c = h->c;
    if (!src) return pfail(c, KATA_ERR_ARG, "import needs a source context");
    kata::Ctx& a = kata::ctx_of(src);
    if (c.cfg.heads != KATA_HEADS || c.cfg.kv_heads != KATA_KV_HEADS || c.cfg.head_dim != KATA_HEAD_DIM || a.cfg.kv_mode != c.cfg.kv_mode || a.cfg.device != c.cfg.device) return pfail(c, KATA_ERR_MODE, "import needs the same head layout, cache mode and device on both sides");
    if (a.kvh_n != KATA_KV_HEADS) return pfail(c, KATA_ERR_MODE, "import takes rows of all %d KV heads (the source context writes %d of them)", KATA_KV_HEADS, a.kvh_n);
    if (n_rows < 1) return pfail(c, KATA_ERR_RANGE, "import of %d rows", n_rows);
    if (int rc = check_batch(c, layer, 1, 1, &seq, &slot0, true)) return rc;
    if (int rc = check_slots(c, seq, slot0, (int64_t)slot0 + n_rows)) return rc;
    if (int rc = check_not_shared(c, seq, slot0, n_rows)) return rc;
    if (age0 < 0 || age0 > INT32_MAX - n_rows) return pfail(c, KATA_ERR_RANGE, "age %d", age0);
    if (src_layer < 0 || src_layer >= a.cfg.n_layers || src_seq < 0 || src_seq >= a.cfg.n_seqs) return pfail(c, KATA_ERR_RANGE, "source layer %d / sequence %d out of range", src_layer, src_seq);
    const int64_t row = (int64_t)src_pos - a.pos_off[src_seq];
    if (src_pos < 0 || row < 0 || row + n_rows > a.max_ctx[src_seq]) return pfail(c, KATA_ERR_RANGE, "source positions [%d,%lld) outside the sequence's %d rows", src_pos, (long long)src_pos + n_rows, a.max_ctx[src_seq]);
    DeviceGuard guard(c.cfg.device);
    const cudaError_t e = kata::launch_paged_import(c, layer, seq, slot0, n_rows, age0, a, a.row_of(src_layer, src_seq) + row, (cudaStream_t)stream);
    return e == cudaSuccess ? KATA_OK : pcuda(c, e, "import launch");
}

}  // extern "C"
