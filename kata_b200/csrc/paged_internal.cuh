// Internal declarations of the paged cache: the context object and the launchers of its kernels.
#pragma once
#include "kata_internal.cuh"
#include "page_pool.hpp"

namespace kata {

constexpr int kPagedMaxRot = 128;    // rotary frequencies of a 256-wide head at most

// Angle tables: frequency i turns freq[i] / 2^64 of a full circle per position; axis[i] (0, 1, 2) says which position it takes.
struct RotTab { uint64_t freq[kPagedMaxRot]; int32_t axis[kPagedMaxRot]; };
// Fills the table; false when the sections do not add up to rot_dim / 2 or cannot be interleaved.
bool make_rot_tab(RotTab& t, int rot_dim, double theta, const int32_t* section, int interleaved);

struct PagedCtx {
    kata_paged_config cfg{};
    kata_pages* pages = nullptr;
    int group = 1, elt = 2;               // query heads per KV head; bytes per cached element
    int page_shift = 4, width = 0;        // width: table entries per sequence
    int64_t rows_per_layer = 0;           // n_pages * page_size
    void* plane[KATA_PAGED_PLANES] = {}; bool owned[KATA_PAGED_PLANES] = {};
    void* block = nullptr;                // one allocation for the pointers from d_table to scores
    int32_t* d_table = nullptr;           // [n_seqs][width], the device's copy of the page table
    RotTab* d_rot = nullptr;
    float* part_o = nullptr; float* part_ml = nullptr; int32_t* counters = nullptr; int32_t* d_err = nullptr;   // decode: partial rows of cut segments, their (m, l), tickets
    float* fin_ml = nullptr;              // decode with weights: joined (m, l) of every row of every segment
    float* scores = nullptr;              // decode with weights: fp32 scores [tile][key][8 or 16 rows] of one launch
    std::vector<int32_t> stamp; int32_t stamp_now = 0;   // per sequence: the call it was last named in (finds a sequence named twice)
    CUtensorMap tm_k{}, tm_v{}; int box_groups = 1;     // rank-5 tile views of the K and V pools; 16-row groups per box
    int sm_count = 148;
    uint64_t launches = 0;
    std::string err;
    bool int8() const { return cfg.kv_mode == KATA_KV_INT8; }
    bool weights() const { return (cfg.flags & KATA_PAGED_WEIGHTS) != 0; }
    size_t plane_row_bytes(int p) const {   // bytes per slot of a plane, 0 when the context has none
        const size_t kvh = cfg.kv_heads;
        if (p == KATA_PAGED_K || p == KATA_PAGED_V) return kvh * cfg.head_dim * elt;
        if (p == KATA_PAGED_K_SCALE || p == KATA_PAGED_V_SCALE) return int8() ? kvh * 2 : 0;
        return weights() ? kvh * 4 : 0;
    }
    void* layer_plane(int p, int layer) const { return plane[p] ? (uint8_t*)plane[p] + (size_t)layer * rows_per_layer * plane_row_bytes(p) : nullptr; }
};

// The sequences of one call, handed to a kernel by value.
struct PagedBatch { int32_t n; int32_t seq[KATA_PAGED_MAX_BATCH], slot[KATA_PAGED_MAX_BATCH], age[KATA_PAGED_MAX_BATCH]; };

size_t paged_part_floats(const PagedCtx& c); size_t paged_part_ml_floats(const PagedCtx& c);
int64_t paged_score_slots(const PagedCtx& c);
cudaError_t configure_paged_decode(const PagedCtx& c);
cudaError_t launch_paged_decode(PagedCtx& c, int layer, int n, const int32_t* seq, const int32_t* n_slots, int T, const __half* q16, const float* gate, void* out, int out_dtype, bool accumulate, cudaStream_t s);
cudaError_t launch_paged_prep(PagedCtx& c, int layer, const PagedBatch& b, int T, const int32_t* axis_pos, const void* q, const void* k, const void* v, int act_dtype,
                              const float* qnorm, const float* knorm, __half* q16, float* gate, cudaStream_t s);
cudaError_t configure_paged_evict(const PagedCtx& c);
cudaError_t launch_paged_evict(PagedCtx& c, int layer, int n_layers, const PagedBatch& b /* slot: n_slots, age: seen */, int keep, int sink, int recent, int32_t* src, cudaStream_t s);
cudaError_t launch_paged_import(PagedCtx& c, int layer, int seq, int slot0, int n_rows, int age0, const Ctx& src, int64_t src_row, cudaStream_t s);
bool make_paged_tmap(CUtensorMap* out, void* base, int elt, int64_t rows, int kv_heads, int head_dim, int box_groups);
Ctx& ctx_of(kata_attn_ctx* h);   // the object behind a contiguous context's handle

__device__ __forceinline__ int64_t paged_row(const int32_t* __restrict__ table_row, int slot, int shift) {   // row of a layer's pool that holds a slot
    return ((int64_t)__ldcg(table_row + (slot >> shift)) << shift) + (slot & ((1 << shift) - 1));
}

}  // namespace kata
