// A batch's decode step over a pool of KV-cache pages: launchers of paged.hip, evict.hip and sample_rows.hip.
// They validate nothing: the entry points in capi_batch.cpp check shapes first.
#pragma once
#include "../../include/mlxr.h"
#include "common.h"

namespace mlxr {

typedef mlxr_paged_kv PagedKV;

// Lengths and page numbers are read on the device only, so they are held in bounds here.
__device__ __forceinline__ int paged_len(const PagedKV& kv, int b) {
    const int n = kv.len[b];
    return n < 0 ? 0 : (n > kv.max_len ? kv.max_len : n);
}
// The page of table entry i of sequence b, or -1 where it names none of the pool.
__device__ __forceinline__ int paged_page(const PagedKV& kv, int b, int i) {
    const int p = kv.table[(int64_t)b * kv.table_stride + i];
    return (unsigned)p < (unsigned)kv.n_pages ? p : -1;
}
// Element offset of row `slot` (0 .. 63) of a page.
__device__ __forceinline__ int64_t paged_row(const PagedKV& kv, int page, int kvh, int slot) {
    return (((int64_t)page * kv.nKV + kvh) * MLXR_PAGE + slot) * kv.D;
}
// Element offset of a slot's weight or position.
__device__ __forceinline__ int64_t paged_slot(const PagedKV& kv, int b, int kvh, int slot) {
    return ((int64_t)b * kv.nKV + kvh) * kv.slot_stride + slot;
}

// Inclusive sums over a wave: within rows of 16 lanes, then the rows' last lanes on to the rows behind.
template <int CTRL, int ROWS> __device__ __forceinline__ int lane_before(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false); }
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t lane_before(uint64_t v) {   // 0 where there is no lane before
    const uint32_t lo = (uint32_t)lane_before<CTRL, ROWS>((int)(uint32_t)v), hi = (uint32_t)lane_before<CTRL, ROWS>((int)(uint32_t)(v >> 32));
    return (uint64_t)lo | ((uint64_t)hi << 32);
}
template <int CTRL, int ROWS> __device__ __forceinline__ double lane_before(double v) {
    return __builtin_bit_cast(double, lane_before<CTRL, ROWS>(__builtin_bit_cast(uint64_t, v)));
}
template <typename T> __device__ __forceinline__ T wave_scan(T v) {
    v += lane_before<0x111, 0xF>(v);   // row_shr 1, 2, 4, 8
    v += lane_before<0x112, 0xF>(v);
    v += lane_before<0x114, 0xF>(v);
    v += lane_before<0x118, 0xF>(v);
    v += lane_before<0x142, 0xA>(v);   // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
    v += lane_before<0x143, 0xC>(v);
    return v;
}

struct PagedAppendArgs {
    PagedKV kv;
    const float* qkv; int row_stride;
    const float *inv_freq, *qn, *kn;
    int nH, rot_dim, traditional;
    const int* positions;
    float eps;
    float* q_out; int q_stride;
};
hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s);

struct PagedAttnArgs {
    PagedKV kv;
    const float* q; int q_stride, nH, window;
    float scale;
    float* out; int out_stride;
    const float* weight_in; float decay;
    void* work;
};
size_t paged_attention_work(const PagedKV& kv, int nH);
hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s);

struct PagedEvictArgs {
    PagedKV src, dst;
    int budget, sink, window;
    void* work;
};
size_t paged_evict_work(const PagedKV& src, int budget);
hipError_t launch_paged_evict(const PagedEvictArgs& a, hipStream_t s);

struct SampleRowsArgs {
    const float* logits; int rows, V; int64_t stride;
    const float* temperature; const int* top_k; const float *top_p, *min_p, *u;
    int *tokens, *status;
    void* work;
};
size_t sample_rows_work(int rows, int V);
hipError_t launch_sample_rows(const SampleRowsArgs& a, hipStream_t s);

}  // namespace mlxr
