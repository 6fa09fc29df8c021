// extern "C" entry points of a batch's steps with any number of new tokens a sequence (include/mlxr.h). Arguments are
// checked before the device is asked for anything; nothing is allocated, copied or waited for.
#include <cmath>
#include "batch_checks.h"

using namespace mlxr;

namespace {

constexpr int MAX_ROWS = 1 << 22;

bool same_twice(std::initializer_list<const void*> ptrs) {
    for (auto p = ptrs.begin(); p != ptrs.end(); p++)
        for (auto q = ptrs.begin(); q != p; q++)
            if (*p == *q) return true;
    return false;
}
int check_rows(int rows) { return rows < 1 || rows > MAX_ROWS ? bad("rows: 1 .. 4194304") : MLXR_OK; }
int check_reserve(const mlxr_paged_kv* kv, int rows) {
    if (int rc = check_kv(kv)) return rc;
    if (rows < 0 || rows > MAX_ROWS) return bad("paged_reserve: 0 .. 4194304 rows");
    if ((int64_t)kv->B * ((kv->max_len + MLXR_PAGE - 1) / MLXR_PAGE) >= (int64_t)1 << 30) return set_error(MLXR_E_UNSUPPORTED, "paged_reserve: the batch could hold 2^30 pages");
    return MLXR_OK;
}
int check_attention(const mlxr_paged_kv* kv, int nH, int rows, int q_type) {
    if (int rc = check_kv(kv)) return rc;
    if (int rc = check_heads(kv, nH)) return rc;
    if (int rc = check_rows(rows)) return rc;
    if (q_type != 0 && q_type != 1) return bad("q_type: 0 (fp32) or 1 (the cache's type)");
    if ((int64_t)rows * (nH / kv->nKV) >= (int64_t)1 << 30) return set_error(MLXR_E_UNSUPPORTED, "paged_attention_rows: 2^30 query heads or more a KV head");
    return MLXR_OK;
}

}  // namespace

extern "C" {

int64_t mlxr_k_paged_reserve_work(const mlxr_paged_kv* kv, int rows) {
    if (guarded([&] { return check_reserve(kv, rows); }) != MLXR_OK) return MLXR_E_INVALID_ARG;
    return (int64_t)paged_reserve_work(*kv, rows);
}
int mlxr_k_paged_reserve(const mlxr_paged_kv* kv, const int32_t* want, int32_t* free_pages, const int32_t* n_free, int rows, int32_t* len_out,
                         int32_t* n_free_out, int32_t* start, int32_t* count, int32_t* seq, int32_t* slot, void* work, size_t work_bytes, void* stream) {
    return guarded([&]() -> int {
        if (int rc = check_reserve(kv, rows)) return rc;
        if (!want || !free_pages || !n_free || !len_out || !n_free_out || !start || !count || !seq || !slot) return bad("paged_reserve: null pointer");
        if (!aligned(want, 4) || !aligned(free_pages, 4) || !aligned(n_free, 4) || !aligned(len_out, 4) || !aligned(n_free_out, 4) || !aligned(start, 4) ||
            !aligned(count, 4) || !aligned(seq, 4) || !aligned(slot, 4))
            return bad("paged_reserve: alignment");
        if (same_twice({kv->table, want, free_pages, len_out, n_free_out, start, count, seq, slot}) || want == kv->len || free_pages == n_free ||
            same_twice({kv->len, kv->table, free_pages, n_free_out, start, count, seq, slot}) ||
            same_twice({n_free, kv->table, want, len_out, start, count, seq, slot}))
            return bad("paged_reserve: two arrays are the same (only len_out may be the cache's len, and n_free_out n_free)");
        if (int rc = check_work(work, work_bytes, (int64_t)paged_reserve_work(*kv, rows))) return rc;
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (int rc = check_device({kv->table, kv->len, want, free_pages, n_free, len_out, n_free_out, start, count, seq, slot, work}, s)) return rc;
        return done(launch_paged_reserve(ReserveArgs{*kv, want, free_pages, n_free, rows, len_out, n_free_out, start, count, seq, slot, work}, s));
    });
}

int mlxr_k_paged_append_rows(const mlxr_paged_kv* kv, const float* qkv, int row_stride, int rows, const int32_t* seq, const int32_t* slot,
                             const int32_t* positions, const float* inv_freq, float rope_scale, const float* qn, const float* kn, int nH, int rot_dim,
                             int traditional, float eps, void* q_out, int q_type, int q_stride, void* stream) {
    return guarded([&]() -> int {
        if (int rc = check_kv(kv)) return rc;
        if (int rc = check_heads(kv, nH)) return rc;
        if (int rc = check_rows(rows)) return rc;
        const int D = kv->D;
        if (!qkv || !q_out || !seq || !slot || (rot_dim && !inv_freq) || (qn == nullptr) != (kn == nullptr))
            return bad("paged_append_rows: null pointer (qn and kn go together)");
        if (rot_dim < 0 || rot_dim > D || rot_dim % 2) return bad("paged_append_rows: rot_dim even, 0 .. D");
        if (q_type != 0 && q_type != 1) return bad("q_type: 0 (fp32) or 1 (the cache's type)");
        if (!(rope_scale == rope_scale)) return bad("paged_append_rows: rope_scale is NaN");
        if (row_stride < (int64_t)(nH + 2 * kv->nKV) * D || q_stride < (int64_t)nH * D) return bad("paged_append_rows: strides");
        if (q_out == qkv && (q_type != 0 || q_stride != row_stride)) return bad("paged_append_rows: q_out over qkv needs its type and stride");
        if (!aligned(qkv, 4) || !aligned(q_out, q_type ? 2 : 4) || !aligned(inv_freq, 4) || !aligned(qn, 4) || !aligned(kn, 4) || !aligned(positions, 4) ||
            !aligned(seq, 4) || !aligned(slot, 4))
            return bad("paged_append_rows: alignment");
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (int rc = check_device({kv->k, kv->v, kv->table, kv->weight, kv->position, qkv, seq, slot, rot_dim ? inv_freq : nullptr, qn, kn, positions, q_out}, s)) return rc;
        return done(launch_paged_append_rows(AppendRowsArgs{*kv, qkv, row_stride, rows, seq, slot, positions, inv_freq, rope_scale, qn, kn, nH, rot_dim,
                                                            traditional, eps, q_out, q_type, q_stride}, s));
    });
}

int64_t mlxr_k_paged_attention_rows_work(const mlxr_paged_kv* kv, int nH, int rows, int q_type) {
    if (guarded([&] { return check_attention(kv, nH, rows, q_type); }) != MLXR_OK) return MLXR_E_INVALID_ARG;
    return (int64_t)paged_attention_rows_work(*kv, nH, rows, q_type);
}
int mlxr_k_paged_attention_rows(const mlxr_paged_kv* kv, const int32_t* start, const int32_t* count, int rows, const void* q, int q_type, int q_stride,
                                int nH, int window, float scale, void* out, int out_stride, void* work, size_t work_bytes, void* stream) {
    return guarded([&]() -> int {
        if (int rc = check_attention(kv, nH, rows, q_type)) return rc;
        if (!start || !count || !q || !out) return bad("paged_attention_rows: null pointer");
        const int unit = q_type ? 8 : 4;   // values in 16 bytes
        if (q_stride < (int64_t)nH * kv->D || out_stride < (int64_t)nH * kv->D || q_stride % unit || out_stride % unit || !aligned(q, 16) || !aligned(out, 16))
            return bad("paged_attention_rows: q and out 16-byte aligned, strides whole multiples of 16 bytes and at least nH * D values");
        if (out == q && out_stride != q_stride) return bad("paged_attention_rows: out over q needs its stride");
        if (window < 0) return bad("paged_attention_rows: window");
        if (!(std::fabs(scale) <= 0x1p126f)) return bad("paged_attention_rows: scale is NaN or above 2^126");
        if (!aligned(start, 4) || !aligned(count, 4)) return bad("paged_attention_rows: alignment");
        if (int rc = check_work(work, work_bytes, (int64_t)paged_attention_rows_work(*kv, nH, rows, q_type))) return rc;
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (int rc = check_device({kv->k, kv->v, kv->table, kv->len, start, count, q, out, work}, s)) return rc;
        return done(launch_paged_attention_rows(AttnRowsArgs{*kv, start, count, rows, q, q_type, q_stride, nH, window, scale, out, out_stride, work}, s));
    });
}

}  // extern "C"
