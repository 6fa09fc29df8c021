// extern "C" entry points of a batch's decode step (include/mlxr.h). Arguments are checked before the device
// is asked for anything; nothing is allocated, copied or waited for.
#include <atomic>
#include <initializer_list>
#include <new>
#include <string>
#include "batch.h"
#include "model.h"

using namespace mlxr;

namespace {

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int bad(const char* what) { return set_error(MLXR_E_INVALID_ARG, what); }

int check_kv(const mlxr_paged_kv* kv) {
    if (!kv || !kv->k || !kv->v || !kv->table || !kv->len) return bad("paged cache: null pointer");
    if (kv->D != 64 && kv->D != 128) return set_error(MLXR_E_UNSUPPORTED, "paged cache: D must be 64 or 128");
    if (kv->st != 0 && kv->st != 1) return bad("paged cache: st must be 0 (bf16) or 1 (f16)");
    if (kv->B < 1 || kv->nKV < 1 || kv->n_pages < 1 || kv->table_stride < 1 || kv->max_len < 1) return bad("paged cache: sizes");
    if (kv->nKV > 1024 || kv->B > 65535) return set_error(MLXR_E_UNSUPPORTED, "paged cache: at most 1024 KV heads and 65535 sequences");
    if (kv->max_len > (1 << 24)) return set_error(MLXR_E_UNSUPPORTED, "paged cache: at most 16777216 slots a sequence");
    if (kv->max_len > (int64_t)kv->table_stride * MLXR_PAGE) return bad("paged cache: max_len is more than the table holds");
    if ((kv->weight || kv->position) && kv->slot_stride < kv->max_len) return bad("paged cache: slot_stride is less than max_len");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return bad("paged cache: k and v must be 16-byte aligned");
    if (!aligned(kv->table, 4) || !aligned(kv->len, 4) || !aligned(kv->weight, 4) || !aligned(kv->position, 4)) return bad("paged cache: alignment");
    return MLXR_OK;
}
int check_heads(const mlxr_paged_kv* kv, int nH) {
    if (nH < 1 || nH > 4096 || nH % kv->nKV) return bad("query heads: a multiple of the KV heads, at most 4096");
    return MLXR_OK;
}
// Attention counts the pages of every sequence, KV head and group of 16 query heads in 32 bits.
int check_pages(const mlxr_paged_kv* kv, int nH) {
    const double groups = (nH / kv->nKV + 15) / 16, pages = (kv->max_len + MLXR_PAGE - 1) / MLXR_PAGE + 4;
    if (groups * pages * kv->B * kv->nKV >= 2147483648.0) return set_error(MLXR_E_UNSUPPORTED, "paged_attention: the batch could hold 2^31 pages");
    return MLXR_OK;
}
int check_work(const void* work, size_t have, int64_t need) {
    if (!work || !aligned(work, 256)) return bad("work: null or not 256-byte aligned");
    if (have < (size_t)need) return set_error(MLXR_E_INVALID_ARG, "work: " + std::to_string(have) + " bytes, " + std::to_string(need) + " needed");
    return MLXR_OK;
}
// The call's memory and stream are the current device's: every pointer that a kernel would follow is looked up, null ones
// aside. A lookup is 0.06 us. Tensors of one pool lie in one allocation, so a pointer into the last one found needs none;
// the device's number is asked for where there are several (an append of one sequence, tensors in one pool: 4.5 us a call,
// 4.4 with the pool's keys looked up alone, 5.0 with a lookup for each pointer).
int check_device(std::initializer_list<const void*> ptrs, hipStream_t s) {
    static std::atomic<int> devices{0};   // does not change while the process runs
    int dev = 0, n = devices.load(std::memory_order_relaxed);
    if ((n == 0 && (hipGetDeviceCount(&n) != hipSuccess || n == 0)) || hipGetDevice(&dev) != hipSuccess) {
        (void)hipGetLastError();
        return set_error(MLXR_E_NO_DEVICE, "no HIP GPU available");
    }
    devices.store(n, std::memory_order_relaxed);
    uintptr_t base = 0;
    size_t size = 0;
    for (const void* p : ptrs) {
        if (!p || reinterpret_cast<uintptr_t>(p) - base < size) continue;
        hipDeviceptr_t from = nullptr;
        if (hipMemGetAddressRange(&from, &size, const_cast<void*>(p)) != hipSuccess) {
            (void)hipGetLastError();
            return bad("a pointer is not to device memory");
        }
        base = reinterpret_cast<uintptr_t>(from);
        int of = dev;
        if (n > 1 && hipPointerGetAttribute(&of, HIP_POINTER_ATTRIBUTE_DEVICE_ORDINAL, const_cast<void*>(p)) != hipSuccess) {
            (void)hipGetLastError();
            return bad("a pointer is not to device memory");
        }
        if (of != dev) return bad("a pointer is to another device's memory than the current one's");
    }
    if (s) {
        hipDevice_t sd = 0;
        if (hipStreamGetDevice(s, &sd) != hipSuccess) { (void)hipGetLastError(); return bad("stream"); }
        if ((int)sd != dev) return bad("the stream is another device's than the current one");
    }
    return MLXR_OK;
}
int done(hipError_t e) { return e == hipSuccess ? MLXR_OK : set_error(MLXR_E_GPU, hipGetErrorString(e)); }
// No exception leaves a C entry (an error message that finds no memory is the only one there is).
template <typename F> int guarded(F f) {
    try {
        return f();
    } catch (...) {
        return MLXR_E_OUT_OF_MEMORY;
    }
}

}  // namespace

extern "C" {

int mlxr_k_paged_append(const mlxr_paged_kv* kv, const float* qkv, int row_stride, const float* inv_freq, const float* qn, const float* kn,
                        int nH, int rot_dim, int traditional, const int32_t* positions, float eps, float* q_out, int q_stride, void* stream) {
    return guarded([&]() -> int {
        if (int rc = check_kv(kv)) return rc;
        if (int rc = check_heads(kv, nH)) return rc;
        const int D = kv->D;
        if (!qkv || !q_out || (rot_dim && !inv_freq) || (qn == nullptr) != (kn == nullptr)) return bad("paged_append: null pointer (qn and kn go together)");
        if ((int64_t)(nH + 2 * kv->nKV) * kv->B >= (1 << 26)) return set_error(MLXR_E_UNSUPPORTED, "paged_append: 2^26 heads or more in one call");
        if (rot_dim < 0 || rot_dim > D || rot_dim % 2) return bad("paged_append: rot_dim even, 0 .. D");
        if (row_stride < (int64_t)(nH + 2 * kv->nKV) * D || q_stride < (int64_t)nH * D) return bad("paged_append: strides");
        if (q_out == qkv && q_stride != row_stride) return bad("paged_append: q_out over qkv needs its stride");
        if (!aligned(qkv, 4) || !aligned(q_out, 4) || !aligned(inv_freq, 4) || !aligned(qn, 4) || !aligned(kn, 4) || !aligned(positions, 4))
            return bad("paged_append: alignment");
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (int rc = check_device({kv->k, kv->v, kv->table, kv->len, kv->weight, kv->position, qkv, rot_dim ? inv_freq : nullptr, qn, kn, positions, q_out}, s)) return rc;
        return done(launch_paged_append(PagedAppendArgs{*kv, qkv, row_stride, inv_freq, qn, kn, nH, rot_dim, traditional, positions, eps, q_out, q_stride}, s));
    });
}

int64_t mlxr_k_paged_attention_work(const mlxr_paged_kv* kv, int nH) {
    const int rc = guarded([&]() -> int {
        if (int bad_kv = check_kv(kv)) return bad_kv;
        if (int bad_heads = check_heads(kv, nH)) return bad_heads;
        return check_pages(kv, nH);
    });
    return rc == MLXR_OK ? (int64_t)paged_attention_work(*kv, nH) : MLXR_E_INVALID_ARG;
}
int mlxr_k_paged_attention(const mlxr_paged_kv* kv, const float* q, int q_stride, int nH, int window, float scale, float* out, int out_stride,
                           const float* weight_in, float decay, void* work, size_t work_bytes, void* stream) {
    return guarded([&]() -> int {
        if (int rc = check_kv(kv)) return rc;
        if (int rc = check_heads(kv, nH)) return rc;
        if (int rc = check_pages(kv, nH)) return rc;
        if (!q || !out) return bad("paged_attention: null pointer");
        if (q_stride < (int64_t)nH * kv->D || out_stride < (int64_t)nH * kv->D || q_stride % 4 || out_stride % 4 || !aligned(q, 16) || !aligned(out, 16))
            return bad("paged_attention: q and out 16-byte aligned, strides multiples of 4 and at least nH * D");
        if (out == q && out_stride != q_stride) return bad("paged_attention: out over q needs its stride");
        if (window < 0) return bad("paged_attention: window");
        if (!(scale == scale) || !(decay == decay)) return bad("paged_attention: scale or decay is NaN");
        if (weight_in && !kv->weight) return bad("paged_attention: weight_in without the cache's weight");
        if (!aligned(weight_in, 4)) return bad("paged_attention: alignment");
        if (int rc = check_work(work, work_bytes, (int64_t)paged_attention_work(*kv, nH))) return rc;
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (int rc = check_device({kv->k, kv->v, kv->table, kv->len, kv->weight, q, out, weight_in, work}, s)) return rc;
        return done(launch_paged_attention(PagedAttnArgs{*kv, q, q_stride, nH, window, scale, out, out_stride, weight_in, decay, work}, s));
    });
}

int64_t mlxr_k_paged_evict_work(const mlxr_paged_kv* src, int budget) {
    if (guarded([&] { return check_kv(src); }) != MLXR_OK || budget < 1) return MLXR_E_INVALID_ARG;
    return (int64_t)paged_evict_work(*src, budget);
}
int mlxr_k_paged_evict(const mlxr_paged_kv* src, const mlxr_paged_kv* dst, int budget, int sink, int window, void* work, size_t work_bytes,
                       void* stream) {
    return guarded([&]() -> int {
        if (int rc = check_kv(src)) return rc;
        if (int rc = check_kv(dst)) return rc;
        if (src->B != dst->B || src->nKV != dst->nKV || src->D != dst->D || src->st != dst->st) return bad("paged_evict: src and dst differ in B, nKV, D or st");
        if (!src->weight) return bad("paged_evict: src has no weights");
        if (dst->position && !src->position) return bad("paged_evict: dst has positions, src none");
        if (budget < 1 || sink < 0 || window < 0 || (int64_t)sink + window > budget) return bad("paged_evict: budget >= 1, sink + window <= budget");
        if ((budget < src->max_len ? budget : src->max_len) > dst->max_len) return bad("paged_evict: dst holds fewer slots than the budget");
        if (src->len == dst->len || src->weight == dst->weight || (src->position && src->position == dst->position) || src->table == dst->table)
            return bad("paged_evict: src and dst share an array");
        if (int rc = check_work(work, work_bytes, (int64_t)paged_evict_work(*src, budget))) return rc;
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (int rc = check_device({src->k, src->v, src->table, src->len, src->weight, src->position, dst->k, dst->v, dst->table, dst->len,
                                   dst->weight, dst->position, work}, s)) return rc;
        return done(launch_paged_evict(PagedEvictArgs{*src, *dst, budget, sink, window, work}, s));
    });
}

int64_t mlxr_k_sample_rows_work(int rows, int V) {
    if (rows < 1 || rows > 65535 || V < 1 || V > (1 << 20)) return MLXR_E_INVALID_ARG;
    return (int64_t)sample_rows_work(rows, V);
}
int mlxr_k_sample_rows(const float* logits, int rows, int V, int64_t stride, const float* temperature, const int32_t* top_k, const float* top_p,
                       const float* min_p, const float* u, int32_t* tokens, int32_t* status, void* work, size_t work_bytes, void* stream) {
    return guarded([&]() -> int {
        if (!logits || !temperature || !u || !tokens) return bad("sample_rows: null pointer");
        if (rows < 1 || rows > 65535 || V < 1 || V > (1 << 20)) return bad("sample_rows: 1 .. 65535 rows of 1 .. 1048576 logits");
        if (stride < V) return bad("sample_rows: stride is less than V");
        if (!aligned(logits, 4) || !aligned(temperature, 4) || !aligned(top_k, 4) || !aligned(top_p, 4) || !aligned(min_p, 4) || !aligned(u, 4) ||
            !aligned(tokens, 4) || !aligned(status, 4))
            return bad("sample_rows: alignment");
        if (int rc = check_work(work, work_bytes, (int64_t)sample_rows_work(rows, V))) return rc;
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (int rc = check_device({logits, temperature, top_k, top_p, min_p, u, tokens, status, work}, s)) return rc;
        return done(launch_sample_rows(SampleRowsArgs{logits, rows, V, stride, temperature, top_k, top_p, min_p, u, tokens, status, work}, s));
    });
}

}  // extern "C"
