// What the entry points over a pool of pages check of their arguments (capi_batch.cpp, capi_rows.cpp). Everything but
// check_device runs before a device is asked for anything.
#pragma once
#include <atomic>
#include <initializer_list>
#include <string>
#include "batch.h"
#include "model.h"

namespace mlxr {

inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int bad(const char* what) { return set_error(MLXR_E_INVALID_ARG, what); }

inline int check_kv(const mlxr_paged_kv* kv) {
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
inline int check_heads(const mlxr_paged_kv* kv, int nH) {
    if (nH < 1 || nH > 4096 || nH % kv->nKV) return bad("query heads: a multiple of the KV heads, at most 4096");
    return MLXR_OK;
}
inline int check_work(const void* work, size_t have, int64_t need) {
    if (!work || !aligned(work, 256)) return bad("work: null or not 256-byte aligned");
    if (have < (size_t)need) return set_error(MLXR_E_INVALID_ARG, "work: " + std::to_string(have) + " bytes, " + std::to_string(need) + " needed");
    return MLXR_OK;
}
// The call's memory and stream are the current device's: every pointer that a kernel would follow is looked up, null ones
// aside. A lookup is 0.06 us. Tensors of one pool lie in one allocation, so a pointer into the last one found needs none;
// the device's number is asked for where there are several (an append of one sequence, tensors in one pool: 4.5 us a call,
// 4.4 with the pool's keys looked up alone, 5.0 with a lookup for each pointer).
inline int check_device(std::initializer_list<const void*> ptrs, hipStream_t s) {
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
inline int done(hipError_t e) { return e == hipSuccess ? MLXR_OK : set_error(MLXR_E_GPU, hipGetErrorString(e)); }
// No exception leaves a C entry (an error message that finds no memory is the only one there is).
template <typename F> inline int guarded(F f) {
    try {
        return f();
    } catch (...) {
        return MLXR_E_OUT_OF_MEMORY;
    }
}

}  // namespace mlxr
