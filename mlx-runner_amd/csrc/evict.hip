// Eviction from a paged KV cache by accumulated attention weight.
#include "batch.h"

namespace mlxr {

// A weight's place in the order: larger is heavier, -0 equals 0, NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// ---- selection: one workgroup of 1024 threads per (KV head, sequence) ----
// Of the middle slots (behind the sink, before the window) the `want` heaviest: an 8-bit radix select of the
// want-th largest key, then one ordered pass that keeps every larger key and the first of the equal ones. The
// kept slots go to the list in order, weights and positions straight to dst.
__global__ __launch_bounds__(1024) void evict_select_kernel(PagedEvictArgs a, int* list, int list_stride) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t pick[2];
    __shared__ uint32_t wsum[2][16];
    const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = paged_len(a.src, b), kept = min(n, a.budget);
    if (kvh == 0 && tid == 0) a.dst.len[b] = kept;
    const float* w = a.src.weight + paged_slot(a.src, b, kvh, 0);
    int* out = list + ((int64_t)b * a.src.nKV + kvh) * list_stride;
    const int lo = min(a.sink, n), hi = n - a.window;
    uint32_t prefix = 0, want = 0;
    if (n > kept) {
        want = (uint32_t)(kept - a.sink - a.window);
        uint32_t mask = 0;
        for (int shift = 24; shift >= 0 && want; shift -= 8) {
            for (int i = tid; i < 256; i += 1024) hist[i] = 0;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += 1024) {
                const uint32_t k = weight_key(w[j]);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t run = 0;
                int bin = 255;
                while (bin > 0 && run + hist[bin] < want) run += hist[bin--];
                pick[0] = (uint32_t)bin; pick[1] = want - run;
            }
            __syncthreads();
            prefix |= pick[0] << shift; mask |= 255u << shift; want = pick[1];
            __syncthreads();
        }
        if (a.budget == a.sink + a.window) prefix = 0xffffffffu;   // no middle slot stays (no key is that large)
    }
    // ordered pass: per 1024 slots the kept ones before each, among the equal keys the first `want`
    uint32_t base = 0, equal = 0;
    for (int j0 = 0; j0 < n; j0 += 1024) {
        const int j = j0 + tid;
        uint32_t k = 0;
        bool mid = false, eq = false;
        if (j < n && n > kept && j >= lo && j < hi) { mid = true; k = weight_key(w[j]); eq = k == prefix; }
        const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
        const uint64_t be = __ballot(eq);
        if (lane == 0) wsum[0][wave] = (uint32_t)__popcll(be);
        __syncthreads();
        uint32_t e = equal + (uint32_t)__popcll(be & below);
        for (int i = 0; i < 16; i++) { if (i < wave) e += wsum[0][i]; equal += wsum[0][i]; }
        const bool keep = j < n && (!mid || k > prefix || (eq && e < want));
        const uint64_t bk = __ballot(keep);
        if (lane == 0) wsum[1][wave] = (uint32_t)__popcll(bk);
        __syncthreads();
        uint32_t at = base + (uint32_t)__popcll(bk & below);
        for (int i = 0; i < 16; i++) { if (i < wave) at += wsum[1][i]; base += wsum[1][i]; }
        if (keep && at < (uint32_t)kept) {
            out[at] = j;
            if (a.dst.weight) a.dst.weight[paged_slot(a.dst, b, kvh, (int)at)] = w[j];
            if (a.dst.position) a.dst.position[paged_slot(a.dst, b, kvh, (int)at)] = a.src.position[paged_slot(a.src, b, kvh, j)];
        }
        __syncthreads();
    }
}

// ---- copy: one thread per 16 bytes of a kept slot's key and value rows ----
__global__ __launch_bounds__(256) void evict_copy_kernel(PagedEvictArgs a, const int* list, int list_stride) {
    const int b = blockIdx.z, kvh = blockIdx.y, per = a.src.D / 8;
    const int i = blockIdx.x * 256 + threadIdx.x, to = i / per, c = i % per;
    if (to >= min(paged_len(a.src, b), a.budget)) return;
    const int from = list[((int64_t)b * a.src.nKV + kvh) * list_stride + to];
    const int ps = paged_page(a.src, b, from / MLXR_PAGE), pd = paged_page(a.dst, b, to / MLXR_PAGE);
    if (pd < 0) return;
    uint4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
    if (ps >= 0) {
        const int64_t r = paged_row(a.src, ps, kvh, from % MLXR_PAGE) / 8 + c;
        k = static_cast<const uint4*>(a.src.k)[r];
        v = static_cast<const uint4*>(a.src.v)[r];
    }
    const int64_t r = paged_row(a.dst, pd, kvh, to % MLXR_PAGE) / 8 + c;
    static_cast<uint4*>(a.dst.k)[r] = k;
    static_cast<uint4*>(a.dst.v)[r] = v;
}

static int evict_room(const PagedKV& src, int budget) { return budget < src.max_len ? budget : src.max_len; }

size_t paged_evict_work(const PagedKV& src, int budget) {
    return (size_t)src.B * src.nKV * evict_room(src, budget) * sizeof(int);
}

hipError_t launch_paged_evict(const PagedEvictArgs& a, hipStream_t s) {
    const int room = evict_room(a.src, a.budget);
    int* list = static_cast<int*>(a.work);
    hipLaunchKernelGGL(evict_select_kernel, dim3(a.src.nKV, a.src.B), dim3(1024), 0, s, a, list, room);
    const int64_t threads = (int64_t)room * (a.src.D / 8);
    hipLaunchKernelGGL(evict_copy_kernel, dim3((unsigned)((threads + 255) / 256), a.src.nKV, a.src.B), dim3(256), 0, s, a, list, room);
    return hipGetLastError();
}

}  // namespace mlxr
