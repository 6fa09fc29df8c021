// Eviction from a paged KV cache by accumulated attention weight.
#include "batch.h"

namespace mlxr {

// A weight's place in the order: larger is heavier, -0 equals 0, NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Two launches: the selection leaves a list of kept slots per (KV head, sequence), the copy moves their rows. The copy
// bounds the operator: 24 sequences of 100 to 16001 slots to 4000, 8 heads of 128: 0.7 GB read and written in 142 us
// (4.9 TB/s; a copy of 4 GiB reaches 4.7), behind 21 us of selection. 4096 slots to 2048 of one sequence: 9 and 5 us.

// ---- selection: one workgroup of 1024 threads per (KV head, sequence) ----
// Of the middle slots (behind the sink, before the window) the `want` heaviest. The weights are read once, as keys
// into LDS (of sequences longer than that holds, the rest is read again from memory each time). A radix select finds
// the want-th largest key, 11, 11 and 10 bits at a time, and stops as soon as a bin is kept whole (13, 13 and 6 bits
// took 1.3 us more for 4096 slots, and no less for 16000). Then each wave
// counts in a range of slots of its own, and after one barrier writes what is kept of it in order: every larger key,
// and the first of the equal ones.
constexpr int EV_T = 1024, EV_W = EV_T / 64, EV_BINS = 2048, EV_PER = EV_BINS / EV_T;
constexpr int EV_NEAR = 32768;     // keys in LDS at most
constexpr int EV_DEFAULT = 13000;    // of these, as many as a launch may have without asking for more LDS

template <bool ALL>   // every sequence's keys are in LDS
__global__ __launch_bounds__(EV_T) void evict_select_kernel(PagedEvictArgs a, int* list, int list_stride, int near) {
    extern __shared__ uint32_t keys[];   // [near]
    __shared__ int hist[EV_BINS];
    __shared__ int sums[EV_W], kept_of[EV_W], equal_of[EV_W], pick[3];
    const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* w = a.src.weight + paged_slot(a.src, b, kvh, 0);
    const int n = paged_len(a.src, b), kept = min(n, a.budget);
    if (kvh == 0 && tid == 0) a.dst.len[b] = kept;
    int* out = list + ((int64_t)b * a.src.nKV + kvh) * list_stride;
    const int lo = min(a.sink, n), hi = n - a.window;   // the middle slots, where any goes
    const bool cut = n > kept;
    uint32_t least = 0xffffffffu;   // kept: keys above it, and of the equal ones the first `want`
    int want = 0;
    if (cut) {
        constexpr int UN = 8;   // loads in flight
        const int near_n = min(n, near);
        for (int j = tid; j < near_n; j += EV_T * UN) {
            float x[UN];
#pragma unroll
            for (int u = 0; u < UN; u++) x[u] = gload(w + min(j + EV_T * u, near_n - 1));
#pragma unroll
            for (int u = 0; u < UN; u++) if (j + EV_T * u < near_n) keys[j + EV_T * u] = weight_key(x[u]);
        }
    }
    auto key = [&](int j) { return ALL || j < near ? keys[j] : weight_key(w[j]); };
    if (cut && kept > a.sink + a.window) {
        want = kept - a.sink - a.window;
        uint32_t prefix = 0, mask = 0;
        for (int level = 0; level < 3; level++) {
            const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bins = level == 2 ? 1024 : EV_BINS;
            for (int i = tid; i < EV_BINS; i += EV_T) hist[i] = 0;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += EV_T) {
                const uint32_t k = key(j);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
            }
            __syncthreads();
            // thread t has the EV_PER bins down from EV_BINS - 1 - EV_PER t: the sums above them by a scan
            const int b1 = EV_BINS - 1 - EV_PER * tid;
            int c[EV_PER], v = 0;
#pragma unroll
            for (int h = 0; h < EV_PER; h++) v += c[h] = hist[b1 - h];
            const int own = v;
            v = wave_scan(v);
            if (lane == 63) sums[wave] = v;
            __syncthreads();
            v -= own;
            for (int i = 0; i < wave; i++) v += sums[i];
#pragma unroll
            for (int h = 0; h < EV_PER; h++) {
                if (v < want && v + c[h] >= want) {
                    pick[0] = b1 - h;
                    pick[1] = want - v;              // of this bin's
                    pick[2] = want - v == c[h];      // all of them
                }
                v += c[h];
            }
            __syncthreads();
            prefix |= (uint32_t)pick[0] << shift; mask |= (uint32_t)(bins - 1) << shift;
            want = pick[1];
            least = prefix;
            if (pick[2] && prefix) { least = prefix - 1; want = 0; break; }
        }
    } else if (cut) {
        __syncthreads();
    }
    // each wave's range: how much of it stays for sure, how much is equal to `least`
    const int per = ((n + EV_W - 1) / EV_W + 63) & ~63, j0 = min(n, wave * per), j1 = min(n, j0 + per);
    auto look = [&](int j, bool& sure, bool& equal) {
        const bool mid = cut && j >= lo && j < hi;
        const uint32_t k = mid ? key(j) : 0xffffffffu;
        sure = j < j1 && (k > least || !mid);
        equal = mid && j < j1 && k == least;
    };
    int ks = 0, es = 0;
    for (int j = j0 + lane; j - lane < j1; j += 64) {
        bool sure, equal;
        look(j, sure, equal);
        ks += (int)__popcll(__ballot(sure));
        es += (int)__popcll(__ballot(equal));
    }
    if (lane == 0) { kept_of[wave] = ks; equal_of[wave] = es; }
    __syncthreads();
    int at = 0, seen = 0;
    for (int i = 0; i < wave; i++) { at += kept_of[i]; seen += equal_of[i]; }
    at += min(seen, want);
    const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
    for (int j = j0 + lane; j - lane < j1; j += 64) {
        bool sure, equal;
        look(j, sure, equal);
        const uint64_t be = __ballot(equal);
        const bool keep = sure || (equal && seen + (int)__popcll(be & below) < want);
        const uint64_t bk = __ballot(keep);
        const int to = at + (int)__popcll(bk & below);
        if (keep && to < kept) out[to] = j;
        seen += (int)__popcll(be);
        at += (int)__popcll(bk);
    }
}

// ---- copy: one thread per 16 bytes of a kept slot's key and value rows; two of them its weight and its position too ----
__global__ __launch_bounds__(256) void evict_copy_kernel(PagedEvictArgs a, const int* list, int list_stride) {
    const int b = blockIdx.z, kvh = blockIdx.y, per = a.src.D / 8;
    const int i = blockIdx.x * 256 + threadIdx.x, to = i / per, c = i % per;
    if (to >= min(paged_len(a.src, b), a.budget)) return;
    const int from = list[((int64_t)b * a.src.nKV + kvh) * list_stride + to];
    const int ps = paged_page(a.src, b, from / MLXR_PAGE), pd = paged_page(a.dst, b, to / MLXR_PAGE);
    float w = 0.0f;
    int pos = 0;
    if (c == 0 && a.dst.weight) w = a.src.weight[paged_slot(a.src, b, kvh, from)];
    if (c == 1 && a.dst.position) pos = a.src.position[paged_slot(a.src, b, kvh, from)];
    uint4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
    if (ps >= 0) {
        const int64_t r = paged_row(a.src, ps, kvh, from % MLXR_PAGE) / 8 + c;
        k = static_cast<const uint4*>(a.src.k)[r];
        v = static_cast<const uint4*>(a.src.v)[r];
    }
    if (c == 0 && a.dst.weight) a.dst.weight[paged_slot(a.dst, b, kvh, to)] = w;
    if (c == 1 && a.dst.position) a.dst.position[paged_slot(a.dst, b, kvh, to)] = pos;
    if (pd < 0) return;
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
    const bool all = a.src.max_len <= EV_NEAR;
    const int near = all ? a.src.max_len : EV_NEAR;
    if (near > EV_DEFAULT) {   // asked for each time: it holds for the current device only
        const void* f = all ? reinterpret_cast<const void*>(evict_select_kernel<true>) : reinterpret_cast<const void*>(evict_select_kernel<false>);
        if (hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, EV_NEAR * 4)) return e;
    }
    const dim3 grid(a.src.nKV, a.src.B);
    if (all) hipLaunchKernelGGL(evict_select_kernel<true>, grid, dim3(EV_T), (size_t)near * 4, s, a, list, room, near);
    else hipLaunchKernelGGL(evict_select_kernel<false>, grid, dim3(EV_T), (size_t)near * 4, s, a, list, room, near);
    if (hipError_t e = hipGetLastError()) return e;
    const int64_t threads = (int64_t)room * (a.src.D / 8);
    hipLaunchKernelGGL(evict_copy_kernel, dim3((unsigned)((threads + 255) / 256), a.src.nKV, a.src.B), dim3(256), 0, s, a, list, room);
    return hipGetLastError();
}

}  // namespace mlxr
