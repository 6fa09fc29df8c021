// Pages for the new tokens of a batch and back from what ended: page tables, first rows, and each row's sequence and slot
// from wanted lengths.
#include "batch.h"

namespace mlxr {

// Everything follows from three running sums over the sequences: of new tokens (a sequence's first row), of pages needed and
// of table entries given back. One workgroup makes them, keeps them where a search is quick (LDS for up to RS_NEAR
// sequences, the workspace otherwise), and then goes flat over the entries that come back, over the pages that are taken and
// over the rows, so that one long sequence among many short ones is spread over all threads too. A refusal for want of pages
// ends all later takings of pages, and one for want of rows all later rows, so the pages taken are a prefix of those asked
// for: their places need no sums of their own. All numbers are whole; the sum of new tokens is one of 64 bits.
//
// Bound by latency: a load, a scan behind a barrier and a dependent load or two for each part. 32 sequences of a token each take
// 4.4 us, launch and all; 200 prompts with 0.2 of the sequences ended 8.6, of which 5.8 here and 2.6 for the rows; 4000
// sequences that give back 7896 entries and take 1172 pages 16.0 (12.5 here: 2.0 for the sums, 3 for 4096 entries that come back, 2 for
// the pages taken). From more than RS_T sequences on a thread takes RS_EACH items at once, whose loads, scans and steps of
// the search wait together (4000 sequences: 20.5 us against 31.7 with one; 200 with one 10.1, with four 12.9).
constexpr int RS_T = 1024, RS_WV = RS_T / 64, RS_EACH = 4;
constexpr int RS_NEAR = 4095;      // sequences whose sums stay in LDS (64 KiB; 4000 16.0 us, 20.9 in the workspace)
constexpr int RS_ROWS = 4096;      // rows written by the one workgroup, a us per 1200; more by a launch over the sequences, 3 us (32
                                   // rows 4.4 us against 7.5, 24079 rows 25.5 against 8.6)
constexpr int RS_SLICE = 8192;     // rows of one sequence a wave of that launch writes

__device__ __forceinline__ int rs_pages(int slots) { return (slots + MLXR_PAGE - 1) / MLXR_PAGE; }
__device__ __forceinline__ int rs_held(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }
// A thread's items: wave w has 64 * EACH after each other, lane l the l-th of each 64 of them.
template <int EACH>
__device__ __forceinline__ int rs_item(int e) { return (int)(threadIdx.x >> 6) * 64 * EACH + e * 64 + (int)(threadIdx.x & 63); }

// For each x[e], which rise with the item, the last of n + 1 ascending sums that is at most x[e]. Those of a wave's first and
// last item are found by the whole wave, 64 places a step, and what lies between them by halves.
template <int EACH>
__device__ __forceinline__ void rs_find(const int* sums, int n, const int (&x)[EACH], int (&at)[EACH]) {
    const int lane = threadIdx.x & 63, least = __builtin_amdgcn_readlane(x[0], 0), most = __builtin_amdgcn_readlane(x[EACH - 1], 63);
    int lo = 0, hi = 0;
    for (int left = n + 1; left > 1;) {
        const int step = (left + 63) / 64, i = lo + lane * step, j = hi + lane * step;
        const bool in = lane * step < left;
        const uint64_t upto_lo = __ballot(in && i <= n && sums[min(i, n)] <= least), upto_hi = __ballot(in && j <= n && sums[min(j, n)] <= most);
        lo += ((int)__popcll(upto_lo) - 1) * step;
        hi += ((int)__popcll(upto_hi) - 1) * step;
        left = step;
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) at[e] = lo;
    if (lo == hi) return;
    for (int step = 1 << (31 - __clz(hi - lo)); step; step >>= 1) {
        int v[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) v[e] = sums[min(at[e] + step, hi)];
#pragma unroll
        for (int e = 0; e < EACH; e++) at[e] = v[e] <= x[e] ? min(at[e] + step, hi) : at[e];
    }
}

// Sums in the order of items, each at most 2^24 so that a wave's 64 stay within 32 bits. The first half leaves each wave's
// sum in LDS, and behind a barrier the second turns x[e] into what lies before the item and adds all of it to `total`.
template <typename T, int EACH>
__device__ __forceinline__ void rs_sums(T (&x)[EACH], T* sums) {
    T before = 0;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int own = (int)x[e], upto = wave_scan(own);
        x[e] = before + (upto - own);
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = before;
}
template <typename T, int EACH>
__device__ __forceinline__ void rs_before(T (&x)[EACH], const T* sums, T& total) {
    const int lane = threadIdx.x & 63;
    const T own = lane < RS_WV ? sums[lane] : T(0), upto = wave_scan(own), before = total + __shfl(upto - own, (int)(threadIdx.x >> 6));
#pragma unroll
    for (int e = 0; e < EACH; e++) x[e] += before;
    total += __shfl(upto, 63);
}

template <bool FAR, int EACH>
__global__ __launch_bounds__(RS_T) void reserve_kernel(ReserveArgs a, int own_rows) {
    __shared__ int near[FAR ? 4 : 4 * (RS_NEAR + 1)];
    __shared__ uint64_t add_sums[2][RS_WV];
    __shared__ int need_sums[2][RS_WV], back_sums[2][RS_WV], taken;
    constexpr int AT_ONCE = RS_T * EACH;
    const PagedKV& kv = a.kv;
    const int tid = threadIdx.x, B = kv.B;
    int* table = const_cast<int*>(kv.table);
    const int stride = FAR ? B + 1 : RS_NEAR + 1;
    int *start = FAR ? static_cast<int*>(a.work) : near, *need = start + stride, *back = need + stride, *len = back + stride;
    if (tid == 0) taken = 0;
    int free = rs_held(*a.n_free, kv.n_pages);
    uint64_t all_add = 0;
    int all_need = 0, all_back = 0, have[EACH], want[EACH];
    auto lengths = [&](int c) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int b = c + rs_item<EACH>(e);
            have[e] = b < B ? rs_held(kv.len[b], kv.max_len) : 0;
            want[e] = b < B ? rs_held(a.want[b], kv.max_len) : 0;
        }
    };
    for (int c = 0, i = 0; c < B; c += AT_ONCE, i ^= 1) {
        uint64_t add[EACH];
        int n[EACH], r[EACH];
        lengths(c);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int pages = rs_pages(want[e]) - rs_pages(have[e]);
            add[e] = want[e] > have[e] ? want[e] - have[e] : 0;
            n[e] = want[e] > have[e] ? pages : 0;
            r[e] = want[e] < have[e] ? -pages : 0;
        }
        rs_sums(add, add_sums[i]);
        rs_sums(n, need_sums[i]);
        rs_sums(r, back_sums[i]);
        __syncthreads();
        rs_before(add, add_sums[i], all_add);
        rs_before(n, need_sums[i], all_need);
        rs_before(r, back_sums[i], all_back);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int b = c + rs_item<EACH>(e);
            if (b >= B) break;
            start[b] = (int)min(add[e], (uint64_t)0x7fffffff);
            need[b] = n[e];
            back[b] = r[e];
            len[b] = have[e];
        }
    }
    if (tid == 0) { start[B] = (int)min(all_add, (uint64_t)0x7fffffff); need[B] = all_need; back[B] = all_back; }
    __syncthreads();
    // what comes back goes on the stack, entries outside the pool left out
    for (int e0 = 0, i = 0; e0 < all_back; e0 += AT_ONCE, i ^= 1) {
        int x[EACH], b[EACH], page[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) x[e] = min(e0 + rs_item<EACH>(e), all_back - 1);
        rs_find(back, B, x, b);
#pragma unroll
        for (int e = 0; e < EACH; e++) page[e] = paged_page(kv, b[e], rs_pages(len[b[e]]) - back[b[e] + 1] + x[e]);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            if (e0 + rs_item<EACH>(e) >= all_back) page[e] = -1;
            x[e] = page[e] >= 0;
        }
        rs_sums(x, need_sums[i]);
        __syncthreads();
        rs_before(x, need_sums[i], free);
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (page[e] >= 0 && x[e] < kv.n_pages) a.free_pages[x[e]] = page[e];
        free = min(free, kv.n_pages);
    }
    // who gets what was asked for; a wave's last granted taking reaches furthest
    int reach = 0;
    for (int c = 0; c < B; c += AT_ONCE) {
        if (B > AT_ONCE) lengths(c);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int b = c + rs_item<EACH>(e), from = b < B ? need[b] : 0, upto = b < B ? need[b + 1] : 0, first = b < B ? start[b] : 0;
            const int more = want[e] > have[e] ? want[e] - have[e] : 0;
            const bool granted = more && (int64_t)first + more <= a.rows && (upto == from || upto <= free);
            if (b < B) {
                a.start[b] = first;
                a.count[b] = granted ? more : 0;
                a.len_out[b] = granted || want[e] < have[e] ? want[e] : have[e];
            }
            const uint64_t takes = __ballot(granted && upto > from);
            if (takes) reach = __builtin_amdgcn_readlane(upto, 63 - __clzll(takes));
        }
    }
    if ((tid & 63) == 0 && reach) atomicMax(&taken, reach);
    __syncthreads();
    const int take = taken;
    if (tid == 0) *a.n_free_out = free - take;
    for (int x0 = 0; x0 < take; x0 += AT_ONCE) {   // the pages come off the top in order
        int x[EACH], b[EACH], page[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            x[e] = min(x0 + rs_item<EACH>(e), take - 1);
            page[e] = a.free_pages[free - 1 - x[e]];
        }
        rs_find(need, B, x, b);
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (x0 + rs_item<EACH>(e) < take) table[(int64_t)b[e] * kv.table_stride + rs_pages(len[b[e]]) + x[e] - need[b[e]]] = page[e];
    }
    for (int r0 = 0; r0 < own_rows; r0 += AT_ONCE) {
        int r[EACH], f[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) r[e] = r0 + rs_item<EACH>(e);
        rs_find(start, B, r, f);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            if (r[e] >= own_rows) break;
            const int b = min(f[e], B - 1), next = start[b + 1];
            const bool on = r[e] < next && next <= a.rows && (need[b + 1] == need[b] || need[b + 1] <= free);
            a.seq[r[e]] = on ? b : -1;
            a.slot[r[e]] = on ? len[b] + r[e] - start[b] : -1;
        }
    }
}

// Many rows: a wave per sequence and RS_SLICE of its rows, and all of them over the rows behind the last.
__global__ __launch_bounds__(256) void reserve_rows_kernel(ReserveArgs a) {
    const int lane = threadIdx.x & 63, waves = gridDim.x * 4, w = blockIdx.x * 4 + (threadIdx.x >> 6), B = a.kv.B;
    for (int b = w; b < B; b += waves) {
        const int start = a.start[b], next = b + 1 < B ? a.start[b + 1] : start + a.count[b], on = a.count[b], have = a.len_out[b] - on;
        const int end = min(next, a.rows);
        for (int64_t i = (int64_t)blockIdx.y * RS_SLICE + lane; i < (int64_t)(blockIdx.y + 1) * RS_SLICE && start + i < end; i += 64) {
            a.seq[start + i] = on ? b : -1;
            a.slot[start + i] = on ? have + (int)i : -1;
        }
    }
    const int total = min(a.rows, a.start[B - 1] + a.count[B - 1]);   // a last sequence that was refused has its rows behind this
    for (int64_t r = total + ((int64_t)blockIdx.y * waves + w) * 64 + lane; r < a.rows; r += (int64_t)gridDim.y * waves * 64) { a.seq[r] = -1; a.slot[r] = -1; }
}

size_t paged_reserve_work(const PagedKV& kv, int rows) { return (size_t)(kv.B + 1) * 4 * sizeof(int); }

hipError_t launch_paged_reserve(const ReserveArgs& a, hipStream_t s) {
    const bool far = a.kv.B > RS_NEAR, many = a.rows > RS_ROWS;
    const int own_rows = many ? 0 : a.rows;
    if (far) hipLaunchKernelGGL((reserve_kernel<true, RS_EACH>), dim3(1), dim3(RS_T), 0, s, a, own_rows);
    else if (a.kv.B > RS_T) hipLaunchKernelGGL((reserve_kernel<false, RS_EACH>), dim3(1), dim3(RS_T), 0, s, a, own_rows);
    else hipLaunchKernelGGL((reserve_kernel<false, 1>), dim3(1), dim3(RS_T), 0, s, a, own_rows);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !many) return e;
    const int most = a.rows < a.kv.max_len ? a.rows : a.kv.max_len, waves = a.kv.B < 4096 ? a.kv.B : 4096;
    hipLaunchKernelGGL(reserve_rows_kernel, dim3((waves + 3) / 4, (most + RS_SLICE - 1) / RS_SLICE), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace mlxr
