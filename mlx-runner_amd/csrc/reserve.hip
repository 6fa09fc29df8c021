// Pages for the new tokens of a batch and back from what ended: page tables, first rows, and each row's sequence and slot
// from wanted lengths.
#include "batch.h"

namespace mlxr {

// Everything follows from three running sums over the sequences: of new tokens (a sequence's first row), of pages needed and
// of table entries given back. One workgroup makes them, 1024 sequences at a time, keeps them where a
// binary search is quick (LDS for up to RS_NEAR sequences, the workspace otherwise), and then goes flat over the entries
// that come back, over the pages that are taken and over the rows, so that one long sequence among many short ones is spread over
// all threads too. A refusal for want of pages ends all later takings of pages, and one for want of rows all later rows, so
// the pages taken are a prefix of those asked for: their places need no sums of their own. Bound by latency: a
// load, a scan behind two barriers and a dependent load or two for each part.
constexpr int RS_T = 1024, RS_WV = RS_T / 64;
constexpr int RS_NEAR = 4095;      // sequences whose sums stay in LDS (64 KiB)
constexpr int RS_ROWS = 4096;      // rows written by the one workgroup; more by a launch over the sequences
constexpr int RS_SLICE = 8192;     // rows of one sequence a wave of that launch writes

__device__ __forceinline__ int rs_pages(int slots) { return (slots + MLXR_PAGE - 1) / MLXR_PAGE; }
__device__ __forceinline__ int rs_held(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }
// The last of n + 1 ascending sums that is at most x.
__device__ __forceinline__ int rs_find(const int* sums, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (sums[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <bool FAR>
__global__ __launch_bounds__(RS_T) void reserve_kernel(ReserveArgs a, int* far, int own_rows) {
    __shared__ int near[FAR ? 4 : 4 * (RS_NEAR + 1)];
    __shared__ uint64_t wave_add[2][RS_WV];
    __shared__ int wave_need[2][RS_WV], wave_back[2][RS_WV], taken;
    const PagedKV& kv = a.kv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, B = kv.B;
    int* table = const_cast<int*>(kv.table);
    int *start = FAR ? far : near, *need = start + (FAR ? B + 1 : RS_NEAR + 1), *back = need + (FAR ? B + 1 : RS_NEAR + 1), *len = back + (FAR ? B + 1 : RS_NEAR + 1);
    if (tid == 0) taken = 0;
    uint64_t rows_before = 0;
    int need_before = 0, back_before = 0;
    for (int c = 0, i = 0; c < B; c += RS_T, i ^= 1) {
        const int b = c + tid;
        const int have = b < B ? rs_held(kv.len[b], kv.max_len) : 0, want = b < B ? rs_held(a.want[b], kv.max_len) : 0;
        const int more = want > have ? want - have : 0, pages = rs_pages(want) - rs_pages(have);
        const int n = more ? pages : 0, r = want < have ? -pages : 0;
        const uint64_t add_upto = wave_scan((uint64_t)more);
        const int need_upto = wave_scan(n), back_upto = wave_scan(r);
        if (lane == 63) { wave_add[i][wave] = add_upto; wave_need[i][wave] = need_upto; wave_back[i][wave] = back_upto; }
        __syncthreads();
        uint64_t x = rows_before + add_upto - (uint64_t)more;
        int y = need_before + need_upto - n, z = back_before + back_upto - r;
        for (int v = 0; v < RS_WV; v++) {
            if (v < wave) { x += wave_add[i][v]; y += wave_need[i][v]; z += wave_back[i][v]; }
            rows_before += wave_add[i][v]; need_before += wave_need[i][v]; back_before += wave_back[i][v];
        }
        if (b < B) {
            start[b] = (int)min(x, (uint64_t)0x7fffffff);
            need[b] = y;
            back[b] = z;
            len[b] = have;
        }
    }
    if (tid == 0) { start[B] = (int)min(rows_before, (uint64_t)0x7fffffff); need[B] = need_before; back[B] = back_before; }
    __syncthreads();
    // what comes back goes on the stack, entries outside the pool left out
    int free = rs_held(*a.n_free, kv.n_pages);
    for (int e0 = 0; e0 < back_before; e0 += RS_T) {
        const int e = e0 + tid;
        int page = -1;
        if (e < back_before) {
            const int b = rs_find(back, B, e);
            page = paged_page(kv, b, rs_pages(len[b]) - (back[b + 1] - back[b]) + e - back[b]);
        }
        const uint64_t in = __ballot(page >= 0);
        if (lane == 0) wave_need[0][wave] = (int)__popcll(in);
        __syncthreads();
        int at = free + (int)__popcll(in & (((uint64_t)1 << lane) - 1));
        for (int v = 0; v < RS_WV; v++) {
            at += v < wave ? wave_need[0][v] : 0;
            free += wave_need[0][v];
        }
        if (page >= 0 && at < kv.n_pages) a.free_pages[at] = page;
        free = min(free, kv.n_pages);
        __syncthreads();
    }
    // who gets what was asked for
    for (int b = tid; b < B; b += RS_T) {
        const int have = len[b], want = rs_held(a.want[b], kv.max_len), more = want > have ? want - have : 0;
        const int upto = need[b + 1];
        const bool granted = more && (int64_t)start[b] + more <= a.rows && (upto == need[b] || upto <= free);
        a.start[b] = start[b];
        a.count[b] = granted ? more : 0;
        a.len_out[b] = granted || want < have ? want : have;
        if (granted && upto > need[b]) atomicMax(&taken, upto);
        if (!FAR && far) far[b] = have;
    }
    __syncthreads();
    const int take = taken;
    if (tid == 0) *a.n_free_out = free - take;
    for (int x = tid; x < take; x += RS_T) {   // the pages come off the top in order
        const int b = rs_find(need, B, x);
        table[(int64_t)b * kv.table_stride + rs_pages(len[b]) + x - need[b]] = a.free_pages[free - 1 - x];
    }
    for (int r = tid; r < own_rows; r += RS_T) {
        const int b = min(rs_find(start, B, r), B - 1), next = start[b + 1];
        const bool on = r < next && next <= a.rows && (need[b + 1] == need[b] || need[b + 1] <= free);
        a.seq[r] = on ? b : -1;
        a.slot[r] = on ? len[b] + r - start[b] : -1;
    }
}

// Many rows: a wave per sequence and RS_SLICE of its rows, and all of them over the rows behind the last.
__global__ __launch_bounds__(256) void reserve_rows_kernel(ReserveArgs a, const int* len) {
    const int lane = threadIdx.x & 63, waves = gridDim.x * 4, w = blockIdx.x * 4 + (threadIdx.x >> 6), B = a.kv.B;
    for (int b = w; b < B; b += waves) {
        const int start = a.start[b], next = b + 1 < B ? a.start[b + 1] : start + a.count[b], on = a.count[b], have = len[b];
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
    int* work = static_cast<int*>(a.work);
    if (far) hipLaunchKernelGGL(reserve_kernel<true>, dim3(1), dim3(RS_T), 0, s, a, work, many ? 0 : a.rows);
    else hipLaunchKernelGGL(reserve_kernel<false>, dim3(1), dim3(RS_T), 0, s, a, many ? work : nullptr, many ? 0 : a.rows);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !many) return e;
    const int most = a.rows < a.kv.max_len ? a.rows : a.kv.max_len, waves = a.kv.B < 4096 ? a.kv.B : 4096;
    hipLaunchKernelGGL(reserve_rows_kernel, dim3((waves + 3) / 4, (most + RS_SLICE - 1) / RS_SLICE), dim3(256), 0, s, a, far ? work + 3 * (size_t)(a.kv.B + 1) : work);
    return hipGetLastError();
}

}  // namespace mlxr
