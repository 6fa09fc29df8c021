// Attention of any number of new tokens a sequence over a pool of KV-cache pages.
#include "batch.h"

namespace mlxr {

__device__ __forceinline__ float at_times(float f, float x) { return __builtin_isinf(x) ? x : f * x; }   // for an f above 0 that may have come out as 0

// A wave per (row, query head): keys a page at a time, one a lane, then the page's values, two dims a lane.
template <int ST, bool HQ>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnRowsArgs a) {
    __shared__ float qs[4][128];
    const PagedKV& kv = a.kv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = kv.D;
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int row = (int)(item / a.nH), h = (int)(item % a.nH), kvh = h / (a.nH / kv.nKV);
    if (row >= a.rows) return;
    int b = -1;
    for (int b0 = 0; b0 < kv.B && b < 0; b0 += 64) {
        const int c = b0 + lane;
        const bool in = c < kv.B && row >= a.start[c] && row - a.start[c] < a.count[c];
        const uint64_t m = __ballot(in);
        if (m) b = b0 + (int)__builtin_ctzll(m);
    }
    if (b < 0) return;
    const int len = paged_len(kv, b), at = len - a.count[b] + (row - a.start[b]);
    const int first = a.window > 0 ? max(0, at + 1 - a.window) : 0;
    for (int d = lane; d < D; d += 64) {
        const int64_t i = (int64_t)row * a.q_stride + h * D + d;
        qs[wave][d] = a.scale * (HQ ? kv_float<ST>(static_cast<const uint16_t*>(a.q)[i]) : static_cast<const float*>(a.q)[i]);
    }
    const uint16_t *K = static_cast<const uint16_t*>(kv.k), *V = static_cast<const uint16_t*>(kv.v);
    float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
    for (int p = first / MLXR_PAGE; p * MLXR_PAGE <= at; p++) {
        const int page = paged_page(kv, b, p), key = p * MLXR_PAGE + lane;
        if (page < 0) continue;
        const int64_t base = paged_row(kv, page, kvh, 0);
        float s = -INFINITY;
        if (key >= first && key <= at) {
            s = 0.0f;
            for (int d = 0; d < D; d++) s = fmaf(qs[wave][d], kv_float<ST>(K[base + lane * D + d]), s);
        }
        const bool odd = s != s;
        const float mx = fmaxf(m, wave_max(odd ? -INFINITY : s)), ms = mx == -INFINITY ? 0.0f : mx, c = expf(m - ms), e = odd ? s : expf(s - ms);
        l = l * c + wave_sum(e);
        for (int i = 0; i < 2; i++) o[i] = m == -INFINITY ? o[i] : at_times(c, o[i]);
        m = mx;
        for (int j = 0; j < MLXR_PAGE; j++) {
            if (__shfl(s, j) == -INFINITY) continue;
            const float pj = __shfl(e, j);
            for (int i = 0; i < 2; i++)
                if (lane + 64 * i < D) o[i] += at_times(pj, kv_float<ST>(V[base + j * D + lane + 64 * i]));
        }
    }
    for (int i = 0; i < 2; i++) {
        if (lane + 64 * i >= D) continue;
        const float v = l == 0.0f ? 0.0f : o[i] / l;
        const int64_t to = (int64_t)row * a.out_stride + h * D + lane + 64 * i;
        if (HQ) static_cast<uint16_t*>(a.out)[to] = kv_round<ST>(v);
        else static_cast<float*>(a.out)[to] = v;
    }
}

size_t paged_attention_rows_work(const PagedKV& kv, int nH, int rows, int q_type) { return 256; }

hipError_t launch_paged_attention_rows(const AttnRowsArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(((int64_t)a.rows * a.nH + 3) / 4));
#define AT_GO(ST, HQ) hipLaunchKernelGGL((attn_rows_kernel<ST, HQ>), grid, dim3(256), 0, s, a)
    if (a.kv.st == 0) { if (a.q_type) AT_GO(0, true); else AT_GO(0, false); }
    else { if (a.q_type) AT_GO(1, true); else AT_GO(1, false); }
#undef AT_GO
    return hipGetLastError();
}

}  // namespace mlxr
