// Append and decode attention of a batch of sequences over a pool of KV-cache pages.
#include "batch.h"

namespace mlxr {

template <int ST> __device__ __forceinline__ uint16_t kv_round(float v) { return ST == 0 ? f32_to_bf16(v) : f32_to_f16(v); }
template <int ST> __device__ __forceinline__ float kv_float(uint16_t v) { return ST == 0 ? bf16_to_f32(v) : f16_to_f32(v); }

// ---- append ----
// One wave per (head, sequence). Lane l holds one pair of a head's dims: of the rotated ones those that rotate
// into each other (half-split: l and l + rot / 2; neighbours: 2l and 2l + 1), of the rest two neighbours. So the
// norm is one wave sum and the rotation needs no exchange. The angle is position * frequency: 32 bits would
// leave it 2^-24 of up to 131072 radians off (0.008), so turns are counted in 64 bits, and what is left after
// whole turns goes on in 32. Keys and values are rounded once, to nearest.
template <int ST>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    const PagedKV& kv = a.kv;
    const int heads = a.nH + 2 * kv.nKV, D = kv.D;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int l = threadIdx.x & 63;
    if (item >= (int64_t)heads * kv.B) return;
    const int h = (int)(item % heads), b = (int)(item / heads);
    const int slot = paged_len(kv, b) - 1;
    if (slot < 0) return;
    const bool isQ = h < a.nH, isV = h >= a.nH + kv.nKV, on = l < D / 2;
    const int half = a.rot_dim / 2;
    const bool turns = l < half && !isV;
    const int d0 = l < half ? (a.traditional ? 2 * l : l) : 2 * l, d1 = l < half && !a.traditional ? l + half : d0 + 1;
    const float* x = a.qkv + (int64_t)b * a.row_stride + (int64_t)h * D;
    float v0 = on ? x[d0] : 0.0f, v1 = on ? x[d1] : 0.0f;
    const int pos = a.positions ? a.positions[b] : slot;
    const float* nw = isV ? nullptr : (isQ ? a.qn : a.kn);
    if (nw) {
        const float r = 1.0f / sqrtf(wave_sum(v0 * v0 + v1 * v1) / (float)D + a.eps);
        if (on) { v0 = v0 * r * nw[d0]; v1 = v1 * r * nw[d1]; }
    }
    if (turns) {
        const double t = (double)pos * (double)a.inv_freq[l] * 0.15915494309189533577;   // 1 / (2 pi)
        float sn, c;
        sincospif((float)(2.0 * (t - rint(t))), &sn, &c);
        const float o0 = v0 * c - v1 * sn, o1 = v1 * c + v0 * sn;
        v0 = o0; v1 = o1;
    }
    if (isQ) {
        float* q = a.q_out + (int64_t)b * a.q_stride + (int64_t)h * D;
        if (on) { q[d0] = v0; q[d1] = v1; }
        return;
    }
    const int page = paged_page(kv, b, slot / MLXR_PAGE), kvh = (h - a.nH) % kv.nKV;
    if (!isV && l == 0) {
        if (kv.weight) kv.weight[paged_slot(kv, b, kvh, slot)] = 0.0f;
        if (kv.position) kv.position[paged_slot(kv, b, kvh, slot)] = pos;
    }
    if (page < 0 || !on) return;
    uint16_t* row = static_cast<uint16_t*>(isV ? kv.v : kv.k) + paged_row(kv, page, kvh, slot % MLXR_PAGE);
    row[d0] = kv_round<ST>(v0);
    row[d1] = kv_round<ST>(v1);
}

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    const int64_t items = (int64_t)(a.nH + 2 * a.kv.nKV) * a.kv.B;
    const dim3 grid((unsigned)((items + 3) / 4));
    if (a.kv.st == 0) hipLaunchKernelGGL(paged_append_kernel<0>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(paged_append_kernel<1>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

// ---- attention ----
// One workgroup per (KV head, sequence). A wave takes every fourth key; lane l holds dims l and l + 64. Per head:
// running maximum m, sum and weighted values of one pass over the keys; with weights a second pass for p.
template <int ST>
__global__ __launch_bounds__(256) void paged_attn_simple_kernel(PagedAttnArgs a) {
    __shared__ float ms[4], ls[4], os[4][128], stat[4096][2];   // a head's maximum and sum
    const PagedKV& kv = a.kv;
    const int kvh = blockIdx.x, b = blockIdx.y, D = kv.D, G = a.nH / kv.nKV;
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int L = paged_len(kv, b), first = a.window > 0 && L > a.window ? L - a.window : 0;
    const uint16_t *K = static_cast<const uint16_t*>(kv.k), *V = static_cast<const uint16_t*>(kv.v);
    float* weight = kv.weight ? kv.weight + paged_slot(kv, b, kvh, 0) : nullptr;
    const float* win = a.weight_in ? a.weight_in + paged_slot(kv, b, kvh, 0) : nullptr;
    int g = 0;
    float q0, q1;
    auto query = [&] {
        const float* q = a.q + (int64_t)b * a.q_stride + (int64_t)(kvh * G + g) * D;
        q0 = q[l] * a.scale;
        q1 = D > 64 ? q[l + 64] * a.scale : 0.0f;
    };
    auto score = [&](int j, int64_t& row) {
        const int page = paged_page(kv, b, j / MLXR_PAGE);
        if (page < 0) return -INFINITY;
        row = paged_row(kv, page, kvh, j % MLXR_PAGE);
        return wave_sum(q0 * kv_float<ST>(K[row + l]) + (D > 64 ? q1 * kv_float<ST>(K[row + l + 64]) : 0.0f));
    };
    for (g = 0; g < G; g++) {
        query();
        float m = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
        for (int j = first + w; j < L; j += 4) {
            int64_t row = 0;
            const float s = score(j, row);
            if (s == -INFINITY) continue;
            const float mn = fmaxf(m, s), c = expf(m - mn), p = expf(s - mn);
            o0 = o0 * c + p * kv_float<ST>(V[row + l]);
            if (D > 64) o1 = o1 * c + p * kv_float<ST>(V[row + l + 64]);
            sum = sum * c + p;
            m = mn;
        }
        __syncthreads();
        if (l == 0) { ms[w] = m; ls[w] = sum; }
        os[w][l] = o0; os[w][l + 64] = o1;
        __syncthreads();
        const float M = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
        float total = 0.0f, o = 0.0f;
        for (int i = 0; i < 4; i++) {
            const float c = ms[i] == -INFINITY ? 0.0f : expf(ms[i] - M);
            total += ls[i] * c;
            if (threadIdx.x < D) o += os[i][threadIdx.x] * c;
        }
        if (threadIdx.x < D) a.out[(int64_t)b * a.out_stride + (int64_t)(kvh * G + g) * D + threadIdx.x] = total == 0.0f ? 0.0f : o / total;
        if (threadIdx.x == 0) { stat[g][0] = M; stat[g][1] = total; }
    }
    if (!weight) return;
    __syncthreads();
    for (int j = w; j < L; j += 4) {
        int64_t row = 0;
        float p = 0.0f;
        for (g = 0; g < G && j >= first; g++) {
            query();
            const float s = score(j, row);
            if (s != -INFINITY) p += expf(s - stat[g][0]) / stat[g][1];
        }
        if (l == 0) weight[j] = (win && a.decay != 0.0f ? a.decay * win[j] : 0.0f) + p;
    }
}

size_t paged_attention_work(const PagedKV&, int) { return 256; }

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
    const dim3 grid(a.kv.nKV, a.kv.B);
    if (a.kv.st == 0) hipLaunchKernelGGL(paged_attn_simple_kernel<0>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(paged_attn_simple_kernel<1>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace mlxr
