// Append of any number of new tokens a sequence to a pool of KV-cache pages: norm, rotation, cache rows.
#include "batch.h"

namespace mlxr {

// Sine and cosine of position * frequency. 32 bits would leave the angle 2^-24 of up to 2^17 radians off (0.008), so turns
// are counted in 64 bits, and what is left after whole turns goes on in 32.
__device__ __forceinline__ void ar_turn(int pos, float freq, float scale, float& sn, float& c) {
    const double t = (double)pos * (double)freq * 0.15915494309189533577;   // 1 / (2 pi)
    sincospif((float)(2.0 * (t - rint(t))), &sn, &c);
    sn *= scale;
    c *= scale;
}
struct ArRow { int b, slot, pos, page; };
__device__ __forceinline__ bool ar_row(const AppendRowsArgs& a, int row, ArRow& r) {
    r.b = a.seq[row];
    r.slot = a.slot[row];
    if ((unsigned)r.b >= (unsigned)a.kv.B || (unsigned)r.slot >= (unsigned)a.kv.max_len) return false;
    r.pos = a.positions ? a.positions[row] : r.slot;
    r.page = paged_page(a.kv, r.b, r.slot / MLXR_PAGE);
    return true;
}
__device__ __forceinline__ void ar_mark(const PagedKV& kv, const ArRow& r, int kvh) {
    if (kv.weight) kv.weight[paged_slot(kv, r.b, kvh, r.slot)] = 0.0f;
    if (kv.position) kv.position[paged_slot(kv, r.b, kvh, r.slot)] = r.pos;
}

// A workgroup per row (and, where that makes no more than four workgroups a CU, per AR_T / (D / 8) of its heads: 4 rows of 512 + 2 * 128 heads take 4.9 us, 22
// without; one of 4096 + 2 * 1024 5.1 and 240; 2048 rows 14.9 and 13.8). Eight lanes (D 64) or sixteen have a head, eight
// dims each: of the rotated ones four and those that they rotate into, of the rest neighbours. So a wave asks for eight or
// four heads with two 16-byte loads a lane, the norm is a sum over a row of lanes, and a lane's four sines and cosines, which
// depend on the row alone, serve every head that it comes by. Everything is fp32 up to the one rounding of what is stored in
// the cache's type (half a step). Bound by HBM from a few hundred rows on: 2048 rows of 32 + 2 * 8 heads of 128, fp32 in and
// half out, 13.8 us, 5.5 TB/s; 4019 rows of 40 + 2 * 8 heads with fp32 queries 44.6 us, 4.8 TB/s. Five rows 4.6 us, launch
// and all.
constexpr int AR_T = 256;
template <int ST, int D, bool HQ, bool TRAD>
__global__ __launch_bounds__(AR_T) void append_rows_kernel(AppendRowsArgs a) {
    constexpr int LN = D / 8, AT = AR_T / LN;
    const PagedKV& kv = a.kv;
    const int row = blockIdx.x, l = threadIdx.x % LN, heads = a.nH + 2 * kv.nKV;
    ArRow r;
    if (!ar_row(a, row, r)) return;
    const int quarter = a.rot_dim / 8;               // lanes whose dims rotate
    const bool turns = l < quarter;
    const int dA = TRAD ? 8 * l : (turns ? 4 * l : a.rot_dim + 8 * (l - quarter)), dB = TRAD || !turns ? dA + 4 : dA + a.rot_dim / 2;
    float sn[4] = {0.0f, 0.0f, 0.0f, 0.0f}, c[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    if (turns)
#pragma unroll
        for (int i = 0; i < 4; i++) ar_turn(r.pos, a.inv_freq[4 * l + i], a.rope_scale, sn[i], c[i]);
    float wq[8], wk[8];
    if (a.qn)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = i < 4 ? dA + i : dB + i - 4;
            wq[i] = a.qn[d];
            wk[i] = a.kn[d];
        }
    const float* x = a.qkv + (int64_t)row * a.row_stride;
    for (int h = blockIdx.y * AT + threadIdx.x / LN; h < heads; h += gridDim.y * AT) {
        const bool isQ = h < a.nH, isV = h >= a.nH + kv.nKV;
        const float4 u = gload4(x + h * D + dA), w = gload4(x + h * D + dB);
        float v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
        if (a.qn) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) s += v[i] * v[i];
            s = quad_sum(s);
            s += dpp<0x141>(s);                          // row_half_mirror: 8 lanes
            if (LN == 16) s += dpp<0x140>(s);            // row_mirror: 16 lanes
            const float f = 1.0f / sqrtf(s / (float)D + a.eps);
            if (!isV)
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = v[i] * f * (isQ ? wq[i] : wk[i]);
        }
        if (turns && !isV)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int p = TRAD ? 2 * i : i, q = TRAD ? 2 * i + 1 : i + 4;
                const float o0 = v[p] * c[i] - v[q] * sn[i], o1 = v[q] * c[i] + v[p] * sn[i];
                v[p] = o0; v[q] = o1;
            }
        if (isQ && !HQ) {
            float* q = static_cast<float*>(a.q_out) + (int64_t)row * a.q_stride + h * D;
            *reinterpret_cast<float4*>(q + dA) = float4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<float4*>(q + dB) = float4{v[4], v[5], v[6], v[7]};
            continue;
        }
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = (uint32_t)kv_round<ST>(v[2 * i]) | ((uint32_t)kv_round<ST>(v[2 * i + 1]) << 16);
        uint16_t* to;
        if (isQ) to = static_cast<uint16_t*>(a.q_out) + (int64_t)row * a.q_stride + h * D;
        else {
            const int kvh = (h - a.nH) % kv.nKV;
            if (r.page < 0) continue;                  // the slot holds no key: its weight and position stay too
            if (!isV && l == 0) ar_mark(kv, r, kvh);
            to = static_cast<uint16_t*>(isV ? kv.v : kv.k) + paged_row(kv, r.page, kvh, r.slot % MLXR_PAGE);
        }
        *reinterpret_cast<uint2*>(to + dA) = uint2{o[0], o[1]};
        *reinterpret_cast<uint2*>(to + dB) = uint2{o[2], o[3]};
    }
}

// The same for any even rot_dim and any alignment: a wave per (row, head), one pair a lane (the 2048 rows 20.4 us, the five 7.1).
template <int ST, bool HQ>
__global__ __launch_bounds__(256) void append_rows_any_kernel(AppendRowsArgs a) {
    const PagedKV& kv = a.kv;
    const int heads = a.nH + 2 * kv.nKV, D = kv.D, l = threadIdx.x & 63, row = blockIdx.x, half = a.rot_dim / 2;
    ArRow r;
    if (!ar_row(a, row, r)) return;
    const bool on = l < D / 2, turns = l < half;
    const int d0 = l < half ? (a.traditional ? 2 * l : l) : 2 * l, d1 = l < half && !a.traditional ? l + half : d0 + 1;
    float sn = 0.0f, c = 1.0f;
    if (turns) ar_turn(r.pos, a.inv_freq[l], a.rope_scale, sn, c);
    for (int h = threadIdx.x >> 6; h < heads; h += 4) {
        const bool isQ = h < a.nH, isV = h >= a.nH + kv.nKV;
        const float* x = a.qkv + (int64_t)row * a.row_stride + h * D;
        float v0 = on ? x[d0] : 0.0f, v1 = on ? x[d1] : 0.0f;
        const float* nw = isV ? nullptr : (isQ ? a.qn : a.kn);
        if (nw) {
            const float f = 1.0f / sqrtf(wave_sum(v0 * v0 + v1 * v1) / (float)D + a.eps);
            if (on) { v0 = v0 * f * nw[d0]; v1 = v1 * f * nw[d1]; }
        }
        if (turns && !isV) {
            const float o0 = v0 * c - v1 * sn, o1 = v1 * c + v0 * sn;
            v0 = o0; v1 = o1;
        }
        if (isQ && !HQ) {
            float* q = static_cast<float*>(a.q_out) + (int64_t)row * a.q_stride + h * D;
            if (on) { q[d0] = v0; q[d1] = v1; }
            continue;
        }
        uint16_t* to;
        if (isQ) to = static_cast<uint16_t*>(a.q_out) + (int64_t)row * a.q_stride + h * D;
        else {
            const int kvh = (h - a.nH) % kv.nKV;
            if (r.page < 0) continue;
            if (!isV && l == 0) ar_mark(kv, r, kvh);
            to = static_cast<uint16_t*>(isV ? kv.v : kv.k) + paged_row(kv, r.page, kvh, r.slot % MLXR_PAGE);
        }
        if (on) { to[d0] = kv_round<ST>(v0); to[d1] = kv_round<ST>(v1); }
    }
}

hipError_t launch_paged_append_rows(const AppendRowsArgs& a, hipStream_t s) {
    auto at = [](const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    const bool wide = a.rot_dim % 8 == 0 && a.row_stride % 4 == 0 && a.q_stride % 4 == 0 && at(a.qkv, 16) && at(a.q_out, a.q_type ? 8 : 16);
    const int per = AR_T / (a.kv.D / 8), groups = (a.nH + 2 * a.kv.nKV + per - 1) / per;
    const dim3 grid(a.rows, wide && (int64_t)a.rows * groups <= 4 * 256 ? groups : 1);
#define AR_GO(ST, HQ) do { \
        if (!wide) hipLaunchKernelGGL((append_rows_any_kernel<ST, HQ>), grid, dim3(256), 0, s, a); \
        else if (a.kv.D == 64 && a.traditional) hipLaunchKernelGGL((append_rows_kernel<ST, 64, HQ, true>), grid, dim3(AR_T), 0, s, a); \
        else if (a.kv.D == 64) hipLaunchKernelGGL((append_rows_kernel<ST, 64, HQ, false>), grid, dim3(AR_T), 0, s, a); \
        else if (a.traditional) hipLaunchKernelGGL((append_rows_kernel<ST, 128, HQ, true>), grid, dim3(AR_T), 0, s, a); \
        else hipLaunchKernelGGL((append_rows_kernel<ST, 128, HQ, false>), grid, dim3(AR_T), 0, s, a); \
    } while (0)
    if (a.kv.st == 0) { if (a.q_type) AR_GO(0, true); else AR_GO(0, false); }
    else { if (a.q_type) AR_GO(1, true); else AR_GO(1, false); }
#undef AR_GO
    return hipGetLastError();
}

}  // namespace mlxr
