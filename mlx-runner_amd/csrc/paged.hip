// Append and decode attention of a batch of sequences over a pool of KV-cache pages.
#include "batch.h"

namespace mlxr {

template <int ST> __device__ __forceinline__ uint16_t kv_round(float v) { return ST == 0 ? f32_to_bf16(v) : f32_to_f16(v); }
template <int ST> __device__ __forceinline__ float kv_float(uint16_t v) { return ST == 0 ? bf16_to_f32(v) : f16_to_f32(v); }

// ---- append ----
// One wave per (head, sequence). Lane l holds one pair of a head's dims: of the rotated ones those that rotate
// into each other (half-split: l and l + rot / 2; neighbours: 2l and 2l + 1), of the rest two neighbours. So the
// norm is one wave sum and the rotation needs no exchange. Bound by the launch: 4.4 us for one sequence, 4.9 for
// 200 (10 MB), as launches follow each other. The angle is position * frequency: 32 bits would
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
    if (page < 0) return;   // the slot holds no key: its weight and position stay too
    if (!isV && l == 0) {
        if (kv.weight) kv.weight[paged_slot(kv, b, kvh, slot)] = 0.0f;
        if (kv.position) kv.position[paged_slot(kv, b, kvh, slot)] = pos;
    }
    if (!on) return;
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
//
// out = sum_j p_j v_j, p = softmax of scale q k_j over a sequence's slots, for the G query heads of a KV head at
// once: each key and value row is read once, 4 D bytes a slot, and that read bounds the kernel (G = 4 asks for 4
// multiply-adds a byte, far below what the matrix cores have).
//
// Split. A (sequence, KV head, group of 16 query heads) is a segment of ceil(slots / 64) pages. All segments' pages,
// laid end to end with PA_GAP places behind each segment (what beginning and ending one costs, in pages), are cut into
// equal runs, one per workgroup, so ragged batches keep the card as evenly busy as one long sequence, and lengths may
// stay on the device: each workgroup finds its run by a scan over the batch's page counts. A segment inside one run is
// written out at once; one cut by runs leaves partial results (maximum, sum, unnormalised values), which the last
// workgroup to finish joins in run order: the same bits every time.
//
// Inside. A wave takes 32 keys at a time, straight from memory into the operands of 16x16x32 MFMAs, without LDS:
//   S^T = K q^T: lane (m = l % 16, g = l / 16) holds 8 dims 32 s + 8 g .. of key m (step s); 16 rows of q are the
//   columns. The product leaves a lane with row l % 16's scores of keys 4 g .. 4 g + 3 of both 16-key tiles.
//   O^T = V^T P^T: those eight are what the lane has to hold of P^T as an operand, if slot e of group g stands for
//   key 4 g + e of the first tile (e < 4) or 4 g + e - 4 of the second. So lane (m, g) loads these eight keys'
//   dims (D / 16) m .., transposes them in registers (one byte permute per two values), and maximum, sum and rescale of
//   a row stay within its four lanes.
// q and p are fp32 split into parts that the matrix cores multiply exactly: three bf16 by truncation (24 bits), or
// two f16 (22 bits, q scaled to at most 2^14 by a power of two, p by 2^14). Scores are in powers of two (log2 e is
// in q's scale).
//
// Measured (bf16, D 128): 4 sequences of 99 to 131 thousand slots, 40 / 8 heads 314 us (6.0 TB/s; a copy of 4 GiB reaches
// 4.7); 32 of 0 to 8191, 32 / 8 heads 99 us (5.4 TB/s); one of 4096 11.4 us, of which 2 go by until the first keys are
// asked for, 3 until they are multiplied and 5 to hand over and join. Beside that, each change alone, in us for the three:
// two workgroups of four waves a CU 322, 102, 12.7; 512 workgroups of eight 322, 109, 13.1; no places behind a segment
// 322, 106, and 22 instead of 17.4 for a window of 1024 over 24 sequences of 5 to 16000 slots (short ones cost their ends,
// not their pages); the next keys asked for ahead of these ones' softmax, for more registers and a second copy of the
// step, 340, 121, 15.0; runs found by barriers for up to 64 sequences too 316, 101, 12.1.
constexpr int PA_WV = 8, PA_T = 64 * PA_WV;   // waves and threads of a workgroup
constexpr int PA_MAXW = 256;       // workgroups: one a CU
constexpr int PA_GAP = 4;          // places behind a segment
constexpr int PA_MINPER = 4;       // places of a run at least (one sequence of 4096: 12.1 us; with 6 13.1, with 8 15.5)
constexpr int PA_ROWS = 16;
typedef float pa_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 pa_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_h8 __attribute__((ext_vector_type(8)));
typedef uint32_t pa_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t pa_u2 __attribute__((ext_vector_type(2)));

template <int ST> __device__ __forceinline__ pa_f4 pa_mfma(uint4 a, uint4 b, pa_f4 c) {
    if constexpr (ST == 0) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_b8, a), __builtin_bit_cast(pa_b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pa_h8, a), __builtin_bit_cast(pa_h8, b), c, 0, 0, 0);
}
constexpr int pa_parts(int ST) { return ST == 0 ? 3 : 2; }
// The low (or high) halves of two words as one.
__device__ __forceinline__ uint32_t pa_lo(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t pa_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
// Eight fp32 values as parts whose sum they are (ST 0) or nearly are (ST 1).
template <int ST> __device__ __forceinline__ void pa_split(const float* x, uint4* o) {
    uint32_t w[pa_parts(ST)][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int t = 0; t < pa_parts(ST); t++) {
            if constexpr (ST == 0) {
                w[t][i] = pa_hi(__float_as_uint(a), __float_as_uint(b));
                a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
                b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
            } else {
                const _Float16 ha = (_Float16)a, hb = (_Float16)b;
                w[t][i] = (uint32_t)__builtin_bit_cast(uint16_t, ha) | ((uint32_t)__builtin_bit_cast(uint16_t, hb) << 16);
                a -= (float)ha;
                b -= (float)hb;
            }
        }
    }
#pragma unroll
    for (int t = 0; t < pa_parts(ST); t++) o[t] = uint4{w[t][0], w[t][1], w[t][2], w[t][3]};
}

struct PaWork {
    unsigned* count;      // [PA_MAXW] arrivals at the segment that starts in a run and goes on behind it; zero between calls
    float* stat;          // [B][nH][2] a row's maximum and the inverse of its sum, for the weights
    float* part;          // [2 W] partial results: [16] maxima, [16] sums, [16][D]
    float* score;         // [B][nH][score_stride], for the weights
    int score_stride, W, groups;   // groups: of 16 query heads of a KV head
};
__host__ __device__ __forceinline__ constexpr size_t pa_part_floats(int D) { return PA_ROWS * (D + 2); }

// A sequence's part of the work: keys [first, L), pages p0 .. p0 + n - 1.
struct PaSeq { int L, first, p0, n; };
__device__ __forceinline__ PaSeq pa_seq_of(const PagedAttnArgs& a, int L) {
    PaSeq s;
    s.L = L;
    s.first = a.window > 0 && s.L > a.window ? s.L - a.window : 0;
    s.p0 = s.first / MLXR_PAGE;
    s.n = s.L > 0 ? (s.L - 1) / MLXR_PAGE - s.p0 + 1 : 0;
    return s;
}
__device__ __forceinline__ PaSeq pa_seq(const PagedAttnArgs& a, int b) { return pa_seq_of(a, paged_len(a.kv, b)); }
__device__ __forceinline__ int pa_places(int pages) { return pages ? pages + PA_GAP : 0; }
__device__ __forceinline__ float pa_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float pa_safe(float m) { return m == -INFINITY ? 0.0f : m; }   // -inf - -inf would be NaN
__device__ __forceinline__ float pa_times(float f, float x) { return __builtin_isinf(x) ? x : f * x; }   // for an f above 0 that may have come out as 0
__device__ __forceinline__ void pa_store2(float* p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 pa_load2(const float* p) {
    const uint64_t v = __hip_atomic_load(const_cast<uint64_t*>(reinterpret_cast<const uint64_t*>(p)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return float2{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

template <int ST, int D, bool WT>
__global__ __launch_bounds__(PA_T, 2) void paged_attn_kernel(PagedAttnArgs a, PaWork wk) {
    constexpr int KS = D / 32, NP = pa_parts(ST), DV = D / 16, OS = D + 4;   // k steps; dims of a lane's value rows; LDS row
    constexpr int LDS_O = PA_WV * PA_ROWS * OS, LDS_C = 2 * PA_MAXW * PA_ROWS + 5 * PA_T;
    __shared__ float lds[LDS_O > LDS_C ? LDS_O : LDS_C];
    __shared__ float sm[PA_WV][PA_ROWS], sl[PA_WV][PA_ROWS];
    __shared__ uint32_t wsum[2][PA_WV], found_pre;
    __shared__ int found_b, found_len, last;
    const PagedKV& kv = a.kv;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    const uint32_t w = blockIdx.x;
    const int G = a.nH / kv.nKV;
    const uint32_t per_seq = (uint32_t)(kv.nKV * wk.groups);   // segments of a sequence
    const uint16_t *K = static_cast<const uint16_t*>(kv.k), *V = static_cast<const uint16_t*>(kv.v);

    // This workgroup's run of pages. Up to 64 sequences each wave finds by itself; more are summed 512 at a time, for
    // the total and again for the sequence in which the run begins (the host has checked that all pages of all segments
    // number less than 2^31). Idle rows get their zeros here, from one workgroup each.
    auto zero = [&](uint64_t idle, int b0) {
        for (; idle; idle &= idle - 1) {
            float* o = a.out + (int64_t)(b0 + (int)__builtin_ctzll(idle)) * a.out_stride;
            for (int i = 4 * lane; i < a.nH * D; i += 256) *reinterpret_cast<float4*>(o + i) = float4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    };
    auto run_of = [&](uint32_t places, uint32_t& per, uint32_t& t, uint32_t& t1) {   // false: there are fewer runs than workgroups
        const uint32_t all = places * per_seq;
        per = max((uint32_t)PA_MINPER, (all + wk.W - 1) / (uint32_t)wk.W);
        t = w * per;
        t1 = min(all, t + per);
        return t < all;
    };
    uint32_t per, t, t1, pre;
    int b, L;
    if (kv.B <= 64) {
        const int len = lane < kv.B ? paged_len(kv, lane) : -1, n = len < 0 ? 0 : pa_places(pa_seq_of(a, len).n);
        const uint64_t idle = __ballot(len == 0 && (uint32_t)lane % (uint32_t)wk.W == w);
        if (wave == 0) zero(idle, 0);
        const uint32_t upto = (uint32_t)wave_scan(n), before = upto - n;
        if (!run_of((uint32_t)__builtin_amdgcn_readlane((int)upto, 63), per, t, t1)) return;
        b = (int)__builtin_ctzll(__ballot(before * per_seq <= t && t < upto * per_seq));
        pre = (uint32_t)__builtin_amdgcn_readlane((int)before, b);
        L = __builtin_amdgcn_readlane(len, b);
    } else {
        uint32_t T = 0, before = 0, chunk = 0;
        int n = 0, len = 0;
        auto scan = [&](int c, bool first) {
            len = c + tid < kv.B ? paged_len(kv, c + tid) : -1;
            n = len < 0 ? 0 : pa_places(pa_seq_of(a, len).n);
            if (first) zero(__ballot(len == 0 && (uint32_t)(c + tid) % (uint32_t)wk.W == w), c + 64 * wave);
            const uint32_t v = (uint32_t)wave_scan(n);
            uint32_t* sums = wsum[(c / PA_T) & 1];
            if (lane == 63) sums[wave] = v;
            __syncthreads();
            before = v - n;
            chunk = 0;
#pragma unroll
            for (int i = 0; i < PA_WV; i++) { before += i < wave ? sums[i] : 0; chunk += sums[i]; }
        };
        for (int c = 0; c < kv.B; c += PA_T) { scan(c, true); T += chunk; }
        if (!run_of(T, per, t, t1)) return;
        uint32_t run = 0;
        for (int c = 0; c < kv.B; c += PA_T) {
            if (kv.B > PA_T) { __syncthreads(); scan(c, false); }
            const uint32_t p = run + before;
            if (p * per_seq <= t && t < (p + n) * per_seq) { found_b = c + tid; found_pre = p; found_len = len; }
            run += chunk;
            if (run * per_seq > t) break;
        }
        __syncthreads();
        b = __builtin_amdgcn_readfirstlane(found_b);
        pre = __builtin_amdgcn_readfirstlane(found_pre);
        L = __builtin_amdgcn_readfirstlane(found_len);
    }
    PaSeq sq = pa_seq_of(a, L);
    int slot = 0;   // partial results of this workgroup: its first segment's, then its last one's
    while (true) {
        const uint32_t places = (uint32_t)pa_places(sq.n), local = t - pre * per_seq, seg = local / places;
        const int tile = (int)(local - seg * places), tiles = min(sq.n - tile, (int)(t1 - t));
        // on to the run's next segment: places left of this one, then the sequences behind it
        auto ahead = [&] {
            t += places - (uint32_t)tile;
            if (t >= t1) return false;
            while (t >= (pre + (uint32_t)pa_places(sq.n)) * per_seq) { pre += (uint32_t)pa_places(sq.n); sq = pa_seq(a, ++b); }   // t < t1: another one has pages
            return true;
        };
        if (tiles <= 0) {   // the run begins behind a segment's pages
            if (!ahead()) return;
            slot = 1;            // a segment's first part is in the second place unless the run begins with it
            continue;
        }
        const int kvh = (int)(seg / (uint32_t)wk.groups), h0 = (int)(seg - kvh * wk.groups) * PA_ROWS, rows = min(PA_ROWS, G - h0);
        // page numbers, one a lane, and q's parts
        int have = 0, ids = paged_page(kv, b, sq.p0 + tile + min(lane, tiles - 1));
        uint4 q[KS][NP];
        float x[KS][8], unscale = 1.0f;
        const float* qr = a.q + (int64_t)b * a.q_stride + (int64_t)(kvh * G + h0 + min(r, rows - 1)) * D;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const float4 u = gload4(qr + 32 * s + 8 * g), v = gload4(qr + 32 * s + 8 * g + 4);
            x[s][0] = u.x; x[s][1] = u.y; x[s][2] = u.z; x[s][3] = u.w; x[s][4] = v.x; x[s][5] = v.y; x[s][6] = v.z; x[s][7] = v.w;
        }
        {
            float f = r < rows ? a.scale * 1.4426950408889634f : 0.0f;
            if constexpr (ST == 1) {
                float mx = 0.0f;
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[s][e] * f));
                mx = xor32_max(xor16_max(mx));
                int e2 = 0;
                if (mx > 0.0f && mx < INFINITY) { frexpf(mx, &e2); e2 = 14 - e2; e2 = e2 < -126 ? -126 : (e2 > 126 ? 126 : e2); }
                const float up = ldexpf(1.0f, e2);
                unscale = ldexpf(1.0f, -e2);
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[s][e] = x[s][e] * f * up;
            } else {
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[s][e] *= f;
            }
#pragma unroll
            for (int s = 0; s < KS; s++) pa_split<ST>(x[s], q[s]);
        }
        float m, l;
        pa_f4 o[DV];
        float* score = WT ? wk.score + ((int64_t)b * a.nH + kvh * G + h0 + min(r, rows - 1)) * wk.score_stride : nullptr;
        // the wave's next 32 keys from half page u on (every PA_WV-th is its own): where they are, whether there are any
        int u = wave, key0 = 0;
        int64_t base = 0;
        auto seek = [&] {
            for (; u < 2 * tiles; u += PA_WV) {
                const int tt = u >> 1;
                if ((tt >> 6) != have) {
                    have = tt >> 6;
                    ids = paged_page(kv, b, sq.p0 + tile + min(64 * have + lane, tiles - 1));
                }
                const int page = __builtin_amdgcn_readlane(ids, tt & 63);
                key0 = (sq.p0 + tile) * MLXR_PAGE + u * 32;
                if (key0 + 32 <= sq.first || key0 >= sq.L) continue;
                if (page >= 0) {
                    base = paged_row(kv, page, kvh, key0 & (MLXR_PAGE - 1));
                    return true;
                }
                if constexpr (WT)
                    if (r < rows)
#pragma unroll
                        for (int e = 0; e < 8; e++) score[key0 + (e >> 2) * 16 + 4 * g + (e & 3)] = -INFINITY;
            }
            return false;
        };
        uint4 kr[2][KS];
        uint32_t vr[8][DV / 2];
        auto load_k = [&] {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int s = 0; s < KS; s++) kr[i][s] = __builtin_bit_cast(uint4, gload(reinterpret_cast<const pa_u4*>(K + base + (16 * i + r) * D + 32 * s + 8 * g)));
        };
        auto load_v = [&] {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint16_t* row = V + base + ((e >> 2) * 16 + 4 * g + (e & 3)) * D + DV * r;
                if constexpr (DV == 8) {
                    const pa_u4 x = gload(reinterpret_cast<const pa_u4*>(row));
                    vr[e][0] = x.x; vr[e][1] = x.y; vr[e][2] = x.z; vr[e][3] = x.w;
                } else {
                    const pa_u2 x = gload(reinterpret_cast<const pa_u2*>(row));
                    vr[e][0] = x.x; vr[e][1] = x.y;
                }
            }
        };
        // Products in parts are not what infinite keys and values ask for (a part of 0 times infinity, parts of two signs). A
        // wave with a row that is not finite takes its keys again, with care: tiles that hold something infinite or NaN key by
        // key in fp32, lane (r, g) with row r's dims D / 4 g ... A score of -infinity is a key that takes no part; an infinite
        // value stays, however small its p is. A NaN in a row's query is NaN in its result, whatever the keys are. With one
        // infinite value in each cache, 32 sequences of 0 to 8191 take 185 us in place of 99, 4 of 99 to 131 thousand 515 in
        // place of 315 (900 and 2900 with all of such a wave's keys one by one). Tiles are loaded in a place of their own for
        // the look at them: a branch between loading and multiplying costs every call 2 % (102 and 320 us).
        bool careful = false, odd_q = false;
        auto odd_tile = [&] {
            uint32_t odd = 0;
            constexpr uint32_t EXP = ST == 0 ? 0x7f80u : 0x7c00u;
            auto look = [&](uint32_t w) { odd |= (uint32_t)((w & EXP) == EXP) | (uint32_t)((w >> 16 & EXP) == EXP); };
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int s = 0; s < KS; s++) { look(kr[i][s].x); look(kr[i][s].y); look(kr[i][s].z); look(kr[i][s].w); }
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int d = 0; d < DV / 2; d++) look(vr[e][d]);
            return (bool)__any(odd);
        };
        auto slow_step = [&] {
            const float f = a.scale * 1.4426950408889634f;
#pragma unroll 1
            for (int e = 0; e < 32; e++) {
                const int key = key0 + e;
                if (key < sq.first || key >= sq.L) continue;   // its score in the workspace is -infinity or unread
                const int64_t at = base + e * D + D / 4 * g;
                float sc = 0.0f;
#pragma unroll 1
                for (int d = 0; d < D / 4; d += 8) {
                    const pa_u4 k = gload(reinterpret_cast<const pa_u4*>(K + at + d));
                    const float4 y = gload4(qr + D / 4 * g + d), z = gload4(qr + D / 4 * g + d + 4);
                    const float x8[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
#pragma unroll
                    for (int c = 0; c < 8; c++) sc = fmaf(x8[c] * f, kv_float<ST>((uint16_t)(k[c / 2] >> 16 * (c & 1))), sc);
                }
                sc = xor32_sum(xor16_sum(sc));
                if constexpr (WT) if (g == ((e >> 2) & 3) && r < rows) score[key] = sc;   // the lane that wrote it before
                if (sc == -INFINITY) continue;
                const float mx = fmaxf(m, sc), c = pa_exp2(m - pa_safe(mx)), p = pa_exp2(sc - mx);
                m = mx;
                l = l * c + (g == 0 ? p : 0.0f);   // the four lanes' sums are added in the end
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < DV; j += 2) {
                        const uint32_t v = gload(reinterpret_cast<const uint32_t*>(V + at + DV * i + j));
                        constexpr float up = ST == 0 ? 1.0f : 16384.0f;
                        o[j][i] = pa_times(c, o[j][i]) + pa_times(p * up, kv_float<ST>((uint16_t)v));
                        o[j + 1][i] = pa_times(c, o[j + 1][i]) + pa_times(p * up, kv_float<ST>((uint16_t)(v >> 16)));
                    }
            }
        };
        while (true) {
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int j = 0; j < DV; j++) o[j] = pa_f4{0.0f, 0.0f, 0.0f, 0.0f};
            for (u = wave; seek(); u += PA_WV) {
                if (__builtin_expect(careful, 0)) {   // loaded again below
                    load_k();
                    load_v();
                    if (odd_q || odd_tile()) { slow_step(); continue; }
                }
                load_k();
                load_v();
                const int key = key0;
                pa_f4 sc[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    sc[i] = pa_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int s = 0; s < KS; s++)
#pragma unroll
                        for (int p = 0; p < NP; p++) sc[i] = pa_mfma<ST>(kr[i][s], q[s][p], sc[i]);
                }
                float sv[8];
#pragma unroll
                for (int e = 0; e < 8; e++) sv[e] = ST == 0 ? sc[e >> 2][e & 3] : sc[e >> 2][e & 3] * unscale;
                if (key < sq.first || key + 32 > sq.L) {   // keys outside take no part, whatever their rows hold
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int k = key + (e >> 2) * 16 + 4 * g + (e & 3);
                        if (k < sq.first || k >= sq.L) {
                            sv[e] = -INFINITY;
#pragma unroll
                            for (int d = 0; d < DV / 2; d++) vr[e][d] = 0;
                        }
                    }
                }
                if constexpr (WT)
                    if (r < rows) {
                        float* s = score + key + 4 * g;
                        *reinterpret_cast<float4*>(s) = float4{sv[0], sv[1], sv[2], sv[3]};
                        *reinterpret_cast<float4*>(s + 16) = float4{sv[4], sv[5], sv[6], sv[7]};
                    }
                float mx = fmaxf(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])), fmaxf(fmaxf(sv[4], sv[5]), fmaxf(sv[6], sv[7])));
                mx = fmaxf(m, xor32_max(xor16_max(mx)));
                if (__any(mx > m)) {
                    const float c = pa_exp2(m - pa_safe(mx));
                    l *= c;
                    if (__builtin_expect(careful, 0)) {
#pragma unroll
                        for (int j = 0; j < DV; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) o[j][i] = pa_times(c, o[j][i]);
                    } else {
#pragma unroll
                        for (int j = 0; j < DV; j++) o[j] *= c;
                    }
                    m = mx;
                }
                const float ms = pa_safe(m);
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    p[e] = pa_exp2(sv[e] - ms);
                    l += p[e];
                    if constexpr (ST == 1) p[e] *= 16384.0f;
                }
                uint4 pp[NP];
                pa_split<ST>(p, pp);
#pragma unroll
                for (int j = 0; j < DV; j++) {
                    uint4 vt;
                    if (j & 1) vt = uint4{pa_hi(vr[0][j / 2], vr[1][j / 2]), pa_hi(vr[2][j / 2], vr[3][j / 2]), pa_hi(vr[4][j / 2], vr[5][j / 2]), pa_hi(vr[6][j / 2], vr[7][j / 2])};
                    else vt = uint4{pa_lo(vr[0][j / 2], vr[1][j / 2]), pa_lo(vr[2][j / 2], vr[3][j / 2]), pa_lo(vr[4][j / 2], vr[5][j / 2]), pa_lo(vr[6][j / 2], vr[7][j / 2])};
#pragma unroll
                    for (int i = 0; i < NP; i++) o[j] = pa_mfma<ST>(vt, pp[i], o[j]);
                }
            }
            float odd[4] = {0.0f * l, 0.0f, 0.0f, 0.0f};   // NaN where one of them is not finite
#pragma unroll
            for (int j = 0; j < DV; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) odd[i] = fmaf(0.0f, o[j][i], odd[i]);
            const float any_odd = (odd[0] + odd[1]) + (odd[2] + odd[3]);
            if (careful || !__any(any_odd != any_odd && r < rows)) break;
            // rows whose query holds NaN are what they are; one that holds infinities has no tile in parts
            bool nan_q = false, inf_q = false;
#pragma unroll 1
            for (int d = 0; d < D / 4; d++) {
                const float y = gload(qr + D / 4 * g + d);
                nan_q |= y != y;
                inf_q |= __builtin_isinf(y);
            }
            uint64_t nan_rows = __ballot(nan_q);
            nan_rows |= nan_rows >> 32;
            nan_rows |= nan_rows >> 16;
            const bool mine = r < rows && !((nan_rows >> r) & 1);
            if (!__any(any_odd != any_odd && mine)) break;
            odd_q = __any(inf_q && mine);
            careful = true;
            have = -1;
        }
        // the waves' results: lane (r, g) has row r's dims DV (4 g + i) + j
        l = xor32_sum(xor16_sum(l));
        if (g == 0) { sm[wave][r] = m; sl[wave][r] = l; }
        if (r < rows) {
            float* so = lds + (wave * PA_ROWS + r) * OS;
            constexpr float down = ST == 0 ? 1.0f : 1.0f / 16384.0f;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < DV; j += 4)
                    *reinterpret_cast<float4*>(so + DV * (4 * g + i) + j) = float4{o[j][i] * down, o[j + 1][i] * down, o[j + 2][i] * down, o[j + 3][i] * down};
        }
        __syncthreads();
        const bool whole = tiles == sq.n;
        auto most = [&](int row) {   // of the waves' maxima
            float M = sm[0][row];
#pragma unroll
            for (int v = 1; v < PA_WV; v++) M = fmaxf(M, sm[v][row]);
            return M;
        };
        float* part = wk.part + (size_t)(2 * w + slot) * pa_part_floats(D);
        float* out = a.out + (int64_t)b * a.out_stride + (int64_t)(kvh * G + h0) * D;
        float* stat = WT ? wk.stat + 2 * ((int64_t)b * a.nH + kvh * G + h0) : nullptr;
        auto finish = [&](int row, int d, float M, float sum, float x, float y) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            *reinterpret_cast<float2*>(out + row * D + d) = sum == 0.0f ? float2{0.0f, 0.0f} : float2{x * inv, y * inv};
            if (WT && d == 0) *reinterpret_cast<float2*>(stat + 2 * row) = float2{M, inv};
        };
        for (int i = tid; i < rows * D / 2; i += PA_T) {
            const int row = i / (D / 2), d = 2 * (i % (D / 2));
            const float M = most(row), Ms = pa_safe(M);
            float sum = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
            for (int v = 0; v < PA_WV; v++) {
                const float c = pa_exp2(sm[v][row] - Ms);
                const float2 e = *reinterpret_cast<const float2*>(lds + (v * PA_ROWS + row) * OS + d);
                sum += c * sl[v][row]; x += c * e.x; y += c * e.y;
            }
            if (!isfinite(x + y)) {   // perhaps 0 times infinity
                x = y = 0.0f;
#pragma unroll 1
                for (int v = 0; v < PA_WV; v++) {
                    const float c = pa_exp2(sm[v][row] - Ms);
                    const float2 e = *reinterpret_cast<const float2*>(lds + (v * PA_ROWS + row) * OS + d);
                    x += pa_times(c, e.x); y += pa_times(c, e.y);
                }
            }
            if (whole) finish(row, d, Ms, sum, x, y);
            else {
                pa_store2(part + 2 * PA_ROWS + row * D + d, x, y);
                if (d == 0) pa_store2(part + 2 * row, M, sum);
            }
        }
        if (!whole) {
            // the runs that hold the segment, from the first page's to the last one's
            const uint32_t s0 = pre * per_seq + seg * places, w0 = s0 / per;
            const int parts = (int)((s0 + sq.n - 1) / per - w0) + 1, first_slot = s0 == w0 * per ? 0 : 1;
            parts_stored();
            if (tid == 0) last = part_last(wk.count + w0, parts);
            __syncthreads();
            if (last) {
                auto of = [&](int i) { return wk.part + (size_t)(2 * (w0 + i) + (i == 0 ? first_slot : 0)) * pa_part_floats(D); };
                // a thread has four dims of a row and every ways-th part: all threads have some, most parts are in flight at once
                const int items = rows * D / 4, ways = items >= PA_T ? 1 : PA_T / items;
                constexpr int CB = 8;
                float2* ml = reinterpret_cast<float2*>(lds);
                for (int e0 = 0; e0 < items; e0 += PA_T) {
                    const int at = e0 + tid, way = ways == 1 ? 0 : min(at / items, ways), item = ways == 1 ? min(at, items - 1) : at % items;
                    const int row = item / (D / 4), d = 4 * (item % (D / 4));
                    float2 e[CB][2];
                    auto load = [&](int k) {
#pragma unroll
                        for (int c = 0; c < CB; c++) {
                            const float* p = of(min(k + ways * c, parts - 1)) + 2 * PA_ROWS + row * D + d;
                            e[c][0] = pa_load2(p); e[c][1] = pa_load2(p + 2);
                        }
                    };
                    load(way);
                    if (e0 == 0) {   // all parts' maxima and sums, and the rows' maximum
                        for (int k = tid; k < parts * PA_ROWS; k += 4 * PA_T) {
                            float2 v[4];
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                const int q = min(k + PA_T * c, parts * PA_ROWS - 1);
                                v[c] = pa_load2(of(q / PA_ROWS) + 2 * min(q % PA_ROWS, rows - 1));
                            }
#pragma unroll
                            for (int c = 0; c < 4; c++) if (k + PA_T * c < parts * PA_ROWS) ml[k + PA_T * c] = v[c];
                        }
                        __syncthreads();
                        float M = -INFINITY;
                        for (int k = 4 * wave + g; k < parts; k += 4 * PA_WV) M = fmaxf(M, ml[k * PA_ROWS + r].x);
                        M = xor32_max(xor16_max(M));
                        if (g == 0) sm[wave][r] = M;
                        __syncthreads();
                    }
                    const float M = pa_safe(most(row));
                    float sum = 0.0f;
                    float4 x = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (int k = way; k < parts && way < ways; k += ways * CB) {
#pragma unroll
                        for (int c = 0; c < CB; c++) {
                            const float2 s = ml[min(k + ways * c, parts - 1) * PA_ROWS + row];
                            const float f = pa_exp2(s.x - M);   // a part of NaN counts, whatever its maximum: 0 times NaN is NaN
                            if (k + ways * c < parts) { sum += f * s.y; x.x += f * e[c][0].x; x.y += f * e[c][0].y; x.z += f * e[c][1].x; x.w += f * e[c][1].y; }
                        }
                        if (k + ways * CB < parts) load(k + ways * CB);
                    }
                    if (!isfinite((x.x + x.y) + (x.z + x.w))) {   // perhaps 0 times infinity
                        x = float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
                        for (int k = way; k < parts && way < ways; k += ways) {
                            const float f = pa_exp2(ml[k * PA_ROWS + row].x - M);
                            const float* p = of(k) + 2 * PA_ROWS + row * D + d;
                            const float2 e0 = pa_load2(p), e1 = pa_load2(p + 2);
                            x.x += pa_times(f, e0.x); x.y += pa_times(f, e0.y); x.z += pa_times(f, e1.x); x.w += pa_times(f, e1.y);
                        }
                    }
                    if (ways > 1) {   // the ways' sums, in their order
                        float* all_sums = lds + 2 * PA_ROWS * parts;
                        float* mine = all_sums + 5 * tid;
                        mine[0] = sum; mine[1] = x.x; mine[2] = x.y; mine[3] = x.z; mine[4] = x.w;
                        __syncthreads();
                        for (int v = 1; v < ways && way == 0; v++) {
                            const float* p = all_sums + 5 * (tid + v * items);
                            sum += p[0]; x.x += p[1]; x.y += p[2]; x.z += p[3]; x.w += p[4];
                        }
                    }
                    if (way == 0 && at < items) {
                        finish(row, d, M, sum, x.x, x.y);
                        finish(row, d + 2, M, sum, x.z, x.w);
                    }
                }
                if (tid == 0) part_rearm(wk.count + w0);
            }
        }
        slot = 1;
        if (!ahead()) return;
        __syncthreads();   // the LDS is written again
    }
}

// weight = decay * weight_in + the sum of p over the query heads of a KV head, from the scores that the first launch wrote
// (4 bytes a query head and slot beside 4 D a slot read there) and the rows' statistics. A launch of its own, as p needs
// the whole row's sum: 5.6 us for 16 sequences of 700 to 4100, 40 / 8 heads (8.6 MB).
__global__ __launch_bounds__(256) void paged_weight_kernel(PagedAttnArgs a, PaWork wk) {
    const PagedKV& kv = a.kv;
    const int kvh = blockIdx.y, b = blockIdx.z, G = a.nH / kv.nKV, j = blockIdx.x * 256 + threadIdx.x;
    const PaSeq s = pa_seq(a, b);
    if (j >= s.L) return;
    float p = 0.0f;
    if (j >= s.first) {
        const int64_t row = (int64_t)b * a.nH + kvh * G;
        const float2* stat = reinterpret_cast<const float2*>(wk.stat) + row;
        const float* sc = wk.score + row * wk.score_stride + j;
        for (int h = 0; h < G; h++) { const float2 st = stat[h]; p += pa_exp2(sc[(int64_t)h * wk.score_stride] - st.x) * st.y; }
    }
    const int64_t at = paged_slot(kv, b, kvh, j);
    kv.weight[at] = (a.weight_in && a.decay != 0.0f ? a.decay * a.weight_in[at] : 0.0f) + p;
}

static size_t pa_layout(const PagedKV& kv, int nH, void* base, PaWork& wk) {
    const int G = nH / kv.nKV;
    wk.groups = (G + PA_ROWS - 1) / PA_ROWS;
    const int64_t places = (kv.max_len + MLXR_PAGE - 1) / MLXR_PAGE + 1 + PA_GAP, runs = ((int64_t)kv.B * kv.nKV * wk.groups * places + PA_MINPER - 1) / PA_MINPER;
    wk.W = (int)(runs < PA_MAXW ? runs : PA_MAXW);
    wk.score_stride = (kv.max_len + MLXR_PAGE - 1) / MLXR_PAGE * MLXR_PAGE;
    uint8_t* p = static_cast<uint8_t*>(base);
    size_t at = 0;
    auto take = [&](size_t bytes) { uint8_t* q = p ? p + at : nullptr; at += (bytes + 255) / 256 * 256; return q; };
    wk.count = reinterpret_cast<unsigned*>(take(PA_MAXW * sizeof(unsigned)));   // first: where it is for every size
    wk.part = reinterpret_cast<float*>(take((size_t)2 * wk.W * pa_part_floats(kv.D) * sizeof(float)));
    wk.stat = wk.score = nullptr;
    if (kv.weight) {
        wk.stat = reinterpret_cast<float*>(take((size_t)kv.B * nH * 2 * sizeof(float)));
        wk.score = reinterpret_cast<float*>(take((size_t)kv.B * nH * wk.score_stride * sizeof(float)));
    }
    return at;
}

size_t paged_attention_work(const PagedKV& kv, int nH) {
    PaWork wk;
    return pa_layout(kv, nH, nullptr, wk);
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
    PaWork wk;
    pa_layout(a.kv, a.nH, a.work, wk);
#define PA_GO(ST, D, WT) hipLaunchKernelGGL((paged_attn_kernel<ST, D, WT>), dim3(wk.W), dim3(PA_T), 0, s, a, wk)
#define PA_D(ST, WT) do { if (a.kv.D == 64) PA_GO(ST, 64, WT); else PA_GO(ST, 128, WT); } while (0)
    if (a.kv.weight) { if (a.kv.st == 0) PA_D(0, true); else PA_D(1, true); }
    else { if (a.kv.st == 0) PA_D(0, false); else PA_D(1, false); }
#undef PA_D
#undef PA_GO
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.kv.weight) return e;
    hipLaunchKernelGGL(paged_weight_kernel, dim3((a.kv.max_len + 255) / 256, a.kv.nKV, a.kv.B), dim3(256), 0, s, a, wk);
    return hipGetLastError();
}

}  // namespace mlxr
