// Token selection of many rows from given random numbers: temperature, top-k, top-p and min-p over the whole
// vocabulary.
//
// Every cut and the draw itself are one question, asked of the tokens in rank order (logit descending, equal
// ones by index): where does a running sum of weights w = exp((v - max) / T) (top-k: of ones) reach a target? The
// answer needs the order only where the sum crosses. Two launches:
//   1. sample_groups_kernel, several workgroups a row: the maximum of every 64 logits. One read of the logits, and
//      that read bounds the operator: 0.6 MB a row of 152 thousand.
//   2. sample_pick_kernel. With the row's maximum known, tokens fall into bins of 1/64 of x = (max - v) / T, 2048 of
//      them (what lies behind x = 32 has no weight that counts). Where the sum of a whole row matters (top-p or
//      nothing over all tokens) its workgroups first add up the bins' weights, and the last one goes on alone: it
//      finds the bins in which the sums cross, gathers just their tokens (the groups' maxima say where none are),
//      sorts them and walks. For top-k and min-p alone no sum over the row is needed: the groups' maxima give a
//      bin down to which there are k tokens or more, and these are gathered and sorted at once.
// A bin's weights are a constant times f in (exp(-1/64), 1], added as multiples of 2^-43: no order of the atomic adds
// changes a result, and 2^20 of them stay below 2^63. Everything else is 64-bit floating point: a draw lies next to
// a border only if it is within about 2^-43 of it.
// Rows whose crossing bins hold too many tokens for that (thousands of equal logits, top-k of thousands) take the
// radix descent instead, which asks for no room: a histogram of the order keys' leading bits, the bin in which the
// sum crosses, and again within that bin, until one key is left, whose tokens have one weight.
#include "batch.h"

namespace mlxr {

constexpr double SR_ONE = 8796093022208.0;   // 2^43: the weight of the largest logit
constexpr int SR_T = 1024, SR_BINS = 2048;
constexpr uint32_t SR_MINUS_INF = 0x007fffffu;   // the order key of -infinity; NaN has 0

__device__ __forceinline__ uint32_t sr_key(float v) {
    if (v != v) return 0u;
    const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sr_value(uint32_t k) { return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k); }

struct SrRow {
    const float* v; int V;
    float top;          // the largest logit
    double inv;         // 1 / T
    __device__ __forceinline__ double weight(float x) const { return exp(((double)x - (double)top) * inv); }
    __device__ __forceinline__ uint64_t fixed(float x) const { return (uint64_t)(weight(x) * SR_ONE + 0.5); }
};

// The tokens with a key above `key`, and `n` of those that have it (lowest indices first).
struct SrCut { uint32_t key; uint32_t n; };
__device__ __forceinline__ SrCut sr_min(SrCut a, SrCut b) {   // the shorter of two prefixes of the rank order
    if (a.key != b.key) return a.key > b.key ? a : b;
    return a.n < b.n ? a : b;
}

struct SrShared {
    uint64_t mass[SR_BINS];
    uint32_t count[SR_BINS];
    uint64_t wmass[16], sum;
    uint32_t wcount[16], pick;
    uint64_t above_mass; uint32_t above_count;
};

// Sum over the workgroup, to every thread.
__device__ uint64_t sr_sum(uint64_t v, SrShared& sh) {
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wmass[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < SR_T / 64; i++) t += sh.wmass[i];
    return t;
}
__device__ uint64_t sr_max(uint64_t v, SrShared& sh) {
    for (int o = 1; o < 64; o <<= 1) { const uint64_t p = __shfl_xor(v, o, 64); v = p > v ? p : v; }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wmass[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < SR_T / 64; i++) t = sh.wmass[i] > t ? sh.wmass[i] : t;
    return t;
}
// The sum of the weights within a cut.
__device__ uint64_t sr_mass(const SrRow& r, SrCut cut, SrShared& sh) {
    uint64_t t = 0;
    for (int i = threadIdx.x; i < r.V; i += SR_T) if (sr_key(r.v[i]) > cut.key) t += r.fixed(r.v[i]);
    if (threadIdx.x == 0 && cut.n) t += cut.n * r.fixed(sr_value(cut.key));
    return sr_sum(t, sh);
}

// The shortest prefix of the cut's tokens whose count (by_mass false) or sum of weights reaches `target` (>= 1):
// the whole cut if none does. *mass: its sum of weights.
__device__ SrCut sr_descend(const SrRow& r, SrCut cut, bool by_mass, uint64_t target, SrShared& sh, uint64_t* mass) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t prefix = 0, mask = 0, above_count = 0;
    uint64_t above_mass = 0;
    const uint64_t edge = cut.n ? r.fixed(sr_value(cut.key)) : 0;   // the weight of the tokens at the cut's key
    const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
    for (int level = 0; level < 3; level++) {
        const int shift = shifts[level];
        const uint32_t bins = 1u << bits[level];
        __syncthreads();
        for (int i = tid; i < SR_BINS; i += SR_T) { sh.mass[i] = 0; sh.count[i] = 0; }
        __syncthreads();
        for (int i = tid; i < r.V; i += SR_T) {
            const float x = r.v[i];
            const uint32_t k = sr_key(x);
            if (k > cut.key && (k & mask) == prefix) {
                const uint32_t bin = (k >> shift) & (bins - 1);
                atomicAdd(&sh.count[bin], 1u);
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[bin]), (unsigned long long)r.fixed(x));
            }
        }
        __syncthreads();
        if (tid == 0 && cut.n && (cut.key & mask) == prefix) {
            const uint32_t bin = (cut.key >> shift) & (bins - 1);
            sh.count[bin] += cut.n;
            sh.mass[bin] += cut.n * edge;
        }
        if (tid == 0) { sh.pick = 0xffffffffu; }
        __syncthreads();
        // thread t has bins - 1 - 2t and the one below it: sums of everything above by scans
        const int b1 = (int)bins - 1 - 2 * tid, b0 = b1 - 1;
        const uint32_t c1 = b1 >= 0 ? sh.count[b1] : 0, c0 = b0 >= 0 ? sh.count[b0] : 0;
        const uint64_t m1 = b1 >= 0 ? sh.mass[b1] : 0, m0 = b0 >= 0 ? sh.mass[b0] : 0;
        uint32_t c = c1 + c0;
        uint64_t m = m1 + m0;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t c2 = __shfl_up(c, o, 64);
            const uint64_t m2 = __shfl_up(m, o, 64);
            if (lane >= o) { c += c2; m += m2; }
        }
        if (lane == 63) { sh.wcount[wave] = c; sh.wmass[wave] = m; }
        __syncthreads();
        uint32_t ca = above_count, call = above_count;
        uint64_t ma = above_mass, mall = above_mass;
        for (int i = 0; i < SR_T / 64; i++) {
            if (i < wave) { ca += sh.wcount[i]; ma += sh.wmass[i]; }
            call += sh.wcount[i]; mall += sh.wmass[i];
        }
        if (level == 0 && (by_mass ? mall : (uint64_t)call) < target) { *mass = mall; return cut; }
        ca += c - c1 - c0; ma += m - m1 - m0;   // above this thread's bins
        const uint64_t s0 = by_mass ? ma : ca, s1 = s0 + (by_mass ? m1 : c1), s2 = s1 + (by_mass ? m0 : c0);
        if (s0 < target && s2 >= target) {   // one thread: sums only grow
            const bool upper = s1 >= target;
            sh.pick = (uint32_t)(upper ? b1 : b0);
            sh.above_count = ca + (upper ? 0 : c1);
            sh.above_mass = ma + (upper ? 0 : m1);
        }
        __syncthreads();
        prefix |= sh.pick << shift; mask |= (bins - 1) << shift;
        above_count = sh.above_count; above_mass = sh.above_mass;
    }
    const uint64_t w = r.fixed(sr_value(prefix));
    uint64_t need = target - (by_mass ? above_mass : (uint64_t)above_count);
    if (by_mass) need = w ? (need + w - 1) / w : 1;
    *mass = above_mass + need * w;
    return SrCut{prefix, (uint32_t)need};
}

// The index of the n-th (from 1) token with this key.
__device__ int sr_nth(const SrRow& r, uint32_t key, uint32_t n, SrShared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = ((r.V + 15) / 16 + 63) & ~63;
    const int i0 = min(r.V, wave * per), i1 = min(r.V, i0 + per);
    uint32_t c = 0;
    for (int i = i0; i < i1; i += 64) c += (uint32_t)__popcll(__ballot(i + lane < i1 && sr_key(r.v[min(i + lane, r.V - 1)]) == key));
    __syncthreads();
    if (lane == 0) sh.wcount[wave] = c;
    if (threadIdx.x == 0) sh.pick = 0;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; w++) before += sh.wcount[w];
    if (before < n && before + c >= n) {
        for (int i = i0; i < i1; i += 64) {
            const bool hit = i + lane < i1 && sr_key(r.v[min(i + lane, r.V - 1)]) == key;
            const uint64_t m = __ballot(hit);
            const uint32_t at = before + (uint32_t)__popcll(m & (lane ? ~0ull >> (64 - lane) : 0ull)) + 1;
            if (hit && at == n) sh.pick = (uint32_t)(i + lane);
            before += (uint32_t)__popcll(m);
            if (before >= n) break;
        }
    }
    __syncthreads();
    return (int)sh.pick;
}

// A target a fraction of a sum: the least whole number not below it, at least 1.
__device__ __forceinline__ uint64_t sr_target(double share, uint64_t sum) {
    const double t = ceil(share * (double)sum);
    if (!(t >= 1.0)) return 1;
    return t >= (double)sum ? sum : (uint64_t)t;
}

// The radix descent over a whole row: any parameters, one workgroup.
__device__ int sr_descent_token(const SampleRowsArgs& a, int row, const SrRow& r, uint32_t top, SrShared& sh) {
    const int tid = threadIdx.x;
    uint64_t mass = 0, kept_mass = 0;
    SrCut cut{SR_MINUS_INF, 0};
    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < r.V) cut = sr_descend(r, cut, false, (uint64_t)k, sh, &mass);
    else mass = sr_mass(r, cut, sh);
    SrCut end = cut;
    kept_mass = mass;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    if (p < 1.0f) end = sr_descend(r, cut, true, sr_target((double)p, mass), sh, &kept_mass);
    const float low = a.min_p ? a.min_p[row] : 0.0f;
    if (low > 0.0f) {
        uint64_t least = 0;   // the complement of the smallest key that stays
        for (int i = tid; i < r.V; i += SR_T) {
            const uint32_t key = sr_key(r.v[i]);
            if (key > SR_MINUS_INF && r.weight(r.v[i]) >= (double)low) { const uint64_t c = (uint32_t)~key; least = c > least ? c : least; }
        }
        least = sr_max(least, sh);
        const SrCut by = least ? SrCut{~(uint32_t)least, 0xffffffffu} : SrCut{top, 1u};
        const SrCut both = sr_min(end, by);
        if (both.key != end.key || both.n != end.n) {
            end = both;
            if (end.n == 0xffffffffu) {   // every token with that key
                uint64_t c = 0;
                for (int i = tid; i < r.V; i += SR_T) c += sr_key(r.v[i]) == end.key;
                end.n = (uint32_t)sr_sum(c, sh);
            }
            kept_mass = sr_mass(r, end, sh);
        }
    }
    uint64_t unused;
    const SrCut at = sr_descend(r, end, true, sr_target((double)a.u[row], kept_mass), sh, &unused);
    return sr_nth(r, at.key, at.n, sh);
}

// ---- bins, gathered tokens and their order ----
constexpr int SR_GROUP = 64, SR_LIST = 2048;
constexpr double SR_WIDTH = 64.0;   // bins per unit of x

struct SrWork {
    float* gmax;        // [rows][groups]
    uint64_t* mass;     // [rows][SR_BINS]: sums of f, cleared by the first launch where the second adds to them
    unsigned* count;    // [rows]: the workgroups that have added theirs
    int groups, spans, per;   // groups of a row; workgroups of a row and the groups of each
};

// What a row asks for.
enum SrKind { SR_GREEDY, SR_TOP, SR_SUM };   // the first rank; the first ones by count or weight; sums over the row
struct SrAsk { SrKind kind; int k; float p, low; };
__device__ __forceinline__ SrAsk sr_ask(const SampleRowsArgs& a, int row) {
    SrAsk q;
    q.k = a.top_k ? a.top_k[row] : 0;
    if (q.k <= 0 || q.k > a.V) q.k = a.V;
    q.p = a.top_p ? a.top_p[row] : 1.0f;
    q.low = a.min_p ? a.min_p[row] : 0.0f;
    const float T = a.temperature[row];
    if (!(T > 0.001f)) q.kind = SR_GREEDY;
    else q.kind = q.k == a.V && (q.p < 1.0f || !(q.low > 0.0f)) && a.V > SR_LIST ? SR_SUM : SR_TOP;
    return q;
}

struct SrBins {
    double top, inv;   // the largest logit, bins per unit of logit
    __device__ __forceinline__ double x(float v) const { return (top - (double)v) * inv; }   // in bins; NaN or infinite outside
};
// exp(-y / 64) for y in [0, 1): the Taylor sum to the fifth power is off by 2^-45.
__device__ __forceinline__ double sr_small_exp(double y) {
    y *= 1.0 / SR_WIDTH;
    return 1.0 - y * (1.0 - y * (0.5 - y * (1.0 / 6 - y * (1.0 / 24 - y * (1.0 / 120)))));
}
__device__ __forceinline__ uint64_t sr_fixed(double x, int bin) { return (uint64_t)(sr_small_exp(x - (double)bin) * SR_ONE + 0.5); }

// Per 64 logits the maximum (NaN ignored). A lane has four neighbours, 16 lanes a group.
template <bool VEC>
__global__ __launch_bounds__(256) void sample_groups_kernel(SampleRowsArgs a, SrWork wk) {
    const int row = blockIdx.y, span = blockIdx.x, tid = threadIdx.x;
    const float* v = a.logits + (int64_t)row * a.stride;
    if (tid == 0 && span == 0) wk.count[row] = 0;
    if (sr_ask(a, row).kind == SR_SUM)
        for (int i = span * 256 + tid; i < SR_BINS; i += wk.spans * 256) wk.mass[(int64_t)row * SR_BINS + i] = 0;
    const int g1 = min(wk.groups, (span + 1) * wk.per);
    constexpr int UN = 4;   // loads in flight
    for (int g = span * wk.per + (tid >> 4); g < g1; g += 16 * UN) {
        float4 x[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int i = (g + 16 * u) * SR_GROUP + 4 * (tid & 15);
            x[u] = float4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (g + 16 * u < g1) {
                if (i + 4 <= a.V) {
                    if constexpr (VEC) x[u] = gload4(v + i);
                    else x[u] = float4{gload(v + i), gload(v + i + 1), gload(v + i + 2), gload(v + i + 3)};
                } else {
                    if (i < a.V) x[u].x = v[i];
                    if (i + 1 < a.V) x[u].y = v[i + 1];
                    if (i + 2 < a.V) x[u].z = v[i + 2];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const float m = row16_max(fmaxf(fmaxf(fmaxf(-INFINITY, x[u].x), x[u].y), fmaxf(fmaxf(-INFINITY, x[u].z), x[u].w)));
            if ((tid & 15) == 0 && g + 16 * u < g1) wk.gmax[(int64_t)row * wk.groups + g + 16 * u] = m;
        }
    }
}

struct SrPick {
    uint64_t list[SR_LIST], ranked[SR_LIST];
    double run[SR_LIST], wave_sum[16];
    int ids[SR_T];
    int n, nids, first;
    uint32_t best;
    float wave_top[16];
};

// Running sums (inclusive) of two values a thread, 2 tid and 2 tid + 1, over the workgroup: into run.
__device__ void sr_scan(double a0, double a1, SrPick& s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    double v = a0 + a1;
    for (int o = 1; o < 64; o <<= 1) { const double u = __shfl_up(v, o, 64); if (lane >= o) v += u; }
    __syncthreads();
    if (lane == 63) s.wave_sum[wave] = v;
    __syncthreads();
    double before = 0.0;
    for (int i = 0; i < wave; i++) before += s.wave_sum[i];
    const double up = __shfl_up(v, 1, 64);
    if (lane) before += up;
    s.run[2 * tid] = before + a0;
    s.run[2 * tid + 1] = (before + a0) + a1;
    __syncthreads();
}
// The first i < n with run[i] + base >= target; n if there is none.
__device__ int sr_first(double target, double base, int n, SrPick& s) {
    __syncthreads();
    if (threadIdx.x == 0) s.first = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += SR_T)
        if (s.run[i] + base >= target && (i == 0 || !(s.run[i - 1] + base >= target))) atomicMin(&s.first, i);
    __syncthreads();
    return s.first;
}
// The first i < n whose weight is below `low` (in [.., n]); the ranked tokens' weights fall.
__device__ int sr_first_below(double low, int n, const SrBins& bins, SrPick& s) {
    __syncthreads();
    if (threadIdx.x == 0) s.first = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += SR_T)
        if (exp(-bins.x(sr_value((uint32_t)(s.ranked[i] >> 32))) / SR_WIDTH) < low) atomicMin(&s.first, i);
    __syncthreads();
    return s.first;
}

// Gathers the tokens of bins b0 .. b1, ranked, with running sums of their weights in run. Returns how many there
// are; more than SR_LIST: nothing else is done.
__device__ int sr_gather(const SrRow& r, const SrBins& bins, const float* gmax, int groups, int b0, int b1, SrPick& s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __syncthreads();
    if (tid == 0) s.n = 0;
    for (int base = 0; base < groups; base += SR_T) {
        if (tid == 0) s.nids = 0;
        __syncthreads();
        const int g = base + tid;
        const bool has = g < groups && bins.x(gmax[g]) < (double)(b1 + 1);
        const uint64_t m = __ballot(has);
        int at = 0;
        if (lane == 0 && m) at = atomicAdd(&s.nids, (int)__popcll(m));
        at = __shfl(at, 0, 64) + (int)__popcll(m & (lane ? ~0ull >> (64 - lane) : 0ull));
        if (has) s.ids[at] = g;
        __syncthreads();
        const int n = s.nids;
        constexpr int UN = 4;
        for (int i = wave; i < n; i += 16 * UN) {
            float v[UN];
            int idx[UN];
#pragma unroll
            for (int u = 0; u < UN; u++) {
                idx[u] = i + 16 * u < n ? s.ids[i + 16 * u] * SR_GROUP + lane : r.V;
                v[u] = idx[u] < r.V ? r.v[idx[u]] : -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < UN; u++) {
                const double x = bins.x(v[u]);
                const bool in = x >= (double)b0 && x < (double)(b1 + 1);
                const uint64_t mi = __ballot(in);
                if (!mi) continue;
                int to = 0;
                if (lane == 0) to = atomicAdd(&s.n, (int)__popcll(mi));
                to = __shfl(to, 0, 64) + (int)__popcll(mi & (lane ? ~0ull >> (64 - lane) : 0ull));
                if (in && to < SR_LIST) s.list[to] = ((uint64_t)sr_key(v[u]) << 32) | (uint32_t)~(uint32_t)idx[u];
            }
        }
        __syncthreads();
    }
    const int n = s.n;
    if (n > SR_LIST) return n;
    // each wave sorts its runs of 64 in registers; a key's rank is its place in its run and, for every other run, how
    // many of that run's keys are larger
    const int runs = (n + 63) / 64;
    uint64_t mine[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int q = wave + 16 * h;
        mine[h] = 0;
        if (q < runs) {
            mine[h] = 64 * q + lane < n ? s.list[64 * q + lane] : 0;
            uint64_t k = mine[h];
#pragma unroll
            for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
                for (int d = size >> 1; d > 0; d >>= 1) {
                    const uint64_t p = __shfl_xor(k, d, 64);
                    const bool lower = (lane & d) == 0, desc = size == 64 || (lane & size) == 0;
                    k = (lower == desc) ? (p > k ? p : k) : (p < k ? p : k);
                }
            mine[h] = k;
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; h++) if (wave + 16 * h < runs) s.list[64 * (wave + 16 * h) + lane] = mine[h];
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int q = wave + 16 * h;
        if (q >= runs) continue;
        int rank = lane;
        for (int o = 0; o < runs; o++) {
            if (o == q) continue;
            const uint64_t* run = s.list + 64 * o;
            int lo = 0;
#pragma unroll
            for (int step = 32; step > 0; step >>= 1) lo += run[lo + step - 1] > mine[h] ? step : 0;
            lo += run[lo] > mine[h] ? 1 : 0;
            rank += lo;
        }
        if (mine[h]) s.ranked[rank] = mine[h];
    }
    __syncthreads();
    double w[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        w[h] = 0.0;
        if (2 * tid + h < n) {
            const double x = bins.x(sr_value((uint32_t)(s.ranked[2 * tid + h] >> 32)));
            const int bin = (int)x;
            w[h] = exp((double)-bin / SR_WIDTH) * (double)sr_fixed(x, bin);   // as the bins' sums have it
        }
    }
    sr_scan(w[0], w[1], s);
    return n;
}

__global__ __launch_bounds__(SR_T) void sample_pick_kernel(SampleRowsArgs a, SrWork wk) {
    __shared__ union { SrShared sh; SrPick pick; } u;
    __shared__ int go;
    SrPick& s = u.pick;
    const int row = blockIdx.y, span = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const SrAsk ask = sr_ask(a, row);
    if (span && ask.kind != SR_SUM) return;
    SrRow r;
    r.v = a.logits + (int64_t)row * a.stride;
    r.V = a.V;
    const float* gmax = wk.gmax + (int64_t)row * wk.groups;
    float top = -INFINITY;
    for (int g = tid; g < wk.groups; g += SR_T) top = fmaxf(top, gmax[g]);
    top = wave_max(top);
    if (lane == 0) s.wave_top[wave] = top;
    __syncthreads();
    for (int i = 0; i < 16; i++) top = fmaxf(top, s.wave_top[i]);
    if (!isfinite(top)) {   // none, or infinite
        if (span == 0 && tid == 0) { a.tokens[row] = 0; if (a.status) a.status[row] = 1; }
        return;
    }
    r.top = top;
    const float T = a.temperature[row];
    r.inv = 1.0 / (double)T;
    const SrBins bins{(double)top, SR_WIDTH / (double)T};
    if (ask.kind == SR_SUM) {
        // the span's share of the bins' sums
        uint64_t* hist = s.list;
        for (int i = tid; i < SR_BINS; i += SR_T) hist[i] = 0;
        __syncthreads();
        const int i1 = min(r.V, (span + 1) * wk.per * SR_GROUP);
        for (int i = span * wk.per * SR_GROUP + tid; i < i1; i += SR_T) {
            const double x = bins.x(r.v[i]);
            if (x < (double)SR_BINS) {   // not NaN, not -infinity
                const int bin = (int)x;
                atomicAdd(reinterpret_cast<unsigned long long*>(&hist[bin]), (unsigned long long)sr_fixed(x, bin));
            }
        }
        __syncthreads();
        uint64_t* all = wk.mass + (int64_t)row * SR_BINS;
        for (int i = tid; i < SR_BINS; i += SR_T)
            if (hist[i]) __hip_atomic_fetch_add(&all[i], hist[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        parts_stored();
        if (tid == 0) go = part_last(wk.count + row, wk.spans);
        __syncthreads();
        if (!go) return;
    }
    if (tid == 0 && a.status) a.status[row] = 0;
    if (ask.kind == SR_GREEDY || (ask.low > 1.0f)) {   // no weight is above 1
        if (tid == 0) s.best = 0xffffffffu;
        __syncthreads();
        for (int g = tid; g < wk.groups; g += SR_T) if (gmax[g] == top) atomicMin(&s.best, (uint32_t)g);
        __syncthreads();
        const int i = (int)s.best * SR_GROUP + lane;
        const uint64_t m = __ballot(wave == 0 && i < r.V && r.v[min(i, r.V - 1)] == top);
        if (tid == 0) a.tokens[row] = (int)s.best * SR_GROUP + (int)__builtin_ctzll(m);
        return;
    }
    double goal = (double)a.u[row];
    goal = goal > 0.0 ? (goal < 1.0 ? goal : 1.0) : 0.0;
    int token = -1;
    if (ask.kind == SR_TOP) {
        int b1 = SR_BINS - 1;
        if (r.V > SR_LIST) {
            // the bin down to which there are k tokens: that of the k-th largest group maximum; with min-p no further than its own
            if (ask.k < r.V) {
                uint32_t* cnt = reinterpret_cast<uint32_t*>(s.list);
                for (int i = tid; i < SR_BINS; i += SR_T) cnt[i] = 0;
                __syncthreads();
                for (int g = tid; g < wk.groups; g += SR_T) {
                    const double x = bins.x(gmax[g]);
                    if (x < (double)SR_BINS) atomicAdd(&cnt[(int)x], 1u);
                }
                __syncthreads();
                sr_scan((double)cnt[2 * tid], (double)cnt[2 * tid + 1], s);
                b1 = min(b1, sr_first((double)ask.k, 0.0, SR_BINS, s));
            }
            if (ask.low > 0.0f && ask.p >= 1.0f) b1 = min(b1, (int)(-log((double)ask.low) * SR_WIDTH) + 1);
        }
        const int n = sr_gather(r, bins, gmax, wk.groups, 0, b1, s);
        if (n <= SR_LIST) {
            const int k = min(ask.k, n);
            int end = k;
            if (ask.p < 1.0f) end = min(end, sr_first((double)ask.p * s.run[k - 1], 0.0, k, s) + 1);
            if (ask.low > 0.0f) end = min(end, sr_first_below((double)ask.low, k, bins, s));
            end = max(end, 1);
            const int at = min(sr_first(goal * s.run[end - 1], 0.0, end, s), end - 1);
            token = (int)~(uint32_t)s.ranked[at];
        }
    } else {
        const uint64_t* all = wk.mass + (int64_t)row * SR_BINS;
        double w[2];
#pragma unroll
        for (int h = 0; h < 2; h++)
            w[h] = exp((double)-(2 * tid + h) / SR_WIDTH) * (double)__hip_atomic_load(const_cast<uint64_t*>(&all[2 * tid + h]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sr_scan(w[0], w[1], s);
        const double sum = s.run[SR_BINS - 1], p_goal = (double)ask.p * sum;
        int bp = SR_BINS, bm = SR_BINS;
        if (ask.p < 1.0f) bp = min(sr_first(p_goal, 0.0, SR_BINS, s), SR_BINS - 1);
        if (ask.low > 0.0f) { const double x = -log((double)ask.low) * SR_WIDTH; if (x < (double)SR_BINS) bm = (int)x; }
        const int be = min(bp, bm);   // the bin in which the kept tokens end
        double kept = sum, before = 0.0;
        int draw = -1;
        double draw_before = 0.0;
        if (be == SR_BINS) draw = min(sr_first(goal * kept, 0.0, SR_BINS, s), SR_BINS - 1);
        else {
            before = be ? s.run[be - 1] : 0.0;
            // where the draw falls if it falls before that bin: looked up now, while the bins' sums are there
        }
        int n = 0, end = 0;
        if (be < SR_BINS) {
            const double keep_run0 = s.run[2 * tid], keep_run1 = s.run[2 * tid + 1];
            n = sr_gather(r, bins, gmax, wk.groups, be, be, s);
            if (n <= SR_LIST) {
                end = n;
                if (bp == be) end = min(end, sr_first(p_goal, before, n, s) + 1);
                if (bm == be) end = min(end, sr_first_below((double)ask.low, n, bins, s));
                kept = before + (end ? s.run[end - 1] : 0.0);
                if (before == 0.0) end = max(end, 1);
                if (end && (goal * kept > before || before == 0.0)) {
                    const int at = min(sr_first(goal * kept, before, end, s), end - 1);
                    token = (int)~(uint32_t)s.ranked[at];
                } else {
                    __syncthreads();
                    s.run[2 * tid] = keep_run0; s.run[2 * tid + 1] = keep_run1;
                    draw = min(sr_first(goal * kept, 0.0, be, s), be - 1);
                }
            }
        }
        if (draw >= 0) {
            draw_before = draw ? s.run[draw - 1] : 0.0;
            n = sr_gather(r, bins, gmax, wk.groups, draw, draw, s);
            if (n > 0 && n <= SR_LIST) token = (int)~(uint32_t)s.ranked[min(sr_first(goal * kept, draw_before, n, s), n - 1)];
        }
    }
    if (token < 0) {
        __syncthreads();
        token = sr_descent_token(a, row, r, sr_key(top), u.sh);
    }
    if (tid == 0) a.tokens[row] = token;
}

static size_t sr_layout(int rows, int V, void* base, SrWork& wk) {
    wk.groups = (V + SR_GROUP - 1) / SR_GROUP;
    // about a thousand workgroups, of 64 groups each at least
    const int most = (wk.groups + 63) / 64, want = (1024 + rows - 1) / rows;
    wk.spans = want < most ? want : most;
    wk.per = (wk.groups + wk.spans - 1) / wk.spans;
    wk.spans = (wk.groups + wk.per - 1) / wk.per;
    uint8_t* p = static_cast<uint8_t*>(base);
    size_t at = 0;
    auto take = [&](size_t bytes) { uint8_t* q = p ? p + at : nullptr; at += (bytes + 255) / 256 * 256; return q; };
    wk.count = reinterpret_cast<unsigned*>(take((size_t)rows * 4));
    wk.gmax = reinterpret_cast<float*>(take((size_t)rows * wk.groups * 4));
    wk.mass = reinterpret_cast<uint64_t*>(take((size_t)rows * SR_BINS * 8));
    return at;
}

size_t sample_rows_work(int rows, int V) {
    SrWork wk;
    return sr_layout(rows, V, nullptr, wk);
}

hipError_t launch_sample_rows(const SampleRowsArgs& a, hipStream_t s) {
    SrWork wk;
    sr_layout(a.rows, a.V, a.work, wk);
    const dim3 grid(wk.spans, a.rows);
    const bool vec = a.stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
    if (vec) hipLaunchKernelGGL(sample_groups_kernel<true>, grid, dim3(256), 0, s, a, wk);
    else hipLaunchKernelGGL(sample_groups_kernel<false>, grid, dim3(256), 0, s, a, wk);
    hipLaunchKernelGGL(sample_pick_kernel, grid, dim3(SR_T), 0, s, a, wk);
    return hipGetLastError();
}

}  // namespace mlxr
