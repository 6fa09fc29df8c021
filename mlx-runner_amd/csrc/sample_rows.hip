// Token selection of many rows from given random numbers: temperature, top-k, top-p and min-p over the whole
// vocabulary.
//
// Every cut and the draw itself are one question, asked of the tokens in rank order (logit descending, equal
// ones by index): where does a running sum reach a target? For top-k the sum counts, for the others it adds
// weights w = exp((v - max) / T). It is answered by a radix descent over the logits' order keys: a histogram of
// the leading bits (counts and sums of w per bin), the bin in which the sum passes the target, and again within
// that bin, until one key is left; its tokens have one weight, so the rest is a division. Weights are rounded to
// multiples of 2^-43 of exp() in 64 bits and added as integers: no order of the atomic adds changes a result,
// a sum of 2^20 weights stays below 2^63, and the rounding moves a border by 2^-44 a token.
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

__global__ __launch_bounds__(SR_T) void sample_rows_kernel(SampleRowsArgs a) {
    __shared__ SrShared sh;
    const int row = blockIdx.x, tid = threadIdx.x;
    SrRow r;
    r.v = a.logits + (int64_t)row * a.stride;
    r.V = a.V;
    uint64_t best = 0;
    for (int i = tid; i < r.V; i += SR_T) {
        const uint64_t k = ((uint64_t)sr_key(r.v[i]) << 32) | (uint32_t)~(uint32_t)i;
        best = k > best ? k : best;
    }
    best = sr_max(best, sh);
    const uint32_t top = (uint32_t)(best >> 32);
    r.top = sr_value(top);
    const bool none = top <= SR_MINUS_INF || !isfinite(r.top);
    if (tid == 0 && a.status) a.status[row] = none ? 1 : 0;
    const float T = a.temperature[row];
    if (none || !(T > 0.001f)) {
        if (tid == 0) a.tokens[row] = none ? 0 : (int)~(uint32_t)best;
        return;
    }
    r.inv = 1.0 / (double)T;
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
            if (key > SR_MINUS_INF && r.weight(r.v[i]) >= (double)low) { const uint64_t c = ~key; least = c > least ? c : least; }
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
    const int token = sr_nth(r, at.key, at.n, sh);
    if (tid == 0) a.tokens[row] = token;
}

size_t sample_rows_work(int, int) { return 256; }

hipError_t launch_sample_rows(const SampleRowsArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(sample_rows_kernel, dim3(a.rows), dim3(SR_T), 0, s, a);
    return hipGetLastError();
}

}  // namespace mlxr
