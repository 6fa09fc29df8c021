// Token selection of many rows from given random numbers: temperature, top-k, top-p and min-p over the whole
// vocabulary.
//
// Every cut and the draw itself are one question, asked of the tokens in rank order (logit descending, equal
// ones by index): where does a running sum of weights w = exp((v - max) / T) (top-k: of ones) reach a target? The
// answer needs the order only where the sum crosses. Three launches:
//   1. sample_groups_kernel, about a thousand workgroups: the maximum of every 64 logits. The one read of the logits that
//      every row needs: 0.6 MB a row of 152 thousand, 37 us for 256 of them (4.2 TB/s), 3 us for one.
//   2. sample_sums_kernel, for rows that ask for a sum over all their tokens (top-p, or nothing, without top-k). With the
//      row's maximum known, tokens fall into 2048 bins of x = (max - v) / T, 64 to a unit (finer ones above a temperature
//      of 1), and what lies behind x = 32 into the last one. Each bin's weights are added up, and each token's bin is
//      written down. 27 us for 102 rows of 152 thousand, in which no unit is busy: of the waves' cycles half go by waiting
//      for memory or a barrier and a quarter waiting to issue, LDS is in use a sixth of the time, most of it for bank
//      conflicts; there are three workgroups a CU and each is a chain of two dependent reads. Other rows leave at once (2 us).
//   3. sample_pick_kernel, one workgroup a row. A row with sums: the bins in which the sums cross are found, just their
//      tokens are gathered (through the groups' maxima, or by the bin numbers where most groups qualify), ranked and
//      walked. A row without: the groups' maxima give a bin down to which there are k tokens or more, or min-p does, and
//      these are gathered. Bound by what waits for what in one workgroup: 9 us for a top-k of 40, about 20 us where a cut lies
//      among the bulk of the tokens (13 us to look through 152 thousand bin numbers).
// A bin's weights are a constant times f in (exp(-1/64), 1], added as multiples of 2^-43: no order of the atomic adds
// changes a result, and 2^20 of them stay below 2^63. So a weight is off by 2^-43 of itself at most (the largest logit's is
// exact), and everything else is 64-bit floating point: a token differs from the exact sums' only if the draw, or a cut, is
// within about 2^-42 of a border, as a share of the sum.
// Rows whose tokens to be ranked are more than the list holds (2048) take the radix descent instead, which asks for no room: a
// histogram of the order keys' leading bits, the bin in which the sum crosses, and again within that bin, until one key is
// left, whose tokens have one weight. These are rows with a top-k of more than about one token in 64 (from 125 at a vocabulary
// of 8000, 490 at 32000 and 1400 at 152 thousand with normally spread logits: the groups' maxima cannot tell the k-th), with
// thousands of equal logits where a sum crosses, of a bulk so flat that a bin holds thousands (2^20 logits of deviation 2 at a
// temperature of 1, 152 thousand from about 35), and sums that cross behind the bins. Up to 16 passes of one workgroup over
// the row: 38 us for a top-k of 100 of 4097, 415 for 5000 of 152 thousand (570 with every cut), 2.7 ms for 40000 of 2^20.
#include "batch.h"

namespace mlxr {

constexpr double SR_ONE = 8796093022208.0;   // 2^43: the weight of the largest logit
constexpr int SR_T = 1024, SR_W = SR_T / 64;   // threads and waves of a workgroup
constexpr int SR_BINS = 2048, SR_PER = SR_BINS / SR_T;
constexpr uint32_t SR_MINUS_INF = 0x007fffffu;   // the order key of -infinity; NaN has 0

__device__ __forceinline__ uint32_t sr_key(float v) {
    if (v != v) return 0u;
    const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sr_value(uint32_t k) { return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k); }

// Bins: 64 to a unit of x at temperatures up to 1, and as many to a unit of the logits at those up to 8, where the bulk's
// logits lie closer in x (at 3, two bins of 64 a unit may hold 3000 of 152 thousand tokens; one row with a top-p of 0.9 then
// took 475 us through the radix descent, and takes 44). Sums are kept of those up to x = 32 or, above 1, of the logits. Tokens
// behind them have weight, up to x = 52 (`reach`): 2^20 tokens of e^-52 are less than 2^-54 of the sum. The row's numbers are
// in scalar registers: the last launch has no others to spare (14 vector registers spilled without, 28 scalar ones are kept
// in lanes of vector registers with; 38.7 and 38.1 us for 256 mixed rows).
struct SrBins {
    double top, inv, width;   // the largest logit; bins per unit of logit, and the other way round
    double per, inv_per;      // bins per unit of x
    int reach;                // the first bin whose tokens have no weight that counts
    __device__ __forceinline__ double x(float v) const { return (top - (double)v) * inv; }   // in bins; NaN or infinite outside
};
// A value that all lanes hold, in scalar registers.
__device__ __forceinline__ double sr_uniform(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)b), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32));
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ SrBins sr_bins(float top, float T, double inv_T) {
    const double per = T > 1.0f ? 64.0 * fmin((double)T, 8.0) : 64.0, inv_per = T > 1.0f ? fmax(inv_T, 0.125) / 64.0 : 1.0 / 64.0;
    return SrBins{(double)top, sr_uniform(per * inv_T), sr_uniform((double)T * inv_per), sr_uniform(per), sr_uniform(inv_per),
                  __builtin_amdgcn_readfirstlane((int)(52.0 * per))};
}
// 2^43 exp(-y / per) for y = x - bin in [0, 1), rounded to a whole number: the Taylor sum to the fifth power is off by
// 2^-45 at most; added to 2^52 it is rounded into the mantissa's low bits.
__device__ __forceinline__ uint64_t sr_fixed(double x, int bin, double inv_per) {
    const double y = (x - (double)bin) * inv_per;
    const double e = fma(y, fma(y, fma(y, fma(y, fma(y, -SR_ONE / 120, SR_ONE / 24), -SR_ONE / 6), SR_ONE / 2), -SR_ONE), SR_ONE);
    return __builtin_bit_cast(uint64_t, e + 0x1p52) & 0xfffffffffffffull;
}
// exp(-64 i / per) and exp(-i / per): a bin's constant is one of each.
struct SrTables { double whole[32], part[64]; };
__device__ __forceinline__ double sr_constant(const SrTables& t, int bin) { return t.whole[bin >> 6] * t.part[bin & 63]; }
// A logit's weight in units of 2^-43, as the bins' sums have it.
__device__ __forceinline__ double sr_weight(const SrBins& bins, const SrTables& t, float v) {
    double x = bins.x(v), c = 1.0;
    if (!(x < (double)bins.reach)) return 0.0;
    for (; x >= (double)SR_BINS; x -= 64.0 * 31) c *= t.whole[31];   // behind the bins: powers of the tables' last entry
    const int bin = (int)x;
    return c * sr_constant(t, bin) * (double)sr_fixed(x, bin, bins.inv_per);
}

// A sum of weights in the radix descent: multiples of 2^-43 and, beside them, of 2^-76. So no order of the atomic adds
// changes it, and of 2^20 weights, at most 1 each, it loses 2^-56 at most.
typedef unsigned __int128 sr_u128;
constexpr double SR_LOW = 8589934592.0;   // 2^33
struct SrMass {
    uint64_t high, low;
    __device__ __forceinline__ void add(SrMass m, uint32_t times = 1) { high += times * m.high; low += times * m.low; }
    __device__ __forceinline__ sr_u128 sum() const { return ((sr_u128)high << 33) + low; }
};

struct SrRow {
    const float* v; int V;
    bool vec;           // 16-byte loads of four neighbours from indices divisible by four
};
// Weights in the radix descent.
struct SrScale {
    SrBins bins;
    const SrTables& t;
    __device__ __forceinline__ double weight(float v) const { return sr_weight(bins, t, v); }
    __device__ __forceinline__ SrMass fixed(float v) const {
        const double w = weight(v), whole = floor(w);
        return SrMass{(uint64_t)whole, (uint64_t)((w - whole) * SR_LOW)};
    }
};

// Four neighbours from index i (divisible by four); -infinity behind the row.
__device__ __forceinline__ void sr_load4(const SrRow& r, int i, float* o) {
    if (r.vec && i + 4 <= r.V) {
        const float4 x = gload4(r.v + i);
        o[0] = x.x; o[1] = x.y; o[2] = x.z; o[3] = x.w;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = i + e < r.V ? gload(r.v + i + e) : -INFINITY;
}

// The tokens with a key above `key`, and `n` of those that have it (lowest indices first).
struct SrCut { uint32_t key; uint32_t n; };
__device__ __forceinline__ SrCut sr_min(SrCut a, SrCut b) {   // the shorter of two prefixes of the rank order
    if (a.key != b.key) return a.key > b.key ? a : b;
    return a.n < b.n ? a : b;
}

struct SrShared {
    uint64_t high[SR_BINS], low[SR_BINS];
    uint32_t count[SR_BINS];
    SrMass wmass[SR_W], above_mass;
    uint64_t wsum[SR_W];
    uint32_t wcount[SR_W], pick, above_count;
};

// Sum over the workgroup, to every thread.
__device__ uint64_t sr_sum(uint64_t v, SrShared& sh) {
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wsum[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < SR_W; i++) t += sh.wsum[i];
    return t;
}
__device__ uint64_t sr_max(uint64_t v, SrShared& sh) {
    for (int o = 1; o < 64; o <<= 1) { const uint64_t p = __shfl_xor(v, o, 64); v = p > v ? p : v; }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wsum[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < SR_W; i++) t = sh.wsum[i] > t ? sh.wsum[i] : t;
    return t;
}
// What the waves before this one and all of them have, from one value a wave in LDS.
__device__ __forceinline__ uint64_t sr_lane(uint64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return (uint64_t)lo | ((uint64_t)hi << 32);
}
__device__ __forceinline__ void sr_waves(const SrMass* w, SrMass& before, SrMass& all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const SrMass m = lane < SR_W ? w[lane] : SrMass{0, 0}, upto = {wave_scan(m.high), wave_scan(m.low)};
    before.add(SrMass{sr_lane(upto.high - m.high, wave), sr_lane(upto.low - m.low, wave)});
    all.add(SrMass{sr_lane(upto.high, SR_W - 1), sr_lane(upto.low, SR_W - 1)});
}
// The sum of the weights within a cut.
__device__ sr_u128 sr_mass(const SrRow& r, const SrScale& sc, SrCut cut, SrShared& sh) {
    SrMass t = {0, 0};
    for (int i = threadIdx.x; i < r.V; i += SR_T) if (sr_key(r.v[i]) > cut.key) t.add(sc.fixed(r.v[i]));
    if (threadIdx.x == 0 && cut.n) t.add(sc.fixed(sr_value(cut.key)), cut.n);
    t = SrMass{wave_scan(t.high), wave_scan(t.low)};
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.wmass[threadIdx.x >> 6] = t;
    __syncthreads();
    SrMass before = {0, 0}, all = {0, 0};
    sr_waves(sh.wmass, before, all);
    return all.sum();
}

// How many weights w reach `need`: the quotient rounded up, at least 1. The quotient of doubles is off by one at most.
__device__ uint32_t sr_times(sr_u128 need, sr_u128 w) {
    if (w == 0) return 1;
    auto real = [](sr_u128 v) { return (double)(uint64_t)(v >> 64) * 0x1p64 + (double)(uint64_t)v; };
    uint32_t n = (uint32_t)(real(need) / real(w));
    while (n * w < need) n++;
    while (n > 1 && (n - 1) * w >= need) n--;
    return n ? n : 1;
}

// The order keys' bits that a level of the descent takes.
struct SrLevel {
    int shift; uint32_t bins;
    __device__ __forceinline__ SrLevel(int level) : shift(level == 0 ? 21 : level == 1 ? 10 : 0), bins(level == 2 ? 1024 : 2048) {}
    __device__ __forceinline__ uint32_t bin(uint32_t key) const { return (key >> shift) & (bins - 1); }
};
// What a wave's lanes at work on one key each add to its bin: lanes with one key (ties by the thousand) add once, as many adds
// to one place would wait for each other. Calls add(times) in the lanes that do.
template <typename F> __device__ __forceinline__ void sr_add(uint32_t k, F add) {
    const uint64_t lanes = __ballot(true), equal = __ballot(k == (uint32_t)__builtin_amdgcn_readfirstlane((int)k));
    const bool one = equal == lanes;
    if (!one || (threadIdx.x & 63) == (unsigned)__builtin_ctzll(lanes)) add(one ? (uint32_t)__popcll(lanes) : 1u);
}

// The first k tokens (1 .. V - 1 of them), all of those above -infinity where there are fewer.
__device__ SrCut sr_first(const SrRow& r, uint32_t k, SrShared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t prefix = 0, mask = 0, above = 0;
#pragma unroll 1
    for (int l = 0; l < 3; l++) {
        const SrLevel level(l);
        __syncthreads();
        for (int i = tid; i < SR_BINS; i += SR_T) sh.count[i] = 0;
        __syncthreads();
        for (int i = tid; i < r.V; i += SR_T) {
            const uint32_t key = sr_key(gload(r.v + i));
            if (key > SR_MINUS_INF && (key & mask) == prefix) sr_add(key, [&](uint32_t times) { atomicAdd(&sh.count[level.bin(key)], times); });
        }
        __syncthreads();
        // thread t has SR_PER bins from bins - 1 - SR_PER t down: sums of everything above by scans
        const int b1 = (int)level.bins - 1 - SR_PER * tid;
        int own = 0;
#pragma unroll
        for (int h = 0; h < SR_PER; h++) if (b1 - h >= 0) own += (int)sh.count[b1 - h];
        const int c = wave_scan(own);
        if (lane == 63) sh.wcount[wave] = (uint32_t)c;
        __syncthreads();
        uint32_t before = above + (uint32_t)(c - own), all = above;
        for (int i = 0; i < SR_W; i++) {
            if (i < wave) before += sh.wcount[i];
            all += sh.wcount[i];
        }
        if (all < k) return SrCut{SR_MINUS_INF, 0};   // the first level's only
        for (int h = 0; h < SR_PER && b1 - h >= 0; h++) {
            const uint32_t with = before + sh.count[b1 - h];
            if (before < k && with >= k) { sh.pick = (uint32_t)(b1 - h); sh.above_count = before; }
            before = with;
        }
        __syncthreads();
        prefix |= sh.pick << level.shift; mask |= (level.bins - 1) << level.shift;
        above = sh.above_count;
    }
    return SrCut{prefix, k - above};
}

// The shortest prefix of the cut's tokens whose sum of weights reaches `target` (>= 1): the whole cut if none does. *mass: its
// sum of weights.
__device__ SrCut sr_descend(const SrRow& r, const SrScale& sc, SrCut cut, sr_u128 target, SrShared& sh, sr_u128* mass) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t prefix = 0, mask = 0;
    SrMass above = {0, 0};
    const SrMass edge = cut.n ? sc.fixed(sr_value(cut.key)) : SrMass{0, 0};   // the weight of the tokens at the cut's key
    auto bin_mass = [&](int i) { return SrMass{sh.high[i], sh.low[i]}; };
#pragma unroll 1
    for (int l = 0; l < 3; l++) {
        const SrLevel level(l);
        __syncthreads();
        for (int i = tid; i < SR_BINS; i += SR_T) { sh.high[i] = 0; sh.low[i] = 0; }
        __syncthreads();
        for (int i = tid; i < r.V; i += SR_T) {
            const float x = gload(r.v + i);
            const uint32_t key = sr_key(x);
            if (key > cut.key && (key & mask) == prefix)
                sr_add(key, [&](uint32_t times) {
                    const SrMass m = sc.fixed(x);
                    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.high[level.bin(key)]), (unsigned long long)(times * m.high));
                    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.low[level.bin(key)]), (unsigned long long)(times * m.low));
                });
        }
        __syncthreads();
        if (tid == 0 && cut.n && (cut.key & mask) == prefix) {
            const uint32_t bin = level.bin(cut.key);
            sh.high[bin] += cut.n * edge.high;
            sh.low[bin] += cut.n * edge.low;
        }
        if (tid == 0) { sh.pick = 0xffffffffu; }
        __syncthreads();
        const int b1 = (int)level.bins - 1 - SR_PER * tid;
        SrMass own = {0, 0};
#pragma unroll
        for (int h = 0; h < SR_PER; h++) if (b1 - h >= 0) own.add(bin_mass(b1 - h));
        const SrMass m = {wave_scan(own.high), wave_scan(own.low)};
        if (lane == 63) sh.wmass[wave] = m;
        __syncthreads();
        SrMass before = above, all = above;
        before.add(m);
        before.high -= own.high; before.low -= own.low;
        sr_waves(sh.wmass, before, all);
        if (l == 0 && all.sum() < target) { *mass = all.sum(); return cut; }
#pragma unroll 1
        for (int h = 0; h < SR_PER && b1 - h >= 0; h++) {   // one bin of one thread: sums only grow
            SrMass with = before;
            with.add(bin_mass(b1 - h));
            if (before.sum() < target && with.sum() >= target) { sh.pick = (uint32_t)(b1 - h); sh.above_mass = before; }
            before = with;
        }
        __syncthreads();
        prefix |= sh.pick << level.shift; mask |= (level.bins - 1) << level.shift;
        above = sh.above_mass;
    }
    const sr_u128 w = sc.fixed(sr_value(prefix)).sum();
    const uint32_t need = sr_times(target - above.sum(), w);
    *mass = above.sum() + need * w;
    return SrCut{prefix, need};
}

// The index of the n-th (from 1) token with this key.
__device__ int sr_nth(const SrRow& r, uint32_t key, uint32_t n, SrShared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = ((r.V + SR_W - 1) / SR_W + 63) & ~63;
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

// A target a fraction of a sum: the least whole number not below it, at least 1. The fraction is 24 bits over a power of two,
// a sum less than 2^97.
__device__ __forceinline__ sr_u128 sr_target(float share, sr_u128 sum) {
    if (!(share > 0.0f)) return 1;
    if (share >= 1.0f) return sum;
    int e;
    const uint32_t bits = (uint32_t)(frexpf(share, &e) * 16777216.0f);
    const int down = 24 - e;
    if (down > 126) return 1;
    const sr_u128 t = (sum * bits + (((sr_u128)1 << down) - 1)) >> down;
    return t > 0 ? t : 1;
}

// The radix descent over a whole row: any parameters, one workgroup. A call of its own: its code is as long as all the rest.
__device__ __noinline__ int sr_descent_token(const float* v, int V, float largest, float T, const SrTables& tables, int k, float p, float low,
                                             float given, SrShared& sh) {
    const int tid = threadIdx.x;
    const SrRow r{v, V, false};
    const SrScale sc{sr_bins(largest, T, 1.0 / (double)T), tables};
    const uint32_t top = sr_key(largest);
    sr_u128 mass = 0, kept_mass = 0;
    SrCut cut{SR_MINUS_INF, 0};
    if (k < r.V) cut = sr_first(r, (uint32_t)k, sh);
    mass = sr_mass(r, sc, cut, sh);
    SrCut end = cut;
    kept_mass = mass;
    if (p < 1.0f) end = sr_descend(r, sc, cut, sr_target(p, mass), sh, &kept_mass);
    if (low > 0.0f) {
        uint64_t least = 0;   // the complement of the smallest key that stays
        for (int i = tid; i < r.V; i += SR_T) {
            const uint32_t key = sr_key(r.v[i]);
            if (key > SR_MINUS_INF && sc.weight(r.v[i]) >= (double)low * SR_ONE) { const uint64_t c = (uint32_t)~key; least = c > least ? c : least; }
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
            kept_mass = sr_mass(r, sc, end, sh);
        }
    }
    sr_u128 unused;
    const SrCut at = sr_descend(r, sc, end, sr_target(given, kept_mass), sh, &unused);
    return sr_nth(r, at.key, at.n, sh);
}

// ---- bins, gathered tokens and their order ----
constexpr int SR_GROUP = 64, SR_LIST = 2048;
typedef uint32_t sr_w4 __attribute__((ext_vector_type(4)));
typedef uint16_t sr_h2 __attribute__((ext_vector_type(2)));

struct SrWork {
    float* gmax;        // [rows][groups]
    uint16_t* bin;      // [rows][groups][64]: the tokens' bins (65535: none), written where sums over the row are needed
    uint64_t* mass;     // [rows][sum_spans][SR_BINS]: sums of f
    int groups;               // of a row
    int spans, per;           // the first launch's workgroups of a row, and the groups of each
    int sum_spans, sum_per;   // the second's, where it adds up bins
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

__host__ __device__ __forceinline__ bool sr_vec(const SampleRowsArgs& a) { return a.stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0; }

// Per 64 logits the maximum (NaN ignored). A lane has four neighbours, 16 lanes a group.
template <bool VEC>
__global__ __launch_bounds__(256) void sample_groups_kernel(SampleRowsArgs a, SrWork wk) {
    const int row = blockIdx.y, span = blockIdx.x, tid = threadIdx.x;
    const float* v = a.logits + (int64_t)row * a.stride;
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

// The bins' sums of the rows that need them, several workgroups a row, and each token's bin. What lies behind the last bin
// goes to it (no sum may cross in it then): up to SR_WIDE bins are added up like the others (all that have weight, at
// temperatures up to 1) and then as multiples of the last one's constant, tokens behind those one by one.
constexpr int SR_SUM_T = 512, SR_WIDE = 52 * 64;
__global__ __launch_bounds__(SR_SUM_T) void sample_sums_kernel(SampleRowsArgs a, SrWork wk) {
    __shared__ uint64_t hist[SR_WIDE];
    __shared__ double wave_tail[SR_SUM_T / 64];
    __shared__ float wave_top[SR_SUM_T / 64];
    const int row = blockIdx.y, tid = threadIdx.x;
    if (sr_ask(a, row).kind != SR_SUM) return;
    const float* gmax = wk.gmax + (int64_t)row * wk.groups;
    float top = -INFINITY;
#pragma unroll 4
    for (int g = tid; g < wk.groups; g += SR_SUM_T) top = fmaxf(top, gload(gmax + g));
    for (int i = tid; i < SR_WIDE; i += SR_SUM_T) hist[i] = 0;
    top = wave_max(top);
    if ((tid & 63) == 0) wave_top[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SR_SUM_T / 64; i++) top = fmaxf(top, wave_top[i]);
    if (!isfinite(top)) return;
    const SrRow r{a.logits + (int64_t)row * a.stride, a.V, sr_vec(a)};
    const SrBins bins = sr_bins(top, a.temperature[row], 1.0 / (double)a.temperature[row]);
    const double inv_per = bins.inv_per;
    bool far = false;
    uint16_t* out = wk.bin + (int64_t)row * wk.groups * SR_GROUP;
    const int i1 = min(a.V, ((int)blockIdx.x + 1) * wk.sum_per * SR_GROUP);
    constexpr int UN = 4;
#pragma unroll 1
    for (int i = blockIdx.x * wk.sum_per * SR_GROUP + 4 * tid; i < i1; i += 4 * SR_SUM_T * UN) {
        float v[UN][4];
#pragma unroll
        for (int k = 0; k < UN; k++) sr_load4(r, i + 4 * SR_SUM_T * k < i1 ? i + 4 * SR_SUM_T * k : a.V, v[k]);
#pragma unroll
        for (int k = 0; k < UN; k++) {
            uint32_t bin[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double x = bins.x(v[k][e]);
                bin[e] = 0xffffu;
                if (x < (double)SR_WIDE) {   // not NaN, not -infinity
                    bin[e] = (uint32_t)(int)x;
                    atomicAdd(reinterpret_cast<unsigned long long*>(&hist[bin[e]]), (unsigned long long)sr_fixed(x, (int)bin[e], inv_per));
                } else if (x < (double)bins.reach) {
                    far = true;
                }
            }
            const int at = i + 4 * SR_SUM_T * k;
            if (at < i1) *reinterpret_cast<uint2*>(out + at) = uint2{bin[0] | (bin[1] << 16), bin[2] | (bin[3] << 16)};
        }
    }
    __syncthreads();
    double tail = 0.0;
    for (int i = SR_BINS + tid; i < SR_WIDE; i += SR_SUM_T)
        if (hist[i]) tail += exp((double)(SR_BINS - 1 - i) * inv_per) * (double)hist[i];
    if (far)
        for (int i = blockIdx.x * wk.sum_per * SR_GROUP + 4 * tid; i < i1; i += 4 * SR_SUM_T)
            for (int e = i; e < min(i + 4, i1); e++) {
                const double x = bins.x(r.v[e]);
                if (x >= (double)SR_WIDE && x < (double)bins.reach) tail += exp(((double)(SR_BINS - 1) - x) * inv_per) * SR_ONE;
            }
    tail = wave_scan(tail);
    if ((tid & 63) == 63) wave_tail[tid >> 6] = tail;
    __syncthreads();
    if (tid == 0) {
        tail = 0.0;
        for (int i = 0; i < SR_SUM_T / 64; i++) tail += wave_tail[i];
        hist[SR_BINS - 1] += (uint64_t)(tail + 0.5);
    }
    __syncthreads();
    uint64_t* mine = wk.mass + ((int64_t)row * wk.sum_spans + blockIdx.x) * SR_BINS;
    for (int i = tid; i < SR_BINS; i += SR_SUM_T) mine[i] = hist[i];
}

// What one workgroup keeps of its row. Code that runs once is paid for by its size (instructions come from memory
// like data: the same steps unrolled, in 76 KB, took 21 us for one row where these 22 KB take 14), so loops here stay
// rolled and exponentials are looked up.
constexpr int SR_MAXGROUPS = (1 << 20) / SR_GROUP, SR_NEAR = 4096;   // groups of the longest row; of these kept in LDS
struct SrPick {
    uint64_t list[SR_LIST];
    union {
        struct { uint64_t ranked[SR_LIST]; double run[SR_LIST]; };
        uint16_t ids[SR_MAXGROUPS];   // while tokens are gathered, before they are ranked
    };
    float gmax[SR_NEAR];
    double wave_sum[2][SR_W];
    int wave_count[2][4][SR_W];
    float wave_top[SR_W];
    int n, nids, found;
    uint32_t best;
};
static_assert(SR_LIST == SR_BINS && SR_BINS == 32 * 64, "run holds the bins' sums and the gathered tokens'");

// The logits within [lo, hi] or [lo2, hi2] of the given groups, as keys, to the list (as many as it holds; n counts all).
// A wave reads four groups at a time, four neighbours a lane, UN such loads in flight.
template <int UN>
__device__ __forceinline__ void sr_collect(const float* v, int V, bool vec, const uint16_t* ids, int count, float lo, float hi, float lo2, float hi2,
                                           uint64_t* list, int* n) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t before = lane ? ~0ull >> (64 - lane) : 0ull;
    const SrRow r{v, V, vec};
#pragma unroll 1
    for (int i = 4 * wave; i < count; i += 4 * SR_W * UN) {
        float x[UN][4];
        int idx[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int q = i + 4 * SR_W * u + (lane >> 4);
            idx[u] = q < count ? ids[q] * SR_GROUP + 4 * (lane & 15) : V;
            sr_load4(r, idx[u], x[u]);
        }
#pragma unroll
        for (int u = 0; u < UN; u++) {
            uint64_t in[4];
            int total = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                in[e] = __ballot((x[u][e] >= lo && x[u][e] <= hi) || (x[u][e] >= lo2 && x[u][e] <= hi2));
                total += (int)__popcll(in[e]);
            }
            if (!total) continue;
            int to = 0;
            if (lane == 0) to = atomicAdd(n, total);
            to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int at = to + (int)__popcll(in[e] & before);
                if (((in[e] >> lane) & 1) && at < SR_LIST) list[at] = ((uint64_t)sr_key(x[u][e]) << 32) | (uint32_t)~(uint32_t)(idx[u] + e);
                to += (int)__popcll(in[e]);
            }
        }
    }
}
// The same over a row's bin numbers, as the first pass over it has left them: the logits of bins b0 and `also`. Eight
// numbers a lane and load, found by packed minima of their differences; a lane with a hit goes on by itself.
__device__ __noinline__ void sr_collect_bins(const float* v, const uint16_t* bin, int V, int b0, int also, uint64_t* list, int* n) {
    const uint32_t t0 = (uint32_t)b0 * 0x10001u, t1 = (uint32_t)(also < 0 ? b0 : also) * 0x10001u;
    auto least = [](uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(sr_h2, a), __builtin_bit_cast(sr_h2, b))); };
    constexpr int UN = 4;
#pragma unroll 1
    for (int i = 8 * (int)threadIdx.x; i < V; i += 8 * SR_T * UN) {
        sr_w4 x[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int at = i + 8 * SR_T * u;   // rows of numbers are padded to eight
            x[u] = sr_w4{0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
            if (at < V) x[u] = gload(reinterpret_cast<const sr_w4*>(bin + at));
        }
#pragma unroll 1
        for (int u = 0; u < UN; u++) {
            const sr_w4 w = x[0];
#pragma unroll
            for (int k = 0; k + 1 < UN; k++) x[k] = x[k + 1];
            uint32_t m[4];
#pragma unroll
            for (int k = 0; k < 4; k++) m[k] = least(w[k] ^ t0, w[k] ^ t1);
            const uint32_t all = least(least(m[0], m[1]), least(m[2], m[3]));
            if ((all & 0xffffu) && (all >> 16)) continue;
            uint32_t hits = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) hits |= (m[k] & 0xffffu ? 0u : 1u << (2 * k)) | (m[k] >> 16 ? 0u : 2u << (2 * k));
            while (hits) {
                const int at = i + 8 * SR_T * u + __builtin_ctz(hits);
                hits &= hits - 1;
                if (at >= V) break;   // the last eight may reach behind the row, where nothing was written
                const int to = atomicAdd(n, 1);
                if (to < SR_LIST) list[to] = (uint32_t)~(uint32_t)at;
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(*n, SR_LIST); i += SR_T) list[i] |= (uint64_t)sr_key(gload(v + (int)~(uint32_t)list[i])) << 32;
}

// The n > 256 gathered tokens, ranked: each wave sorts runs of 64 in registers; a key's rank is its place in its run
// and, for every other run, how many of that run's keys are larger.
__device__ __noinline__ void sr_rank_many(uint64_t* list, uint64_t* ranked, int n) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), runs = (n + 63) / 64;
    for (int q = wave; q < runs; q += SR_W) {
        uint64_t k = 64 * q + lane < n ? list[64 * q + lane] : 0;
#pragma unroll 1
        for (int size = 2; size <= 64; size <<= 1)
#pragma unroll 1
            for (int d = size >> 1; d > 0; d >>= 1) {
                const uint64_t p = __shfl_xor(k, d, 64);
                const bool lower = (lane & d) == 0, desc = size == 64 || (lane & size) == 0;
                k = (lower == desc) ? (p > k ? p : k) : (p < k ? p : k);
            }
        list[64 * q + lane] = k;
    }
    __syncthreads();
    for (int q = wave; q < runs; q += SR_W) {
        const uint64_t k = list[64 * q + lane];
        int at = lane;
#pragma unroll 1
        for (int o = 0; o < runs; o++) {
            if (o == q) continue;
            const uint64_t* run = list + 64 * o;
            int lo = 0;
#pragma unroll
            for (int step = 32; step > 0; step >>= 1) lo += run[lo + step - 1] > k ? step : 0;
            at += lo + (run[lo] > k ? 1 : 0);
        }
        if (k) ranked[at] = k;
    }
}

// One workgroup at work on a row. The helpers alternate between two places for what waves tell each other, so that
// each needs one barrier: a place is written again only behind the next one's.
struct SrTeam {
    SrPick& s;
    const SrTables& tables;
    const SrRow& r;
    SrBins bins;
    const float* gmax; int groups;
    const uint16_t* bin;   // the bins of the row's tokens, where they were written down
    int tid, lane, wave, flip;

    __device__ __forceinline__ float group(int g) const { return g < SR_NEAR ? s.gmax[g] : gmax[g]; }
    __device__ __forceinline__ double constant(int bin) const { return sr_constant(tables, bin); }
    __device__ __forceinline__ double weight(float v) const { return sr_weight(bins, tables, v); }
    __device__ __forceinline__ float ranked(int i) const { return sr_value((uint32_t)(s.ranked[i] >> 32)); }
    __device__ __forceinline__ int token(int i) const { return (int)~(uint32_t)s.ranked[i]; }

    // Running sums (inclusive) of SR_PER values a thread, SR_PER tid .., over the workgroup: into run.
    __device__ __forceinline__ void scan(const double* a) {
        double v = 0.0;
#pragma unroll
        for (int h = 0; h < SR_PER; h++) v += a[h];
        v = wave_scan(v);
        double* sums = s.wave_sum[flip ^= 1];
        if (lane == 63) sums[wave] = v;
        __syncthreads();
        double before = lane_before<0x138, 0xF>(v);   // the lane before
        for (int i = 0; i < wave; i++) before += sums[i];
#pragma unroll
        for (int h = 0; h < SR_PER; h++) s.run[SR_PER * tid + h] = before += a[h];
        __syncthreads();
    }
    // Over the workgroup, how often each of up to four conditions holds for an i < n.
    template <int C, typename F> __device__ __forceinline__ void counts(int n, F yes, int* c) {
        for (int q = 0; q < C; q++) c[q] = 0;
        for (int i = tid; i - lane < n; i += SR_T) {
            bool b[C];
            for (int q = 0; q < C; q++) b[q] = false;
            if (i < n) yes(i, b);
#pragma unroll
            for (int q = 0; q < C; q++) c[q] += (int)__popcll(__ballot(b[q]));
        }
        flip ^= 1;
        if (lane == 0)
#pragma unroll
            for (int q = 0; q < C; q++) s.wave_count[flip][q][wave] = c[q];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < C; q++) {
            c[q] = 0;
#pragma unroll
            for (int i = 0; i < SR_W; i++) c[q] += s.wave_count[flip][q][i];
        }
    }
    // The first i < n with run[i] + base >= target (n if there is none): the sums only grow.
    __device__ __forceinline__ int first(double target, double base, int n) {
        int c;
        counts<1>(n, [&](int i, bool* b) { b[0] = s.run[i] + base < target; }, &c);
        return c;
    }
    // The first i < n whose weight is below `low`: the ranked tokens' weights only fall.
    __device__ __forceinline__ int first_below(double low, int n) {
        int c;
        counts<1>(n, [&](int i, bool* b) { b[0] = weight(ranked(i)) >= low * SR_ONE; }, &c);
        return c;
    }

    // Ranks the n gathered tokens.
    __device__ __forceinline__ void rank(int n) {
        if (n <= 256) {   // each against all (256 mixed rows: 89 us; only up to 64: 94, up to 1024: 101)
            for (int i = tid; i - lane < n; i += SR_T) {
                const uint64_t k = i < n ? s.list[i] : 0;
                int above = 0;
#pragma unroll 4
                for (int o = 0; o < n; o++) above += s.list[o] > k;
                if (i < n) s.ranked[above] = k;
            }
        } else {
            sr_rank_many(s.list, s.ranked, n);
        }
        __syncthreads();
    }
    // The logits of bins b0 .. b1 lie in [lo, hi]; a few of the neighbouring bins may too.
    __device__ __forceinline__ void range(int b0, int b1, float& lo, float& hi) const {
        const double top = bins.top, slack = fabs(top) * 0x1p-22 + 0x1p-120;
        const double l = top - (double)(b1 + 1) * bins.width, h = top - (double)b0 * bins.width;
        lo = fmaxf((float)(l - fabs(l) * 0x1p-22 - slack), -3.402823466e38f);
        hi = (float)fmin(h + fabs(h) * 0x1p-22 + slack, top);
        if (!(hi <= (float)top)) hi = (float)top;   // T infinite: 0 times infinity
    }
    // Gathers the tokens of bins b0 .. b1 and of bin `also` (before them, or -1), and perhaps a few of the bins next to
    // them, ranked, with the running sums of their weights in run. Returns how many; above SR_LIST nothing else is done.
    __device__ __forceinline__ int gather(int also, int b0, int b1) {
        const uint64_t before = lane ? ~0ull >> (64 - lane) : 0ull;
        float lo, hi, lo2 = 1.0f, hi2 = 0.0f;
        range(b0, b1, lo, hi);
        if (also >= 0) range(also, also, lo2, hi2);
        __syncthreads();
        for (int g = tid; g - lane < groups; g += SR_T) {
            const uint64_t has = __ballot(g < groups && group(g) >= lo);
            if (!has) continue;
            int at = 0;
            if (lane == 0) at = atomicAdd(&s.nids, (int)__popcll(has));
            at = __builtin_amdgcn_readfirstlane(at) + (int)__popcll(has & before);
            if ((has >> lane) & 1) s.ids[at] = (uint16_t)g;
        }
        __syncthreads();
        const int ids = s.nids;
        // few groups: theirs (2 or 8 loads a wave for 128 or 512 of them); most groups, in the bulk: all bin numbers at once,
        // half the bytes and a quarter of the work a token (2374 groups of 64: 13 us, 29 us by groups)
        if (ids <= 8 * SR_W || !bin) sr_collect<1>(r.v, r.V, r.vec, s.ids, ids, lo, hi, lo2, hi2, s.list, &s.n);
        else sr_collect_bins(r.v, bin, r.V, b0, also, s.list, &s.n);
        __syncthreads();
        const int n = s.n;
        if (n > SR_LIST) return n;
        rank(n);
        double w[SR_PER];
#pragma unroll 1
        for (int h = 0; h < SR_PER; h++) w[h] = SR_PER * tid + h < n ? weight(ranked(SR_PER * tid + h)) : 0.0;
        scan(w);
        return n;
    }
};

// The bin down to which there are `want` groups, by their maxima. Where the bins of the tables hold fewer it is looked for
// once more in wider ones, up to where no token has weight that counts: that is the answer if there are fewer still.
__device__ __forceinline__ int sr_bin_of(SrTeam& t, int want) {
    SrPick& s = t.s;
    int* cnt = reinterpret_cast<int*>(s.list);
    int shift = 0;
#pragma unroll 1
    while (true) {
        for (int i = t.tid; i < SR_BINS; i += SR_T) cnt[i] = 0;
        if (t.tid == 0) s.found = -1;
        __syncthreads();
        for (int g = t.tid; g < t.groups; g += SR_T) {
            const double x = t.bins.x(t.group(g));
            if (x < (double)t.bins.reach && ((int)x >> shift) < SR_BINS) atomicAdd(&cnt[(int)x >> shift], 1);
        }
        __syncthreads();
        int c[SR_PER], v = 0;
#pragma unroll
        for (int h = 0; h < SR_PER; h++) v += c[h] = cnt[SR_PER * t.tid + h];
        const int own = v;
        v = wave_scan(v);
        int* sums = s.wave_count[t.flip ^= 1][0];
        if (t.lane == 63) sums[t.wave] = v;
        __syncthreads();
        v -= own;
        for (int i = 0; i < t.wave; i++) v += sums[i];
#pragma unroll
        for (int h = 0; h < SR_PER; h++) {
            if (v < want && v + c[h] >= want) s.found = SR_PER * t.tid + h;
            v += c[h];
        }
        __syncthreads();
        const int found = s.found;
        if (found >= 0) return ((found + 1) << shift) - 1;
        if (shift) return t.bins.reach;
        while ((t.bins.reach >> shift) >= SR_BINS) shift++;
        __syncthreads();   // all have read what is written again
    }
}

__global__ __launch_bounds__(SR_T) void sample_pick_kernel(SampleRowsArgs a, SrWork wk) {
    __shared__ union { SrShared sh; SrPick pick; } u;
    __shared__ SrTables tables;
    SrPick& s = u.pick;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* gmax = wk.gmax + (int64_t)row * wk.groups;
    constexpr int GU = SR_NEAR / SR_T;
    float near[GU];
#pragma unroll
    for (int k = 0; k < GU; k++) near[k] = gload(gmax + min(tid + k * SR_T, wk.groups - 1));   // in flight while the rest is looked up
    const SrAsk ask = sr_ask(a, row);
    const float T = a.temperature[row], given = a.u[row];
    SrRow r;
    r.v = a.logits + (int64_t)row * a.stride;
    r.V = a.V;
    r.vec = sr_vec(a);
    SrTeam t{s, tables, r, sr_bins(0.0f, T, 1.0 / (double)T), gmax, wk.groups, ask.kind == SR_SUM ? wk.bin + (int64_t)row * wk.groups * SR_GROUP : nullptr, tid, lane, wave, 0};
    if (wave < 2) {
        const double e = exp((wave ? -64.0 * (double)(lane & 31) : (double)-lane) * t.bins.inv_per);
        if (!wave) tables.part[lane] = e;
        else if (lane < 32) tables.whole[lane] = e;
    }
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < GU; k++) { s.gmax[tid + k * SR_T] = near[k]; top = fmaxf(top, near[k]); }
    for (int g = SR_NEAR + tid; g < wk.groups; g += SR_T) top = fmaxf(top, gload(gmax + g));
    top = wave_max(top);
    if (lane == 0) s.wave_top[wave] = top;
    if (tid == 0) { s.best = 0xffffffffu; s.n = 0; s.nids = 0; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SR_W; i++) top = fmaxf(top, s.wave_top[i]);
    if (!isfinite(top)) {   // none, or infinite
        if (tid == 0) { a.tokens[row] = 0; if (a.status) a.status[row] = 1; }
        return;
    }
    t.bins.top = sr_uniform((double)top);
    double goal = (double)given;
    goal = goal > 0.0 ? (goal < 1.0 ? goal : 1.0) : 0.0;
    int token = -1;
    if (ask.kind == SR_GREEDY || ask.low > 1.0f) {   // no weight is above 1
        for (int g = tid; g < wk.groups; g += SR_T) if (t.group(g) == top) atomicMin(&s.best, (uint32_t)g);
        __syncthreads();
        const int i = (int)s.best * SR_GROUP + lane;
        const uint64_t m = __ballot(i < r.V && r.v[min(i, r.V - 1)] == top);
        token = (int)s.best * SR_GROUP + (int)__builtin_ctzll(m);
    } else {
        // Where the kept tokens end and the draw falls among them. One gather does for most rows, and a second one if
        // the draw falls in another bin than was guessed.
        int also = -1, b0 = 0, b1 = t.bins.reach;
        int bp = SR_BINS, bm = SR_BINS;      // the bins in which top-p and min-p cut
        double p_goal = 0.0, kept = 0.0, before = 0.0, also_before = 0.0;
        double sums[SR_PER];                 // the bins' running sums, which the gathered tokens' take the place of
        bool drawing = false;                // the gathered bin is the draw's
        if (ask.kind == SR_TOP) {
            // all tokens down to a bin: that of the k-th largest group maximum, with min-p no further than its own
            if (r.V > SR_LIST) {
                if (ask.k < r.V) b1 = sr_bin_of(t, ask.k);
                if (ask.low > 0.0f && ask.p >= 1.0f) b1 = min(b1, (int)(-log((double)ask.low) * t.bins.per) + 1);
            }
        } else {
            const uint64_t* all = wk.mass + (int64_t)row * wk.sum_spans * SR_BINS + SR_PER * tid;
            uint64_t mass[SR_PER] = {};
#pragma unroll 4
            for (int k = 0; k < wk.sum_spans; k++)
#pragma unroll
                for (int h = 0; h < SR_PER; h++) mass[h] += gload(all + (int64_t)k * SR_BINS + h);
#pragma unroll
            for (int h = 0; h < SR_PER; h++) sums[h] = t.constant(SR_PER * tid + h) * (double)mass[h];
            t.scan(sums);
#pragma unroll
            for (int h = 0; h < SR_PER; h++) sums[h] = s.run[SR_PER * tid + h];
            kept = s.run[SR_BINS - 1];
            p_goal = (double)ask.p * kept;
            if (ask.p < 1.0f) bp = min(t.first(p_goal, 0.0, SR_BINS), SR_BINS - 1);
            if (ask.low > 0.0f) { const double x = -log((double)ask.low) * t.bins.per; if (x < (double)SR_BINS) bm = (int)x; }
            b0 = min(bp, bm);
            drawing = b0 == SR_BINS;         // nothing is cut
            // the draw's bin, if all tokens of the bin that the kept ones end in were kept: most often that is it
            const int last = min(b0, SR_BINS - 1), guess = min(t.first(goal * s.run[last], 0.0, last + 1), last);
            if (drawing || guess == b0) b0 = guess;
            else also = guess;
            b1 = b0;
            before = b0 ? s.run[b0 - 1] : 0.0;
            also_before = also > 0 ? s.run[also - 1] : 0.0;
        }
#pragma unroll 1
        while (b0 < SR_BINS - 1) {   // else a sum crosses behind the bins
            const int n = t.gather(also, b0, b1);
            if (n > SR_LIST) {
                if (also < 0) break;
                also = -1;   // without the guessed bin there may be room
                __syncthreads();
                if (tid == 0) { s.n = 0; s.nids = 0; }
                __syncthreads();
                continue;
            }
            if (ask.kind == SR_TOP) {
                const int k = min(ask.k, n);
                int end = k;
                if (ask.p < 1.0f) end = min(end, t.first((double)ask.p * s.run[k - 1], 0.0, k) + 1);
                if (ask.low > 0.0f) end = min(end, t.first_below((double)ask.low, k));
                end = max(end, 1);
                token = t.token(min(t.first(goal * s.run[end - 1], 0.0, end), end - 1));
                break;
            }
            int c[4];   // the list holds bin b0's tokens at c[0] .. c[1] - 1, those of `also` at c[2] .. c[3] - 1
            t.counts<4>(n, [&](int i, bool* b) {
                const double x = t.bins.x(t.ranked(i));
                b[0] = x < (double)b0; b[1] = x < (double)(b0 + 1); b[2] = x < (double)also; b[3] = x < (double)(also + 1);
            }, c);
            const double base = before - (c[0] ? s.run[c[0] - 1] : 0.0);
            int end = c[1];
            if (!drawing) {
                if (bp == b0) end = min(end, max(c[0], t.first(p_goal, base, c[1])) + 1);
                if (bm == b0) end = min(end, max(c[0], t.first_below((double)ask.low, c[1])));
                if (b0 == 0) end = max(end, 1);
                kept = end > c[0] ? base + s.run[end - 1] : before;
            }
            if (drawing || goal * kept > before || b0 == 0) {
                if (end > c[0]) token = t.token(min(max(c[0], t.first(goal * kept, base, end)), end - 1));
                break;
            }
            if (also >= 0 && goal * kept > also_before) {
                if (c[3] > c[2]) token = t.token(min(max(c[2], t.first(goal * kept, also_before - (c[2] ? s.run[c[2] - 1] : 0.0), c[3])), c[3] - 1));
                break;
            }
            __syncthreads();
#pragma unroll
            for (int h = 0; h < SR_PER; h++) s.run[SR_PER * tid + h] = sums[h];
            if (tid == 0) { s.n = 0; s.nids = 0; }
            __syncthreads();
            b1 = b0 = min(t.first(goal * kept, 0.0, b0), b0 - 1);
            before = b0 ? s.run[b0 - 1] : 0.0;
            also = -1;
            drawing = true;
        }
    }
    if (token < 0) {
        __syncthreads();
        token = sr_descent_token(r.v, r.V, top, T, tables, ask.k, ask.p, ask.low, given, u.sh);
    }
    if (tid == 0) { a.tokens[row] = token; if (a.status) a.status[row] = 0; }
}

// Groups of a workgroup that adds up bins, at least: it also clears and stores 2048 of them (33 rows: 34 us, with 64 39 us).
constexpr int SR_SUM_LEAST = 256;
static size_t sr_layout(int rows, int V, void* base, SrWork& wk) {
    wk.groups = (V + SR_GROUP - 1) / SR_GROUP;
    auto cut = [&](int wgs, int least, int& spans, int& per) {   // about wgs workgroups in all, of `least` groups each or more
        const int most = (wk.groups + least - 1) / least, want = (wgs + rows - 1) / rows;
        per = (wk.groups + (want < most ? want : most) - 1) / (want < most ? want : most);
        spans = (wk.groups + per - 1) / per;
    };
    cut(1024, 64, wk.spans, wk.per);
    cut(2048, SR_SUM_LEAST, wk.sum_spans, wk.sum_per);   // each adds all of its bins to the row's in the end
    uint8_t* p = static_cast<uint8_t*>(base);
    size_t at = 0;
    auto take = [&](size_t bytes) { uint8_t* q = p ? p + at : nullptr; at += (bytes + 255) / 256 * 256; return q; };
    wk.gmax = reinterpret_cast<float*>(take((size_t)rows * wk.groups * 4));
    wk.bin = reinterpret_cast<uint16_t*>(take((size_t)rows * wk.groups * SR_GROUP * 2));
    wk.mass = reinterpret_cast<uint64_t*>(take((size_t)rows * wk.sum_spans * SR_BINS * 8));
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
    if (sr_vec(a)) hipLaunchKernelGGL(sample_groups_kernel<true>, grid, dim3(256), 0, s, a, wk);
    else hipLaunchKernelGGL(sample_groups_kernel<false>, grid, dim3(256), 0, s, a, wk);
    // which rows need sums is on the device: the others' workgroups leave at once
    hipLaunchKernelGGL(sample_sums_kernel, dim3(wk.sum_spans, a.rows), dim3(SR_SUM_T), 0, s, a, wk);
    hipLaunchKernelGGL(sample_pick_kernel, dim3(a.rows), dim3(SR_T), 0, s, a, wk);
    return hipGetLastError();
}

}  // namespace mlxr
