// Attention of any number of new tokens a sequence over a pool of KV-cache pages.
#include <type_traits>
#include "batch.h"

namespace mlxr {

// out = sum_j p_j v_j, p = softmax of scale q k_j over the slots up to a row's own: 4 D flops a (row, query head, slot), and
// 4 D bytes a slot and KV head once. One token a sequence is bound by those reads, a chunk by the matrix cores.
//
// Split. The (token, query head of the KV head) pairs of a sequence and KV head, tokens first, are its queries; AR_M of them
// are an item, so a page is read once for all heads of a group and several tokens. An item walks the pages from the first
// that its first token attends to its last token's own. All items' pages (pairs of pages, see below), laid end to end, are
// cut into equal runs, one per workgroup, so chunks, prompts and single tokens of one call keep the card evenly busy, and
// counts and lengths may stay on the device: each workgroup finds its run by a scan over the sequences. How many pages an
// item has follows from rounding twice, so its length here is a bound that adds up in closed form (AtPlaces): up to two
// places of an item hold no page, and AR_GAP more stand for what beginning and ending one costs. An item inside one run is
// written out at once; one cut by runs leaves partial results (maximum, sum, unnormalised values), which the last workgroup
// to finish joins in run order: the same bits every time. A part is 2.5 us of a join by one workgroup, so where a wave would
// have more than AR_GROUP of them they are joined in groups, and then the groups (180 tokens after 594 and 52 after 11387,
// five heads of one KV head: 63 us, 185 with one join).
//
// Inside. Eight waves have 32 queries each and read the same page from LDS; where an item has 128 queries or fewer, four do, and
// the other four take every other page, joined through LDS at the end. Pages are copied there straight from the cache, three
// ahead (or two, in pairs), 16-byte pieces XOR-swizzled by the key. 32x32x16 MFMAs:
//   S^T = K q^T: lane (r = l % 32, h = l / 32) has query r's scores of keys 8 (i / 4) + 4 h + i % 4 of both 32-key halves.
//   O^T = V^T P^T: a lane's eight scores of 16 keys are what it has to hold of P^T as an operand, if element e of
//   half h stands for key 8 (e / 4) + 4 h + e % 4. V^T has its keys in that order from the LDS transpose read.
// So maximum, sum and rescaling of a query stay within two lanes. Products and softmax take about as long as each other, so
// the two waves of a SIMD are half a page apart: between two barriers one multiplies (the last page's values, the next one's keys)
// while the other has its softmax. Queries in the cache's type enter as they are, and
// p is rounded to it; fp32 ones, and their p, are split into parts that the matrix cores multiply exactly: three bf16 by
// truncation (24 bits), or two f16 (22 bits, q scaled to at most 2^14 by a power of two). Scores are in powers of two.
// A query's reference point for p moves only when a page's maximum is LAZY or more above it: until then p is up to
// 2^LAZY, and nothing has to be rescaled. f16 ends 2^-24 below one, so that a long tail of small p would lose its bits, and with
// one sign where keys are alike (131072 equal ones that weigh as much as one in front of them: 2^-12 of the result): with such a
// cache the point moves down to a page's maximum as well when that is LAZY or more below, so that what ends is 2^-24 (2^-28 of
// fp32 queries) of the largest p of its own page, whatever the length (fp32 queries: by whole powers of two, so that moves round nothing). That costs nothing at D 128 and 3% at D 64 (24 windows
// in fp32 67 -> 69 us); LAZY of 5, 6 and 7 are alike.
//
// Roundings. Scores, sums and values are fp32. Queries of the cache's type and p rounded to it (half a step, 2^-8 of p in
// bf16; the sum is of the unrounded p) cost one product a key and dim each; fp32 ones three (bf16) or two (f16), and are
// right to 24 and 22 bits. A lane sums p page by page and adds the pages' sums: 131072 equal keys that weigh as much as one key in
// front of them are 1e-4 off, 2e-3 with one addition a key, in the same time.
//
// Measured, and what bounds it. 2048 tokens after 30000, 40 heads of 128, 8 KV heads, bf16: 1.24 ms, 1.05 PF/s: the matrix
// cores are busy for 57% of the cycles, at the 1.8 to 1.85 GHz that the power limit leaves (1.10 ms without the copies, 1.04
// without the softmax), and a page's turn is 2.05 us: 0.6 for the keys' products, 0.35 to 0.45 for the values', 0.75 to 0.9
// for the softmax, 0.2 for what the copies need, 0.1 for barriers. 2048 after 0: 62 us, 0.55 PF/s: 1.7 parts of items a run, of
// 10 pages each. A part costs 10 us beside its pages: 4 until the first ones are there, 1.3 for the queries, 1.3 for the look
// for what is not finite, 3.5 to hand its results over (2.2 to write a whole item's); a join, in 159 of the 251 runs, 6.7 more.
// 32 sequences, 24 with one new token and 8 with up to 400, after up to 7000: 207 us, matrix cores busy for 37% of the cycles: a
// run has 2.7 parts and 103 pages, half of them in pairs for four queries; 53 at 2.05 us, 25 pairs at 2.5, 11 until first pages are
// there, 18 for beginnings and ends, 5 for joins. 24 windows of 1024, 64 dims, f16: 58 us, two parts of 12 pages a run, 1.55 us a page, a
// quarter of the places without one. fp32 queries over bf16: a page 4.5 us, a part 16 beside its pages (8 for the
// queries, 2.6 for the look, 5.2 to hand over), a join 7.5. Five tokens of fp32 after 7000: 33 us, of which 5 are the launch, 2.6 the
// search for the run, 5 the queries, 13 two turns behind each other, 4 partial results and 3 to 5 the join: one round trip after
// another; its reads alone would be 6.
// What is not finite sends its run's part of the item through the pages again: one infinite value in 2048 tokens after 0 makes 62 us 370
// (fp32 queries 117 and 1270), 2048 after 30000 1.24 ms 4.2, five tokens 33 us 145. The fp32 kernels of 128 dims spill
// registers on that way (580 bytes a lane over bf16, 332 over f16); in the page loops two are read back, where a page is masked.
// More than 64 sequences are scanned by the workgroup, twice: 32 single tokens of up to 8192 slots take as long among 512 sequences as
// alone, among 32768 90 to 100 us longer.
// Both sides of the choices. Pages in pairs where an item has AR_M / 2 queries or fewer: 34.4 us against 38.5 for the five
// tokens, 208 against 227 for the 32 sequences, 58 against 62 for the windows. Each wave looks for its run by itself
// (up to 64 sequences): 34.4 against 35.6 and 58 against 59. Items of AR_M queries rather than of half as many read a page
// for twice as many products.
constexpr int AR_WV = 8, AR_TH = 64 * AR_WV, AR_M = 32 * AR_WV;   // waves and threads of a workgroup, queries of an item
constexpr int AR_MAXW = 256;       // workgroups: one a CU
// Places behind an item. Of 128 dims 4 to 6 are alike; of 64 dims 5 is 1 to 5% faster than 7 in six of nine batches (2048 tokens
// after 0: 48 us against 50, with 9 52; 10 chunks with a window of 300: 40 against 42) and 2% slower in one (24 windows of 1024).
constexpr int AR_GAP = 5;
constexpr int AR_COUNTS = 4 * AR_MAXW;
constexpr int AR_GROUP = 8;        // parts that a wave joins one after another
constexpr int AR_MINPER = 2;       // places of a run at least
constexpr int AR_RING = 4;         // pages of keys, and of values, in LDS
#define AT_IN __attribute__((always_inline))   // what holds the operands' registers has to stay in the kernel
typedef float at_f16 __attribute__((ext_vector_type(16)));
typedef __bf16 at_b8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_b2 __attribute__((ext_vector_type(2)));
typedef _Float16 at_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 at_h2 __attribute__((ext_vector_type(2)));
typedef uint32_t at_u4 __attribute__((ext_vector_type(4)));
typedef short at_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* at_lptr;
typedef __attribute__((address_space(3))) at_s4* at_lv4;

template <int ST> __device__ __forceinline__ at_f16 at_mfma(at_u4 a, at_u4 b, at_f16 c) {
    if constexpr (ST == 0) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(at_b8, a), __builtin_bit_cast(at_b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(at_h8, a), __builtin_bit_cast(at_h8, b), c, 0, 0, 0);
}
constexpr int at_parts(int ST, bool HQ) { return HQ ? 1 : (ST == 0 ? 3 : 2); }
// Two fp32 values as dword i of operands: rounded once (HQ), or parts whose sum they are (bf16) or nearly are (f16).
template <int ST, bool HQ> __device__ __forceinline__ void at_split2(float a, float b, int i, at_u4* o) {
#pragma unroll
    for (int t = 0; t < at_parts(ST, HQ); t++) {
        if constexpr (ST == 0 && HQ) o[t][i] = __builtin_bit_cast(uint32_t, at_b2{(__bf16)a, (__bf16)b});
        else if constexpr (ST == 0) {
            o[t][i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
            a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
            b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
        } else {
            const at_h2 h = {(_Float16)a, (_Float16)b};
            o[t][i] = __builtin_bit_cast(uint32_t, h);
            a -= (float)h[0];
            b -= (float)h[1];
        }
    }
}
template <int ST, bool HQ> __device__ __forceinline__ void at_split(const float* x, at_u4* o) {
#pragma unroll
    for (int i = 0; i < 4; i++) at_split2<ST, HQ>(x[2 * i], x[2 * i + 1], i, o);
}
__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float at_safe(float m) { return m == -INFINITY ? 0.0f : m; }   // -inf - -inf would be NaN
__device__ __forceinline__ float at_times(float f, float x) { return __builtin_isinf(x) ? x : f * x; }   // for an f above 0 that may have come out as 0
__device__ __forceinline__ void at_store2(float* p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 at_load2(const float* p) {
    const uint64_t v = __hip_atomic_load(const_cast<uint64_t*>(reinterpret_cast<const uint64_t*>(p)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return float2{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

// The LDS transpose read. Of a pointer of its own (__restrict__): otherwise the compiler, which cannot tell what it reads from
// what copies write, waits for every copy in flight in front of it.
__device__ __forceinline__ uint2 at_read_tr(const uint8_t* __restrict__ p) { return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lv4)p)); }
// Values that are the same in all lanes, for the scalar registers: addresses and loops that are not known to be so cost many times more.
__device__ __forceinline__ int at_one(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t at_one(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)at_one((int)(uint32_t)v) | (uint64_t)(uint32_t)at_one((int)(v >> 32)) << 32);
}
__device__ __forceinline__ uint64_t at_one(uint64_t v) { return (uint64_t)at_one((int64_t)v); }

// a / b for a below 2^52: the compiler's own division of 64 bits is a page of code.
__device__ __forceinline__ uint64_t at_div(uint64_t a, uint64_t b) {
    uint64_t q = (uint64_t)((double)a / (double)b);
    if (q * b > a) q--;
    if (a - q * b >= b) q++;
    return q;
}

struct AtShared {
    uint64_t sums[2][AR_WV], found_pre;
    int found_b, last, odd[AR_WV];
    float m[AR_WV][64], l[AR_WV][64];
};
struct AtWork {
    unsigned* count;      // [AR_COUNTS] arrivals; zero between calls. [w0]: at the item that starts in run w0 and goes on behind it;
                          // [AR_MAXW + w0], [2 AR_MAXW + run]: at its first group of parts, at the group that starts with the run
    float* part;          // [2 W] partial results: [AR_WV][D / 4 + 1][64][2]: 32 queries' values, then maximum and sum
    int W;
};
__host__ __device__ __forceinline__ constexpr size_t at_part_floats(int D) { return (size_t)AR_WV * (D / 4 + 1) * 128; }

// A sequence's rows: c of them, the first at row `row` and slot `base`; `none` rows in front of these have no slot.
struct AtSeq { int c, base, row, none; };
__device__ __forceinline__ AtSeq at_seq(const AttnRowsArgs& a, int b) {
    const int64_t n = max(0, a.count[b]), s = a.start[b], len = paged_len(a.kv, b);
    const int64_t i0 = max((int64_t)0, -s), i1 = min(n, (int64_t)a.rows - s);   // tokens whose rows are in the array
    const int64_t first = min(max(i0, n - len), max(i0, i1));                   // the first of them with a slot
    return AtSeq{(int)max((int64_t)0, i1 - first), (int)max((int64_t)0, len - n + first), (int)(s + first), (int)max((int64_t)0, first - i0)};
}
__device__ __forceinline__ AtSeq at_one(const AtSeq& s) { return AtSeq{at_one(s.c), at_one(s.base), at_one(s.row), at_one(s.none)}; }
// How many items a sequence has, and their places: min(A + floor(S i / G), cap) + GAP for item i, S pages of queries (AR_M / 64);
// half as many pages for a last item of AR_M / 2 queries or fewer, whose pages go in pairs.
template <int D> struct AtPlaces {
    static constexpr int S = AR_M / MLXR_PAGE, GAP = AR_GAP;
    int64_t A, cap, bend;   // from item `bend` on the cap holds
    int G, items;
    bool few;
    __device__ __forceinline__ AtPlaces(const AttnRowsArgs& a, int G_, const AtSeq& s) : G(G_) {
        const int64_t spread = (AR_M - 1) / G, queries = (int64_t)s.c * G;
        items = (int)((queries + AR_M - 1) / AR_M);
        few = queries - (int64_t)(items - 1) * AR_M <= AR_M / 2;
        A = (s.base + spread) / MLXR_PAGE + 2;
        cap = a.window > 0 ? (a.window + spread + MLXR_PAGE - 1) / MLXR_PAGE + 1 : (int64_t)1 << 40;
        bend = cap <= A ? 0 : ((cap - A) * G + S - 1) / S;
    }
    __device__ __forceinline__ int64_t pages(int item) const { return min(A + (int64_t)((uint32_t)item * (uint32_t)S / (uint32_t)G), cap); }   // items are below 2^23
    __device__ __forceinline__ int64_t of(int item) const { return (few && item == items - 1 ? (pages(item) + 1) / 2 : pages(item)) + GAP; }
    __device__ __forceinline__ int64_t steps(int v) const {   // sum of floor(S i / G) over i < v <= G
        int64_t n = 0;
#pragma unroll
        for (int k = 1; k < S; k++) n += max(0, v - (k * G + S - 1) / S);
        return n;
    }
    __device__ __forceinline__ int64_t cum(int n) const {     // of items 0 .. n - 1, n < items or the last of them counted whole
        const int64_t m = min((int64_t)n, bend);
        const uint32_t u = (uint32_t)m / (uint32_t)G, v = (uint32_t)m % (uint32_t)G;
        return (int64_t)n * GAP + m * A + (int64_t)S * G * ((int64_t)u * ((int64_t)u - 1) / 2) + u * steps(G) + (int64_t)S * u * v + steps((int)v) + (n - m) * cap;
    }
    __device__ __forceinline__ int64_t all() const { return cum(items - 1) + of(items - 1); }
};

// Where a key's 16-byte pieces lie in LDS: piece c at c ^ this. Sixteen keys' same piece, and four keys' same four pieces, are in
// different banks.
template <int D> __device__ __forceinline__ int at_swz_k(int key) { return D == 128 ? key & 15 : (key >> 1) & 7; }
template <int D> __device__ __forceinline__ int at_swz_v(int key) { return 4 * (D == 128 ? key & 3 : (key >> 1) & 1) + ((key >> 2) & 3); }

template <int ST, int D, bool HQ>
__global__ __launch_bounds__(AR_TH, 2) void attn_rows_kernel(AttnRowsArgs a, AtWork wk) {
    constexpr int NP = at_parts(ST, HQ), KS = D / 16, NV = D / 32, TILE = 64 * D * 2, ROW = 2 * D, CH = D / 8;   // CH: 16-byte pieces of a row
    constexpr int PW = TILE / 1024 / AR_WV;   // copies a wave and page of keys (or values)
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];   // [AR_RING] pages of keys, then of values (partial results in between); AtShared
    AtShared& sh = *reinterpret_cast<AtShared*>(lds + 2 * AR_RING * TILE);
    const PagedKV& kv = a.kv;
    const int tid = threadIdx.x, lane = tid & 63, wave = at_one(tid >> 6), r = lane & 31, h = lane >> 5;
    const int G = a.nH / kv.nKV, W = wk.W;
    // neighbouring runs share keys: those of an XCD (workgroups 8 apart) are neighbours
    const int w = W % 8 == 0 ? (int)(blockIdx.x % 8) * (W / 8) + (int)blockIdx.x / 8 : (int)blockIdx.x;
    const void *K = kv.k, *V = kv.v;

    // this workgroup's run of places
    auto places_of = [&](const AtSeq& s) AT_IN -> uint64_t { return s.c ? (uint64_t)(AtPlaces<D>(a, G, s).all() * kv.nKV) : 0; };
    auto zero = [&](const AtSeq& s) AT_IN {   // rows without a slot
        const int per = a.nH * D * (HQ ? 2 : 4) / 16;
        for (int64_t i = lane; i < (int64_t)s.none * per; i += 64) {
            const int64_t row = s.row - s.none + i / per;
            *reinterpret_cast<at_u4*>(static_cast<uint8_t*>(a.out) + row * a.out_stride * (HQ ? 2 : 4) + i % per * 16) = at_u4{0, 0, 0, 0};
        }
    };
    uint64_t total = 0, per, t, t1, pre;
    int b;
    AtSeq sq;
    auto zeros = [&](const AtSeq& s, int first) AT_IN {   // of the sequences first + lane, each by one workgroup
        for (uint64_t idle = __ballot(s.none > 0 && (first + lane) % W == w); idle; idle &= idle - 1) {
            const int i = (int)__builtin_ctzll(idle);
            zero(AtSeq{0, 0, __builtin_amdgcn_readlane(s.row, i), __builtin_amdgcn_readlane(s.none, i)});
        }
    };
    auto run_of = [&]() AT_IN {   // false: there are fewer runs than workgroups
        per = max((uint64_t)AR_MINPER, at_one(at_div(total + W - 1, W)));
        t = (uint64_t)w * per;
        t1 = min(total, t + per);
        return t < total;
    };
    if (kv.B <= 64) {   // each wave by itself
        const AtSeq s = lane < kv.B ? at_seq(a, lane) : AtSeq{0, 0, 0, 0};
        const uint64_t n = places_of(s), upto = wave_scan(n);
        if (wave == 0) zeros(s, 0);
        total = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)upto, 63) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(upto >> 32), 63) << 32;
        if (!run_of()) return;
        b = (int)__builtin_ctzll(__ballot(upto - n <= t && t < upto));
        const uint64_t before = upto - n;
        pre = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)before, b) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(before >> 32), b) << 32;
        sq = AtSeq{__builtin_amdgcn_readlane(s.c, b), __builtin_amdgcn_readlane(s.base, b), __builtin_amdgcn_readlane(s.row, b), 0};
    } else {
        uint64_t before = 0, n = 0, chunk = 0;
        int step = 0;
        auto scan = [&](int c, bool first) AT_IN {
            const AtSeq s = c + tid < kv.B ? at_seq(a, c + tid) : AtSeq{0, 0, 0, 0};
            n = places_of(s);
            if (first) zeros(s, c + 64 * wave);
            const uint64_t v = wave_scan(n);
            uint64_t* sums = sh.sums[step++ & 1];
            if (lane == 63) sums[wave] = v;
            __syncthreads();
            before = v - n;
            chunk = 0;
#pragma unroll
            for (int i = 0; i < AR_WV; i++) { before += i < wave ? sums[i] : 0; chunk += sums[i]; }
        };
#pragma unroll 1
        for (int c = 0; c < kv.B; c += AR_TH) { scan(c, true); total += chunk; }
        total = at_one(total);
        if (!run_of()) return;
        uint64_t run = 0;
#pragma unroll 1
        for (int c = 0; c < kv.B; c += AR_TH) {
            scan(c, false);
            const uint64_t p = run + before;
            if (p <= t && t < p + n) { sh.found_b = c + tid; sh.found_pre = p; }
            run += chunk;
            if (run > t) break;
        }
        __syncthreads();
        b = at_one(sh.found_b);
        pre = at_one(sh.found_pre);
        sq = at_one(at_seq(a, b));
    }
    // the item in which the run begins
    int kvh, item, items;
    {
        const AtPlaces<D> pl(a, G, sq);
        items = at_one(pl.items);
        const uint64_t each = at_one((uint64_t)pl.all()), local = t - pre;
        kvh = at_one((int)at_div(local, each));
        pre += kvh * each;
        const int64_t at = (int64_t)(t - pre);
        int lo = 0, step = 1;
        while (step * 64 < items) step *= 64;
        for (;; step /= 64) {   // the last item that begins at or before the place
            const int i = lo + lane * step;
            lo += step * (63 - (int)__builtin_clzll(__ballot(i < items && i >= lo && pl.cum(i) <= at)));
            if (step == 1) break;
        }
        item = at_one(lo);
        pre += at_one(pl.cum(item));
    }
    while (true) {
        // pre: the item's first place
        const AtPlaces<D> pl(a, G, sq);
        const int f0 = item * AR_M, R = min((int64_t)AR_M, (int64_t)sq.c * G - f0);
        auto first_of = [&](int tok) AT_IN { return a.window > 0 ? max(0, sq.base + tok + 1 - a.window) : 0; };
        const int p0 = at_one(first_of(f0 / G) / MLXR_PAGE), pages = at_one((sq.base + (f0 + R - 1) / G) / MLXR_PAGE - p0 + 1);
        const bool two = R <= AR_M / 2;   // pages go in pairs
        const int pair = two ? 2 : 1, place = (int)(t - pre), places = (pages + pair - 1) / pair, tile = place * pair;   // the run's first page of the item
        const int tiles = (int)min((int64_t)(pages - tile), (int64_t)(t1 - t) * pair);
        // on to the run's next item; where the next sequence has no rows, 256 counts a step (eight sequences of 11 to
        // 15 pages, 7500 idle ones between each two of them: 181 us, 2050 with one a step)
        auto next_sequence = [&]() AT_IN {
            while (++b < kv.B) {
                sq = at_one(at_seq(a, b));
                if (sq.c) return true;
                uint64_t on[4] = {};
                for (b++; b < kv.B; b += 256) {
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const int i = b + 64 * u + lane;
                        on[u] = __ballot(a.count[min(i, kv.B - 1)] > 0 && i < kv.B);
                    }
                    if (on[0] | on[1] | on[2] | on[3]) break;
                }
                const int u = on[0] ? 0 : on[1] ? 1 : on[2] ? 2 : 3;
                b += 64 * u + (on[u] ? (int)__builtin_ctzll(on[u]) : 0) - 1;
            }
            return false;      // not with t < t1 <= total, which is of sequences that have rows
        };
        auto ahead = [&]() AT_IN {
            const uint64_t n = at_one((uint64_t)pl.of(item));
            t = pre + n;
            if (t >= t1) return false;
            pre = t;
            if (++item == items) {
                item = 0;
                if (++kvh == kv.nKV) {
                    kvh = 0;
                    if (!next_sequence()) return false;
                    items = at_one(AtPlaces<D>(a, G, sq).items);
                }
            }
            return true;
        };
        if (tiles <= 0) {   // the run begins behind an item's pages
            if (!ahead()) return;
            continue;
        }
        // this wave's queries, and the other pages' of few
        const int turn = two ? wave >> 2 : 0, block = two ? wave & 3 : wave, blocks = (R + 31) / 32;
        const int mine = min(32, R - 32 * block);                 // how many, if above 0
        const bool active = mine > 0;
        const int f = f0 + (active ? 32 * block + min(r, mine - 1) : 0), tok = f / G, head = kvh * G + f % G;
        const int lim = sq.base + tok, low = first_of(tok);       // the slots that this lane's query attends: low .. lim
        const int lim0 = __builtin_amdgcn_readlane(lim, 0), lim1 = __builtin_amdgcn_readlane(lim, 31), low0 = __builtin_amdgcn_readlane(low, 0), low1 = __builtin_amdgcn_readlane(low, 31);
        const int64_t q_at = (int64_t)(sq.row + tok) * a.q_stride + (int64_t)head * D;
        // where pages are in the pools (bytes), one a lane, 64 at a time; below 0 where there is none
        int have = 0;
        int64_t offs;
        auto look = [&]() AT_IN {
            const int page = paged_page(kv, b, p0 + tile + min(64 * have + lane, tiles - 1));
            offs = page < 0 ? -1 : ((int64_t)page * kv.nKV + kvh) * TILE;
        };
        look();
        auto page_of = [&](int i) AT_IN -> int64_t {
            if ((i >> 6) != have) {
                have = i >> 6;
                look();
            }
            return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)offs, i & 63) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(offs >> 32), i & 63) << 32);
        };
        // a KiB of this wave's share of a page's copy: what lies in its first `bytes`, and zeros behind (nothing is read of a page
        // that is not there)
        auto copy = [&](const void* pool, bool values, int64_t off, int bytes, uint32_t to, int j) AT_IN {
            const uint8_t* from = static_cast<const uint8_t*>(pool) + off;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, at_one(off < 0 ? 0 : bytes), 0x00020000);
            uint8_t* dst = lds + to;
            const int piece = wave * PW + j, key = piece * (64 / CH) + lane / CH, swz = values ? at_swz_v<D>(key) : at_swz_k<D>(key);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (at_lptr)(dst + piece * 1024), 16, key * ROW + 16 * (lane % CH ^ swz), 0, 0, 0);
        };
        const int end = sq.base + sq.c;
        auto rows_of = [&](int i) AT_IN { return max(0, min(MLXR_PAGE, end - (p0 + tile + i) * MLXR_PAGE)) * ROW; };   // bytes of page i in front of the sequence's end
        // queries as operands: dims 16 s + 8 h .. + 7 of query r
        at_u4 q[KS][NP];
        float cl = HQ ? fabsf(a.scale) * 1.4426950408889634f : 1.0f;   // scores to powers of two
        {   // of all waves, those without queries too: what one keeps for the next item costs registers
            if constexpr (HQ) {
                const uint16_t* p = static_cast<const uint16_t*>(a.q) + q_at + 8 * h;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) q[ks][0] = gload(reinterpret_cast<const at_u4*>(p + 16 * ks));
                if (a.scale < 0.0f)
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) q[ks][0] ^= 0x80008000u;
                cl = fmaxf(cl, 0x1p-126f);   // a scale of 0: scores of 0, and -infinity stays what it is
            } else {
                float x[KS][8], mx = 0.0f;
                const float* p = static_cast<const float*>(a.q) + q_at + 8 * h;
                const float by = a.scale * 1.4426950408889634f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const float4 u = gload4(p + 16 * ks), v = gload4(p + 16 * ks + 4);
                    x[ks][0] = u.x; x[ks][1] = u.y; x[ks][2] = u.z; x[ks][3] = u.w; x[ks][4] = v.x; x[ks][5] = v.y; x[ks][6] = v.z; x[ks][7] = v.w;
                }
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[ks][e] *= by;
                        if (ST == 1) mx = fmaxf(mx, fabsf(x[ks][e]));
                    }
                if constexpr (ST == 1) {
                    mx = xor32_max(mx);
                    int e2 = 0;
                    if (mx > 0.0f && mx < INFINITY) { frexpf(mx, &e2); e2 = 14 - e2; e2 = e2 < -126 ? -126 : (e2 > 126 ? 126 : e2); }
                    const float up = ldexpf(1.0f, e2);
                    cl = ldexpf(1.0f, -e2);
#pragma unroll
                    for (int ks = 0; ks < KS; ks++)
#pragma unroll
                        for (int e = 0; e < 8; e++) x[ks][e] *= up;
                }
#pragma unroll
                for (int ks = 0; ks < KS; ks++) at_split<ST, HQ>(x[ks], q[ks]);
            }
        }
        at_f16 o[NV];        // dims 32 n + 8 (i / 4) + 4 h + i % 4 of query r
        float m, l;          // the point of reference; this lane's keys' sum
        constexpr float LAZY = ST == 1 && !HQ ? 6.0f : 8.0f;   // how far p's point of reference may be from a page's maximum
        constexpr float UP = ST == 0 ? 0.0f : 15.0f - LAZY;         // p times 2^UP: up to 2^15
        at_f16 s[2];         // scores of a page, keys 32 kb + 8 (i / 4) + 4 h + i % 4
        at_u4 pr[4];         // p of a page, rounded (HQ; s otherwise)
        constexpr uint32_t VALUES = AR_RING * TILE;
        auto first_key = [&](int i) AT_IN { return (p0 + tile + i) * MLXR_PAGE; };
        constexpr int KA = HQ ? 3 : 2, VA = HQ ? 5 : 3;      // fragments in registers: read KA - 1 (VA - 1) steps of NP products ahead
        at_u4 kf[KA][2];
        uint32_t kaddr;
        auto kread = [&](int ks) AT_IN {
#pragma unroll
            for (int kb = 0; kb < 2; kb++) kf[ks % KA][kb] = *reinterpret_cast<const at_u4*>(lds + ((kaddr ^ (32u * ks)) + 32u * ROW * kb));
        };
        auto find_k = [&](uint32_t at) AT_IN {
            int ln = lane;
            asm volatile("" : "+v"(ln));   // addresses are made here, not kept across pages
            const uint32_t lr = ln & 31, lh = ln >> 5;
            kaddr = at + lr * ROW + 16 * (lh ^ at_swz_k<D>(lr));              // ^ 32 ks, + 32 ROW kb
        };
        auto begin_k = [&]() AT_IN {
#pragma unroll
            for (int ks = 0; ks < KA - 1; ks++) kread(ks);
        };
        auto products_k = [&](auto beside) AT_IN {   // beside(ks): what else each step asks for
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                __builtin_amdgcn_sched_barrier(0);
                if (ks + KA - 1 < KS) kread(ks + KA - 1);
                beside(ks);
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int kb = 0; kb < 2; kb++) s[kb] = at_mfma<ST>(kf[ks % KA][kb], q[ks][p], ks + p ? s[kb] : at_f16{0.0f});
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto softmax = [&](auto CARE, int k0) AT_IN {
            if (__builtin_expect(k0 + MLXR_PAGE - 1 > lim0 || k0 < low1, 0))   // some query does not attend all of the page
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int key = k0 + 32 * kb + 8 * (e >> 2) + 4 * h + (e & 3);
                        if (key > lim || key < low) s[kb][e] = -INFINITY;
                    }
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int e = 0; e < 16; e++) mx = fmaxf(mx, s[kb][e]);
            mx = xor32_max(mx);
            if (HQ || ST == 1) mx *= cl;
            bool move = mx > m + LAZY;
            if (ST == 1) move |= mx < m - LAZY && mx > -INFINITY;
            if (__any(move)) {
                const float to = ST == 1 && !HQ ? rintf(mx) : mx;   // whole: any number of moves up and down rounds nothing
                float mn = fmaxf(m, to);
                if (ST == 1 && to < m && to > -INFINITY && xor32_max(l) * at_exp2(m - to) < 0x1p64f) mn = to;   // what goes before stays far from overflow
                const float c = at_exp2(m - at_safe(mn));
                l *= c;
#pragma unroll
                for (int n = 0; n < NV; n++)
#pragma unroll
                    for (int e = 0; e < 16; e++) o[n][e] = decltype(CARE)::value ? at_times(c, o[n][e]) : c * o[n][e];
                m = mn;
            }
            const float ms = at_safe(m) - UP;
            float sum[4];        // of the page: many small p would lose bits one after another beside a large one in l
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    s[kb][e] = at_exp2(HQ || ST == 1 ? fmaf(s[kb][e], cl, -ms) : s[kb][e] - ms);
                    sum[e & 3] = kb == 0 && e < 4 ? s[kb][e] : sum[e & 3] + s[kb][e];
                }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if constexpr (HQ)
#pragma unroll
                for (int st = 0; st < 4; st++) {
                    float p8[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) p8[e] = s[st >> 1][8 * (st & 1) + e];
                    at_split<ST, HQ>(p8, &pr[st]);
                }
        };
        uint2 vf[VA][2];   // V^T fragments (16 keys st, 32 dims n) f = NV st + n
        uint32_t vaddr;
        auto vread = [&](int f) AT_IN {
#pragma unroll
            for (int u = 0; u < 2; u++) vf[f % VA][u] = at_read_tr(lds + ((vaddr ^ (64u * (f % NV)) ^ (32u * u)) + 8u * ROW * u + 16u * ROW * (f / NV)));
        };
        auto begin_v = [&](uint32_t at) AT_IN {
            int ln = lane;
            asm volatile("" : "+v"(ln));
            const uint32_t lh = ln >> 5, j = ln & 15;
            vaddr = at + (4 * lh + (j >> 2)) * ROW + 16 * ((2 * (ln >> 4 & 1) + ((j & 3) >> 1)) ^ (4 * (j >> (D == 128 ? 2 : 3)) + lh)) + 8 * (j & 1);
#pragma unroll
            for (int f = 0; f < VA - 1; f++) vread(f);
        };
        auto products_v = [&](auto beside) AT_IN {   // beside(f): what else each step asks for or reads
            at_u4 pp[2][NP];   // p of 16 keys; the next ones' are split among these ones' products
            auto split = [&](int st, int i) AT_IN { at_split2<ST, HQ>(s[st >> 1][8 * (st & 1) + 2 * i], s[st >> 1][8 * (st & 1) + 2 * i + 1], i, pp[st & 1]); };
            if constexpr (!HQ)
#pragma unroll
                for (int i = 0; i < 4; i++) split(0, i);
#pragma unroll
            for (int f = 0; f < 4 * NV; f++) {
                const int st = f / NV, n = f % NV;
                __builtin_amdgcn_sched_barrier(0);
                if (f + VA - 1 < 4 * NV) vread(f + VA - 1);
                beside(f);
                const at_u4 vt = {vf[f % VA][0].x, vf[f % VA][0].y, vf[f % VA][1].x, vf[f % VA][1].y};
                if constexpr (HQ) o[n] = at_mfma<ST>(vt, pr[st], o[n]);
                else {
#pragma unroll
                    for (int p = 0; p < NP; p++) o[n] = at_mfma<ST>(vt, pp[st & 1][p], o[n]);
                    if (st < 3)
#pragma unroll
                        for (int i = 0; i < 4 / NV; i++) split(st + 1, 4 / NV * n + i);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        // pages of the run that some query attends some of: lo .. hi - 1
        const int lo = active ? low0 / MLXR_PAGE - (p0 + tile) : 0, hi = active ? min(tiles, lim1 / MLXR_PAGE - (p0 + tile) + 1) : 0;
        // The run's pages, `STEP` of them a turn, two barriers a turn: behind the first one waves 0 .. 3 multiply (the values of the turn before,
        // then its keys), behind the second one waves 4 .. 7. Among turn j's products a wave asks for turn j + FAR's keys and the values
        // of the turn in front of that, into what all waves have read before turn j's first barrier.
        auto pages_through = [&](auto STEPC) AT_IN {
            constexpr int STEP = decltype(STEPC)::value, FAR = AR_RING / STEP - 1;
            const int turns = (tiles + STEP - 1) / STEP;
            const bool late = wave >= 4;
            int64_t keys[STEP], values[STEP];   // the pages of the turn that is asked for, and of the one before
            int key_at[STEP], value_at[STEP], value_bytes[STEP];
            uint32_t valid = 0;        // whether the pages asked for are there, the last one's bit lowest
#pragma unroll
            for (int g = 0; g < STEP; g++) keys[g] = -1;
            auto plan = [&](int j) AT_IN {    // turn j's keys, turn j - 1's values
#pragma unroll
                for (int g = 0; g < STEP; g++) {
                    const int i = j * STEP + g;
                    values[g] = keys[g];
                    value_bytes[g] = rows_of(i - STEP);
                    value_at[g] = VALUES + ((i - STEP) & (AR_RING - 1)) * TILE;
                    keys[g] = i < tiles ? page_of(i) : -1;
                    key_at[g] = (i & (AR_RING - 1)) * TILE;
                    valid = 2 * valid + (keys[g] >= 0);
                }
            };
            constexpr int PIECES = 2 * STEP * PW;
            auto ask = [&](int n) AT_IN {     // of PIECES, values first
                const int g = n / PW % STEP, c = n % PW;
                if (n < PIECES / 2) copy(V, true, values[g], value_bytes[g], value_at[g], c);
                else copy(K, false, keys[g], TILE, key_at[g], c);
            };
            // a turn's copies among its products, evenly: values beside the values' products, keys beside the keys'
            auto beside_v = [&](int f) AT_IN {
                constexpr int EACH = 8 * NV / PIECES;
                if (f % EACH == EACH / 2) ask(f / EACH);
                if (f >= 4 * NV - KA + 1) kread(f - (4 * NV - KA + 1));
            };
            auto beside_k = [&](int ks) AT_IN {
                constexpr int EACH = 2 * KS / PIECES;
                if (ks % EACH == EACH / 2) ask(PIECES / 2 + ks / EACH);
            };
            auto first_barrier = [&](auto MORE) AT_IN {
                // in front of turn j: this wave's copies of its keys and of the values before landed, and of its values where they are asked for
                // in time (STEP 1: all but turn j + 1's keys and what turn j + 2 asked for)
                constexpr int LATER = STEP == 2 ? 0 : PIECES / 2 + PIECES;
                static_assert(LATER + decltype(MORE)::value < 16, "the low bits of the count");
                __builtin_amdgcn_s_waitcnt(0x0F70 | (LATER + decltype(MORE)::value));
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            };
            auto second_barrier = [&]() AT_IN {
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            };
#pragma unroll
            for (int j = 0; j <= FAR; j++) {
                plan(j);
#pragma unroll
                for (int n = j ? 0 : PIECES / 2; n < PIECES; n++) ask(n);
            }
            first_barrier(std::integral_constant<int, PIECES>{});           // one turn more has been asked for than behind turn 0's products in the loop
            if (late) second_barrier();
            find_k(turn * TILE);
            begin_k();
            products_k([](int) {});          // of a page that is not there: not used
#pragma unroll 1
            for (int j = 0; j < turns; j++) {
                const int i = j * STEP + turn;
                const bool on = i >= lo && i < hi && (valid >> ((FAR + 1) * STEP - 1 - turn) & 1);
                if (late) first_barrier(std::integral_constant<int, 0>{});
                else second_barrier();
                plan(j + 1 + FAR);
                auto then = [&]() AT_IN {
                    if (late) second_barrier();
                    else first_barrier(std::integral_constant<int, 0>{});
                    __builtin_amdgcn_s_setprio(1);
                    find_k(((i + STEP) & (AR_RING - 1)) * TILE);
                };
                if (on) {
                    if (STEP == 1) begin_v(VALUES + (i & (AR_RING - 1)) * TILE);
                    softmax(std::false_type{}, first_key(i));
                    // all of it in front of the barrier: a computation in registers may be moved behind one
                    if constexpr (HQ) asm volatile("" : "+v"(pr[0]), "+v"(pr[1]), "+v"(pr[2]), "+v"(pr[3]), "+v"(l));
                    else asm volatile("" : "+v"(s[0]), "+v"(s[1]), "+v"(l));
                    then();
                    if (STEP == 2) begin_v(VALUES + (i & (AR_RING - 1)) * TILE);
                    products_v(beside_v);
                } else {
                    then();
#pragma unroll
                    for (int n = 0; n < PIECES / 2; n++) ask(n);
                    begin_k();
                }
                products_k(beside_k);
                __builtin_amdgcn_s_setprio(0);
            }
            if (!late) second_barrier();
            __builtin_amdgcn_s_waitcnt(0);   // copies of nothing
        };
        // Infinities and NaN. A product of 0 and infinity, or of a masked p and NaN, is not what the formula has, nor are parts of an
        // infinite query or key. Where a result is not finite the item's pages are taken again, with care: a page that holds something
        // infinite or NaN (keys only matter in parts) key by key in fp32; a score of -infinity is a key that takes no part, an infinite value
        // stays, however small its p is.
        bool odd_q = false;
        auto odd_page = [&]() AT_IN {
            uint32_t odd = 0;
            constexpr uint32_t EXP = ST == 0 ? 0x7f80u : 0x7c00u;
#pragma unroll 1
            for (int i = lane * 16; i < TILE; i += 1024)
#pragma unroll
                for (int u = HQ ? 1 : 0; u < 2; u++) {
                    const at_u4 x = *reinterpret_cast<const at_u4*>(lds + u * VALUES + i);
#pragma unroll
                    for (int e = 0; e < 4; e++) odd |= (uint32_t)((x[e] & EXP) == EXP) | (uint32_t)((x[e] >> 16 & EXP) == EXP);
                }
            return (bool)__any(odd);
        };
        auto slow_page = [&](int k0) AT_IN {
            const float by = a.scale * 1.4426950408889634f;
#pragma unroll 1
            for (int e = 0; e < MLXR_PAGE; e++) {
                const int key = k0 + e;
                if (key > lim1 || key < low0) continue;
                float sc = 0.0f;
#pragma unroll 1
                for (int ks = 0; ks < KS; ks++) {
                    const at_u4 k = *reinterpret_cast<const at_u4*>(lds + e * ROW + 16 * ((2 * ks + h) ^ at_swz_k<D>(e)));
                    float x[8];
                    if constexpr (HQ) {
                        const at_u4 y = gload(reinterpret_cast<const at_u4*>(static_cast<const uint16_t*>(a.q) + q_at + 16 * ks + 8 * h));
#pragma unroll
                        for (int c = 0; c < 8; c++) x[c] = kv_float<ST>((uint16_t)(y[c / 2] >> 16 * (c & 1)));
                    } else {
                        const float4 u = gload4(static_cast<const float*>(a.q) + q_at + 16 * ks + 8 * h), v = gload4(static_cast<const float*>(a.q) + q_at + 16 * ks + 8 * h + 4);
                        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
                    }
#pragma unroll
                    for (int c = 0; c < 8; c++) sc = fmaf(x[c] * by, kv_float<ST>((uint16_t)(k[c / 2] >> 16 * (c & 1))), sc);
                }
                sc = xor32_sum(sc);
                const bool in = key <= lim && key >= low && sc != -INFINITY;
                const float mx = in ? fmaxf(m, sc) : m, c = at_exp2(m - at_safe(mx)), p = in ? at_exp2(sc - at_safe(mx) + UP) : 0.0f;
                m = mx;
                l = l * c + (h == 0 ? p : 0.0f);   // the two lanes' sums are added in the end
#pragma unroll
                for (int n = 0; n < NV; n++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const uint2 v = *reinterpret_cast<const uint2*>(lds + VALUES + e * ROW + 16 * ((4 * n + g) ^ at_swz_v<D>(e)) + 8 * h);
                        const float v4[4] = {kv_float<ST>((uint16_t)v.x), kv_float<ST>((uint16_t)(v.x >> 16)), kv_float<ST>((uint16_t)v.y), kv_float<ST>((uint16_t)(v.y >> 16))};
#pragma unroll
                        for (int d = 0; d < 4; d++) o[n][4 * g + d] = at_times(c, o[n][4 * g + d]) + (in ? at_times(p, v4[d]) : 0.0f);
                    }
            }
        };
        auto clear = [&]() AT_IN {
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int n = 0; n < NV; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[n][e] = 0.0f;
        };
        clear();
        if (two) pages_through(std::integral_constant<int, 2>{});
        else pages_through(std::integral_constant<int, 1>{});
        bool careful = false;
        {
            float odd4[4] = {0.0f * l, 0.0f, 0.0f, 0.0f};   // NaN where one is not finite
#pragma unroll
            for (int n = 0; n < NV; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) odd4[e & 3] = fmaf(0.0f, o[n][e], odd4[e & 3]);
            const float any = (odd4[0] + odd4[1]) + (odd4[2] + odd4[3]);
            bool again = active && any != any;
            if (__builtin_expect(__any(again), 0)) {   // a query that holds NaN has NaN results, whatever the keys are
                bool nan_q = false;
#pragma unroll 1
                for (int d = 0; d < D / 2; d++) {
                    const int64_t at = q_at + D / 2 * h + d;
                    const float x = HQ ? kv_float<ST>(gload(static_cast<const uint16_t*>(a.q) + at)) : gload(static_cast<const float*>(a.q) + at);
                    nan_q |= x != x;
                    odd_q |= !HQ && __builtin_isinf(x * a.scale * 1.4426950408889634f);
                }
                uint64_t nan_rows = __ballot(nan_q);
                nan_rows |= nan_rows >> 32;
                again = again && !((nan_rows >> r) & 1);
                odd_q = __any(odd_q);
            }
            if (lane == 0) sh.odd[wave] = 0;
            if (__any(again) && lane == 0) sh.odd[wave] = 1;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < AR_WV; i++) careful |= sh.odd[i] != 0;
        }
        if (__builtin_expect(careful, 0)) {
            clear();
#pragma unroll 1
            for (int i = 0; i < tiles; i++) {
                const int64_t page = page_of(i);
                const int k0 = first_key(i);
                if (page < 0) continue;
#pragma unroll
                for (int n = 0; n < PW; n++) {
                    copy(K, false, page, TILE, 0, n);
                    copy(V, true, page, rows_of(i), VALUES, n);
                }
                __builtin_amdgcn_s_waitcnt(0);
                __syncthreads();
                if ((!two || (i & 1) == turn) && i >= lo && i < hi) {
                    if (odd_q || odd_page()) slow_page(k0);
                    else {
                        find_k(0);
                        begin_k();
                        products_k([](int) {});
                        softmax(std::true_type{}, k0);
                        begin_v(VALUES);
                        products_v([](int) {});
                    }
                }
                __syncthreads();
            }
        }
        // Where several waves have the same queries (each other's pages; later other runs'), all eight lay down what they have and take eight of a lane's
        // values of 32 queries at a time, added in the order of `way`.
        constexpr int NR = 16 * NV;
        int way = turn, ways = two ? 2 : 1, blk = block;
        l = xor32_sum(l);
        // four dims 32 n + 8 g + 4 h .. of the queries 32 qb + r
        auto result_of = [&](int qb) AT_IN {
            const int fq = f0 + min(32 * qb + r, R - 1), tq = fq / G;
            return (int64_t)(sq.row + tq) * a.out_stride + (int64_t)(kvh * G + fq - tq * G) * D + 4 * h;
        };
        auto put = [&](int64_t to, int n, int g, float inv, float x0, float x1, float x2, float x3) AT_IN {
            float y[8] = {x0 * inv, x1 * inv, x2 * inv, x3 * inv, 0.0f, 0.0f, 0.0f, 0.0f};
            if (inv == 0.0f)   // no key: nothing times 0
#pragma unroll
                for (int d = 0; d < 4; d++) y[d] = 0.0f;
            if constexpr (HQ) {
                at_u4 y4[1];
                at_split<ST, true>(y, y4);
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + to + 32 * n + 8 * g) = uint2{y4[0][0], y4[0][1]};
            } else *reinterpret_cast<float4*>(static_cast<float*>(a.out) + to + 32 * n + 8 * g) = float4{y[0], y[1], y[2], y[3]};
        };
        // the runs that hold the item, from the first page's to the last one's
        const bool whole = tiles == pages;
        const int w0 = whole ? 0 : at_one((int)at_div(pre, per));
        const int parts = whole ? 1 : at_one((int)at_div(pre + places - 1, per)) - w0 + 1, first_slot = pre == (uint64_t)w0 * per ? 0 : 1;
        // a run has two parts at most: of what it begins with, and of an item that starts behind that
        auto part_of = [&](int run, int qb) AT_IN {
            return wk.part + (size_t)(2 * run + (run == w0 ? first_slot : 0)) * at_part_floats(D) + (size_t)qb * (D / 4 + 1) * 128 + 2 * lane;
        };
        // How parts are joined: a wave has 32 queries and every ways-th part. Above AR_GROUP a wave, the last workgroup of each
        // group of parts joins these where the group's first part was, and the last of those the groups.
        const int join_ways = blocks > 4 ? 1 : blocks > 2 ? 2 : blocks > 1 ? 4 : 8, group = AR_GROUP * join_ways;
        const bool grouped = parts > group;
        const int g0 = grouped ? w0 + (w - w0) / group * group : w0;   // the first run of this one's group
        int to_run = w;
#pragma unroll 1
        for (int pass = 0;; pass++) {
            const bool out = whole || pass == (grouped ? 2 : 1), here = blk < blocks;
            if (ways > 1) {
                const int of = AR_WV / ways;   // blocks' places
                float* all = reinterpret_cast<float*>(lds) + lane;
                if (here) {
                    float* mine = all + (way * of + blk) * NR * 64;
#pragma unroll
                    for (int n = 0; n < NV; n++)
#pragma unroll
                        for (int e = 0; e < 16; e++) mine[(16 * n + e) * 64] = o[n][e];
                    sh.m[way * of + blk][lane] = m;
                    sh.l[way * of + blk][lane] = l;
                }
                __syncthreads();
#pragma unroll 1
                for (int id = wave; id < blocks * (NR / 8); id += AR_WV) {
                    const int qb = id % blocks, pc = id / blocks;
                    float M = -INFINITY, L = 0.0f, x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                    for (int k = 0; k < ways; k++) M = fmaxf(M, sh.m[k * of + qb][lane]);
#pragma unroll 2
                    for (int k = 0; k < ways; k++) {
                        const float c = at_exp2(sh.m[k * of + qb][lane] - at_safe(M));   // a part of NaN counts, whatever its maximum: 0 times NaN is NaN
                        const float* v = all + ((k * of + qb) * NR + 8 * pc) * 64;
                        L += c * sh.l[k * of + qb][lane];
#pragma unroll
                        for (int e = 0; e < 8; e++) x[e] += at_times(c, v[e * 64]);
                    }
                    if (out) {
                        if (32 * qb + r < R) {
                            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                            const int64_t to = result_of(qb);
                            put(to, pc >> 1, 2 * (pc & 1), inv, x[0], x[1], x[2], x[3]);
                            put(to, pc >> 1, 2 * (pc & 1) + 1, inv, x[4], x[5], x[6], x[7]);
                        }
                    } else {
                        float* to = part_of(to_run, qb);
#pragma unroll
                        for (int e = 0; e < 4; e++) at_store2(to + (4 * pc + e) * 128, x[2 * e], x[2 * e + 1]);
                        if (pc == 0) at_store2(to + D / 4 * 128, M, L);
                    }
                }
            } else if (here) {
                if (out) {
                    if (32 * blk + r < R) {
                        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                        const int64_t to = result_of(blk);
#pragma unroll
                        for (int n = 0; n < NV; n++)
#pragma unroll
                            for (int g = 0; g < 4; g++) put(to, n, g, inv, o[n][4 * g], o[n][4 * g + 1], o[n][4 * g + 2], o[n][4 * g + 3]);
                    }
                } else {
                    float* to = part_of(to_run, blk);
#pragma unroll
                    for (int n = 0; n < NV; n++)
#pragma unroll
                        for (int e = 0; e < 8; e++) at_store2(to + (8 * n + e) * 128, o[n][2 * e], o[n][2 * e + 1]);
                    at_store2(to + D / 4 * 128, m, l);
                }
            }
            if (out) break;
            parts_stored();
            const bool last_join = pass == 1 || !grouped;   // of groups, or of all parts
            unsigned* count = wk.count + (last_join ? w0 : g0 == w0 ? AR_MAXW + w0 : 2 * AR_MAXW + g0);
            const int n = !grouped ? parts : pass ? (parts + group - 1) / group : min(group, parts - (g0 - w0));
            if (tid == 0) sh.last = part_last(count, n);
            __syncthreads();
            if (!sh.last) break;
            const int from = last_join ? w0 : g0, stride = pass ? group : 1;
            ways = join_ways;
            blk = wave % (AR_WV / ways);
            way = wave / (AR_WV / ways);
            clear();
#pragma unroll 1
            for (int k = way; k < n && blk < blocks; k += ways) {
                const float* p = part_of(from + k * stride, blk);
                float2 x[NV][8];
                const float2 st = at_load2(p + D / 4 * 128);
#pragma unroll
                for (int n = 0; n < NV; n++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[n][e] = at_load2(p + (8 * n + e) * 128);
                const float M = fmaxf(m, st.x), c = at_exp2(m - at_safe(M)), c2 = at_exp2(st.x - at_safe(M));
                m = M;
                l = c * l + c2 * st.y;
#pragma unroll
                for (int n = 0; n < NV; n++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        o[n][2 * e] = at_times(c, o[n][2 * e]) + at_times(c2, x[n][e].x);
                        o[n][2 * e + 1] = at_times(c, o[n][2 * e + 1]) + at_times(c2, x[n][e].y);
                    }
            }
            if (tid == 0) part_rearm(count);
            to_run = g0;
        }
        if (!ahead()) return;
        lds_barrier();     // the LDS is written again; results may still be on their way
    }
}

static size_t at_layout(const PagedKV& kv, int nH, int rows, void* base, AtWork& wk) {
    const int64_t G = nH / kv.nKV, items = ((int64_t)rows * G + AR_M - 1) / AR_M + kv.B, places = (kv.max_len + MLXR_PAGE - 1) / MLXR_PAGE + 4 + AR_GAP;
    const double runs = (double)items * (double)kv.nKV * (double)places / AR_MINPER + 1.0;
    wk.W = runs < AR_MAXW ? (int)runs : AR_MAXW;
    uint8_t* p = static_cast<uint8_t*>(base);
    wk.count = reinterpret_cast<unsigned*>(p);   // first: where it is for every size
    wk.part = reinterpret_cast<float*>(p + AR_COUNTS * sizeof(unsigned));
    return AR_COUNTS * sizeof(unsigned) + (size_t)2 * wk.W * at_part_floats(kv.D) * sizeof(float);
}

size_t paged_attention_rows_work(const PagedKV& kv, int nH, int rows, int q_type) {
    AtWork wk;
    return at_layout(kv, nH, rows, nullptr, wk);
}

hipError_t launch_paged_attention_rows(const AttnRowsArgs& a, hipStream_t s) {
    AtWork wk;
    at_layout(a.kv, a.nH, a.rows, a.work, wk);
    // more LDS than a launch has by itself is asked for each time: it holds for the current device only
#define AT_GO(ST, D, HQ) do { \
        constexpr int LDS = 2 * AR_RING * 64 * D * 2 + (int)sizeof(AtShared); \
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_rows_kernel<ST, D, HQ>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS)) return e; \
        hipLaunchKernelGGL((attn_rows_kernel<ST, D, HQ>), dim3(wk.W), dim3(AR_TH), LDS, s, a, wk); \
    } while (0)
#define AT_D(ST, HQ) do { if (a.kv.D == 64) AT_GO(ST, 64, HQ); else AT_GO(ST, 128, HQ); } while (0)
    if (a.kv.st == 0) { if (a.q_type) AT_D(0, true); else AT_D(0, false); }
    else { if (a.q_type) AT_D(1, true); else AT_D(1, false); }
#undef AT_D
#undef AT_GO
    return hipGetLastError();
}

}  // namespace mlxr
