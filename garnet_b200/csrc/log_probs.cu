// Log probabilities of given tokens, their ranks, entropies and the top alternatives of rows of logits, in one pass over the logits.
//
//   y = x log2(e) / T, a reference r near the row's maximum of y, S = sum 2^(y - r), W = sum 2^(y - r) (y - r):
//   log p(t) = ln 2 ((y_t - r) - log2 S),  H = ln 2 (log2 S - W / S),  rank = 1 + #{x > x_t}.
//
// A row is cut into 1, 2, 4 or 8 parts, one CTA each, that meet through distributed shared memory.  The warps of a CTA take blocks of 2 KB in
// turn: four 16-byte loads per lane, the block's maximum (NaN wins) by packed maxima and one warp reduction, which also says whether the
// warp's reference has to grow (by more than 2^8, so that this is rare: S and W are rescaled then), then per value one conversion,
// half of a packed multiply-add, one exponential and half of two packed additions; the rank is counted in packed 16-bit numbers,
// in blocks whose maximum is above the target's logit or NaN.
// The block maxima stay in shared memory.  The top_k-th largest of the threads' own maxima is no larger than the top_k-th
// largest logit, so that only blocks that reach it - few more than top_k - are read a second time (from L2) for the alternatives: every
// value that reaches it becomes a candidate, (value, lowest index) as one 64-bit number, and the candidates larger than it say its place.
// Where too many are equal for that, every warp keeps a sorted list across its lanes.
// Everything is added in an order that depends on sizes only.  A row whose maximum lies beyond +-2^100 (a mask of the type's lowest
// value over all of it) or, in y, beyond +-2^20 (a temperature next to zero) is summed again, value by value, against its maximum.
//
// Bound: HBM in principle (every logit once).  For 16-bit logits the exponentials, 16 per clock and SM, take nearly as long: 67 us of the
// unit at 1965 MHz for 2048 rows of 151936 bf16, beside 95 us of the measured bandwidth.  That call takes 127 us (0.75 of the bandwidth; a
// profiled launch of 126 us at its own clock counted the unit, with all that goes through it, busy for 64 %), fp16 130 us (its values
// are converted and bounded one by one), 1024 rows of fp32 108 us (0.88).  One row of 151936 and 64 rows of 32003 fp32 take 11.5 us each,
// the latency of launch, loads, two meetings of the cluster and the alternatives' order.
#include <cfloat>
#include <cmath>
#include <cooperative_groups.h>
#include <cstdint>

#include "tc_common.cuh"

namespace gb200 {

namespace {

namespace cg = cooperative_groups;

constexpr int kLpMaxTop = 32, kLpMaxParts = 8;
constexpr int kLpVecs = 4, kLpBlockBytes = kLpVecs * 32 * 16;
constexpr int kLpEntries = 128;   // block maxima that a warp keeps; more blocks share them
constexpr float kLpHuge = 1.2676506002282294e30f;   // 2^100
constexpr float kLpFar = 1048576.f;                 // 2^20: the reference, an fp32 number, is then within 2^-4 of the y that it stands for

struct LogProbs {
    const void* logits;
    long long stride;
    const int* targets;
    float* log_probs;
    int* ranks;
    float* entropy;
    float* top_log_probs;
    int* top_ids;
    int vocab, top_k, parts;
    float scale;   // 1 / temperature
};

// Sixteen bytes of logits: packed maxima, and their values.
template <typename T>
struct LpVec;
template <>
struct LpVec<float> {
    static constexpr int n = 4;
    __device__ static float top(const uint4& v) { return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w))); }
    __device__ static float max_nan(float a, float b)
    {
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
        return r;
    }
    __device__ static void values(const uint4& v, float (&x)[4]) { x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w); }
    // values with -inf and what lies below -2^100 as -2^100
    __device__ static void finite(const uint4& v, float (&x)[4])
    {
        values(v, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = fmaxf(x[i], -kLpHuge);
    }
    struct Count {
        int n = 0;
        float than;
        __device__ explicit Count(float t) : than(t) {}
        __device__ void add(const uint4& v)
        {
            float x[4];
            values(v, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) n += x[i] > than;
        }
        __device__ void settle() {}
    };
};
template <typename T2>
struct LpPairs {
    static constexpr int n = 8;
    __device__ static T2 pair(uint32_t w) { return *reinterpret_cast<const T2*>(&w); }
    __device__ static uint32_t word(T2 p) { return *reinterpret_cast<const uint32_t*>(&p); }
    __device__ static float low(T2 p);
    __device__ static float high(T2 p);
    __device__ static T2 same(float x);
    __device__ static float top(const uint4& v)
    {
        const T2 m = __hmax2_nan(__hmax2_nan(pair(v.x), pair(v.y)), __hmax2_nan(pair(v.z), pair(v.w)));
        const float a = low(m), b = high(m);
        return LpVec<float>::max_nan(a, b);
    }
    __device__ static void values(const uint4& v, float (&x)[8])
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = low(pair(w[i])), x[2 * i + 1] = high(pair(w[i]));
    }
    // values with -inf and what lies below -2^100 as -2^100
    __device__ static void finite(const uint4& v, float (&x)[8]);
    // counted as 16-bit floating-point numbers: exact up to 256, and a vector adds at most 4 to either half
    struct Count {
        int n = 0;
        T2 than, halves;
        __device__ explicit Count(float t) : than(same(t)), halves(same(0.f)) {}
        __device__ void add(const uint4& v)
        {
            halves = __hadd2(halves, __hadd2(__hadd2(__hgt2(pair(v.x), than), __hgt2(pair(v.y), than)), __hadd2(__hgt2(pair(v.z), than), __hgt2(pair(v.w), than))));
        }
        __device__ void settle()
        {
            n += int(low(halves)) + int(high(halves));
            halves = same(0.f);
        }
    };
};
template <> __device__ __forceinline__ float LpPairs<__nv_bfloat162>::low(__nv_bfloat162 p) { return __uint_as_float(word(p) << 16); }
template <> __device__ __forceinline__ float LpPairs<__nv_bfloat162>::high(__nv_bfloat162 p) { return __uint_as_float(word(p) & 0xffff0000u); }
template <> __device__ __forceinline__ __nv_bfloat162 LpPairs<__nv_bfloat162>::same(float x) { return __float2bfloat162_rn(x); }
template <> __device__ __forceinline__ float LpPairs<__half2>::low(__half2 p) { return __low2float(p); }
template <> __device__ __forceinline__ float LpPairs<__half2>::high(__half2 p) { return __high2float(p); }
template <> __device__ __forceinline__ __half2 LpPairs<__half2>::same(float x) { return __float2half2_rn(x); }
template <>
__device__ __forceinline__ void LpPairs<__nv_bfloat162>::finite(const uint4& v, float (&x)[8])
{
    const __nv_bfloat162 least = same(-kLpHuge);
    values(make_uint4(word(__hmax2(pair(v.x), least)), word(__hmax2(pair(v.y), least)), word(__hmax2(pair(v.z), least)), word(__hmax2(pair(v.w), least))), x);
}
template <>
__device__ __forceinline__ void LpPairs<__half2>::finite(const uint4& v, float (&x)[8])   // fp16 has no -2^100
{
    values(v, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaxf(x[i], -kLpHuge);
}
template <>
struct LpVec<__nv_bfloat16> : LpPairs<__nv_bfloat162> {};
template <>
struct LpVec<__half> : LpPairs<__half2> {};

__device__ __forceinline__ float lp_value(const float* x, long long i) { return x[i]; }
__device__ __forceinline__ float lp_value(const __nv_bfloat16* x, long long i) { return __bfloat162float(x[i]); }
__device__ __forceinline__ float lp_value(const __half* x, long long i) { return __half2float(x[i]); }

// Larger for larger values, the same for +0 and -0; 0 for NaN.
__device__ __forceinline__ uint32_t lp_key(float x)
{
    if (isnan(x)) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// A value and its place: larger values first, then lower places.
__device__ __forceinline__ unsigned long long lp_entry(float x, long long i) { return (static_cast<unsigned long long>(lp_key(x)) << 32) | (0xffffffffu - uint32_t(i)); }
__device__ __forceinline__ float lp_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The values of a part of a row: S and W against `ref`, the largest value, how many are above the target, and whether there is a NaN.
struct LpSum {
    float ref, s, w, top;
    int above, nan;
};
__device__ __forceinline__ LpSum lp_join(const LpSum& a, const LpSum& b)
{
    LpSum r;
    r.ref = fmaxf(a.ref, b.ref);
    const float da = a.ref - r.ref, db = b.ref - r.ref, fa = ex2(da), fb = ex2(db);
    r.s = fa * a.s + fb * b.s;
    r.w = (fa > 0.f ? fa * (a.w + da * a.s) : 0.f) + (fb > 0.f ? fb * (b.w + db * b.s) : 0.f);
    r.top = fmaxf(a.top, b.top);
    r.above = a.above + b.above, r.nan = a.nan | b.nan;
    return r;
}

// The same over 8 lanes' sums, in a fixed order; every lane of the warp that asks gets the result.
__device__ __forceinline__ LpSum lp_join_lanes(LpSum v)
{
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        LpSum o;
        o.ref = __shfl_xor_sync(0xffffffffu, v.ref, d), o.s = __shfl_xor_sync(0xffffffffu, v.s, d), o.w = __shfl_xor_sync(0xffffffffu, v.w, d);
        o.top = __shfl_xor_sync(0xffffffffu, v.top, d);
        o.above = __shfl_xor_sync(0xffffffffu, v.above, d), o.nan = __shfl_xor_sync(0xffffffffu, v.nan, d);
        v = (threadIdx.x & d) ? lp_join(o, v) : lp_join(v, o);   // the lower lanes' sum first
    }
    return v;
}

// A part's results in shared memory, read by the first of its cluster.
struct LpPart {
    LpSum sum;
    unsigned long long top[kLpMaxTop];
};
template <int kThreads>
struct LpShared {
    static constexpr int warps = kThreads / 32, candidates = kThreads;
    LpPart part;
    LpSum sums[8];
    int found;                                               // candidates in `keys`, or more than there is room for
    unsigned long long keys[kLpMaxParts * kLpMaxTop];        // candidates in no order; or lists of 32, one per warp; or the parts' lists
    unsigned long long out[kLpMaxTop];
    alignas(16) uint32_t lane_tops[kThreads];                // as keys
    uint32_t bound;
    float maxima[kLpEntries * warps];                        // [entry][warp]
    static_assert(warps <= 8 && candidates <= kLpMaxParts * kLpMaxTop, "room for sums and keys");
};

// The largest `most` of `count` different keys, up to one per thread, to out[0 ..] in descending order; 0 where there are fewer.
__device__ __forceinline__ void lp_rank(const unsigned long long* keys, int count, int most, unsigned long long* out)
{
    if (int(threadIdx.x) >= count && int(threadIdx.x) < most) out[threadIdx.x] = 0;
    if (int(threadIdx.x & ~31u) >= count) return;
    const unsigned long long key = int(threadIdx.x) < count ? keys[threadIdx.x] : 0;
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < count; ++i) place += keys[i] > key;
    if (key && place < most) out[place] = key;
}

// The same of `lists` descending lists of 32, which 0 may follow: a key's place is its place in its list and the numbers of larger keys in
// the others.  Out's 32 entries are 0 before.
template <int kThreads>
__device__ __forceinline__ void lp_merge(const unsigned long long* keys, int lists, int most, unsigned long long* out)
{
    for (int i = threadIdx.x; i < lists * 32; i += kThreads) {
        const unsigned long long key = keys[i];
        int larger[kLpMaxParts] = {};
#pragma unroll
        for (int step = 16; step; step >>= 1)
#pragma unroll
            for (int l = 0; l < kLpMaxParts; ++l)
                if (l < lists && keys[l * 32 + larger[l] + step - 1] > key) larger[l] += step;
        int place = 0;
#pragma unroll
        for (int l = 0; l < kLpMaxParts; ++l) place += l < lists ? larger[l] + (larger[l] == 31 && keys[l * 32 + 31] > key) : 0;
        if (key && place < most) out[place] = key;
    }
}

template <typename T, int kLpThreads>
__global__ void __launch_bounds__(kLpThreads, 1024 / kLpThreads) log_probs_kernel(const LogProbs p)
{
    using Vec = LpVec<T>;
    constexpr int kBlock = kLpBlockBytes / int(sizeof(T)), kLpWarps = kLpThreads / 32, kLpCandidates = LpShared<kLpThreads>::candidates;
    __shared__ LpShared<kLpThreads> sh;
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = int(blockIdx.x) % p.parts;
    const size_t r = blockIdx.x / unsigned(p.parts);
    const T* row = static_cast<const T*>(p.logits) + r * p.stride;
    // whole blocks from the row's first 16-byte boundary on; the first part has the values before them, the last part those behind
    const int head = min(p.vocab, int((16 - (reinterpret_cast<uintptr_t>(row) & 15)) % 16 / sizeof(T)));
    const int blocks = (p.vocab - head) / kBlock, tail = head + blocks * kBlock;
    const int block0 = int((long long)part * blocks / p.parts), block1 = int((long long)(part + 1) * blocks / p.parts);
    const int loose0 = part == 0 ? head : 0, loose = loose0 + (part + 1 == p.parts ? p.vocab - tail : 0);   // single values of this part
    const auto loose_at = [&](int i) { return i < loose0 ? i : tail + i - loose0; };
    const uint4* row_blocks = reinterpret_cast<const uint4*>(row + head) + lane;
    const auto block_at = [&](int b) { return row_blocks + (long long)b * (kLpBlockBytes / 16); };
    const float scale = p.scale * 1.4426950408889634f;

    const int rounds = (block1 - block0 + kLpWarps - 1) / kLpWarps;          // blocks of a warp
    if (rounds > 1 && rounds <= 8) {
        // a short part: all of it is asked for at once, sixteen lanes per block of 2 KB
        for (int i = lane >> 4; i < rounds; i += 2)
            if (block0 + i * kLpWarps + warp < block1)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(row + head) + (long long)(block0 + i * kLpWarps + warp) * kLpBlockBytes + (lane & 15) * 128));
    }
    const int shared_by = max(1, (rounds + kLpEntries - 1) / kLpEntries), entries = (rounds + shared_by - 1) / shared_by;
    float ref = -kLpHuge * scale, entry = -INFINITY, top = -INFINITY, lane_top = -INFINITY;   // ref: in powers of two
    int nan = 0;
    uint64_t s2[2] = {0, 0}, w2[2] = {0, 0};
    const uint64_t scale2 = f32x2(scale, scale);
    uint4 v[kLpVecs];
    int b = block0 + warp;
    const uint4* from = block_at(b);
    if (b < block1) {   // asked for before the two dependent loads of the target's logit
#pragma unroll
        for (int k = 0; k < kLpVecs; ++k) v[k] = __ldg(from + 32 * k);
    }
    const int target = p.targets ? p.targets[r] : -1;
    const bool given = target >= 0 && target < p.vocab;
    const float x_t = given ? lp_value(row, target) : INFINITY;
    typename Vec::Count count(x_t);
    // the warp's reference grows to its new maximum m (a NaN is noted)
    const auto grow = [&](float m) {
        const float y = m * scale;
        if (y <= ref + 8.f) return;
        if (isnan(m)) {
            nan = 1;
        } else if (m <= kLpHuge) {   // beyond that the row is summed again
            const float d = ref - y, f = ex2(d);
            const uint64_t f2 = f32x2(f, f), d2 = f32x2(fmaxf(d, -1e30f), fmaxf(d, -1e30f));
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                w2[k] = mul2(f2, fma2(d2, s2[k], w2[k]));
                s2[k] = mul2(f2, s2[k]);
            }
            ref = y;
        }
    };
    float* to = sh.maxima + warp;
    int left = shared_by, unsettled = 256 / (2 * Vec::n * kLpVecs / 4);
#pragma unroll 1
    for (; b < block1; b += kLpWarps) {
        float m = Vec::top(v[0]);
#pragma unroll
        for (int k = 1; k < kLpVecs; ++k) m = LpVec<float>::max_nan(m, Vec::top(v[k]));
        lane_top = fmaxf(lane_top, m);   // a NaN loses
        asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(m));
        grow(m);
        if (!(m <= x_t)) {   // else none of the block is larger than the target's; beside a NaN there may be larger ones
#pragma unroll
            for (int k = 0; k < kLpVecs; ++k) count.add(v[k]);
        }
        const uint64_t minus2 = f32x2(-ref, -ref);
        if (b + kLpWarps < block1) from += kLpWarps * (kLpBlockBytes / 16);   // the last block is asked for twice
#pragma unroll
        for (int k = 0; k < kLpVecs; ++k) {
            float x[Vec::n];
            Vec::finite(v[k], x);
            v[k] = __ldg(from + 32 * k);
#pragma unroll
            for (int e = 0; e < Vec::n; e += 2) {
                const uint64_t d = fma2(f32x2(x[e], x[e + 1]), scale2, minus2);
                float a, c;
                f32x2_split(d, a, c);
                const uint64_t p2 = f32x2(ex2(a), ex2(c));
                s2[(e >> 1) & 1] = add2(s2[(e >> 1) & 1], p2);
                w2[(e >> 1) & 1] = fma2(p2, d, w2[(e >> 1) & 1]);
            }
        }
        if (--unsettled == 0) {
            count.settle();
            unsettled = 256 / (2 * Vec::n * kLpVecs / 4);
        }
        entry = LpVec<float>::max_nan(entry, m);   // a block with a NaN counts as one that may hold alternatives
        top = fmaxf(top, m);
        if (--left == 0) {
            if (lane == 0) *to = entry;
            to += kLpWarps;
            left = shared_by, entry = -INFINITY;
        }
    }
    if (lane == 0 && to < sh.maxima + entries * kLpWarps) *to = entry;
    for (int i0 = warp * 32; i0 < loose; i0 += kLpThreads) {
        const float x = i0 + lane < loose ? lp_value(row, loose_at(i0 + lane)) : -INFINITY;
        float m = x;
        lane_top = fmaxf(lane_top, x);
        asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(m));
        grow(m);
        top = fmaxf(top, m);
        count.n += x > x_t;
        const float d = fmaf(fmaxf(x, -kLpHuge), scale, -ref), e = i0 + lane < loose ? ex2(d) : 0.f;
        s2[0] = add2(s2[0], f32x2(e, 0.f));
        w2[0] = fma2(f32x2(e, 0.f), f32x2(d, 0.f), w2[0]);
    }
    count.settle();
    if (p.top_k) sh.lane_tops[threadIdx.x] = lp_key(lane_top);
    {
        LpSum mine;
        float a, b, c, d;
        f32x2_split(add2(s2[0], s2[1]), a, b);
        f32x2_split(add2(w2[0], w2[1]), c, d);
        mine.s = a + b, mine.w = c + d;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            mine.s += __shfl_xor_sync(0xffffffffu, mine.s, o);
            mine.w += __shfl_xor_sync(0xffffffffu, mine.w, o);
        }
        mine.ref = ref, mine.top = top, mine.nan = nan;
        mine.above = __reduce_add_sync(0xffffffffu, count.n);
        if (lane == 0) sh.sums[warp] = mine;
    }
    if (threadIdx.x == 0) sh.found = 0, sh.bound = 0xffffffffu;
    __syncthreads();

    // ---- alternatives of the part
    if (p.top_k) {
        // the top_k-th largest of the threads' maxima
        const uint32_t mine = lp_key(lane_top);
        int larger = 0;
#pragma unroll 8
        for (int i = 0; i < kLpThreads; i += 4) {
            const uint4 o = *reinterpret_cast<const uint4*>(&sh.lane_tops[i]);
            larger += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
        }
        if (larger < p.top_k) atomicMin(&sh.bound, mine);
        __syncthreads();
        const float bound = sh.bound ? lp_unkey(sh.bound) : -INFINITY;
        // what reaches the bound, in any order
        const auto every_block = [&](auto&& take) {
            for (int e = 0; e < entries; ++e) {
                if (sh.maxima[e * kLpWarps + warp] < bound) continue;   // not for NaN
                for (int i = e * shared_by; i < min(rounds, (e + 1) * shared_by); ++i) {
                    const int b = block0 + i * kLpWarps + warp;
                    if (b >= block1) break;
#pragma unroll
                    for (int k = 0; k < kLpVecs; ++k) v[k] = __ldg(block_at(b) + 32 * k);
#pragma unroll
                    for (int k = 0; k < kLpVecs; ++k) take(v[k], head + b * kBlock + (k * 32 + lane) * Vec::n);
                }
            }
        };
        const auto candidate = [&](float x, int i) {
            const int to = atomicAdd(&sh.found, 1);
            if (to < kLpCandidates) sh.keys[to] = lp_entry(x, i);
        };
        every_block([&](const uint4& vec, int at) {
            float x[Vec::n];
            Vec::values(vec, x);
            uint32_t hits = 0;
#pragma unroll
            for (int n = 0; n < Vec::n; ++n) hits |= x[n] >= bound ? 1u << n : 0u;
            for (; hits; hits &= hits - 1) {   // seldom more than one lane's
                const int i = at + __ffs(hits) - 1;
                candidate(lp_value(row, i), i);
            }
        });
        for (int i = threadIdx.x; i < loose; i += kLpThreads)
            if (lp_value(row, loose_at(i)) >= bound) candidate(lp_value(row, loose_at(i)), loose_at(i));
        __syncthreads();
        const int found = sh.found;
        if (found > kLpCandidates) {
            // many equal values: every warp keeps a sorted list of 32 across its lanes instead
            __syncthreads();
            unsigned long long list = 0, least = 0;   // the lane's entry; the top_k-th
            const auto keep = [&](float x, int i) {
                const unsigned long long key = x >= bound ? lp_entry(x, i) : 0;
                for (uint32_t todo = __ballot_sync(0xffffffffu, key > least); todo; todo &= todo - 1) {
                    const unsigned long long in = __shfl_sync(0xffffffffu, key, __ffs(todo) - 1);
                    if (in <= least) continue;
                    const int place = __popc(__ballot_sync(0xffffffffu, list > in));
                    const unsigned long long before = __shfl_up_sync(0xffffffffu, list, 1);
                    list = lane < place ? list : lane == place ? in : before;
                    least = __shfl_sync(0xffffffffu, list, p.top_k - 1);
                }
            };
            every_block([&](const uint4& vec, int at) {
                if (!__any_sync(0xffffffffu, !(Vec::top(vec) < bound))) return;
                float x[Vec::n];
                Vec::values(vec, x);
#pragma unroll 1
                for (int n = 0; n < Vec::n; ++n) {
                    float mine = x[0];
#pragma unroll
                    for (int t = 1; t < Vec::n; ++t) mine = n == t ? x[t] : mine;
                    keep(mine, at + n);
                }
            });
            for (int i0 = warp * 32; i0 < loose; i0 += kLpThreads) {
                const bool there = i0 + lane < loose;
                const int i = there ? loose_at(i0 + lane) : 0;
                keep(there ? lp_value(row, i) : NAN, i);
            }
            sh.keys[threadIdx.x] = list;
            if (threadIdx.x < kLpMaxTop) sh.part.top[threadIdx.x] = 0;
            __syncthreads();
            lp_merge<kLpThreads>(sh.keys, kLpWarps, p.top_k, sh.part.top);
        } else {
            lp_rank(sh.keys, found, p.top_k, sh.part.top);
        }
    }
    if (warp == kLpWarps - 1) {
        const LpSum all = lp_join_lanes((lane & 7) < kLpWarps ? sh.sums[lane & 7] : LpSum{-kLpHuge, 0.f, 0.f, -INFINITY, 0, 0});
        if (lane == 0) sh.part.sum = all;
    }

    // ---- the parts of the row
    cg::cluster_group cluster = cg::this_cluster();
    if (p.parts > 1) cluster.sync();
    else __syncthreads();
    const auto part_of = [&](int c) -> const LpPart& { return p.parts > 1 ? *cluster.map_shared_rank(&sh.part, c) : sh.part; };
    const auto all_parts = [&] {   // a lane asks for each part's sum; lanes without a part have a sum of nothing
        LpSum v{-kLpHuge, 0.f, 0.f, -INFINITY, 0, 0};
        if ((lane & 7) < p.parts) v = part_of(lane & 7).sum;
        return p.parts > 1 ? lp_join_lanes(v) : sh.part.sum;
    };
    LpSum all = all_parts();
    const bool empty = all.top == -INFINITY && !all.nan;   // a row of -inf
    const bool huge = !all.nan && !empty && !(fabsf(all.top) <= kLpHuge && fabsf(all.top) * scale <= kLpFar);
    if (huge) {
        // summed again against the maximum, value by value
        if (p.parts > 1) cluster.sync();   // the others have read this part's sums
        else __syncthreads();
        float s = 0.f, w = 0.f;
        const auto add = [&](int i) {
            const float d = (lp_value(row, i) - all.top) * scale, e = ex2(d);
            s += e;
            w += e > 0.f ? e * d : 0.f;   // inf - inf is NaN, and s with it
        };
        for (int i = block0 * kBlock + int(threadIdx.x); i < block1 * kBlock; i += kLpThreads) add(head + i);
        for (int i = threadIdx.x; i < loose; i += kLpThreads) add(loose_at(i));
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            w += __shfl_xor_sync(0xffffffffu, w, o);
        }
        if (lane == 0) sh.sums[warp].s = s, sh.sums[warp].w = w;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int k = 1; k < kLpWarps; ++k) s += sh.sums[k].s, w += sh.sums[k].w;
            sh.part.sum.s = s, sh.part.sum.w = w, sh.part.sum.ref = 0.f;   // all against the same maximum
        }
        if (p.parts > 1) cluster.sync();
        else __syncthreads();
        const LpSum again = all_parts();
        all.s = again.s, all.w = again.w;
    }
    if (part == 0) {
        const float log2_s = log2f(all.s);
        constexpr float kLn2 = 0.6931471805599453f;
        const auto log_prob = [&](float x) -> float {
            if (all.nan || isnan(all.s)) return NAN;
            if (empty || x == -INFINITY) return -INFINITY;
            // rounding may leave a sole value's a little above 0
            if (huge || x < -kLpHuge) return fminf(0.f, (x - all.top) * p.scale - log2_s * kLn2);
            return fminf(0.f, (fmaf(x, scale, -all.ref) - log2_s) * kLn2);
        };
        if (threadIdx.x == 0) {
            if (p.targets) {
                p.log_probs[r] = given ? log_prob(x_t) : 0.f;
                p.ranks[r] = given ? all.above + 1 : 0;
            }
            if (p.entropy) p.entropy[r] = all.nan || isnan(all.s) ? NAN : empty ? 0.f : fmaxf(0.f, (log2_s - all.w / all.s) * kLn2);
        }
        if (p.top_k) {
            const unsigned long long* result = sh.part.top;
            if (p.parts > 1) {
                // the candidates' place is free: every warp of this CTA has come through the barrier above
                if (warp == 0) sh.out[lane] = 0;
                for (int c = warp; c < p.parts; c += kLpWarps) sh.keys[c * 32 + lane] = lane < p.top_k ? part_of(c).top[lane] : 0;
                __syncthreads();
                lp_merge<kLpThreads>(sh.keys, p.parts, p.top_k, sh.out);
                __syncthreads();
                result = sh.out;
            }
            if (int(threadIdx.x) < p.top_k) {
                const unsigned long long key = result[threadIdx.x];
                p.top_ids[r * p.top_k + threadIdx.x] = key ? int(0xffffffffu - uint32_t(key)) : -1;
                p.top_log_probs[r * p.top_k + threadIdx.x] = key ? log_prob(lp_unkey(uint32_t(key >> 32))) : NAN;
            }
        }
    }
    if (p.parts > 1) cluster.sync();   // the first part may still read this one
}

template <int kThreads>
auto lp_kernel(int dtype)
{
    return dtype == GARNET_B200_BF16 ? log_probs_kernel<__nv_bfloat16, kThreads>
           : dtype == GARNET_B200_FP16 ? log_probs_kernel<__half, kThreads> : log_probs_kernel<float, kThreads>;
}

}  // namespace

}  // namespace gb200

using namespace gb200;

extern "C" {

int garnet_b200_log_probs(const void* d_logits, int dtype, int64_t row_stride, const int* d_targets, int rows, int vocab, int top_k,
                          float temperature, float* d_log_probs, int* d_ranks, float* d_entropy, float* d_top_log_probs, int* d_top_ids,
                          unsigned flags, void* stream)
{
    if (!d_logits || rows <= 0 || vocab <= 0 || row_stride < vocab) return fail(GARNET_B200_INVALID_VALUE, "log_probs: bad argument");
    if (dtype != GARNET_B200_BF16 && dtype != GARNET_B200_FP16 && dtype != GARNET_B200_FP32)
        return fail(GARNET_B200_INVALID_VALUE, "log_probs: unknown dtype %d", dtype);
    if (reinterpret_cast<uintptr_t>(d_logits) & (dtype == GARNET_B200_FP32 ? 3 : 1))
        return fail(GARNET_B200_INVALID_VALUE, "log_probs: the logits are not aligned to their values");
    if (!(temperature >= 1e-6f && temperature <= 1e6f))
        return fail(GARNET_B200_INVALID_VALUE, "log_probs: the temperature must lie between 1e-6 and 1e6");
    if (!d_targets != !d_log_probs || !d_targets != !d_ranks)
        return fail(GARNET_B200_INVALID_VALUE, "log_probs: targets, log_probs and ranks are given together");
    if (top_k < 0 || top_k > vocab || (top_k > 0 && (!d_top_log_probs || !d_top_ids)))
        return fail(GARNET_B200_INVALID_VALUE, "log_probs: bad top_k %d, or no arrays for it", top_k);
    if (top_k > kLpMaxTop) return fail(GARNET_B200_NOT_SUPPORTED, "log_probs: top_k above %d", kLpMaxTop);
    // Few rows: as many parts as run at once, four CTAs of 256 threads to an SM, each with a block for every warp (one row of 151936 bf16
    // 11.2 us in 8 parts, 17.0 in one).  More rows than such CTAs run at once: CTAs of 128 threads, of which the last to end leave less
    // idle (2048 rows 125 us, 131 with 256 threads; one row 13.2 us with 128).
    const long long blocks = (long long)vocab * (dtype == GARNET_B200_FP32 ? 4 : 2) / kLpBlockBytes;
    int parts = 1;
    while (parts < kLpMaxParts && (long long)rows * parts * 2 <= 4 * kSmCount && blocks >= 2 * parts * 8) parts *= 2;
    const int threads = rows > 4 * kSmCount ? 128 : 256;
    if ((long long)rows * parts > 0x7fffffffll) return fail(GARNET_B200_NOT_SUPPORTED, "log_probs: too many rows");
    const LogProbs p{d_logits, row_stride, d_targets, d_log_probs, d_ranks, d_entropy, d_top_log_probs, d_top_ids, vocab, top_k, parts, 1.f / temperature};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(rows) * unsigned(parts));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {unsigned(parts), 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = (flags & 1u) ? 2 : 1;
    GB_CUDA(cudaLaunchKernelEx(&cfg, threads == 128 ? lp_kernel<128>(dtype) : lp_kernel<256>(dtype), p));
    return GARNET_B200_OK;
}

}  // extern "C"
