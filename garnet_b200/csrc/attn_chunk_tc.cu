// Chunk attention over the paged cache on the tensor cores: S = Q K^T and O += P V as tcgen05 MMAs, the softmax in fp32.
//
// A CTA owns one kv head and one or two tiles of 128 query rows; a tile's rows are (token, q head of the group), so that the K and V
// rows it stages serve all the q heads of the group.  Per step of 64 keys:
//   loader warps    look up the page of every key and copy its K and V rows by cp.async into a ring of units (the keys of step u, the
//                   values of step u - 2): halves of 64 dims, 128-byte rows, swizzled - the K-major operand of Q K^T and the MN-major
//                   operand of P V.  Rows that do not exist, and those behind the last key that a row of the CTA sees, are filled
//                   with zeros (what the cache holds there could be NaN).  TMA boxes of a page took the loader 120 clocks each to ask
//                   for (16 rows x 128 bytes; 4000 clocks per 128 keys, more than all the rest);
//   MMA warps       one thread per tile: P V of step u - 2, then the scores of step u into the set that its P leaves;
//   scout warps     one per tile: wait for the MMAs' barrier in shared memory and pass it on to a named one;
//   softmax warps   one thread per query row: scores into registers, running maximum, p = 2^(s c - m c), the row's sum in fp32, P as
//                   two bf16 numbers each over the scores in tensor memory; O stays in tensor memory for kChSumSteps steps and is
//                   rescaled only when a row's maximum has grown by more than 2^8 since the last time (the final division makes that
//                   exact).  The fp32 work runs two values per instruction.  Two tiles take turns with their exponentials.
// Few rows after a long context: a cluster of up to 8 CTAs shares the keys; every CTA sends its part of row i to CTA i % splits by
// stores to distributed shared memory, which joins and writes it (launch_plan.h says when).
//
// Bound: a step of two tiles costs 1860 clocks of the tensor pipe (N = 64 takes 50 clocks per MMA of Q K^T instead of 33, since both
// operands come from shared memory; P V, twice for a weight's two numbers, 66) and 1024 of the exponential unit (16 per clock); it takes
// 2100 to 2350 (1.07 to 1.20 us): one tile's scores -> maximum -> exponentials -> two numbers beside the MMAs of the other.  B200, 16 / 8
// heads, norms and cache append included, at 1965 MHz: a prompt of 8192 tokens 350 us (0.47 of the measured bf16 peak over the visible
// pairs), 512 tokens at 30000 166 us (0.46), a prompt of 2048 46 us, 24 x 5 tokens at up to 3500 51 us (0.59 of the measured bandwidth), 4
// tokens at 1000 11 us.  Call after call the power limit takes the clock down to 1590 MHz: 410 and 191 us for the two long ones.
// With one number per weight, steps of 128 keys with one set of scores (MMAs of N = 128, P handed over in pieces of 32 keys, 128 or 192
// registers to a softmax thread) took 293 to 300 us for 8192 tokens where these took 286; part of the exponentials as polynomials, and
// two softmax threads per row and tile, were no faster either.
// Numerics: q, k and v are bf16 (exact products), scores, statistics and sums fp32.  The tensor core cuts towards zero what it adds to a
// sum: O is taken out of tensor memory every kChSumSteps steps and added in fp32, in memory of the workspace (19 MB, which stay in L2)
// of which a tile holds a slot while it runs.  A weight of P meets V as two bf16 numbers, its first bits and the rest: 2^-15 of it is lost
// at most, where one number (half as many MMAs of P V: 315 instead of 383 us a call of 8192 rows before sums were kept apart) loses
// 2^-8, about what the result's own rounding takes.  A row that comes out NaN though its scores are numbers, and that does not see one of
// the block's values that is not finite (its weight of zero makes NaN of it), is computed again by the row loop.
#include <algorithm>
#include <cooperative_groups.h>

#include "attn_chunk.cuh"
#include "chunk_barriers.h"
#include "tc_common.cuh"

namespace gb200 {

namespace {

namespace cg = cooperative_groups;

constexpr int kChRows = kChTileRows;   // query rows of a tile (UMMA M, one softmax thread each)
constexpr int kChMaxSplits = 8;
// Named barriers between the warps of a tile: a barrier in shared memory takes its waiter 200 clocks beside warps that keep the
// exponential unit busy, also when it is there already; a named one 30.  Every warp comes to all of its barriers, in the order of
// chunk_barriers.h, also after a wait that gave up.
constexpr int kBarTurn = 1, kBarScores = 3, kBarP = 7;
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
constexpr int kKeys = 64;         // keys of a step (UMMA N of Q K^T, K of P V)
constexpr int kChRounds = kKeys / 32;   // P is handed over, and rows are copied, 32 keys at a time
// A weight of P enters P V as two bf16 numbers, cut off and rest: both of them positive, the rest by 2^-20 of the weight where nothing is
// left, so that an infinite value stays infinite (of two numbers of opposite signs, or a zero, it would make NaN).
constexpr int kPieces = 2;
constexpr float kNearlyOne = 1.f - 0x1p-20f;
__device__ __forceinline__ uint32_t bf16x2_cut(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
constexpr int kChExists = 16;     // steps whose key bits are kept

template <int kTiles, int kUnits>
struct ChShape {
    // warps are allocated four at a time: 14, as well as twice 8, leave a thread 128 registers
    static constexpr int softmax_warps = 4 * kTiles, mma_warp = softmax_warps, scout_warp = mma_warp + kTiles, load_warp = scout_warp + kTiles, loaders = 2;
    static constexpr int threads = (load_warp + loaders) * 32;
    static constexpr int ahead = kUnits > 2 ? kUnits - 2 : 1;                      // units under way when the next is asked for
    static constexpr int q_half = kChRows * 128, q_tile = 2 * q_half;    // 64 dims of a tile of queries; all of them
    static constexpr int half = kKeys * 128, slot = 2 * half, unit = 2 * slot;   // the same of a step's keys (or values); keys and values
    static constexpr int q = 0, ring = kTiles * q_tile, exists = ring + kUnits * unit, bars = exists + kChExists * kChRounds * 4;
    static constexpr int total = bars + 512 + 1024;                      // barriers, and slack for 1024-byte alignment
    // the parts of the rows that this CTA of a split call finishes, over the queries and the ring: [row][CTA] rows of 128 floats, 16 bytes
    // apart in the banks; maxima and sums
    static constexpr int part_row = (kChDim + 4) * 4, parts = kTiles * kChRows + 8, stats = parts * part_row;
    static_assert(stats + parts * 8 <= exists, "the parts fit where the queries and the ring were");
    static_assert(total <= 227 * 1024, "shared memory budget");
    // the key bits of step u are written when unit u - kUnits - 1 is done, and with it the softmax of two steps before that
    static_assert(kUnits + 3 <= kChExists, "key bits");
    // tensor memory of a tile: two sets of scores (P replaces them), O
    static constexpr uint32_t col_o = 2 * kKeys, tile_cols = col_o + kChDim, cols = kTiles * tile_cols;
    static_assert(kTiles * tile_cols <= 512, "tensor memory");
};

__device__ __forceinline__ float chunk_warp_sum(float v)
{
#pragma unroll
    for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// One (row, q head) by one warp, eight slots at a time: running maximum and sum in fp32, four dims per lane.  A score of NaN or +inf makes
// the row NaN; one of -inf has weight 0, whatever the value there.
__device__ __noinline__ void chunk_row(const Chunk& p, int b, int row, int head, int slot, int lane)
{
    constexpr int kAtOnce = 8;
    const int group = p.q_heads / p.kv_heads, kv = head / group;
    const uint2 qr = *(reinterpret_cast<const uint2*>(p.queries + ((size_t(kv) * p.tokens + row) * group + head % group) * kChDim) + lane);
    const float q[4] = {__uint_as_float(qr.x << 16), __uint_as_float(qr.x & 0xffff0000u), __uint_as_float(qr.y << 16), __uint_as_float(qr.y & 0xffff0000u)};
    float top = -INFINITY, sum = 0.f, o[4] = {};
    for (int s0 = 0; s0 <= slot; s0 += kAtOnce) {
        uint2 kr[kAtOnce], vr[kAtOnce];
        uint32_t there = 0;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const long long at = s0 + i <= slot ? chunk_cache_offset(p, b, s0 + i, kv) : -1;
            kr[i] = vr[i] = make_uint2(0, 0);
            if (at < 0) continue;
            there |= 1u << i;
            kr[i] = *(reinterpret_cast<const uint2*>(p.keys + at) + lane), vr[i] = *(reinterpret_cast<const uint2*>(p.values + at) + lane);
        }
        float score[kAtOnce], next = top;
        bool wild = false;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            score[i] = chunk_warp_sum(q[0] * __uint_as_float(kr[i].x << 16) + q[1] * __uint_as_float(kr[i].x & 0xffff0000u) +
                                      q[2] * __uint_as_float(kr[i].y << 16) + q[3] * __uint_as_float(kr[i].y & 0xffff0000u)) * 0.08838834764831845f;
            if (!((there >> i) & 1)) score[i] = -INFINITY;
            wild = wild || !(score[i] < INFINITY);
            next = fmaxf(next, score[i]);
        }
        if (wild) {   // the same for all lanes
            sum = NAN;
            break;
        }
        if (next == -INFINITY) continue;
        const float old = top == next ? 1.f : expf(top - next);
        sum *= old;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] *= old;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (score[i] == -INFINITY) continue;   // weight 0
            const float w = expf(score[i] - next);
            const float v[4] = {__uint_as_float(vr[i].x << 16), __uint_as_float(vr[i].x & 0xffff0000u), __uint_as_float(vr[i].y << 16), __uint_as_float(vr[i].y & 0xffff0000u)};
#pragma unroll
            for (int d = 0; d < 4; ++d) o[d] += w * v[d];
            sum += w;
        }
        top = next;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const __nv_bfloat162 r[2] = {__floats2bfloat162_rn(o[0] * inv, o[1] * inv), __floats2bfloat162_rn(o[2] * inv, o[3] * inv)};
    *(reinterpret_cast<uint2*>(p.out + (size_t(row) * p.q_heads + head) * kChDim) + lane) = *reinterpret_cast<const uint2*>(r);
}

// The last of the slots [from, to) of sequence b at which a head's value is not finite, -1 without one; by one warp, eight at a time.
__device__ __noinline__ int chunk_last_wild(const Chunk& p, int b, int kv, int from, int to, int lane)
{
    constexpr int kAtOnce = 8;
    const auto wild = [](uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; };
    for (int s0 = to - 1; s0 >= from; s0 -= kAtOnce) {
        uint2 v[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const long long at = s0 - i >= from ? chunk_cache_offset(p, b, s0 - i, kv) : -1;
            v[i] = at >= 0 ? *(reinterpret_cast<const uint2*>(p.values + at) + lane) : make_uint2(0, 0);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (__any_sync(0xffffffffu, wild(v[i].x) || wild(v[i].y))) return s0 - i;
    }
    return -1;
}

// A warp takes a slot, the first free one from `from` on: there are as many as there can be tiles that hold tensor memory, as this one
// does.  (One that all want first takes the last of 256 tiles 15 us; looking at one after the other, 1 us each.)
__device__ __noinline__ int take_slot(unsigned* bits, int from, int lane)
{
    constexpr int kWords = (kChSumSlots + 31) / 32;
    static_assert(kWords <= 32, "a lane looks at a word");
    const unsigned there = lane + 1 < kWords ? 0xffffffffu : lane + 1 == kWords ? 0xffffffffu >> (31 - (kChSumSlots - 1) % 32) : 0u;
    for (int i = 0; i < 256; ++i) {
        unsigned free = lane < kWords ? ~__ldcg(bits + lane) & there : 0u, behind = lane == from / 32 ? free & (0xffffffffu << (from & 31)) : lane > from / 32 ? free : 0u;
        const unsigned words = __ballot_sync(0xffffffffu, behind != 0u), all = __ballot_sync(0xffffffffu, free != 0u);
        if (!words) behind = free;
        const int word = __ffs(words ? words : all) - 1;
        int slot = -1;
        if (lane == word) {
            const unsigned bit = behind & (0u - behind);
            if (!(atomicOr(bits + word, bit) & bit)) slot = word * 32 + __ffs(bit) - 1;
            __threadfence();
        }
        slot = __shfl_sync(0xffffffffu, slot, max(word, 0));
        if (word >= 0 && slot >= 0) return slot;
    }
    return -1;
}

// 32 dims of a row's kept sums; and o += f times them
__device__ __forceinline__ void load_kept(const float4* from, float4 (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __ldcg(from + i * kChRows);
}
__device__ __forceinline__ void add_kept(const float4 (&v)[8], float f, uint32_t (&o)[32])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        o[4 * i] = __float_as_uint(fmaf(v[i].x, f, __uint_as_float(o[4 * i])));
        o[4 * i + 1] = __float_as_uint(fmaf(v[i].y, f, __uint_as_float(o[4 * i + 1])));
        o[4 * i + 2] = __float_as_uint(fmaf(v[i].z, f, __uint_as_float(o[4 * i + 2])));
        o[4 * i + 3] = __float_as_uint(fmaf(v[i].w, f, __uint_as_float(o[4 * i + 3])));
    }
}

// mbar_wait_warp without suspending: the softmax has its scores a hundred clocks sooner.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag)
{
    const bool all = __all_sync(0xffffffffu, mbar_wait(bar, parity));
    if (!all) *abort_flag = 1;
    return all;
}

template <int kTiles, int kUnits>
__global__ void __launch_bounds__(ChShape<kTiles, kUnits>::threads, kUnits == 2 ? 2 : 1)
    attn_chunk_tc_kernel(const __grid_constant__ Chunk p, const __grid_constant__ CUtensorMap q_map, const int splits)
{
    using S = ChShape<kTiles, kUnits>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint32_t* exists = reinterpret_cast<uint32_t*>(smem + S::exists);       // [steps][kChRounds]: bits of the keys that have a page
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::bars);           // [units]
    uint64_t* empty = full + kUnits;                                        // [units]
    uint64_t* q_full = empty + kUnits;
    uint64_t* s_full = q_full + 1;                                          // [tiles][2 sets] scores written, and P V of two steps before done
    uint64_t* drained = s_full + kTiles * 2;                                // [tiles]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + kTiles);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* sum_slot = abort_flag + 1;                                // [tiles]: the tile's place in p.sums, -1 without one

    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int group = p.q_heads / p.kv_heads, tile_tokens = kChRows / group;
    const int split = int(blockIdx.x) % splits, kv = int(blockIdx.x) / splits % p.kv_heads, y = int(blockIdx.x) / splits / p.kv_heads;
    if (threadIdx.x == 0) {
        for (int u = 0; u < kUnits; ++u) mbar_init(&full[u], S::loaders), mbar_init(&empty[u], kTiles);
        mbar_init(q_full, 1);
        for (int i = 0; i < kTiles * 2; ++i) mbar_init(&s_full[i], 1);
        for (int q = 0; q < kTiles; ++q) mbar_init(&drained[q], 1);
        *abort_flag = 0;
        for (int q = 0; q < kTiles; ++q) sum_slot[q] = -1;
        fence_barrier_init();
    }
    pdl_wait();   // queries, cache rows and lists come from the kernels before this one
    const ChunkBlock blk = p.blocks[y];
    if (blk.b < 0) return;   // no rows for this CTA, and none for the others of its cluster
    // Tensor memory is taken behind the wait, and the kernels behind this one come up when all of its CTAs have theirs: a CTA that holds
    // tensor memory while it waits for another kernel could keep it from that kernel's CTA on the same SM, and both would wait for ever.
    if (warp == S::load_warp) {
        tmem_alloc(tmem_slot, S::cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    // keys that a tile's last row sees, and the steps of this CTA
    int ends[kTiles], steps[kTiles], most = 0;
#pragma unroll
    for (int q = 0; q < kTiles; ++q) {
        const int t0 = blk.first + q * tile_tokens, t1 = min(blk.len, t0 + tile_tokens);
        ends[q] = t0 >= t1 || blk.pos0 < 0 || blk.pos0 > p.max_context - 1 - t0 ? 0 : min(p.max_context, blk.pos0 + t1);
        most = max(most, ends[q]);
    }
    const int all_steps = (most + kKeys - 1) / kKeys;
    const int step0 = int((long long)split * all_steps / splits), step1 = int((long long)(split + 1) * all_steps / splits);
    int most_steps = 0;
#pragma unroll
    for (int q = 0; q < kTiles; ++q) {
        steps[q] = max(0, min(step1, (ends[q] + kKeys - 1) / kKeys) - step0);
        most_steps = max(most_steps, steps[q]);
    }

    if (warp >= S::load_warp) {
        // --------------------------------------------------------------- loaders
        const int lw = warp - S::load_warp;
        if (most_steps) {
            if (lw == 0 && elect_one()) {
                mbar_expect_tx(q_full, kTiles * S::q_tile);
                for (int q = 0; q < kTiles; ++q)
                    for (int h = 0; h < 2; ++h)
                        tma_load_2d(smem + S::q + q * S::q_tile + h * S::q_half, &q_map, h * 64,
                                    (kv * p.tokens + blk.row0 + blk.first + q * tile_tokens) * group, q_full);
            }
            __syncwarp();
            // Rounds of 32 keys go round the loaders; a lane looks up the page of one key of each round.
            const int* table = p.tables + size_t(blk.b) * p.width;
            constexpr int kMine = (kChRounds + S::loaders - 1) / S::loaders;
            int page[kMine], row[kMine], logical[kMine], within[kMine];   // of the step looked up last
            const int step_pages = kKeys / p.page_size, step_rest = kKeys % p.page_size;
            const auto look_up = [&](int j) {
#pragma unroll
                for (int u = 0; u < kMine; ++u) {
                    const int round = u * S::loaders + lw, pos = (step0 + j) * kKeys + round * 32 + lane;
                    if (j == 0) {
                        logical[u] = pos / p.page_size, within[u] = pos % p.page_size;
                    } else {
                        logical[u] += step_pages, within[u] += step_rest;
                        if (within[u] >= p.page_size) within[u] -= p.page_size, ++logical[u];
                    }
                    page[u] = round < kChRounds && j < most_steps && pos < most ? table[logical[u]] : -1;
                }
            };
            const size_t row_bytes = size_t(p.kv_heads) * kChDim * 2;
            const int piece = lane & 15, upper = lane >> 4;
            const size_t column = size_t(kv) * kChDim * 2 + piece * 16;
            uint32_t to_off[4];   // where a lane's 16 bytes of rows 0 and 1, 2 and 3, ... of eight go: the swizzle
#pragma unroll
            for (int i = 0; i < 4; ++i) to_off[i] = (piece >> 3) * S::half + (2 * i + upper) * 128 + (((piece & 7) ^ (2 * i + upper)) << 4);
            // two rows of 256 bytes per copy instruction; rows that do not exist are filled with zeros
            const auto copy = [&](const __nv_bfloat16* cache, const int (&rows)[kMine], uint32_t to) {
                const char* from = reinterpret_cast<const char*>(cache) + column;
#pragma unroll
                for (int u = 0; u < kMine; ++u) {
                    const int round = u * S::loaders + lw;
                    if (round >= kChRounds) break;
                    int r[16];   // all at once: a copy that waits for its own row's number takes 50 clocks
#pragma unroll
                    for (int i = 0; i < 16; ++i) r[i] = __shfl_sync(0xffffffffu, rows[u], 2 * i + upper);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        cp_async16(to + to_off[i & 3] + (round * 4 + (i >> 2)) * 1024, from + size_t(max(r[i], 0)) * row_bytes, r[i] >= 0);
                }
            };
            const auto announce = [&](int u) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[u % kUnits]);
            };
            look_up(0);
            int before[kMine], before_that[kMine];   // rows of the last two steps
#pragma unroll
            for (int u = 0; u < kMine; ++u) before[u] = before_that[u] = -1;
            int sent = 0;
            for (; sent < most_steps + 2; ++sent) {
#pragma unroll
                for (int u = 0; u < kMine; ++u) {
                    const bool there = page[u] >= 0 && page[u] < p.physical_pages;
                    row[u] = there ? page[u] * p.page_size + within[u] : -1;
                    const uint32_t bits = __ballot_sync(0xffffffffu, there);
                    if (lane == 0 && u * S::loaders + lw < kChRounds) exists[(sent % kChExists) * kChRounds + u * S::loaders + lw] = bits;
                }
                look_up(sent + 1);   // asked for a step ahead
                if (sent >= kUnits && !mbar_wait_warp(&empty[sent % kUnits], ((sent / kUnits) - 1) & 1, abort_flag)) break;
                const uint32_t to = smem_u32(smem + S::ring + sent % kUnits * S::unit);
                if (sent < most_steps) copy(p.keys, row, to);
                if (sent >= 2) copy(p.values, before_that, to + S::slot);
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group %0;" ::"n"(S::ahead) : "memory");
                if (sent >= S::ahead) announce(sent - S::ahead);
#pragma unroll
                for (int u = 0; u < kMine; ++u) before_that[u] = before[u], before[u] = row[u];
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (sent == most_steps + 2)
                for (int u = max(0, sent - S::ahead); u < sent; ++u) announce(u);
            // nothing is in flight when the CTA gives its memory back, also after a wait that gave up
            if (lw == 0) mbar_wait_suspended(q_full, 0);
            __syncwarp();
        }
    } else if (warp >= S::scout_warp) {
        // -------------- scouts, one per tile: pass on that scores (and P V of two steps before) are done
        const int q = warp - S::scout_warp;
        int my_steps = 0;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) my_steps = i == q ? steps[i] : my_steps;
        if (my_steps > kChSumSteps) {   // the softmax reads it behind the scores' barriers
            const int taken = take_slot(p.sum_slots, int((blockIdx.x * kTiles + q) % kChSumSlots), lane);
            sum_slot[q] = taken;
            if (taken < 0) *abort_flag = 1;
            __syncwarp();
        }
        bool good = true;
        chunk_scout(
            my_steps, [&](int i) { bar_sync(kBarP + q * 2 + (i & 1), kWeightsThreads); },
            [&](int i) { good = good && wait_warp(&s_full[q * 2 + (i & 1)], (i >> 1) & 1, abort_flag); },
            [&](int i) {
                tc_fence_after();
                tc_fence_before();
                bar_arrive(kBarScores + q * 2 + (i & 1), kScoresThreads);
            });
    } else if (warp >= S::mma_warp) {
        // ------------------------------------------- MMA issuers, one per tile
        constexpr uint32_t idesc_qk = umma_idesc_f16(1, kChRows, kKeys);
        constexpr uint32_t idesc_pv = umma_idesc_f16(1, kChRows, kChDim) | (1u << 16);   // V: MN-major
        const int q = warp - S::mma_warp;
        int my_steps = 0;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) my_steps = i == q ? steps[i] : my_steps;
        const uint32_t tile = tmem_base + q * S::tile_cols;
        const uint32_t q_lo = umma_desc_lo(smem_u32(smem + S::q + q * S::q_tile)), k_lo = umma_desc_lo(smem_u32(smem + S::ring));
        const uint32_t v_lo = ((smem_u32(smem + S::ring + S::slot) & 0x3FFFFu) >> 4) | (uint32_t(S::half >> 4) << 16);   // the halves of 64 dims
        // Unit u brings the keys of step u and the values of step u - 2: P V of that one, then the scores of step u into the set
        // that its P leaves.
        bool good = most_steps == 0 || mbar_wait_warp(q_full, 0, abort_flag);
        uint32_t unit = 0, parity = 0;
        for (int u = 0; most_steps && u < most_steps + 2; ++u) {
            const uint32_t set = (u & 1) * kKeys;
            good = good && wait_warp(&full[unit], parity, abort_flag);
            const bool pv = u >= 2 && u < my_steps + 2;
            if (pv) bar_sync(kBarP + q * 2 + (u & 1), kWeightsThreads);
            if (good && elect_one()) {
                tc_fence_after();
                if (pv) {
                    const uint32_t v = v_lo + unit * (S::unit >> 4);
#pragma unroll
                    for (int k16 = 0; k16 < kKeys / 16; ++k16)
#pragma unroll
                        for (int piece = 0; piece < kPieces; ++piece)
                            umma_f16_ts(tile + S::col_o, tile + set + piece * (kKeys / 2) + k16 * 8, v + k16 * (2048 >> 4), idesc_pv, (u - 2) % kChSumSteps != 0 || k16 + piece > 0);
                }
                if (u < my_steps) {
                    const uint32_t k = k_lo + unit * (S::unit >> 4);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int k16 = 0; k16 < 4; ++k16)
                            umma_f16_ss(tile + set, q_lo + h * (S::q_half >> 4) + k16 * 2, k + h * (S::half >> 4) + k16 * 2, idesc_qk, h + k16 > 0);
                }
                if (u < my_steps + 2) umma_commit(&s_full[q * 2 + (u & 1)]);
                umma_commit(&empty[unit]);
            }
            __syncwarp();
            if (++unit == kUnits) unit = 0, parity ^= 1;
        }
        if (most_steps && elect_one()) {
            umma_commit(&drained[q]);   // no MMA is in flight when the CTA gives its memory back, also after a wait that gave up
            mbar_wait_suspended(&drained[q], 0);
        }
        __syncwarp();
    } else {
        // -------------------------------------------------------------- softmax
        const int q = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t tm = tmem_base + q * S::tile_cols + (uint32_t((warp & 3) * 32) << 16);
        const int in_tile = r / group, t = blk.first + q * tile_tokens + in_tile, head = kv * group + r % group;
        const bool mine = in_tile < tile_tokens && t < blk.len;
        const int end = !mine || blk.pos0 < 0 || blk.pos0 > p.max_context - 1 - t ? 0 : blk.pos0 + t + 1;   // keys that the row sees
        int my_steps = 0;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) my_steps = i == q ? steps[i] : my_steps;
        // the scores of step i, and with them P V of step i - 2; behind the last steps that alone
        const auto scores_of = [&](int i) { bar_sync(kBarScores + q * 2 + (i & 1), kScoresThreads); };
        constexpr float kScale = 0.08838834764831845f * 1.4426950408889634f;   // 1 / sqrt(128), in powers of two
        float ref = -INFINITY, sum = 0.f;                                      // what the exponents are taken against; the weights' sum
        // steps in which the tiles take turns with their exponentials: left alone they fall into step, first both on the exponential
        // unit, then neither
        const int turns = kTiles == 2 ? min(steps[0], steps[kTiles - 1]) : 0;
        const bool any = __any_sync(0xffffffffu, end > 0);
        float kept = -INFINITY;   // what the weights of the kept sums stand against
        const auto sums_of = [&] { return p.sums + size_t(sum_slot[q]) * (kChSumBytes / 16) + r; };
        // O, the sum of up to kChSumSteps steps, is added to the steps' before; the next P V starts a sum of its own
        const auto keep_sums = [&](int j) {
            // O is complete when the scores of the next step are there
            if (!*abort_flag) wait_warp(&s_full[q * 2 + ((j + 1) & 1)], ((j + 1) >> 1) & 1, abort_flag);
            __syncwarp();
            tc_fence_after();
            if (sum_slot[q] < 0) return;   // and the call gives up
            float4* to = sums_of();
            const bool first = j == kChSumSteps, grown = __any_sync(0xffffffffu, kept != ref);
            const float f = kept == ref ? 1.f : ex2(kept - ref);
#pragma unroll 1
            for (int c = 0; c < kChDim / 32; ++c) {
                uint32_t o[32];
                tmem_ld_32x32(tm + S::col_o + 32 * c, o);
                if (!first && grown) {   // seldom
                    float4 v[8];
                    load_kept(to + 8 * c * kChRows, v);
                    tmem_ld_wait();
                    add_kept(v, f, o);
                }
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float4* at = to + (8 * c + i) * kChRows;
                    const float4 v = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                    if (first || grown) __stcg(at, v);
                    else asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
                }
            }
            kept = ref;
        };
        for (int j = 0; j < my_steps; ++j) {
            const int kb = (step0 + j) * kKeys;
            const uint32_t ts = tm + (j & 1) * kKeys;
            scores_of(j);
            if (!any) {   // none of the warp's rows sees a key: their weights may be what they are
                if (j < turns && (q == 1 || j > 0)) bar_sync(kBarTurn + q, 256);
                if (j < turns && !(q == 1 && j + 1 == turns)) bar_arrive(kBarTurn + 1 - q, 256);
                bar_arrive(kBarP + q * 2 + (j & 1), kWeightsThreads);
                continue;
            }
            tc_fence_after();
            uint32_t s[kChRounds][32];
#pragma unroll
            for (int c = 0; c < kChRounds; ++c) tmem_ld_32x32(ts + 32 * c, s[c]);
            uint32_t there[kChRounds], all = 0xffffffffu;
#pragma unroll
            for (int c = 0; c < kChRounds; ++c) {
                there[c] = exists[(j % kChExists) * kChRounds + c];
                all &= there[c];
            }
            tmem_ld_wait();
            if (!__all_sync(0xffffffffu, end >= kb + kKeys && all == 0xffffffffu)) {
#pragma unroll
                for (int c = 0; c < kChRounds; ++c) {
                    const uint32_t vis = there[c] & bit_range(0, end - kb - 32 * c);
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[c][i] = (vis >> i) & 1 ? s[c][i] : 0xff800000u;   // -inf
                }
            }
            float m[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) m[i] = -INFINITY;
#pragma unroll
            for (int c = 0; c < kChRounds; ++c)
#pragma unroll
                for (int i = 0; i < 32; i += 2) m[(i >> 1) & 7] = max3(m[(i >> 1) & 7], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
            const float top = max3(max3(m[0], m[1], m[2]), max3(m[3], m[4], m[5]), fmaxf(m[6], m[7])) * kScale;
            const bool grow = top > ref + 8.f;
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? ex2(ref - top) : 1.f;
                if (grow) ref = top;
                sum *= f;
                if (j > 0) {
                    // O holds the steps up to the one before this when the next scores are there
                    if (!*abort_flag) wait_warp(&s_full[q * 2 + ((j + 1) & 1)], ((j + 1) >> 1) & 1, abort_flag);
                    __syncwarp();
                    tc_fence_after();
                    const uint64_t f2 = f32x2(f, f);
#pragma unroll 1
                    for (int c = 0; c < kChDim / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld_32x16(tm + S::col_o + 16 * c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float lo, hi;
                            f32x2_split(mul2(f32x2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), f2), lo, hi);
                            o[2 * i] = __float_as_uint(lo), o[2 * i + 1] = __float_as_uint(hi);
                        }
                        tmem_st_32x16(tm + S::col_o + 16 * c, o);
                    }
                }
            }
            const float base = ref == -INFINITY ? 0.f : ref;
            const uint64_t scale2 = f32x2(kScale, kScale), base2 = f32x2(-base, -base), minus1 = f32x2(-kNearlyOne, -kNearlyOne);
            uint64_t part2[2] = {0, 0};
            if (j < turns && (q == 1 || j > 0)) bar_sync(kBarTurn + q, 256);
#pragma unroll
            for (int c = 0; c < kChRounds; ++c) {
                uint32_t w[16], rest[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float a, d;
                    f32x2_split(fma2(f32x2(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])), scale2, base2), a, d);
                    const uint64_t both = f32x2(ex2(a), ex2(d));
                    part2[i & 1] = add2(part2[i & 1], both);
                    f32x2_split(both, a, d);
                    w[i] = bf16x2_cut(a, d);
                    f32x2_split(fma2(f32x2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)), minus1, both), a, d);
                    rest[i] = bf16x2_of(a, d);
                }
                tmem_st_32x16(ts + 16 * c, w);
                tmem_st_32x16(ts + kKeys / 2 + 16 * c, rest);
            }
            if (j < turns && !(q == 1 && j + 1 == turns)) bar_arrive(kBarTurn + 1 - q, 256);
            tmem_st_wait();
            if (j > 0 && j % kChSumSteps == 0) keep_sums(j);
            tc_fence_before();
            bar_arrive(kBarP + q * 2 + (j & 1), kWeightsThreads);
            float part[2];
            f32x2_split(add2(part2[0], part2[1]), part[0], part[1]);
            sum += part[0] + part[1];
        }
        if (my_steps) scores_of(my_steps), scores_of(my_steps + 1);
        tc_fence_after();
        // a wait that gave up leaves NaNs, which no caller can take for a result
        const bool good = !*abort_flag;
        if (!good) sum = NAN;
        const bool used = __any_sync(0xffffffffu, mine);
        // 32 dims of O, with what was kept
        const float kept_scale = kept == ref ? 1.f : ex2(kept - ref);
        const bool with_kept = my_steps > kChSumSteps && any && sum_slot[q] >= 0;
        float4 next[8];   // a trip to L2 ahead
        if (with_kept) load_kept(sums_of(), next);
        const auto load_o = [&](int c, uint32_t (&o)[32]) {
            tmem_ld_32x32(tm + S::col_o + 32 * c, o);
            tmem_ld_wait();
            if (with_kept) {
                add_kept(next, kept_scale, o);
                if (c + 1 < kChDim / 32) load_kept(sums_of() + 8 * (c + 1) * kChRows, next);
            }
        };
        if (splits == 1) {
            const float inv = end == 0 || sum == 0.f ? 0.f : 1.f / sum;
            __nv_bfloat16* out = p.out + (size_t(blk.row0 + t) * p.q_heads + head) * kChDim;
            bool bad = false;
#pragma unroll 1
            for (int c = 0; used && c < kChDim / 32; ++c) {
                uint32_t o[32];
                if (my_steps) load_o(c, o);
                if (mine) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float a = my_steps && end ? __uint_as_float(o[8 * i + 2 * k]) * inv : 0.f, d = my_steps && end ? __uint_as_float(o[8 * i + 2 * k + 1]) * inv : 0.f;
                            bad = bad || isnan(a) || isnan(d);
                            w[k] = bf16x2_of(a, d);
                        }
                        *reinterpret_cast<uint4*>(out + 32 * c + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            __syncwarp();
            // a sum of weights that is NaN says so rightly; another, only where no value that the row does not see is to blame
            bad = bad && good && !isnan(sum);
            uint32_t redo = __ballot_sync(0xffffffffu, bad);
            if (redo) {
                const int wild = chunk_last_wild(p, blk.b, kv, __reduce_min_sync(0xffffffffu, bad ? end : most), most, lane);
                redo = __ballot_sync(0xffffffffu, bad && (end <= wild || sum == 0.f));
            }
            for (; redo; redo &= redo - 1) {
                const int from = __ffs(redo) - 1;
                chunk_row(p, blk.b, __shfl_sync(0xffffffffu, blk.row0 + t, from), __shfl_sync(0xffffffffu, head, from), __shfl_sync(0xffffffffu, end, from) - 1, lane);
            }
        } else {
            // Row i is finished by CTA i % splits of the cluster: its part goes there, as row i / splits.
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();   // every CTA's copies and MMAs are done: their operands may be written over
            const int i = q * kChRows + r, at = i / splits * splits + split;
            uint8_t* there = reinterpret_cast<uint8_t*>(cluster.map_shared_rank(smem, i % splits));
#pragma unroll 1
            for (int c = 0; used && c < kChDim / 32; ++c) {
                uint32_t o[32];
                if (my_steps) load_o(c, o);
                if (mine) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        *reinterpret_cast<uint4*>(there + at * S::part_row + (32 * c + 4 * k) * 4) = my_steps ? make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]) : make_uint4(0, 0, 0, 0);
                }
            }
            if (mine) *reinterpret_cast<float2*>(there + S::stats + at * 8) = make_float2(my_steps ? ref : -INFINITY, my_steps ? sum : 0.f);
        }
    }
    if (splits > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (warp >= S::softmax_warps) cluster.sync();   // with the softmax warps above
        cluster.sync();
        // ---- this CTA's rows from the parts of all: four rows to a warp, eight lanes each
        constexpr int kWarps = S::threads / 32;
        // rows of the tiles up to the last that is a token's
        const int tokens = blk.len - blk.first, used = kTiles == 2 && tokens > tile_tokens ? kChRows + min(tokens - tile_tokens, tile_tokens) * group : min(tokens, tile_tokens) * group;
        const int most_rows = (used - split + splits - 1) / splits, l = lane & 7;
        for (int base = warp * 4; base < most_rows; base += kWarps * 4) {
            const int local = min(base + (lane >> 3), most_rows - 1), i = local * splits + split;
            const int q = i / kChRows, r = i % kChRows, in_tile = r / group, t = blk.first + q * tile_tokens + in_tile, head = kv * group + r % group;
            const bool mine = base + (lane >> 3) < most_rows && in_tile < tile_tokens && t < blk.len;
            const int end = !mine || blk.pos0 < 0 || blk.pos0 > p.max_context - 1 - t ? 0 : blk.pos0 + t + 1;
            const float2 st = l < splits ? *reinterpret_cast<const float2*>(smem + S::stats + (local * splits + l) * 8) : make_float2(-INFINITY, 0.f);
            float top = st.x;
#pragma unroll
            for (int d = 1; d < kChMaxSplits; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float f = st.y == 0.f ? 0.f : ex2(st.x - top);   // 0: nothing visible there
            float total = f * st.y;
#pragma unroll
            for (int d = 1; d < kChMaxSplits; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
            const float factor = total == 0.f || end == 0 ? 0.f : f / total;
            float4 o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < splits; ++c) {
                const float w = __shfl_sync(0xffffffffu, factor, (lane & 24) + c);
                const float4* from = reinterpret_cast<const float4*>(smem + (local * splits + c) * S::part_row) + l;
                if (w == 0.f) continue;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float4 v = from[8 * k];
                    o[k].x += w * v.x, o[k].y += w * v.y, o[k].z += w * v.z, o[k].w += w * v.w;
                }
            }
            bool bad = false;
            const int row = blk.row0 + t;
            if (mine) {
                uint2* out = reinterpret_cast<uint2*>(p.out + (size_t(row) * p.q_heads + head) * kChDim) + l;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    bad = bad || isnan(o[k].x) || isnan(o[k].y) || isnan(o[k].z) || isnan(o[k].w);
                    out[8 * k] = make_uint2(bf16x2_of(o[k].x, o[k].y), bf16x2_of(o[k].z, o[k].w));
                }
            }
            __syncwarp();
            bad = bad && !*abort_flag && !isnan(total);
            uint32_t redo = __ballot_sync(0xffffffffu, bad);
            if (redo) {   // as above
                const int wild = chunk_last_wild(p, blk.b, kv, __reduce_min_sync(0xffffffffu, bad ? end : most), most, lane);
                redo = __ballot_sync(0xffffffffu, bad && end <= wild);
            }
            if (redo)
                for (int g = 0; g < 4; ++g)
                    if ((redo >> (8 * g)) & 0xffu)
                        chunk_row(p, blk.b, __shfl_sync(0xffffffffu, row, 8 * g), __shfl_sync(0xffffffffu, head, 8 * g), __shfl_sync(0xffffffffu, end, 8 * g) - 1, lane);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == S::load_warp) {
        if (lane < kTiles && sum_slot[lane] >= 0) {   // nobody of this CTA reads or writes there any more
            __threadfence();
            atomicAnd(p.sum_slots + sum_slot[lane] / 32, ~(1u << (sum_slot[lane] & 31)));
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, S::cols);
    }
}

template <int kTiles, int kUnits>
int launch(const Chunk& p, int splits, cudaStream_t stream)
{
    using S = ChShape<kTiles, kUnits>;
    CUtensorMap q_map;
    if (int rc = make_tensor_map_2d_16bit(&q_map, p.queries, uint64_t(p.tokens) * p.q_heads, kChDim, kChRows)) return rc;
    const auto kernel = attn_chunk_tc_kernel<kTiles, kUnits>;
    GB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::total));
    const long long ctas = (long long)p.block_count * p.kv_heads * splits;
    if (ctas > 0x7fffffffll) return fail(GARNET_B200_NOT_SUPPORTED, "attention_chunk: too many blocks of rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ctas));
    cfg.blockDim = dim3(S::threads);
    cfg.dynamicSmemBytes = S::total;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {unsigned(splits), 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    GB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p, q_map, splits));
    return GARNET_B200_OK;
}

}  // namespace

int chunk_attention_launch(const Chunk& p, const ChunkPlan& plan, cudaStream_t stream)
{
    if (plan.tiles == 2) return launch<2, 5>(p, plan.splits, stream);
    return plan.units == 2 ? launch<1, 2>(p, plan.splits, stream) : launch<1, 6>(p, plan.splits, stream);
}

}  // namespace gb200
