// Chunk attention over the paged cache on the tensor cores: S = Q K^T and O += P V as tcgen05 MMAs, the softmax in fp32.
//
// A CTA owns one kv head and one or two tiles of 128 query rows; a tile's rows are (token, q head of the group), so that the K and V
// rows it stages serve all the q heads of the group.  Per step of 128 (or 64) keys:
//   loader warp     looks up the pages of the step, one lane per box of rows that lie together in the cache, and copies K and V by TMA
//                   into a ring of slots: two halves of 64 dims, 128-byte rows, swizzled - the K-major operand of Q K^T and the
//                   MN-major operand of P V.  Rows that do not exist, and those behind the last key that a row of the CTA sees, come
//                   from behind the end of the tensor, which reads as zeros (what the cache holds there could be NaN);
//   MMA warp        one thread: P V of a step when its P is there, then Q K^T of the next step, tile by tile: the tensor pipe works on
//                   one tile while the other tile's softmax runs;
//   softmax warps   one thread per query row: scores into registers, running maximum, p = 2^(s c - m c), the row's sum in fp32, P as
//                   bf16 over the scores in tensor memory; O stays in tensor memory and is rescaled only when a row's maximum has
//                   grown by more than 2^8 since the last time (the final division makes that exact; the conditional rescaling of
//                   FlashAttention-4).  The fp32 work runs two values per instruction.
// Few rows after a long context: a cluster of up to 8 CTAs shares the keys, and their partial results meet in distributed shared
// memory; every CTA finishes some of the rows.
// Numerics: q, k and v are bf16 (exact products), scores, statistics and sums fp32.  P is rounded to bf16 where it meets V, 2^-8 of each
// weight at most: the errors of the weights are independent of one another, so that a result is off by about what its own rounding
// to bf16 takes (P in two pieces would cost half as many MMAs again).  A row that comes out NaN (infinities in places that it does not
// see meet weights of zero) is computed again by the row loop.
#include <algorithm>
#include <cooperative_groups.h>

#include "attn_chunk.cuh"
#include "tc_common.cuh"

namespace gb200 {

namespace {

namespace cg = cooperative_groups;

constexpr int kChRows = 128;      // query rows of a tile (UMMA M, one softmax thread each)
constexpr int kChMaxSplits = 8;

template <int kTiles, int kKeys, int kSlots>
struct ChShape {
    static constexpr int softmax_warps = 4 * kTiles, mma_warp = softmax_warps, load_warp = mma_warp + 1, threads = (load_warp + 1) * 32;
    static constexpr int q_half = kChRows * 128, q_tile = 2 * q_half;    // 64 dims of a tile of queries; all of them
    static constexpr int half = kKeys * 128, slot = 2 * half;            // the same of a step's keys (or values)
    static constexpr int q = 0, ring = kTiles * q_tile, exists = ring + kSlots * slot, bars = exists + 4 * (kKeys / 32) * 4;
    static constexpr int total = bars + 192 + 1024;                      // barriers, and slack for 1024-byte alignment
    // partial results of a split call, over the queries and the ring: rows of 128 floats, 16 bytes apart in the banks; maxima, sums
    static constexpr int part_row = (kChDim + 4) * 4, stats = kTiles * kChRows * part_row;
    static_assert(stats + kTiles * kChRows * 8 <= exists, "the partial results fit where the queries and the ring were");
    static_assert(total <= 227 * 1024, "shared memory budget");
    // tensor memory of a tile: the scores (P replaces them), O
    static constexpr uint32_t col_o = kKeys, tile_cols = kKeys + kChDim, cols = kTiles * tile_cols <= 256 ? 256 : 512;
    static_assert(kTiles * tile_cols <= 512, "tensor memory");
};

struct ChMaps {
    CUtensorMap q;                // [kv head][token][q head of the group] rows of 128
    CUtensorMap k, v;             // boxes of `box` cache rows of a kv head
    CUtensorMap k_row, v_row;     // boxes of one row
};

// The query rows of a CTA: up to `rows` tokens of sequence b from its token `first` on.
struct ChBlock {
    int b, first, len, row0, pos0;
};

// Block y counted from the last sequence's last block (the blocks with the most keys come first).  One warp.
__device__ __forceinline__ ChBlock chunk_block(const Chunk& p, int y, int rows, int lane)
{
    int base = 0;
    for (int i0 = 0; i0 < p.batch; i0 += 32) {
        const int b = p.batch - 1 - (i0 + lane);
        int lo = 0, len = 0;
        if (b >= 0) {
            lo = min(max(p.row_starts[b], 0), p.tokens);
            len = min(max(p.row_starts[b + 1], lo), p.tokens) - lo;
        }
        const int n = (len + rows - 1) / rows;
        int upto = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        const int total = __shfl_sync(0xffffffffu, upto, 31);
        if (y < base + total) {
            const int at = y - base;
            const int from = __ffs(__ballot_sync(0xffffffffu, at < upto)) - 1;   // the first lane whose blocks reach so far
            ChBlock r;
            r.b = __shfl_sync(0xffffffffu, b, from);
            r.len = __shfl_sync(0xffffffffu, len, from);
            r.row0 = __shfl_sync(0xffffffffu, lo, from);
            r.first = (__shfl_sync(0xffffffffu, upto, from) - 1 - at) * rows;
            r.pos0 = p.positions[r.b];
            return r;
        }
        base += total;
    }
    return ChBlock{-1, 0, 0, 0, 0};
}

template <int kTiles, int kKeys, int kSlots>
__global__ void __launch_bounds__(ChShape<kTiles, kKeys, kSlots>::threads, kTiles == 1 ? 2 : 1)
    attn_chunk_tc_kernel(const Chunk p, const __grid_constant__ ChMaps maps, const int box, const int splits)
{
    using S = ChShape<kTiles, kKeys, kSlots>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint32_t* exists = reinterpret_cast<uint32_t*>(smem + S::exists);       // [4 steps][kKeys / 32]: bits of the keys that have a page
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::bars);           // [slots]
    uint64_t* empty = full + kSlots;                                        // [slots]
    uint64_t* q_full = empty + kSlots;
    uint64_t* s_full = q_full + 1;                                          // [tiles] scores written (and the P V before them done)
    uint64_t* p_full = s_full + kTiles;                                     // [tiles] P written
    uint64_t* o_full = p_full + kTiles;                                     // [tiles] the last P V done
    uint64_t* drained = o_full + kTiles;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    ChBlock* block_s = reinterpret_cast<ChBlock*>(tmem_slot + 2);

    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int group = p.q_heads / p.kv_heads, tile_tokens = kChRows / group;
    const int split = int(blockIdx.x) % splits, kv = int(blockIdx.x) / splits % p.kv_heads, y = int(blockIdx.x) / splits / p.kv_heads;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kSlots; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        mbar_init(q_full, 1);
        for (int q = 0; q < kTiles; ++q) mbar_init(&s_full[q], 1), mbar_init(&p_full[q], 4), mbar_init(&o_full[q], 1);
        mbar_init(drained, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == S::mma_warp) {
        tmem_alloc(tmem_slot, S::cols);
        tmem_relinquish();
    }
    pdl_launch_dependents();
    pdl_wait();   // queries, cache rows and lists come from the kernels before this one
    if (warp == S::load_warp) {
        const ChBlock found = chunk_block(p, y, tile_tokens * kTiles, lane);
        if (lane == 0) *block_s = found;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const ChBlock blk = *block_s;
    if (blk.b < 0) {   // no rows for this CTA, and none for the others of its cluster
        if (warp == S::mma_warp) tmem_dealloc(tmem_base, S::cols);
        return;
    }
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

    if (warp == S::load_warp) {
        // ---------------------------------------------------------------- loader
        if (most_steps) {
            if (lane == 0) {
                mbar_expect_tx(q_full, kTiles * S::q_tile);
                for (int q = 0; q < kTiles; ++q)
                    for (int h = 0; h < 2; ++h)
                        tma_load_2d(smem + S::q + q * S::q_tile + h * S::q_half, &maps.q, h * 64,
                                    (kv * p.tokens + blk.row0 + blk.first + q * tile_tokens) * group, q_full);
            }
            const int* table = p.tables + size_t(blk.b) * p.width;
            const int boxes = kKeys / box, nowhere = p.physical_pages * p.page_size;
            constexpr int kMost = kKeys / 32;
            // first cache row of a lane's boxes, `nowhere` for those without a page
            int at[kMost], next[kMost];
            const auto look_up = [&](int j, int (&r)[kMost]) {
#pragma unroll
                for (int u = 0; u < kMost; ++u) {
                    const int i = u * 32 + lane, pos = (step0 + j) * kKeys + i * box;
                    r[u] = nowhere;
                    if (i < boxes && j < most_steps && pos < most) {
                        const int page = table[pos / p.page_size];
                        if (page >= 0 && page < p.physical_pages) r[u] = page * p.page_size + pos % p.page_size;
                    }
                }
            };
            const auto request = [&](const CUtensorMap* map, const CUtensorMap* row_map, int n, int j) -> bool {
                const int slot = n % kSlots;
                if (n >= kSlots && !mbar_wait_warp(&empty[slot], ((n / kSlots) - 1) & 1, abort_flag)) return false;
                if (lane == 0) mbar_expect_tx(&full[slot], S::slot);
                __syncwarp();
                uint8_t* to = smem + S::ring + slot * S::slot;
#pragma unroll
                for (int u = 0; u < kMost; ++u) {
                    const int i = u * 32 + lane, pos = (step0 + j) * kKeys + i * box;
                    if (i >= boxes) continue;
                    if (pos + box <= most || pos >= most || at[u] == nowhere) {
                        tma_load_3d(to + i * box * 128, map, 0, kv, at[u], &full[slot]);
                        tma_load_3d(to + S::half + i * box * 128, map, 64, kv, at[u], &full[slot]);
                    } else {
                        for (int r = 0; r < box; ++r) {
                            const int from = pos + r < most ? at[u] + r : nowhere;
                            tma_load_3d(to + (i * box + r) * 128, row_map, 0, kv, from, &full[slot]);
                            tma_load_3d(to + S::half + (i * box + r) * 128, row_map, 64, kv, from, &full[slot]);
                        }
                    }
                }
                return true;
            };
            look_up(0, at);
            int n = 0;
            for (int j = 0; j < most_steps; ++j) {
                look_up(j + 1, next);
                // which keys there are: the softmax of step j - 4 has long been done when the ring takes step j
                uint32_t there[kMost], all = 0xffffffffu;
#pragma unroll
                for (int u = 0; u < kMost; ++u) {
                    there[u] = __ballot_sync(0xffffffffu, u * 32 + lane >= boxes || at[u] != nowhere);
                    all &= there[u];
                }
                if (lane < kKeys / 32) {
                    uint32_t bits = 0xffffffffu;
                    if (all != 0xffffffffu) {
                        bits = 0;
                        for (int k = 0; k < 32; k += min(box, 32)) {
                            const int i = (lane * 32 + k) / box;
                            uint32_t word = 0;
#pragma unroll
                            for (int u = 0; u < kMost; ++u) word = (i >> 5) == u ? there[u] : word;
                            if ((word >> (i & 31)) & 1) bits |= (box >= 32 ? 0xffffffffu : (1u << box) - 1u) << k;
                        }
                    }
                    exists[(j & 3) * (kKeys / 32) + lane] = bits;
                }
                __syncwarp();
                if (!request(&maps.k, &maps.k_row, n, j) || !request(&maps.v, &maps.v_row, n + 1, j)) break;
                n += 2;
#pragma unroll
                for (int u = 0; u < kMost; ++u) at[u] = next[u];
            }
            // nothing is in flight when the CTA gives its memory back, also after a wait that gave up
            mbar_wait_suspended(q_full, 0);
            ring_wait_landed(full, kSlots, uint32_t(n % kSlots), uint32_t(n / kSlots));
            __syncwarp();
        }
    } else if (warp == S::mma_warp) {
        // ----------------------------------------------------------- MMA issuer
        if (most_steps && elect_one()) {
            constexpr uint32_t idesc_qk = umma_idesc_f16(1, kChRows, kKeys);
            constexpr uint32_t idesc_pv = umma_idesc_f16(1, kChRows, kChDim) | (1u << 16);   // V: MN-major
            const uint32_t q_lo = umma_desc_lo(smem_u32(smem + S::q)), k_lo = umma_desc_lo(smem_u32(smem + S::ring));
            const uint32_t v_lo = ((smem_u32(smem + S::ring) & 0x3FFFFu) >> 4) | (uint32_t(S::half >> 4) << 16);   // the halves of 64 dims
            const auto scores = [&](int q, uint32_t slot) {
                const uint32_t a = q_lo + q * (S::q_tile >> 4), k = k_lo + slot * (S::slot >> 4);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k16 = 0; k16 < 4; ++k16)
                        umma_f16_ss(tmem_base + q * S::tile_cols, a + h * (S::q_half >> 4) + k16 * 2, k + h * (S::half >> 4) + k16 * 2, idesc_qk, h + k16 > 0);
                umma_commit(&s_full[q]);
            };
            const auto wait_slot = [&](int n) {
                const bool ok = mbar_wait_suspended(&full[n % kSlots], (n / kSlots) & 1);
                tc_fence_after();
                return ok;
            };
            bool good = mbar_wait_suspended(q_full, 0) && wait_slot(0);
            if (good) {
#pragma unroll
                for (int q = 0; q < kTiles; ++q)
                    if (steps[q] > 0) scores(q, 0);
                umma_commit(&empty[0]);
            }
            for (int j = 0; j < most_steps && good; ++j) {
                const int nv = 2 * j + 1, nk = 2 * j + 2;
                good = wait_slot(nv) && (j + 1 >= most_steps || wait_slot(nk));
#pragma unroll
                for (int q = 0; q < kTiles; ++q) {
                    if (!good || j >= steps[q]) continue;
                    good = mbar_wait_suspended(&p_full[q], j & 1);
                    if (!good) continue;
                    tc_fence_after();
                    const uint32_t tile = tmem_base + q * S::tile_cols, v = v_lo + (nv % kSlots) * (S::slot >> 4);
#pragma unroll
                    for (int k16 = 0; k16 < kKeys / 16; ++k16)
                        umma_f16_ts(tile + S::col_o, tile + k16 * 8, v + k16 * (2048 >> 4), idesc_pv, j > 0 || k16 > 0);
                    if (j + 1 < steps[q]) scores(q, nk % kSlots);
                    else umma_commit(&o_full[q]);
                }
                umma_commit(&empty[nv % kSlots]);
                if (j + 1 < most_steps) umma_commit(&empty[nk % kSlots]);
            }
            if (!good) *abort_flag = 1;
            umma_commit(drained);   // no MMA is in flight when the CTA gives its memory back, also after a wait that gave up
            mbar_wait_suspended(drained, 0);
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
        constexpr float kScale = 0.08838834764831845f * 1.4426950408889634f;   // 1 / sqrt(128), in powers of two
        float ref = -INFINITY, sum = 0.f;                                      // what the exponents are taken against; the weights' sum
        bool good = true;
        for (int j = 0; j < my_steps; ++j) {
            const int kb = (step0 + j) * kKeys;
            good = mbar_wait_warp(&s_full[q], j & 1, abort_flag);
            if (!good) break;
            tc_fence_after();
            uint32_t s[kKeys / 32][32];
#pragma unroll
            for (int c = 0; c < kKeys / 32; ++c) tmem_ld_32x32(tm + 32 * c, s[c]);
            uint32_t there[kKeys / 32], all = 0xffffffffu;
#pragma unroll
            for (int c = 0; c < kKeys / 32; ++c) {
                there[c] = exists[(j & 3) * (kKeys / 32) + c];
                all &= there[c];
            }
            tmem_ld_wait();
            if (!__all_sync(0xffffffffu, end >= kb + kKeys && all == 0xffffffffu)) {
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) {
                    const uint32_t vis = there[c] & bit_range(0, end - kb - 32 * c);
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[c][i] = (vis >> i) & 1 ? s[c][i] : 0xff800000u;   // -inf
                }
            }
            float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kKeys / 32; ++c)
#pragma unroll
                for (int i = 0; i < 32; i += 2) m[(i >> 1) & 3] = max3(m[(i >> 1) & 3], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
            const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * kScale;
            const bool grow = top > ref + 8.f;
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? ex2(ref - top) : 1.f;
                if (grow) ref = top;
                sum *= f;
                if (j > 0) {   // the P V of the step before is done: its commit came before that of these scores
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
            const uint64_t scale2 = f32x2(kScale, kScale), base2 = f32x2(-base, -base);
            uint64_t part2[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < kKeys / 32; ++c) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float a, d;
                    f32x2_split(fma2(f32x2(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])), scale2, base2), a, d);
                    a = ex2(a), d = ex2(d);
                    part2[i & 1] = add2(part2[i & 1], f32x2(a, d));
                    w[i] = bf16x2_of(a, d);
                }
                tmem_st_32x16(tm + 16 * c, w);
            }
            float part[2];
            f32x2_split(add2(part2[0], part2[1]), part[0], part[1]);
            sum += part[0] + part[1];
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[q]);
        }
        if (my_steps && good) good = mbar_wait_warp(&o_full[q], 0, abort_flag);
        tc_fence_after();
        // a wait that gave up leaves NaNs, which no caller can take for a result
        if (!good) sum = NAN;
        if (splits == 1) {
            const float inv = end == 0 || sum == 0.f ? 0.f : 1.f / sum;
            __nv_bfloat16* out = p.out + (size_t(blk.row0 + t) * p.q_heads + head) * kChDim;
            bool bad = false;
#pragma unroll 1
            for (int c = 0; c < kChDim / 32; ++c) {
                uint32_t o[32];
                if (my_steps) {
                    tmem_ld_32x32(tm + S::col_o + 32 * c, o);
                    tmem_ld_wait();
                }
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
            for (uint32_t redo = __ballot_sync(0xffffffffu, bad && good); redo; redo &= redo - 1) {
                const int from = __ffs(redo) - 1;
                chunk_row(p, blk.b, __shfl_sync(0xffffffffu, blk.row0 + t, from), __shfl_sync(0xffffffffu, head, from), __shfl_sync(0xffffffffu, end, from) - 1, lane);
            }
        } else {
            __syncthreads();   // all of the CTA's copies and MMAs are done: their operands may be written over
            float* row = reinterpret_cast<float*>(smem + (q * kChRows + r) * S::part_row);
#pragma unroll 1
            for (int c = 0; c < kChDim / 32; ++c) {
                uint32_t o[32];
                if (my_steps) {
                    tmem_ld_32x32(tm + S::col_o + 32 * c, o);
                    tmem_ld_wait();
                }
                if (mine) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4*>(row + 32 * c + 4 * i) = my_steps ? make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]) : make_uint4(0, 0, 0, 0);
                }
            }
            *reinterpret_cast<float2*>(smem + S::stats + (q * kChRows + r) * 8) = make_float2(my_steps ? ref : -INFINITY, my_steps ? sum : 0.f);
        }
    }
    if (splits > 1) {
        // ---- the CTAs' partial results; the rows go round the cluster's warps
        if (warp >= S::softmax_warps) __syncthreads();   // with the softmax warps above
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        constexpr int kWarps = S::threads / 32;
        for (int i = split * kWarps + warp; i < kTiles * kChRows; i += splits * kWarps) {
            const int q = i / kChRows, r = i % kChRows, in_tile = r / group, t = blk.first + q * tile_tokens + in_tile, head = kv * group + r % group;
            if (in_tile >= tile_tokens || t >= blk.len) continue;
            const int end = blk.pos0 < 0 || blk.pos0 > p.max_context - 1 - t ? 0 : blk.pos0 + t + 1;
            float2 st[kChMaxSplits];
            float4 part[kChMaxSplits];
#pragma unroll
            for (int c = 0; c < kChMaxSplits; ++c) {
                const int from = c < splits ? c : 0;
                st[c] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(smem + S::stats + i * 8, from));
                part[c] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(smem + i * S::part_row + lane * 16, from));
                if (c >= splits) st[c] = make_float2(-INFINITY, 0.f);
            }
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < kChMaxSplits; ++c) top = fmaxf(top, st[c].x);
            float total = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < kChMaxSplits; ++c) {
                if (st[c].y == 0.f) continue;   // nothing visible there
                const float f = ex2(st[c].x - top);
                total += f * st[c].y;
                o.x += f * part[c].x, o.y += f * part[c].y, o.z += f * part[c].z, o.w += f * part[c].w;
            }
            const float inv = end == 0 || total == 0.f ? 0.f : 1.f / total;
            o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
            const int row = blk.row0 + t;
            *reinterpret_cast<uint2*>(p.out + (size_t(row) * p.q_heads + head) * kChDim + lane * 4) = make_uint2(bf16x2_of(o.x, o.y), bf16x2_of(o.z, o.w));
            const bool bad = isnan(o.x) || isnan(o.y) || isnan(o.z) || isnan(o.w);
            __syncwarp();
            if (__any_sync(0xffffffffu, bad) && !*abort_flag) chunk_row(p, blk.b, row, head, end - 1, lane);
        }
        cluster.sync();   // peers may still read this CTA's results
    }
    tc_fence_before();
    __syncthreads();
    if (warp == S::mma_warp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, S::cols);
    }
}

// [physical pages x page size] cache rows of kv_heads x 128, boxes of `rows` rows x 64 dims of one kv head, 128-byte swizzle.
int cache_map(CUtensorMap* map, const void* base, const Chunk& p, int rows)
{
    TensorMapEncodeFn enc = tensor_map_encoder();
    if (!enc) return fail(GARNET_B200_NOT_SUPPORTED, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[3] = {kChDim, cuuint64_t(p.kv_heads), cuuint64_t(p.physical_pages) * p.page_size};
    const cuuint64_t strides[2] = {kChDim * 2, cuuint64_t(p.kv_heads) * kChDim * 2};
    const cuuint32_t box[3] = {64, 1, cuuint32_t(rows)}, ones[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GARNET_B200_CUDA_ERROR, "cuTensorMapEncodeTiled (cache) failed with code %d", int(r));
    return GARNET_B200_OK;
}

template <int kTiles, int kKeys, int kSlots>
int launch(const Chunk& p, int splits, cudaStream_t stream)
{
    using S = ChShape<kTiles, kKeys, kSlots>;
    int box = kKeys;   // rows that lie together in every page: the largest power of two that divides the page size, up to a step
    while (p.page_size % box) box /= 2;
    ChMaps maps;
    if (int rc = make_tensor_map_2d_16bit(&maps.q, p.queries, uint64_t(p.tokens) * p.q_heads, kChDim, kChRows)) return rc;
    if (int rc = cache_map(&maps.k, p.keys, p, box)) return rc;
    if (int rc = cache_map(&maps.v, p.values, p, box)) return rc;
    if (int rc = cache_map(&maps.k_row, p.keys, p, 1)) return rc;
    if (int rc = cache_map(&maps.v_row, p.values, p, 1)) return rc;
    const auto kernel = attn_chunk_tc_kernel<kTiles, kKeys, kSlots>;
    GB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::total));
    // blocks of a sequence's rows: ceil(rows / block) summed over the sequences, of whose lengths the host knows the sum's limit only
    const int rows = kChRows / (p.q_heads / p.kv_heads) * kTiles;
    const long long blocks = std::min<long long>(p.tokens, (long long)p.tokens / rows + p.batch);
    if (blocks * p.kv_heads * splits > 0x7fffffffll) return fail(GARNET_B200_NOT_SUPPORTED, "attention_chunk: too many blocks of rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(blocks * p.kv_heads * splits));
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
    GB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p, maps, box, splits));
    return GARNET_B200_OK;
}

}  // namespace

int chunk_attention_launch(const Chunk& p, cudaStream_t stream)
{
    const ChunkPlan plan = chunk_plan(p.batch, p.kv_heads, p.tokens, kChRows / (p.q_heads / p.kv_heads), p.max_context);
    return plan.tiles == 2 ? launch<2, 128, 5>(p, plan.splits, stream) : launch<1, 64, 4>(p, plan.splits, stream);
}

}  // namespace gb200
