// What the chunk attention kernels share: the operands of one call and the addressing of the paged cache.
#pragma once
#include "common.cuh"

namespace gb200 {

constexpr int kChDim = 128;
constexpr int kChTileRows = 128;   // (token, q head of the group) rows of a tile of the attention

// Rows that a CTA of the attention takes: tokens `first` .. of sequence b, which has `len` of them from row `row0` on, the first of
// them at slot pos0; b is -1 where there is nothing to do.
struct alignas(16) ChunkBlock {
    int b, first, len, row0, pos0, unused[3];
};

// Steps of 64 keys whose weights times values are added in the tensor core before the sum is added to those before in fp32.  The tensor
// core cuts what it adds to a sum, eight times a step (16 keys to an MMA, two bf16 numbers to a weight), each time towards zero: sums of
// positive terms lost 2^-28.5 of themselves per key and bf16 number, 2^-12.2 over 65536 keys and one number.  Sixty-four steps lose 2^-15.5,
// a hundredth of the step between two results (8192 rows: 386 us a call with no such limit, 402 with 64 steps, 424 with 32).
constexpr int kChSumSteps = 64;
constexpr int kChSumSlots = 2 * kSmCount;                          // tiles that hold tensor memory at once: a tile has half of an SM's
constexpr size_t kChSumBytes = size_t(kChTileRows) * kChDim * 4;   // a tile's sums

struct Chunk {
    const __nv_bfloat16* qkv;        // [tokens, (q_heads + 2 kv_heads) * 128]
    const __nv_bfloat16* q_norm_w;   // [128]
    const __nv_bfloat16* k_norm_w;
    const float* rope_cos;           // [positions, 64]
    const float* rope_sin;
    __nv_bfloat16* keys;             // [physical pages][page size][kv heads][128]
    __nv_bfloat16* values;
    const int* tables;               // [batch, width]
    const int* positions;            // [batch]: slot of a sequence's first new row
    const int* row_starts;           // [batch + 1]
    __nv_bfloat16* out;              // [tokens, q_heads * 128]
    __nv_bfloat16* queries;          // workspace: [kv head][token][q head of the group][128]
    ChunkBlock* blocks;              // workspace: the attention's blocks of rows, those that see the most keys first
    unsigned* sum_slots;             // workspace: a bit for each of kChSumSlots, set while a tile holds it
    float4* sums;                    // workspace: [slot][4 dims][row], where a context can be that long
    int batch, tokens, q_heads, kv_heads, page_size, width, physical_pages, max_context;
    int block_rows, block_count;     // tokens of a block; entries of `blocks`
    float eps;
};

#if defined(__CUDACC__)
// The sequence of a row, -1 where it has none.
__device__ __forceinline__ int chunk_sequence(const Chunk& p, int row)
{
    int lo = 0, hi = p.batch;   // the last b with row_starts[b] <= row
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.row_starts[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo < p.batch && p.row_starts[lo] <= row && row < p.row_starts[lo + 1] ? lo : -1;
}
// The slot of a row, -1 where it appends and sees nothing.
__device__ __forceinline__ int chunk_slot(const Chunk& p, int b, int row)
{
    const long long slot = (long long)p.positions[b] + (row - p.row_starts[b]);
    return p.positions[b] >= 0 && slot < p.max_context ? int(slot) : -1;
}
// Offset of a slot's K and V of a head; -1 where it has no page.
__device__ __forceinline__ long long chunk_cache_offset(const Chunk& p, int b, int slot, int head)
{
    const int page = p.tables[size_t(b) * p.width + slot / p.page_size];
    if (page < 0 || page >= p.physical_pages) return -1;
    return (((long long)page * p.page_size + slot % p.page_size) * p.kv_heads + head) * kChDim;
}
#endif

struct ChunkPlan;
// attn_chunk_tc.cu: the attention of rows whose queries and blocks lie in the workspace and whose keys and values lie in the cache.
int chunk_attention_launch(const Chunk& p, const ChunkPlan& plan, cudaStream_t stream);

}  // namespace gb200
