// Attention of a chunk of new tokens of each of several sequences over the paged bf16 KV cache (128-wide heads): the many-row
// companion of the one-token kernel in decode_glue.cu, with the same head norms, RoPE, cache append and score scale
// 1 / sqrt(128) (src/backends/tensorrt/trt_builder.cpp:7565-7726, src/cuda/text_kv_attention_kernel.cu:640-840).
//
// Two launches: attn_chunk_rows_kernel normalises and rotates q and k of every row, appends k and v to the cache and leaves the
// queries in the workspace, a kv head's rows together; the kernel of attn_chunk_tc.cu does the attention.
#include <algorithm>
#include <cstdint>

#include "attn_chunk.cuh"
#include "tc_common.cuh"

namespace gb200 {

namespace {

// a cos + b sin of two values at once with one rounding's error: what the second product is short of is added back.
__device__ __forceinline__ uint64_t turned(uint64_t a, uint64_t cosine, uint64_t b, uint64_t sine, uint64_t minus_sine)
{
    const uint64_t p = mul2(b, sine);
    return fma2(fma2(b, minus_sine, p), f32x2(-1.f, -1.f), fma2(a, cosine, p));
}
// two bf16 numbers as two fp32 numbers; and rounded back
__device__ __forceinline__ uint64_t wide(uint32_t w) { return f32x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t narrow(uint64_t v)
{
    float lo, hi;
    f32x2_split(v, lo, hi);
    return bf16x2_of(lo, hi);
}

// A warp takes four heads of a row, eight lanes each: dims 8 l .. 8 l + 7 and the eight 64 further on, which RoPE turns together.
// Rounded to bf16 after the norm and after the rotation, as a bf16 network does; the fp32 steps in between carry what the sum of
// squares, the products and the root are short of: of 10^6 keys of normal rows 1.7 differ from the float64 result rounded to fp32 and then to
// bf16 (25 by plain fp32 steps).
// Bound: HBM in principle, the rows in and q, k and v out; in practice its instructions, some 250 for four heads with two values to an
// instruction.
constexpr int kRowThreads = 128;

// One CTA beside the rows': the attention's blocks of rows by the keys that they see, the most first, so that the last CTAs to start
// are short ones (24 ragged sequences of 5 rows at up to 3500: 45 instead of 65 us, a ragged batch of 8 prompts 58 instead of 74 us with
// the sequences in their own order, before weights entered as two numbers).  A counting sort; blocks that see equally much (within 1 / 511 of max_context) come in any order.
constexpr int kOrderBuckets = 4 * kRowThreads;
__device__ __forceinline__ void chunk_order(const Chunk& p)
{
    __shared__ int places[kOrderBuckets], sums[kRowThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < (kChSumSlots + 31) / 32) p.sum_slots[threadIdx.x] = 0;   // beside it: nobody holds a slot yet
    for (int i = threadIdx.x; i < kOrderBuckets; i += kRowThreads) places[i] = 0;
    __syncthreads();
    const auto every_block = [&](auto&& take) {   // take(block, its bucket)
        for (int b0 = 0; b0 < p.batch; b0 += kRowThreads) {
            const int b = b0 + int(threadIdx.x);
            int row0 = 0, len = 0, pos0 = 0;
            if (b < p.batch) {
                row0 = min(max(p.row_starts[b], 0), p.tokens);
                len = min(max(p.row_starts[b + 1], row0), p.tokens) - row0;
                pos0 = p.positions[b];
            }
            const int n = (len + p.block_rows - 1) / p.block_rows;
            const auto one = [&](int b, int row0, int len, int pos0, int k) {
                const int first = k * p.block_rows;
                const long long end = pos0 < 0 || pos0 > p.max_context - 1 - first ? 0 : min((long long)p.max_context, (long long)pos0 + min(len, first + p.block_rows));
                take(ChunkBlock{b, first, len, row0, pos0, {}}, kOrderBuckets - 1 - int(end * (kOrderBuckets - 1) / p.max_context));
            };
            if (n == 1) one(b, row0, len, pos0, 0);
            for (uint32_t many = __ballot_sync(0xffffffffu, n > 1); many; many &= many - 1) {   // the warp together
                const int from = __ffs(many) - 1, of = __shfl_sync(0xffffffffu, n, from), r0 = __shfl_sync(0xffffffffu, row0, from);
                const int l = __shfl_sync(0xffffffffu, len, from), p0 = __shfl_sync(0xffffffffu, pos0, from);
                for (int k = lane; k < of; k += 32) one(b0 + warp * 32 + from, r0, l, p0, k);
            }
        }
    };
    every_block([&](const ChunkBlock&, int bucket) { atomicAdd(&places[bucket], 1); });
    __syncthreads();
    // a bucket's first place: the blocks of those before it
    int mine[4], total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) mine[i] = total, total += places[4 * threadIdx.x + i];
    int upto = total;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int before = upto - total, all = 0;
#pragma unroll
    for (int w = 0; w < kRowThreads / 32; ++w) before += w < warp ? sums[w] : 0, all += sums[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) places[4 * threadIdx.x + i] = before + mine[i];
    __syncthreads();
    every_block([&](const ChunkBlock& block, int bucket) {
        const int at = atomicAdd(&places[bucket], 1);
        if (at < p.block_count) p.blocks[at] = block;   // lists that do not ascend may ask for more
    });
    for (int i = all + int(threadIdx.x); i < p.block_count; i += kRowThreads) p.blocks[i].b = -1;
}

__global__ void __launch_bounds__(kRowThreads, 8) attn_chunk_rows_kernel(const Chunk p, const int early)
{
    // few rows: the attention's CTAs come up beside these; many: they would only take their place
    if (early) pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0) {
        chunk_order(p);
        if (!early) pdl_launch_dependents();
        return;
    }
    const int lane = threadIdx.x & 31, l = lane & 7, heads = p.q_heads + 2 * p.kv_heads, quads = (heads + 3) / 4, group = p.q_heads / p.kv_heads;
    const long long task = (long long)(blockIdx.x - 1) * (kRowThreads / 32) + (threadIdx.x >> 5);
    const int row = int(task / quads), h = int(task % quads) * 4 + (lane >> 3);
    if (row >= p.tokens) return;
    const bool has = h < heads, is_q = h < p.q_heads, turns = h < p.q_heads + p.kv_heads;
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo, wlo = lo, whi = lo;
    if (has) {
        const uint4* from = reinterpret_cast<const uint4*>(p.qkv + (size_t(row) * heads + h) * kChDim);
        lo = __ldg(from + l), hi = __ldg(from + 8 + l);
    }
    if (turns) {
        const uint4* w = reinterpret_cast<const uint4*>(is_q ? p.q_norm_w : p.k_norm_w);
        wlo = __ldg(w + l), whi = __ldg(w + 8 + l);
    }
    const int b = chunk_sequence(p, row);
    const int slot = b < 0 ? -1 : chunk_slot(p, b, row);
    if (slot < 0) return;   // the whole warp
    float4 cs[2], sn[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        cs[i] = __ldg(reinterpret_cast<const float4*>(p.rope_cos + size_t(slot) * (kChDim / 2)) + 2 * l + i);
        sn[i] = __ldg(reinterpret_cast<const float4*>(p.rope_sin + size_t(slot) * (kChDim / 2)) + 2 * l + i);
    }
    uint4* to = nullptr;
    if (is_q) {
        to = reinterpret_cast<uint4*>(p.queries + ((size_t(h / group) * p.tokens + row) * group + h % group) * kChDim);
    } else if (has) {
        const long long at = chunk_cache_offset(p, b, slot, (h - p.q_heads) % p.kv_heads);
        if (at >= 0) to = reinterpret_cast<uint4*>((turns ? p.keys : p.values) + at);
    }
    if (__any_sync(0xffffffffu, turns)) {
        // packed: dims 8 l + 2 i, 8 l + 2 i + 1, and from i = 4 on those 64 further on
        const uint32_t xs[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        uint32_t ws[8] = {wlo.x, wlo.y, wlo.z, wlo.w, whi.x, whi.y, whi.z, whi.w};
        const uint64_t minus1 = f32x2(-1.f, -1.f);
        uint64_t sum2 = 0, rest2 = 0;   // the sum of squares and what it is short of
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint64_t x = wide(xs[i]), next = fma2(x, x, sum2);
            rest2 = add2(rest2, fma2(x, x, fma2(next, minus1, sum2)));
            sum2 = next;
        }
        float sum, rest;
        {
            float s0, s1, r0, r1;
            f32x2_split(sum2, s0, s1), f32x2_split(rest2, r0, r1);
            const float a = fmaxf(s0, s1), c = fminf(s0, s1);
            sum = __fadd_rn(a, c);
            rest = r0 + r1 + __fsub_rn(c, __fsub_rn(sum, a));
        }
#pragma unroll
        for (int off = 4; off; off >>= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, sum, off), a = fmaxf(sum, other), c = fminf(sum, other);
            rest += __shfl_xor_sync(0xffffffffu, rest, off);
            sum = __fadd_rn(a, c);
            rest = __fadd_rn(rest, __fsub_rn(c, __fsub_rn(sum, a)));
        }
        const float high = sum * (1.f / kChDim), low = __fmaf_rn(rest, 1.f / kChDim, p.eps), mean = __fadd_rn(high, low);
        const float short_of = __fsub_rn(low, __fsub_rn(mean, high));
        float r = 1.f / sqrtf(mean);
        const float square = __fmul_rn(mean, r);
        // what r is short of 1 / sqrt(mean)
        float c = 0.5f * r * (__fmaf_rn(-square, r, 1.f) - __fmaf_rn(mean, r, -square) * r - short_of * r * r);
        if (sum == INFINITY) {   // squares beyond fp32: numbers become 0, infinities NaN
            r = c = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ws[i] = 0x3f803f80u;   // one: a product with the weight could be infinite
        }
        if (turns) {
            const uint64_t r2 = f32x2(r, r), c2 = f32x2(c, c);
            uint64_t n[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint64_t v = mul2(wide(xs[i]), wide(ws[i]));   // exact: products of two bf16 numbers
                n[i] = wide(narrow(fma2(v, r2, mul2(v, c2))));
            }
            uint32_t y[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float* cosine = reinterpret_cast<const float*>(cs) + 2 * i;
                const float* sine = reinterpret_cast<const float*>(sn) + 2 * i;
                const uint64_t c2 = f32x2(cosine[0], cosine[1]), s2 = f32x2(sine[0], sine[1]), m2 = f32x2(-sine[0], -sine[1]);
                y[i] = narrow(turned(n[i], c2, n[i + 4], m2, s2));
                y[i + 4] = narrow(turned(n[i + 4], c2, n[i], s2, m2));
            }
            lo = make_uint4(y[0], y[1], y[2], y[3]), hi = make_uint4(y[4], y[5], y[6], y[7]);
        }
    }
    if (to) to[l] = lo, to[8 + l] = hi;
    if (!early) pdl_launch_dependents();
}

int validate_chunk(const garnet_b200_attention_options* o)
{
    if (!o) return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: null options");
    if (o->abi != GARNET_B200_ABI || o->struct_size != int(sizeof(garnet_b200_attention_options)))
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: options abi/size mismatch (abi %d, size %d)", o->abi, o->struct_size);
    if (o->head_dim != kChDim) return fail(GARNET_B200_NOT_SUPPORTED, "attention_chunk: head_dim must be %d", kChDim);
    if (o->q_heads <= 0 || o->kv_heads <= 0 || o->q_heads % o->kv_heads)
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: q_heads must be a positive multiple of kv_heads");
    if (o->q_heads / o->kv_heads > 128) return fail(GARNET_B200_NOT_SUPPORTED, "attention_chunk: more than 128 q heads per kv head");
    if (o->page_size <= 0 || o->max_logical_pages <= 0 || o->max_context <= 0 || o->rope_positions <= 0 || !(o->norm_eps > 0.f))
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: page_size, max_logical_pages, max_context, rope_positions and norm_eps must be positive");
    if (o->max_context > (long long)o->max_logical_pages * o->page_size || o->max_context > o->rope_positions)
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: max_context exceeds the page table or the rope tables");
    return GARNET_B200_OK;
}

// The workspace: queries, a block's entry per row at most, the slots' bits, and sums where a context is long enough for them.
struct ChunkSpace {
    size_t blocks, slots, sums, bytes;
};
ChunkSpace chunk_space(const garnet_b200_attention_options& o, int tokens)
{
    ChunkSpace s;
    s.blocks = size_t(tokens) * o.q_heads * kChDim * 2;
    s.slots = s.blocks + size_t(tokens) * sizeof(ChunkBlock);
    s.sums = (s.slots + (kChSumSlots + 31) / 32 * 4 + 255) & ~size_t(255);
    s.bytes = s.sums + (o.max_context > kChSumSteps * 64 ? kChSumSlots * kChSumBytes : 0);
    return s;
}

}  // namespace

}  // namespace gb200

using namespace gb200;

extern "C" {

int garnet_b200_attention_chunk_workspace(const garnet_b200_attention_options* o, int tokens, size_t* bytes)
{
    if (int rc = validate_chunk(o)) return rc;
    if (!bytes || tokens <= 0) return fail(GARNET_B200_INVALID_VALUE, "attention_chunk_workspace: bad argument");
    *bytes = chunk_space(*o, tokens).bytes;
    return GARNET_B200_OK;
}

int garnet_b200_attention_chunk(const garnet_b200_attention_options* o, const void* d_qkv, const void* d_q_norm_weight,
                                const void* d_k_norm_weight, const float* d_rope_cos, const float* d_rope_sin, void* d_key_pages,
                                void* d_value_pages, const int* d_page_tables, const int* d_positions, const int* d_row_starts,
                                void* d_out, void* d_workspace, size_t workspace_bytes, int batch, int tokens, int physical_pages,
                                unsigned flags, void* stream)
{
    if (int rc = validate_chunk(o)) return rc;
    if (!d_qkv || !d_q_norm_weight || !d_k_norm_weight || !d_rope_cos || !d_rope_sin || !d_key_pages || !d_value_pages || !d_page_tables ||
        !d_positions || !d_row_starts || !d_out || batch <= 0 || tokens <= 0 || physical_pages <= 0)
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: null pointer, or batch, tokens or physical_pages not positive");
    const ChunkSpace space = chunk_space(*o, tokens);
    if (!d_workspace || workspace_bytes < space.bytes || (reinterpret_cast<uintptr_t>(d_workspace) & 255))
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: the workspace is missing, too small (%zu < %zu) or not 256-byte aligned", workspace_bytes,
                    space.bytes);
    if ((reinterpret_cast<uintptr_t>(d_qkv) | reinterpret_cast<uintptr_t>(d_key_pages) | reinterpret_cast<uintptr_t>(d_value_pages) |
         reinterpret_cast<uintptr_t>(d_out) | reinterpret_cast<uintptr_t>(d_rope_cos) | reinterpret_cast<uintptr_t>(d_rope_sin) |
         reinterpret_cast<uintptr_t>(d_q_norm_weight) | reinterpret_cast<uintptr_t>(d_k_norm_weight)) & 15)
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: rows, cache pages, norm weights, rope tables and output must be 16-byte aligned");
    if ((long long)physical_pages * o->page_size > 0x7fff0000ll || (long long)tokens * o->q_heads > 0x7fff0000ll)
        return fail(GARNET_B200_NOT_SUPPORTED, "attention_chunk: more than 2^31 cache slots or query rows");
    Chunk p;
    p.qkv = static_cast<const __nv_bfloat16*>(d_qkv);
    p.q_norm_w = static_cast<const __nv_bfloat16*>(d_q_norm_weight);
    p.k_norm_w = static_cast<const __nv_bfloat16*>(d_k_norm_weight);
    p.rope_cos = d_rope_cos, p.rope_sin = d_rope_sin;
    p.keys = static_cast<__nv_bfloat16*>(d_key_pages);
    p.values = static_cast<__nv_bfloat16*>(d_value_pages);
    p.tables = d_page_tables, p.positions = d_positions, p.row_starts = d_row_starts;
    p.out = static_cast<__nv_bfloat16*>(d_out);
    char* ws = static_cast<char*>(d_workspace);
    p.queries = reinterpret_cast<__nv_bfloat16*>(ws);
    p.blocks = reinterpret_cast<ChunkBlock*>(ws + space.blocks);
    p.sum_slots = reinterpret_cast<unsigned*>(ws + space.slots);
    p.sums = reinterpret_cast<float4*>(ws + space.sums);
    p.batch = batch, p.tokens = tokens, p.q_heads = o->q_heads, p.kv_heads = o->kv_heads, p.page_size = o->page_size;
    p.width = o->max_logical_pages, p.physical_pages = physical_pages, p.max_context = o->max_context;
    p.eps = o->norm_eps;
    const int tile_tokens = kChTileRows / (o->q_heads / o->kv_heads);
    const ChunkPlan plan = chunk_plan(batch, o->kv_heads, tokens, tile_tokens, o->max_context);
    p.block_rows = tile_tokens * plan.tiles;
    // blocks of a sequence's rows: ceil(rows / block) summed over the sequences, of whose lengths the host knows the sum's limit only
    p.block_count = int(std::min<long long>(tokens, (long long)tokens / p.block_rows + batch));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long long warps = (long long)tokens * ((o->q_heads + 2 * o->kv_heads + 3) / 4), ctas = (warps * 32 + kRowThreads - 1) / kRowThreads + 1;
    if (ctas > 0x7fffffffll) return fail(GARNET_B200_NOT_SUPPORTED, "attention_chunk: too many rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ctas));
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = (flags & 1u) ? 1 : 0;
    GB_CUDA(cudaLaunchKernelEx(&cfg, attn_chunk_rows_kernel, p, int(ctas <= 4 * kSmCount)));
    return chunk_attention_launch(p, plan, s);
}

}  // extern "C"
