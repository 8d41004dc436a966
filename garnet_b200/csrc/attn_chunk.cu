// Attention of a chunk of new tokens of each of several sequences over the paged bf16 KV cache (128-wide heads): the many-row
// companion of the one-token kernel in decode_glue.cu, with the same head norms, RoPE, cache append and score scale
// 1 / sqrt(128) (src/backends/tensorrt/trt_builder.cpp:7565-7726, src/cuda/text_kv_attention_kernel.cu:640-840).
//
// Two launches: attn_chunk_rows_kernel normalises and rotates q and k of every row, appends k and v to the cache and leaves the
// queries in the workspace, a kv head's rows together; the kernel of attn_chunk_tc.cu does the attention.
#include <algorithm>
#include <cstdint>

#include "attn_chunk.cuh"

namespace gb200 {

namespace {

// a cos + b sin with one rounding's error: the second product's own is added back.
__device__ __forceinline__ float turned(float a, float cosine, float b, float sine)
{
    const float p = __fmul_rn(b, sine);
    return __fadd_rn(__fmaf_rn(a, cosine, p), __fmaf_rn(b, sine, -p));
}
__device__ __forceinline__ void unpack(__nv_bfloat162 v, float& a, float& b)
{
    const float2 f = __bfloat1622float2(v);
    a = f.x, b = f.y;
}

// One CTA per row, a warp per head: a lane holds dims 2 lane, 2 lane + 1 and the two 64 further on, which RoPE turns together.
// Rounded to bf16 after the norm and after the rotation, as a bf16 network does; the fp32 steps in between carry what
// their products and the root are short of, and the sum of squares is exact in double: some 1 of 10^6 results is the other bf16
// neighbour of the float64 result (10 to 20 of 10^6 by plain fp32 steps).
__global__ void __launch_bounds__(256) attn_chunk_rows_kernel(const Chunk p)
{
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = chunk_sequence(p, row);
    if (b < 0) return;
    const int slot = chunk_slot(p, b, row);
    if (slot < 0) return;
    const int heads = p.q_heads + 2 * p.kv_heads, group = p.q_heads / p.kv_heads;
    const float2 cs = reinterpret_cast<const float2*>(p.rope_cos + size_t(slot) * (kChDim / 2))[lane];
    const float2 sn = reinterpret_cast<const float2*>(p.rope_sin + size_t(slot) * (kChDim / 2))[lane];
    for (int h = warp; h < heads; h += 8) {
        const __nv_bfloat162* from = reinterpret_cast<const __nv_bfloat162*>(p.qkv + (size_t(row) * heads + h) * kChDim);
        __nv_bfloat162 lo = from[lane], hi = from[lane + 32];
        __nv_bfloat162* to;
        if (h < p.q_heads) {
            to = reinterpret_cast<__nv_bfloat162*>(p.queries + ((size_t(h / group) * p.tokens + row) * group + h % group) * kChDim);
        } else {
            const long long at = chunk_cache_offset(p, b, slot, (h - p.q_heads) % p.kv_heads);
            if (at < 0) continue;
            to = reinterpret_cast<__nv_bfloat162*>((h < p.q_heads + p.kv_heads ? p.keys : p.values) + at);
        }
        if (h < p.q_heads + p.kv_heads) {
            const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(h < p.q_heads ? p.q_norm_w : p.k_norm_w);
            float x[4], wt[4];
            unpack(lo, x[0], x[1]), unpack(hi, x[2], x[3]);
            unpack(w[lane], wt[0], wt[1]), unpack(w[lane + 32], wt[2], wt[3]);
            double mean = double(x[0] * x[0]) + double(x[1] * x[1]) + double(x[2] * x[2]) + double(x[3] * x[3]);   // exact
#pragma unroll
            for (int off = 16; off; off >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, off);
            mean = mean / kChDim + p.eps;
            const float r = 1.f / sqrtf(float(mean));
            const float c = 0.5f * r * float(__fma_rn(-mean, double(r) * r, 1.0));   // what r is short of 1 / sqrt(mean)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = __fmul_rn(x[i], wt[i]);   // exact: two bf16 numbers
                x[i] = bf16_round_f(__fmaf_rn(v, r, __fmul_rn(v, c)));
            }
            lo = __floats2bfloat162_rn(turned(x[0], cs.x, -x[2], sn.x), turned(x[1], cs.y, -x[3], sn.y));
            hi = __floats2bfloat162_rn(turned(x[2], cs.x, x[0], sn.x), turned(x[3], cs.y, x[1], sn.y));
        }
        to[lane] = lo, to[lane + 32] = hi;
    }
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

size_t chunk_workspace(const garnet_b200_attention_options& o, int tokens) { return size_t(tokens) * o.q_heads * kChDim * 2; }

cudaError_t chunk_launch(void (*kernel)(Chunk), dim3 grid, cudaStream_t stream, bool dependent, const Chunk& p)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

}  // namespace gb200

using namespace gb200;

extern "C" {

int garnet_b200_attention_chunk_workspace(const garnet_b200_attention_options* o, int tokens, size_t* bytes)
{
    if (int rc = validate_chunk(o)) return rc;
    if (!bytes || tokens <= 0) return fail(GARNET_B200_INVALID_VALUE, "attention_chunk_workspace: bad argument");
    *bytes = chunk_workspace(*o, tokens);
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
    if (!d_workspace || workspace_bytes < chunk_workspace(*o, tokens) || (reinterpret_cast<uintptr_t>(d_workspace) & 255))
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: the workspace is missing, too small (%zu < %zu) or not 256-byte aligned", workspace_bytes,
                    chunk_workspace(*o, tokens));
    if ((reinterpret_cast<uintptr_t>(d_qkv) | reinterpret_cast<uintptr_t>(d_key_pages) | reinterpret_cast<uintptr_t>(d_value_pages) |
         reinterpret_cast<uintptr_t>(d_out) | reinterpret_cast<uintptr_t>(d_rope_cos) | reinterpret_cast<uintptr_t>(d_rope_sin)) & 15)
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: rows, cache pages, rope tables and output must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(d_q_norm_weight) | reinterpret_cast<uintptr_t>(d_k_norm_weight)) & 3)
        return fail(GARNET_B200_INVALID_VALUE, "attention_chunk: the norm weights must be 4-byte aligned");
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
    p.queries = static_cast<__nv_bfloat16*>(d_workspace);
    p.batch = batch, p.tokens = tokens, p.q_heads = o->q_heads, p.kv_heads = o->kv_heads, p.page_size = o->page_size;
    p.width = o->max_logical_pages, p.physical_pages = physical_pages, p.max_context = o->max_context;
    p.eps = o->norm_eps;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    GB_CUDA(chunk_launch(attn_chunk_rows_kernel, dim3(unsigned(tokens)), s, (flags & 1u) != 0, p));
    return chunk_attention_launch(p, s);
}

}  // extern "C"
