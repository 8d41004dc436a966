// Log probabilities of given tokens, their ranks, entropies and the top alternatives of rows of logits.
//
//   z = x / temperature, m = max z, S = sum e^(z - m):   log p(t) = z_t - m - log S,   H = log S - sum e^(z - m) (z - m) / S,
//   rank = 1 + #{x > x_t}.
//
// One CTA per row: the maximum, then the sums and the rank, then one pass over the row for every alternative.
// Bound: HBM in principle (every logit once).
#include <cmath>
#include <cstdint>

#include "common.cuh"

namespace gb200 {

namespace {

constexpr int kLpThreads = 256;
constexpr int kLpMaxTop = 32;

struct LogProbs {
    const void* logits;
    long long stride;
    const int* targets;
    float* log_probs;
    int* ranks;
    float* entropy;
    float* top_log_probs;
    int* top_ids;
    int vocab, top_k;
    float scale;   // 1 / temperature
};

__device__ __forceinline__ float lp_value(const float* x, size_t i) { return x[i]; }
__device__ __forceinline__ float lp_value(const __nv_bfloat16* x, size_t i) { return __bfloat162float(x[i]); }
__device__ __forceinline__ float lp_value(const __half* x, size_t i) { return __half2float(x[i]); }

// Larger for larger values, the same for +0 and -0; 0 for NaN.
__device__ __forceinline__ uint32_t lp_key(float x)
{
    if (isnan(x)) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

template <typename V, typename Op>
__device__ __forceinline__ V lp_reduce(V v, Op op)
{
    __shared__ V part[kLpThreads / 32];
    __shared__ V all;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kLpThreads / 32; ++w) v = op(v, part[w]);
        all = v;
    }
    __syncthreads();
    return all;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) log_probs_kernel(const LogProbs p)
{
    pdl_launch_dependents();
    pdl_wait();
    const size_t r = blockIdx.x;
    const T* row = static_cast<const T*>(p.logits) + r * p.stride;
    const auto larger = [](auto a, auto b) { return a > b ? a : b; };
    const auto plus = [](auto a, auto b) { return a + b; };
    const int target = p.targets ? p.targets[r] : -1;
    const bool given = target >= 0 && target < p.vocab;
    const float x_t = given ? lp_value(row, target) : 0.f;
    float top = -INFINITY;
    for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) top = fmaxf(top, lp_value(row, i));
    top = lp_reduce(top, larger);
    const bool empty = top == -INFINITY;   // a row of -inf (or of -inf and NaN)
    float sum = 0.f, weighted = 0.f;
    int above = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
        const float x = lp_value(row, i);
        above += x > x_t;
        const float d = x == -INFINITY ? -INFINITY : (x - top) * p.scale, e = expf(d);
        sum += e;
        weighted += d == -INFINITY ? 0.f : e * d;
    }
    sum = lp_reduce(sum, plus);
    weighted = lp_reduce(weighted, plus);
    above = lp_reduce(above, plus);
    const float log_sum = logf(sum);
    const auto log_prob = [&](float x) { return isnan(sum) ? sum : empty || x == -INFINITY ? -INFINITY : (x - top) * p.scale - log_sum; };
    if (threadIdx.x == 0) {
        if (p.targets) {
            p.log_probs[r] = given ? log_prob(x_t) : 0.f;
            p.ranks[r] = given ? above + 1 : 0;
        }
        if (p.entropy) p.entropy[r] = isnan(sum) ? sum : empty ? 0.f : log_sum - weighted / sum;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top_k; ++k) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
            const uint32_t key = lp_key(lp_value(row, i));
            const unsigned long long c = (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - uint32_t(i));
            if (key && c < last && c > best) best = c;
        }
        best = lp_reduce(best, larger);
        if (threadIdx.x == 0) {
            p.top_ids[r * p.top_k + k] = best ? int(0xffffffffu - uint32_t(best)) : -1;
            p.top_log_probs[r * p.top_k + k] = best ? log_prob(lp_unkey(uint32_t(best >> 32))) : NAN;
        }
        last = best;
    }
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
    if (!(temperature > 0.f) || !std::isfinite(temperature) || !std::isfinite(1.f / temperature))
        return fail(GARNET_B200_INVALID_VALUE, "log_probs: the temperature must be positive and finite");
    if (!d_targets != !d_log_probs || !d_targets != !d_ranks)
        return fail(GARNET_B200_INVALID_VALUE, "log_probs: targets, log_probs and ranks are given together");
    if (top_k < 0 || top_k > vocab || (top_k > 0 && (!d_top_log_probs || !d_top_ids)))
        return fail(GARNET_B200_INVALID_VALUE, "log_probs: bad top_k %d, or no arrays for it", top_k);
    if (top_k > kLpMaxTop) return fail(GARNET_B200_NOT_SUPPORTED, "log_probs: top_k above %d", kLpMaxTop);
    const LogProbs p{d_logits, row_stride, d_targets, d_log_probs, d_ranks, d_entropy, d_top_log_probs, d_top_ids, vocab, top_k, 1.f / temperature};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(rows));
    cfg.blockDim = dim3(kLpThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = (flags & 1u) ? 1 : 0;
    GB_CUDA(cudaLaunchKernelEx(&cfg, dtype == GARNET_B200_BF16 ? log_probs_kernel<__nv_bfloat16> : dtype == GARNET_B200_FP16 ? log_probs_kernel<__half> : log_probs_kernel<float>, p));
    return GARNET_B200_OK;
}

}  // extern "C"
