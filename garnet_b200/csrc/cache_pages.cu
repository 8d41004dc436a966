// The pages of a paged KV cache: handed out to sequences, shared by forked ones, taken back, moved together and copied.
//
// The state is three integer tables in device memory, owned by the caller: the page table that the attention kernels read, the
// positions that every sequence holds, and how many table entries refer to each physical page (0: the page is free).  All of it
// is integer arithmetic with one outcome, whatever the order in which threads run: pages are given out by ascending page number
// in the order of the list, moved pages keep their order.
//
//   extend   sequence s grows by n positions: ceil((len + n) / page) - ceil(len / page) pages, the lowest free ones
//   fork     a child gets its parent's full pages (one more reference each) and a copy of the positions in its last, partial one
//   free     one reference less for every page of the sequence, the row emptied
//   compact  the i-th live page with a number >= the count of live pages moves to the i-th free page below it
//   copy     pages src[i] -> dst[i] in the order of the list
//
// Bound: what moves pages, HBM (two times the bytes of the pages); the rest, the latency of a chain of a few dependent loads: one
// CTA decides (page lists have one order), and a second launch over the whole GPU moves pages and rewrites tables.  B200: 28 layers of
// 1400 pages of 16 x 8 x 128 bf16, half of them live and scattered, moved together in 234 us (0.84 of the measured copy bandwidth, 1.28 GB),
// 400 of them copied in 251 us (0.89), 16 in 11.5 us (0.78), 16 of 60000 pages of two layers in 3 us; 32 sequences get up to 1500 positions each
// out of 20000 pages and give them back in 15 us, 8 forks of up to 1100 positions and their release take 13 us.
#include <algorithm>
#include <climits>
#include <cstdint>

#include "common.cuh"

namespace gb200 {

namespace {

constexpr int kPoolMaxLayers = 128;
constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr int kCopyThreads = 256, kCopyUnits = 4;                         // 16-byte units of a thread at a time
constexpr int kCopyChunk = kCopyThreads * kCopyUnits;                    // units that a CTA moves at a time (16 KB)
constexpr int kCopyCtas = 8 * kSmCount;
constexpr int kPoolMaxBitmap = 192 * 1024;

struct PoolLayers {
    uint4* pages[2 * kPoolMaxLayers];   // key pages of a layer, value pages of a layer
    int buffers;                        // 2 x layers
    int units_per_token;                // 16-byte units of a position
    int page_size;
    int physical_pages;
};

struct PoolTables {
    int* table;       // [sequences, width]
    int* lengths;     // [sequences]
    int* refs;        // [physical pages]
    int sequences, width, page_size, physical_pages;
};

// Workspace of a call, in ints: claims of the sequences, what a list entry was granted, page lists.
struct PoolWork {
    int* claim;       // [sequences]: first entry that names the sequence
    int* first;       // [count]: extend and fork: pages handed out before this entry's, -1 where the entry is refused
    int* need;        // [count]
    int* page;        // [count]: fork: the new page, -1 where there is none
    int* ids;         // [physical pages]: free pages in order; compact: source pages of the moves
    int* dst;         // [physical pages]: compact: destinations of the moves
    int* map;         // [physical pages]: compact: new number of a page, for those with the number `map_from` or more
    int* moves;       // [1]
    int map_from;     // -1: the count of live pages
};

size_t align64(size_t n) { return (n + 63) & ~size_t(63); }
size_t pool_workspace(const garnet_b200_cache_options& o, int count)
{
    return (align64(size_t(o.sequences)) + 3 * align64(size_t(count)) + 3 * align64(size_t(o.physical_pages)) + 64) * sizeof(int);
}
PoolWork pool_work(const garnet_b200_cache_options& o, int count, void* ws)
{
    PoolWork w;
    int* at = static_cast<int*>(ws);
    const auto take = [&](size_t n) {
        int* p = at;
        at += align64(n);
        return p;
    };
    w.claim = take(size_t(o.sequences));
    w.first = take(size_t(count)), w.need = take(size_t(count)), w.page = take(size_t(count));
    w.ids = take(size_t(o.physical_pages)), w.dst = take(size_t(o.physical_pages)), w.map = take(size_t(o.physical_pages));
    w.moves = take(1);
    w.map_from = -1;
    return w;
}

__device__ __forceinline__ int pages_of(int positions, int page_size) { return positions <= 0 ? 0 : (positions - 1) / page_size + 1; }

// Sum of v over the CTA's threads before this one, and over all of them.
__device__ __forceinline__ long long scan_before(long long v, long long& total)
{
    __shared__ long long sums[kPlanWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long upto = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    long long w = lane < kPlanWarps ? sums[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, w, d);
        if (lane >= d) w += o;
    }
    total = __shfl_sync(0xffffffffu, w, kPlanWarps - 1);
    const long long before = warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
    __syncthreads();
    return before + upto - v;
}

// A warp's share of the pages [from, to), a multiple of 32 pages but for the last warp's.
__device__ __forceinline__ void page_share(int pages, int& from, int& to)
{
    const int words = (pages + 31) / 32, per = (words + kPlanWarps - 1) / kPlanWarps, warp = threadIdx.x >> 5;
    from = min(pages, warp * per * 32), to = min(pages, (warp + 1) * per * 32);
}

// Pages of [from, to) whose reference count is zero (free) or not, counted by a warp.
__device__ __forceinline__ int count_pages(const int* refs, int from, int to, bool free_ones)
{
    int n = 0;
#pragma unroll 8
    for (int p = from + int(threadIdx.x & 31); p < to; p += 32) n += (refs[p] <= 0) == free_ones;
    return __reduce_add_sync(0xffffffffu, n);
}

// Page numbers of [from, to) of that kind in ascending order to list[at], list[at + 1], ... as far as `most` entries of the list.
__device__ __forceinline__ void list_pages(const int* refs, int from, int to, bool free_ones, int* list, long long at, long long most)
{
    const int lane = threadIdx.x & 31;
#pragma unroll 4
    for (int p0 = from; p0 < to; p0 += 32) {
        const int p = p0 + lane;
        const bool is = p < to && (refs[p] <= 0) == free_ones;
        const uint32_t bits = __ballot_sync(0xffffffffu, is);
        const long long to_at = at + __popc(bits & ((1u << lane) - 1u));
        if (is && to_at < most) list[to_at] = p;
        at += __popc(bits);
        if (at >= most) break;
    }
}

// What extend and fork ask for, per entry: pages needed, -1 for an entry that is refused.
struct ExtendAsk {
    PoolTables t;
    const int* sequences;
    const int* tokens;

    __device__ int subject(int i) const { return sequences[i]; }
    __device__ int other(int) const { return -1; }
    __device__ int need(int i, const int* claim) const
    {
        const int s = sequences[i], n = tokens[i];
        if (s < 0 || s >= t.sequences || __ldcg(&claim[s]) != i || n < 0) return -1;
        const int len = t.lengths[s];
        if (len < 0 || (long long)len + n > min((long long)t.width * t.page_size, (long long)INT_MAX)) return -1;
        return pages_of(len + n, t.page_size) - pages_of(len, t.page_size);
    }
};
struct ForkAsk {
    PoolTables t;
    const int* parents;
    const int* children;

    __device__ int subject(int i) const { return children[i]; }
    __device__ int other(int i) const { return parents[i]; }
    __device__ int need(int i, const int* claim) const
    {
        const int p = parents[i], c = children[i];
        if (p < 0 || p >= t.sequences || c < 0 || c >= t.sequences || __ldcg(&claim[c]) != i || __ldcg(&claim[p]) != INT_MAX) return -1;
        const int len = t.lengths[p];
        if (t.lengths[c] != 0 || len < 0 || pages_of(len, t.page_size) > t.width) return -1;
        return len % t.page_size ? 1 : 0;
    }
};

// One CTA: checks the entries, adds up what they need, finds that many free pages and takes them.
template <typename Ask>
__device__ void grant(const Ask& ask, const PoolWork& w, int* status, int count)
{
    __shared__ int free_of[kPlanWarps];
    __shared__ long long wanted;
    const PoolTables& t = ask.t;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const auto named = [&](int s) { return s >= 0 && s < t.sequences; };
    for (int i = threadIdx.x; i < count; i += kPlanThreads) {
        if (named(ask.subject(i))) w.claim[ask.subject(i)] = INT_MAX;
        if (named(ask.other(i))) w.claim[ask.other(i)] = INT_MAX;
    }
    if (threadIdx.x == 0) wanted = 0;
    int from, to;
    page_share(t.physical_pages, from, to);
    const int mine = count_pages(t.refs, from, to, true);
    if (lane == 0) free_of[warp] = mine;
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += kPlanThreads)
        if (named(ask.subject(i))) atomicMin(&w.claim[ask.subject(i)], i);
    long long free_before = 0, free_pages = 0;
    for (int k = 0; k < kPlanWarps; ++k) {
        if (k < warp) free_before += free_of[k];
        free_pages += free_of[k];
    }
    __syncthreads();
    long long base = 0;
    for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
        const int i = i0 + int(threadIdx.x);
        const int need = i < count ? ask.need(i, w.claim) : -1;
        long long total;
        const long long before = base + scan_before(max(need, 0), total);
        base += total;
        if (i < count) {
            const bool enough = need <= 0 || before + need <= free_pages;
            w.first[i] = need < 0 || !enough ? -1 : int(min(before, (long long)INT_MAX));
            w.need[i] = max(need, 0);
            status[i] = need < 0 ? GARNET_B200_INVALID_VALUE : enough ? GARNET_B200_OK : GARNET_B200_OUT_OF_MEMORY;
            if (need > 0 && enough) atomicMax(&wanted, before + need);
        }
    }
    __syncthreads();
    if (free_before < wanted) list_pages(t.refs, from, to, true, w.ids, free_before, wanted);
    __syncthreads();
    for (int i = threadIdx.x; i < wanted; i += kPlanThreads) t.refs[__ldcg(&w.ids[i])] = 1;
}

__global__ void __launch_bounds__(kPlanThreads) pool_extend_kernel(const ExtendAsk ask, const PoolWork w, int* status, int count)
{
    grant(ask, w, status, count);
    const PoolTables& t = ask.t;
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < count; i += kPlanWarps) {
        const int first = __ldcg(&w.first[i]);
        if (first < 0) continue;
        const int s = ask.sequences[i], need = __ldcg(&w.need[i]), len = t.lengths[s];
        int* row = t.table + size_t(s) * t.width + pages_of(len, t.page_size);
        for (int j = lane; j < need; j += 32) row[j] = __ldcg(&w.ids[first + j]);
        __syncwarp();
        if (lane == 0) t.lengths[s] = len + ask.tokens[i];
    }
}

__global__ void __launch_bounds__(kPlanThreads) pool_fork_plan_kernel(const ForkAsk ask, const PoolWork w, int* status, int count)
{
    pdl_launch_dependents();
    grant(ask, w, status, count);
    for (int i = threadIdx.x; i < count; i += kPlanThreads) {
        const int first = __ldcg(&w.first[i]);
        w.page[i] = first >= 0 && __ldcg(&w.need[i]) ? __ldcg(&w.ids[first]) : -1;
    }
}

// Units [chunk * kCopyChunk, + kCopyChunk) of a page of `units` 16-byte units in one buffer, four loads ahead of their stores.
__device__ __forceinline__ void copy_chunk(const uint4* src, uint4* dst, int chunk, int units)
{
    uint4 v[kCopyUnits];
    const int at = chunk * kCopyChunk + int(threadIdx.x);
#pragma unroll
    for (int k = 0; k < kCopyUnits; ++k)
        if (at + k * kCopyThreads < units) v[k] = src[at + k * kCopyThreads];
#pragma unroll
    for (int k = 0; k < kCopyUnits; ++k)
        if (at + k * kCopyThreads < units) dst[at + k * kCopyThreads] = v[k];
}

// blockIdx.y: entry of the list; blockIdx.x: share of its page table row and of its page's buffers.
__global__ void __launch_bounds__(kCopyThreads) pool_fork_kernel(const __grid_constant__ PoolLayers layers, const ForkAsk ask, const PoolWork w, int count)
{
    pdl_wait();
    const PoolTables& t = ask.t;
    for (int i = blockIdx.y; i < count; i += gridDim.y) {
        if (w.first[i] < 0) continue;
        const int p = ask.parents[i], c = ask.children[i], len = t.lengths[p], full = len / t.page_size, part = len % t.page_size;
        const int* from = t.table + size_t(p) * t.width;
        int* row = t.table + size_t(c) * t.width;
        for (int j = blockIdx.x * kCopyThreads + threadIdx.x; j < full; j += gridDim.x * kCopyThreads) {
            const int page = from[j];
            row[j] = page;
            if (page >= 0 && page < t.physical_pages) atomicAdd(&t.refs[page], 1);
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            if (part) row[full] = w.page[i];
            t.lengths[c] = len;
        }
        if (!part) continue;
        const int src = from[full], dst = w.page[i];
        if (src < 0 || src >= t.physical_pages) continue;
        const int units = part * layers.units_per_token, chunks = (units + kCopyChunk - 1) / kCopyChunk;
        const size_t page_units = size_t(t.page_size) * layers.units_per_token;
        for (int k = blockIdx.x; k < layers.buffers * chunks; k += gridDim.x) {
            uint4* buffer = layers.pages[k / chunks];
            copy_chunk(buffer + src * page_units, buffer + dst * page_units, k % chunks, units);
        }
    }
}

__global__ void __launch_bounds__(256) pool_free_kernel(const PoolTables t, const int* sequences)
{
    __shared__ int held;
    const int s = sequences[blockIdx.x];
    if (s < 0 || s >= t.sequences) return;
    if (threadIdx.x == 0) held = min(pages_of(atomicExch(&t.lengths[s], 0), t.page_size), t.width);   // an entry named twice is freed once
    __syncthreads();
    int* row = t.table + size_t(s) * t.width;
    for (int j = threadIdx.x; j < held; j += 256) {
        const int page = row[j];
        row[j] = -1;
        if (page >= 0 && page < t.physical_pages) atomicSub(&t.refs[page], 1);
    }
}

__global__ void __launch_bounds__(kPlanThreads) pool_compact_plan_kernel(const PoolTables t, const PoolWork w, int* live_out)
{
    __shared__ int live_of[kPlanWarps], holes_of[kPlanWarps];
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int from, to;
    page_share(t.physical_pages, from, to);
    const int mine = count_pages(t.refs, from, to, false);
    if (lane == 0) live_of[warp] = mine;
    __syncthreads();
    int live = 0;
    for (int k = 0; k < kPlanWarps; ++k) live += live_of[k];
    // free pages below `live`, live pages from there on: as many of the one as of the other
    const int below = min(to, live), above = max(from, live);
    const int holes = count_pages(t.refs, from, below, true);
    if (lane == 0) holes_of[warp] = holes;
    const int movers = count_pages(t.refs, above, to, false);
    __syncthreads();
    if (lane == 0) live_of[warp] = movers;
    __syncthreads();
    int holes_before = 0, movers_before = 0, moves = 0;
    for (int k = 0; k < kPlanWarps; ++k) {
        if (k < warp) holes_before += holes_of[k], movers_before += live_of[k];
        moves += holes_of[k];
    }
    list_pages(t.refs, from, below, true, w.dst, holes_before, moves);
    list_pages(t.refs, above, to, false, w.ids, movers_before, moves);
    for (int p = (w.map_from < 0 ? live : w.map_from) + int(threadIdx.x); p < t.physical_pages; p += kPlanThreads) w.map[p] = p;
    __syncthreads();
    for (int i = threadIdx.x; i < moves; i += kPlanThreads) {
        const int src = __ldcg(&w.ids[i]), dst = __ldcg(&w.dst[i]);
        w.map[src] = dst;
        t.refs[dst] = t.refs[src];
        t.refs[src] = 0;
    }
    if (threadIdx.x == 0) *w.moves = moves, *live_out = live;
}

__global__ void __launch_bounds__(kCopyThreads) pool_compact_kernel(const __grid_constant__ PoolLayers layers, const PoolTables t, const PoolWork w, const int* live_in)
{
    pdl_wait();
    const int moves = *w.moves, live = *live_in;
    if (!moves) return;
    const size_t entries = size_t(t.sequences) * t.width;
    for (size_t e = size_t(blockIdx.x) * kCopyThreads + threadIdx.x; e < entries; e += size_t(gridDim.x) * kCopyThreads) {
        const int page = t.table[e];
        if (page >= live && page < t.physical_pages) t.table[e] = w.map[page];
    }
    const int units = t.page_size * layers.units_per_token, chunks = (units + kCopyChunk - 1) / kCopyChunk, per_page = layers.buffers * chunks;
    for (size_t k = blockIdx.x; k < size_t(moves) * per_page; k += gridDim.x) {
        const int i = int(k / per_page), r = int(k % per_page);
        uint4* buffer = layers.pages[r / chunks];
        copy_chunk(buffer + size_t(w.ids[i]) * units, buffer + size_t(w.dst[i]) * units, r % chunks, units);
    }
}

// Pairs in the order of the list.  As long as no page is the destination of one pair and named by another, the order does not
// matter and every CTA takes any share of all the pairs' bytes; every CTA finds that out for itself, with a bit per page.
// Otherwise a CTA takes the same bytes of every pair, one pair after the other: a thread then reads what it has written itself.
__global__ void __launch_bounds__(kCopyThreads) pool_copy_kernel(const __grid_constant__ PoolLayers layers, const int* src, const int* dst, int count, int bitmap_words)
{
    extern __shared__ uint32_t named[];
    const auto pair_of = [&](int i, int& s, int& d) {
        s = src[i], d = dst[i];
        return s >= 0 && s < layers.physical_pages && d >= 0 && d < layers.physical_pages && s != d;
    };
    int clash = bitmap_words == 0;
    if (bitmap_words) {
        for (int i = threadIdx.x; i < bitmap_words; i += kCopyThreads) named[i] = 0;
        __syncthreads();
        int s, d;
        for (int i = threadIdx.x; i < count; i += kCopyThreads)
            if (pair_of(i, s, d)) clash |= (atomicOr(&named[d >> 5], 1u << (d & 31)) >> (d & 31)) & 1;
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += kCopyThreads)
            if (pair_of(i, s, d)) clash |= (named[s >> 5] >> (s & 31)) & 1;
    }
    clash = __syncthreads_or(clash);
    const int units = layers.page_size * layers.units_per_token, chunks = (units + kCopyChunk - 1) / kCopyChunk, per_page = layers.buffers * chunks;
    const auto move = [&](int i, int r) {
        int s, d;
        if (!pair_of(i, s, d)) return;
        uint4* buffer = layers.pages[r / chunks];
        copy_chunk(buffer + size_t(s) * units, buffer + size_t(d) * units, r % chunks, units);
    };
    if (clash) {
        for (int r = blockIdx.x; r < per_page; r += gridDim.x)
            for (int i = 0; i < count; ++i) move(i, r);
    } else {
        for (size_t k = blockIdx.x; k < size_t(count) * per_page; k += gridDim.x) move(int(k / per_page), int(k % per_page));
    }
}

int validate_cache(const garnet_b200_cache_options* o)
{
    if (!o) return fail(GARNET_B200_INVALID_VALUE, "cache: null options");
    if (o->abi != GARNET_B200_ABI || o->struct_size != int(sizeof(garnet_b200_cache_options)))
        return fail(GARNET_B200_INVALID_VALUE, "cache: options abi/size mismatch (abi %d, size %d)", o->abi, o->struct_size);
    if (o->layers <= 0 || o->physical_pages <= 0 || o->page_size <= 0 || o->sequences <= 0 || o->max_logical_pages <= 0)
        return fail(GARNET_B200_INVALID_VALUE, "cache: layers, physical_pages, page_size, sequences and max_logical_pages must be positive");
    if (o->token_bytes <= 0 || o->token_bytes % 16) return fail(GARNET_B200_INVALID_VALUE, "cache: token_bytes must be a positive multiple of 16");
    if (o->layers > kPoolMaxLayers) return fail(GARNET_B200_NOT_SUPPORTED, "cache: more than %d layers", kPoolMaxLayers);
    if ((long long)o->page_size * o->token_bytes > (1ll << 30)) return fail(GARNET_B200_NOT_SUPPORTED, "cache: a page of more than 1 GiB");
    return GARNET_B200_OK;
}

int pool_layers(const garnet_b200_cache_options& o, void* const* keys, void* const* values, const char* what, PoolLayers* out)
{
    if (!keys || !values) return fail(GARNET_B200_INVALID_VALUE, "%s: null page pointers", what);
    out->buffers = 2 * o.layers;
    out->units_per_token = o.token_bytes / 16;
    out->page_size = o.page_size;
    out->physical_pages = o.physical_pages;
    for (int i = 0; i < o.layers; ++i) {
        if (!keys[i] || !values[i]) return fail(GARNET_B200_INVALID_VALUE, "%s: the pages of layer %d are null", what, i);
        if ((reinterpret_cast<uintptr_t>(keys[i]) | reinterpret_cast<uintptr_t>(values[i])) & 15)
            return fail(GARNET_B200_INVALID_VALUE, "%s: the pages of layer %d are not 16-byte aligned", what, i);
        out->pages[2 * i] = static_cast<uint4*>(keys[i]);
        out->pages[2 * i + 1] = static_cast<uint4*>(values[i]);
    }
    return GARNET_B200_OK;
}

int pool_check_ws(const garnet_b200_cache_options& o, int count, const void* ws, size_t bytes, const char* what)
{
    if (!ws || bytes < pool_workspace(o, count) || (reinterpret_cast<uintptr_t>(ws) & 255))
        return fail(GARNET_B200_INVALID_VALUE, "%s: the workspace is missing, too small (%zu < %zu) or not 256-byte aligned", what, bytes, pool_workspace(o, count));
    return GARNET_B200_OK;
}

PoolTables pool_tables(const garnet_b200_cache_options& o, int* table, int* lengths, int* refs)
{
    return PoolTables{table, lengths, refs, o.sequences, o.max_logical_pages, o.page_size, o.physical_pages};
}

// The second launch of a call: its CTAs come up while the plan runs and wait for it.
template <typename... Params, typename... Args>
cudaError_t launch_behind(void (*kernel)(Params...), dim3 grid, cudaStream_t stream, const Args&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kCopyThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int pool_chunks(const garnet_b200_cache_options& o)
{
    const int units = o.page_size * (o.token_bytes / 16);
    return 2 * o.layers * ((units + kCopyChunk - 1) / kCopyChunk);
}

}  // namespace

}  // namespace gb200

using namespace gb200;

extern "C" {

int garnet_b200_cache_workspace(const garnet_b200_cache_options* o, int count, size_t* bytes)
{
    if (int rc = validate_cache(o)) return rc;
    if (!bytes || count < 0) return fail(GARNET_B200_INVALID_VALUE, "cache_workspace: bad argument");
    *bytes = pool_workspace(*o, count);
    return GARNET_B200_OK;
}

int garnet_b200_cache_extend(const garnet_b200_cache_options* o, int* d_page_tables, int* d_lengths, int* d_refcounts, const int* d_sequences,
                             const int* d_tokens, int* d_status, int count, void* d_workspace, size_t workspace_bytes, void* stream)
{
    if (int rc = validate_cache(o)) return rc;
    if (!d_page_tables || !d_lengths || !d_refcounts || !d_sequences || !d_tokens || !d_status || count <= 0)
        return fail(GARNET_B200_INVALID_VALUE, "cache_extend: null pointer or empty list");
    if (int rc = pool_check_ws(*o, count, d_workspace, workspace_bytes, "cache_extend")) return rc;
    const ExtendAsk ask{pool_tables(*o, d_page_tables, d_lengths, d_refcounts), d_sequences, d_tokens};
    pool_extend_kernel<<<1, kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(ask, pool_work(*o, count, d_workspace), d_status, count);
    GB_CUDA(cudaGetLastError());
    return GARNET_B200_OK;
}

int garnet_b200_cache_fork(const garnet_b200_cache_options* o, void* const* key_pages, void* const* value_pages, int* d_page_tables, int* d_lengths,
                           int* d_refcounts, const int* d_parents, const int* d_children, int* d_status, int count, void* d_workspace,
                           size_t workspace_bytes, void* stream)
{
    if (int rc = validate_cache(o)) return rc;
    if (!d_page_tables || !d_lengths || !d_refcounts || !d_parents || !d_children || !d_status || count <= 0)
        return fail(GARNET_B200_INVALID_VALUE, "cache_fork: null pointer or empty list");
    PoolLayers layers;
    if (int rc = pool_layers(*o, key_pages, value_pages, "cache_fork", &layers)) return rc;
    if (int rc = pool_check_ws(*o, count, d_workspace, workspace_bytes, "cache_fork")) return rc;
    const ForkAsk ask{pool_tables(*o, d_page_tables, d_lengths, d_refcounts), d_parents, d_children};
    const PoolWork w = pool_work(*o, count, d_workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    pool_fork_plan_kernel<<<1, kPlanThreads, 0, s>>>(ask, w, d_status, count);
    GB_CUDA(cudaGetLastError());
    const int lists = std::min(count, 4096), shares = std::max(1, std::min(pool_chunks(*o), kCopyCtas / lists));
    GB_CUDA(launch_behind(pool_fork_kernel, dim3(unsigned(shares), unsigned(lists)), s, layers, ask, w, count));
    return GARNET_B200_OK;
}

int garnet_b200_cache_free(const garnet_b200_cache_options* o, int* d_page_tables, int* d_lengths, int* d_refcounts, const int* d_sequences, int count,
                           void* stream)
{
    if (int rc = validate_cache(o)) return rc;
    if (!d_page_tables || !d_lengths || !d_refcounts || !d_sequences || count <= 0)
        return fail(GARNET_B200_INVALID_VALUE, "cache_free: null pointer or empty list");
    pool_free_kernel<<<unsigned(count), 256, 0, static_cast<cudaStream_t>(stream)>>>(pool_tables(*o, d_page_tables, d_lengths, d_refcounts), d_sequences);
    GB_CUDA(cudaGetLastError());
    return GARNET_B200_OK;
}

int garnet_b200_cache_compact_ex(const garnet_b200_cache_options* o, void* const* key_pages, void* const* value_pages, int* d_page_tables,
                                 int* d_refcounts, int* d_live, int* d_moved, void* d_workspace, size_t workspace_bytes, void* stream)
{
    if (int rc = validate_cache(o)) return rc;
    if (!d_page_tables || !d_refcounts || !d_live) return fail(GARNET_B200_INVALID_VALUE, "cache_compact: null pointer");
    PoolLayers layers;
    if (int rc = pool_layers(*o, key_pages, value_pages, "cache_compact", &layers)) return rc;
    if (int rc = pool_check_ws(*o, 0, d_workspace, workspace_bytes, "cache_compact")) return rc;
    const PoolTables t = pool_tables(*o, d_page_tables, nullptr, d_refcounts);
    PoolWork w = pool_work(*o, 0, d_workspace);
    if (d_moved) w.map = d_moved, w.map_from = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    pool_compact_plan_kernel<<<1, kPlanThreads, 0, s>>>(t, w, d_live);
    GB_CUDA(cudaGetLastError());
    GB_CUDA(launch_behind(pool_compact_kernel, dim3(unsigned(kCopyCtas)), s, layers, t, w, static_cast<const int*>(d_live)));
    return GARNET_B200_OK;
}

int garnet_b200_cache_compact(const garnet_b200_cache_options* o, void* const* key_pages, void* const* value_pages, int* d_page_tables,
                              int* d_refcounts, int* d_live, void* d_workspace, size_t workspace_bytes, void* stream)
{
    return garnet_b200_cache_compact_ex(o, key_pages, value_pages, d_page_tables, d_refcounts, d_live, nullptr, d_workspace, workspace_bytes, stream);
}

int garnet_b200_cache_copy_pages(const garnet_b200_cache_options* o, void* const* key_pages, void* const* value_pages, const int* d_src,
                                 const int* d_dst, int count, void* stream)
{
    if (int rc = validate_cache(o)) return rc;
    if (!d_src || !d_dst || count <= 0) return fail(GARNET_B200_INVALID_VALUE, "cache_copy_pages: null pointer or empty list");
    PoolLayers layers;
    if (int rc = pool_layers(*o, key_pages, value_pages, "cache_copy_pages", &layers)) return rc;
    const size_t bitmap = size_t(o->physical_pages + 31) / 32 * 4;
    const bool fits = bitmap <= size_t(kPoolMaxBitmap);
    if (fits && bitmap > 48 * 1024)
        GB_CUDA(cudaFuncSetAttribute(pool_copy_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPoolMaxBitmap));
    const long long items = (long long)count * pool_chunks(*o);
    pool_copy_kernel<<<unsigned(std::min(items, (long long)kCopyCtas)), kCopyThreads, fits ? bitmap : 0, static_cast<cudaStream_t>(stream)>>>(
        layers, d_src, d_dst, count, fits ? int(bitmap / 4) : 0);
    GB_CUDA(cudaGetLastError());
    return GARNET_B200_OK;
}

}  // extern "C"
