// Pages of a cache that several requests hold: requests that go on from another's tokens, requests that end, and a pool that
// is put together again.  `shares[page]` is how many requests hold a page beyond the first one; paged_resize, which knows
// nothing of it, is right for every page that has one holder.
#pragma once

#include <algorithm>

#include "paged_cache.cuh"

namespace mt {

constexpr int kSharingThreads = 1024, kSharingCluster = 16;  // where the device has room for so large a cluster, else 8

__device__ __forceinline__ bool page_inside(int id, int pages) { return (unsigned int)id < (unsigned int)pages; }

// Tokens -> blocks, for lengths a table of `width` blocks has room for; else -1.
__device__ __forceinline__ int blocks_held(int length, int width, int page_shift) {
    const long long blocks = ((long long)length + (1 << page_shift) - 1) >> page_shift;
    return length < 0 || blocks > width ? -1 : (int)blocks;
}

// ---------------------------------------------------------------------------------------------
// An empty request becomes the first counts[r] tokens of request sources[r].  Full pages are shared by their ids; the page begun
// is copied, since both will write on, into one from the head of the ring.  Two launches: one CTA deals out the pages, in the
// order of the requests (beside it others copy the shares, where they are not counted in place); then a CTA for every request
// and array of pages.  Sixteen prompts of up to 1000 tokens with eight continuations each in 28 layers, 62 MB read and written:
// 27 us with both launches, 69 % of the copy rate; four answers to one prompt in four layers 4.4 us in a graph, the two launches.
constexpr int kForkNone = -1, kForkRefused = -2;

struct ForkParams {
    int* tables;              // [requests, width], rows `table_stride` apart
    const int *lengths, *sources, *counts;  // [requests]
    const int* ring;          // [pool]
    const int* state;         // [2]
    const int* shares;        // [pages]
    int *lengths_out, *state_out, *shares_out;  // may be lengths, state, shares
    int* plan;                // [requests]: the page for what is begun, kForkNone or kForkRefused
    long long table_stride;
    int width, pool, requests, page_shift, pages;
};

__global__ void __launch_bounds__(kSharingThreads) paged_fork_plan_kernel(const ForkParams p) {
    __shared__ long long scratch[1][32];
    __shared__ long long total;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    if (blockIdx.x > 0) {
        for (long long i = (long long)(blockIdx.x - 1) * blockDim.x + threadIdx.x; i < p.pages; i += (long long)(gridDim.x - 1) * blockDim.x)
            p.shares_out[i] = p.shares[i];
        return;
    }
    int first = p.state[0], available = p.state[1];
    if (first < 0 || first >= p.pool) first = 0;
    available = max(0, min(available, p.pool));
    long long asked = 0;
    for (int base = 0; base < p.requests; base += blockDim.x) {
        const int r = base + threadIdx.x;
        bool valid = false;
        int count = 0;
        if (r < p.requests) {
            const int source = p.sources[r];
            count = p.counts[r];
            if (source >= 0 && source < p.requests && source != r && count > 0 && p.lengths[r] == 0) {
                const int held = p.lengths[source];
                valid = count <= held && blocks_held(held, p.width, p.page_shift) >= 0;
            }
        }
        const int need = valid && (count & ((1 << p.page_shift) - 1)) ? 1 : 0;
        long long reach[1] = {need};
        block_scan(reach, scratch);
        reach[0] += asked;
        if (threadIdx.x == blockDim.x - 1) total = reach[0];
        if (r < p.requests) {
            int plan = kForkRefused;
            if (valid && need == 0) plan = kForkNone;
            if (valid && need && reach[0] <= available) {
                const long long at = first + reach[0] - 1;
                const int id = p.ring[at < p.pool ? at : at - p.pool];
                plan = id < 0 ? kForkRefused : id;  // no page has that name
                if (id < 0) record_index(kPageOutside, r, (unsigned int)id);
            }
            p.plan[r] = plan;
        }
        __syncthreads();
        asked = total;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const long long granted = asked < available ? asked : available, at = first + granted;
        p.state_out[0] = (int)(at < p.pool ? at : at - p.pool);
        p.state_out[1] = (int)(available - granted);
    }
}

constexpr int kForkMaxCaches = 64, kForkThreads = 256;

struct ForkCopyParams {
    ForkParams fork;
    uint16_t* arrays[2 * kForkMaxCaches];  // keys of every cache, then values
    PageStrides key_strides, value_strides;
    int kv_heads, head_dim, first_cache;
};

// Rows [0, part) of all heads of a page, 16 bytes a thread and four of them in flight.
__device__ __forceinline__ void copy_page_rows(const uint16_t* source, uint16_t* target, const PageStrides& strides, int kv_heads, int part, int head_dim) {
    const int vectors = head_dim / 8, rows = kv_heads * part;
    const int stride = max(1, (int)blockDim.x / vectors), first_row = threadIdx.x / vectors;
    if (first_row >= stride) return;
    for (int i = (threadIdx.x - first_row * vectors) * 8; i < head_dim; i += blockDim.x * 8)  // one round, but for very wide heads
        for (int at = first_row; at < rows; at += 4 * stride) {
            uint4 moved[4];
            long long offset[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int one = at + k * stride, head = one / part;
                offset[k] = head * strides.head + (one - head * part) * strides.token + i;
                if (one < rows) moved[k] = ptx::ld_global_dependent_u4(source + offset[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (at + k * stride < rows) *reinterpret_cast<uint4*>(target + offset[k]) = moved[k];
        }
}

// CTA (request, y): y = 0 writes the request's row of the table and counts, y = 1 + 2 c and 2 + 2 c copy keys and values of cache c.
__global__ void __launch_bounds__(kForkThreads) paged_fork_kernel(const __grid_constant__ ForkCopyParams p) {
    const ForkParams& f = p.fork;
    const int r = blockIdx.x;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int plan = f.plan[r];
    if (blockIdx.y == 0) {
        if (p.first_cache > 0) return;
        if (plan == kForkRefused) {
            if (threadIdx.x == 0 && f.lengths_out != f.lengths) f.lengths_out[r] = f.lengths[r];
            return;
        }
        const int count = f.counts[r], whole = count >> f.page_shift;
        const int* from = f.tables + f.sources[r] * f.table_stride;
        int* to = f.tables + r * f.table_stride;
        for (int j = threadIdx.x; j < whole; j += blockDim.x) {
            const int id = from[j];
            to[j] = id;
            if (page_inside(id, f.pages)) atomicAdd(&f.shares_out[id], 1);
            else record_index(kPageOutside, r, (unsigned int)id);
        }
        if (threadIdx.x == 0) {
            if (plan != kForkNone) to[whole] = plan;
            f.lengths_out[r] = count;
        }
        return;
    }
    if (plan < 0) return;
    const int count = f.counts[r], whole = count >> f.page_shift;
    const int source = f.tables[f.sources[r] * f.table_stride + whole];
    if (!page_inside(source, f.pages) || !page_inside(plan, f.pages)) {
        if (threadIdx.x == 0) record_index(kPageOutside, r, (unsigned int)(page_inside(source, f.pages) ? plan : source));
        return;
    }
    const int which = (blockIdx.y - 1) & 1;
    const PageStrides& strides = which ? p.value_strides : p.key_strides;
    uint16_t* pages = p.arrays[which * kForkMaxCaches + (blockIdx.y - 1) / 2];
    copy_page_rows(pages + source * strides.page, pages + plan * strides.page, strides, p.kv_heads, count & ((1 << f.page_shift) - 1), p.head_dim);
}

// ---------------------------------------------------------------------------------------------
// Requests end.  A page goes back when as many requests drop it as hold it (shares + 1), at the place of the first that does,
// in the order of requests and blocks.  The drops of every page are counted and its first one is found; then it is known what goes back,
// how much of that stands in front of an entry of the table, and so its place in the ring.  Small tables are one CTA's, which keeps its
// entries; else every step is a launch over all SMs, since the entries' pages lie anywhere: 500 requests of up to 213 pages, half of which
// end, 13.5 us from Python (28 by a cluster of sixteen CTAs, 60 by one that looked entries up one at a time); two of five requests 3.4 us
// in a graph.
struct FreeParams {
    const int* tables;             // [requests, width], rows `table_stride` apart
    const int* lengths;            // [requests]
    const unsigned char* ended;    // [requests]
    int* ring;                     // [pool]
    const int* state;              // [2]
    const int* shares;             // [pages]
    int *lengths_out, *state_out, *shares_out;  // may be lengths, state, shares
    int *drops, *earliest;         // [pages]
    int* before;                   // [2] the state, [kFreeCtas] what the CTAs' ranges give back
    int* ids;                      // [entries]: the pages that they drop, or -1
    long long table_stride;
    int width, pool, requests, page_shift, pages;
};
constexpr int kFreeCtas = 128, kFreeKept = 8, kFreeNever = 0x7FFFFFFF;
inline long long free_bytes(int requests, int width, int pages) {
    const long long entries = (long long)requests * width;
    return (2ll * pages + (entries > kFreeKept * kSharingThreads ? entries + 2 + kFreeCtas : 0)) * (long long)sizeof(int);
}

// The page that an entry of the table drops, or -1.
__device__ __forceinline__ int dropped_page(const FreeParams& p, int entry) {
    const int r = entry / p.width, block = entry - r * p.width;
    if (!p.ended[r] || block >= blocks_held(p.lengths[r], p.width, p.page_shift)) return -1;
    const int id = p.tables[r * p.table_stride + block];
    if (page_inside(id, p.pages)) return id;
    record_index(kPageOutside, r, (unsigned int)id);
    return -1;
}
__device__ __forceinline__ void free_state_of(const FreeParams& p, const int* state, int& first, int& available) {
    first = state[0];
    if (first < 0 || first >= p.pool) first = 0;
    available = max(0, min(state[1], p.pool));
}
__device__ __forceinline__ int length_left(const FreeParams& p, int r) {
    const int length = p.lengths[r];
    return p.ended[r] && blocks_held(length, p.width, p.page_shift) >= 0 ? 0 : length;
}

// kKept: entries of a thread.
template <int kKept>
__global__ void __launch_bounds__(kSharingThreads) paged_free_kernel(const FreeParams p) {
    __shared__ int counts[kKept * 32], total;  // of what goes back: by round, then by warp; then what stands in front
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, entries = p.requests * p.width;
    int first, available, ids[kKept], own[kKept];
    free_state_of(p, p.state, first, available);
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
        const int i = k * kSharingThreads + (int)threadIdx.x;
        ids[k] = i < entries ? dropped_page(p, i) : -1;
        if (ids[k] >= 0) {
            p.drops[ids[k]] = 0;
            p.earliest[ids[k]] = kFreeNever;
        }
    }
    if (p.shares_out != p.shares)
        for (int i = threadIdx.x; i < p.pages; i += kSharingThreads) p.shares_out[i] = p.shares[i];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kKept; ++k)
        if (ids[k] >= 0) {
            atomicAdd(&p.drops[ids[k]], 1);
            atomicMin(&p.earliest[ids[k]], k * kSharingThreads + (int)threadIdx.x);
        }
    __syncthreads();
    // Of the entries that are the first to drop their page (lower half), those that give it back (upper half).
    unsigned int bits = 0;
#pragma unroll
    for (int k = 0; k < kKept; ++k) own[k] = ids[k] >= 0 ? __ldcg(&p.earliest[ids[k]]) : -1;
#pragma unroll
    for (int k = 0; k < kKept; ++k)
        if (own[k] == k * kSharingThreads + (int)threadIdx.x) bits |= (__ldcg(&p.drops[ids[k]]) > p.shares[ids[k]] ? 0x10001u : 1u) << k;
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
        const unsigned int votes = __ballot_sync(0xFFFFFFFFu, bits >> (16 + k) & 1u);
        if (lane == 0) counts[k * 32 + warp] = __popc(votes);
    }
    __syncthreads();
    if (warp == 0) {  // kKept numbers a lane
        int in_front[kKept], sum = 0;
#pragma unroll
        for (int j = 0; j < kKept; ++j) {
            in_front[j] = sum;
            sum += counts[lane * kKept + j];
        }
        int ahead = sum;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, ahead, offset);
            if (lane >= offset) ahead += other;
        }
#pragma unroll
        for (int j = 0; j < kKept; ++j) counts[lane * kKept + j] = ahead - sum + in_front[j];
        if (lane == 31) total = ahead;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
        const bool goes = bits >> (16 + k) & 1u;
        const unsigned int votes = __ballot_sync(0xFFFFFFFFu, goes);
        if (goes) p.ring[((long long)first + available + counts[k * 32 + warp] + __popc(votes & ((1u << lane) - 1u))) % p.pool] = ids[k];
        // The page's entry in front writes its shares; nobody else looks at them any more.
        if (bits >> k & 1u) p.shares_out[ids[k]] = max(0, p.shares[ids[k]] - __ldcg(&p.drops[ids[k]]));
    }
    for (int r = threadIdx.x; r < p.requests; r += kSharingThreads) p.lengths_out[r] = length_left(p, r);
    if (threadIdx.x == 0) {
        p.state_out[0] = first;
        p.state_out[1] = (int)min((long long)p.pool, (long long)available + total);
    }
}

// The steps of a large table.
__global__ void __launch_bounds__(256) paged_free_clear_kernel(const FreeParams p) {
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const long long worker = (long long)blockIdx.x * blockDim.x + threadIdx.x, workers = (long long)gridDim.x * blockDim.x;
    for (long long i = worker; i < p.pages; i += workers) {
        p.drops[i] = 0;
        p.earliest[i] = kFreeNever;
        if (p.shares_out != p.shares) p.shares_out[i] = p.shares[i];
    }
    if (worker < 2) p.before[worker] = p.state[worker];
}

__global__ void __launch_bounds__(256) paged_free_count_kernel(const FreeParams p) {
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const long long entries = (long long)p.requests * p.width, workers = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < entries; i += workers) {
        const int id = dropped_page(p, (int)i);
        p.ids[i] = id;
        if (id < 0) continue;
        atomicAdd(&p.drops[id], 1);
        atomicMin(&p.earliest[id], (int)i);
    }
}

// The entries of a CTA, in the order of the table.
__device__ __forceinline__ void free_range(const FreeParams& p, int& low, int& high) {
    const long long entries = (long long)p.requests * p.width;
    low = (int)(blockIdx.x * entries / gridDim.x);
    high = (int)((blockIdx.x + 1) * entries / gridDim.x);
}

// A page's first entry writes its shares, and leaves that it is the one to give it back or that nobody is.
__global__ void __launch_bounds__(kSharingThreads) paged_free_settle_kernel(const FreeParams p) {
    __shared__ int warp_counts[32];
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int low, high, mine = 0;
    free_range(p, low, high);
    for (long long i = (long long)low + threadIdx.x; i < high; i += kSharingThreads) {
        const int id = p.ids[i];
        if (id < 0 || __ldcg(&p.earliest[id]) != (int)i) continue;
        const int drops = p.drops[id], shares = p.shares[id];
        if (drops > shares) ++mine;
        else p.earliest[id] = kFreeNever;
        p.shares_out[id] = max(0, shares - drops);
    }
    mine = __reduce_add_sync(0xFFFFFFFFu, mine);
    if (lane == 0) warp_counts[warp] = mine;
    __syncthreads();
    if (warp == 0) {
        const int all = __reduce_add_sync(0xFFFFFFFFu, warp_counts[lane]);
        if (lane == 0) p.before[2 + blockIdx.x] = all;
    }
}

__global__ void __launch_bounds__(kSharingThreads) paged_free_give_kernel(const FreeParams p) {
    __shared__ int warp_counts[2][32];
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int low, high, first, available;
    free_range(p, low, high);
    free_state_of(p, p.before, first, available);
    long long before = 0, total = 0;
    for (int c = lane; c < gridDim.x; c += 32) {
        const int there = p.before[2 + c];
        total += there;
        if (c < blockIdx.x) before += there;
    }
#pragma unroll
    for (int offset = 16; offset >= 1; offset >>= 1) {
        total += __shfl_xor_sync(0xFFFFFFFFu, total, offset);
        before += __shfl_xor_sync(0xFFFFFFFFu, before, offset);
    }
    int round = 0;
    for (long long start = low; start < high; start += kSharingThreads, round ^= 1) {
        const long long i = start + threadIdx.x;
        const int id = i < high ? p.ids[i] : -1;
        const bool goes = id >= 0 && p.earliest[id] == (int)i;
        const unsigned int votes = __ballot_sync(0xFFFFFFFFu, goes);
        if (lane == 0) warp_counts[round][warp] = __popc(votes);
        __syncthreads();
        const int others = warp_counts[round][lane];
        const int ahead = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? others : 0), here = __reduce_add_sync(0xFFFFFFFFu, others);
        if (goes) p.ring[((long long)first + available + before + ahead + __popc(votes & ((1u << lane) - 1u))) % p.pool] = id;
        before += here;
    }
    for (int r = blockIdx.x * kSharingThreads + threadIdx.x; r < p.requests; r += gridDim.x * kSharingThreads) p.lengths_out[r] = length_left(p, r);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.state_out[0] = first;
        p.state_out[1] = (int)min((long long)p.pool, available + total);
    }
}

inline int launch_paged_free(const FreeParams& params, int sm_count, cudaStream_t stream) {
    const long long entries = (long long)params.requests * params.width;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(1, 1, 1);
    config.blockDim = dim3(kSharingThreads, 1, 1);
    config.stream = stream;
    cudaLaunchAttribute attrs[1];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = 1;
    if (entries <= kFreeKept * kSharingThreads) {
        const bool few = entries <= 2 * kSharingThreads;
        return cudaLaunchKernelEx(&config, few ? paged_free_kernel<2> : paged_free_kernel<kFreeKept>, params) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
    }
    auto blocks = [&](long long items, int threads, long long most) { return dim3((unsigned int)std::min((items + threads - 1) / threads, most), 1, 1); };
    config.blockDim = dim3(256, 1, 1);
    config.gridDim = blocks(params.pages, 256, 8ll * sm_count);
    if (cudaLaunchKernelEx(&config, paged_free_clear_kernel, params) != cudaSuccess) return MT_ERR_LAUNCH;
    config.gridDim = blocks(entries, 256, 8ll * sm_count);
    if (cudaLaunchKernelEx(&config, paged_free_count_kernel, params) != cudaSuccess) return MT_ERR_LAUNCH;
    config.blockDim = dim3(kSharingThreads, 1, 1);
    config.gridDim = blocks(entries, kSharingThreads, kFreeCtas);
    if (cudaLaunchKernelEx(&config, paged_free_settle_kernel, params) != cudaSuccess) return MT_ERR_LAUNCH;
    return cudaLaunchKernelEx(&config, paged_free_give_kernel, params) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------------------------
// The pages that the block tables hold move to the lowest ids, 0 to held - 1: the n-th of those above, in ascending order, to the
// n-th free id below.  Free ids, shares and what is held are taken from the tables alone, so that pages nobody holds any
// more (of beams that were dropped) become free.  One launch for the numbers, one for the copies, none of which reads what another
// writes: sources lie above, targets below.  236 MB read and written in 90 us, 5.3 TB/s with the numbers' launch.
struct CompactParams {
    const int* tables;        // [requests, width], rows `table_stride` apart
    const int* lengths;       // [requests]
    int* tables_out;          // [requests, width], dense
    int *ring_out, *state_out, *shares_out;  // [pages], [2], [pages]
    int *holders, *rank;      // [pages]: requests that hold a page; pages held below it
    int *movers, *holes;      // [pages]
    int* totals;              // [kSharingCluster] held pages of the CTAs' ranges; then how many are held, and of them below that number
    long long table_stride;
    int width, requests, page_shift, pages;
};
constexpr int kCompactHeld = kSharingCluster, kCompactBelow = kSharingCluster + 1, kCompactTotals = kSharingCluster + 2;

__device__ __forceinline__ void sharing_barrier(bool cluster) {
    if (cluster) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    } else {
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kSharingThreads) paged_compact_kernel(const CompactParams p, bool cluster) {
    __shared__ int warp_counts[32];
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int ctas = gridDim.x, cta = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int worker = cta * blockDim.x + threadIdx.x, workers = ctas * blockDim.x;
    const int entries = p.requests * p.width;
    for (int i = worker; i < p.pages; i += workers) p.holders[i] = 0;
    sharing_barrier(cluster);
    auto held_entry = [&](int i, int& r, int& block, bool report) {
        r = i / p.width;
        block = i - r * p.width;
        const int length = p.lengths[r], blocks = blocks_held(length, p.width, p.page_shift);
        if (report && blocks < 0 && block == 0) record_index(kLengthOutside, r, (unsigned int)length);
        return block < blocks;
    };
    for (int i = worker; i < entries; i += workers) {
        int r, block;
        if (!held_entry(i, r, block, true)) continue;
        const int id = p.tables[r * p.table_stride + block];
        if (page_inside(id, p.pages)) atomicAdd(&p.holders[id], 1);
        else record_index(kPageOutside, r, (unsigned int)id);
    }
    sharing_barrier(cluster);
    const int low = (int)((long long)cta * p.pages / ctas), high = (int)((long long)(cta + 1) * p.pages / ctas);
    int mine = 0;
    for (int i = low + threadIdx.x; i < high; i += blockDim.x) mine += __ldcg(&p.holders[i]) > 0;
    mine = __reduce_add_sync(0xFFFFFFFFu, mine);
    if (lane == 0) warp_counts[warp] = mine;
    __syncthreads();
    if (warp == 0) {
        const int all = __reduce_add_sync(0xFFFFFFFFu, warp_counts[lane]);
        if (lane == 0) p.totals[cta] = all;
    }
    sharing_barrier(cluster);
    int before = 0, held = 0;
    for (int c = 0; c < ctas; ++c) {
        const int there = __ldcg(&p.totals[c]);
        held += there;
        if (c < cta) before += there;
    }
    if (worker == 0) {
        p.totals[kCompactHeld] = held;
        if (held == p.pages) p.totals[kCompactBelow] = held;
    }
    for (int start = low; start < high; start += blockDim.x) {
        const int i = start + threadIdx.x;
        const bool used = i < high && __ldcg(&p.holders[i]) > 0;
        const unsigned int votes = __ballot_sync(0xFFFFFFFFu, used);
        __syncthreads();
        if (lane == 0) warp_counts[warp] = __popc(votes);
        __syncthreads();
        const int others = warp_counts[lane];
        const int ahead = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? others : 0), round = __reduce_add_sync(0xFFFFFFFFu, others);
        const int rank = before + ahead + __popc(votes & ((1u << lane) - 1u));
        if (i < high) {
            p.rank[i] = rank;
            if (used && i >= held) p.movers[rank] = i;
            if (!used && i < held) p.holes[i - rank] = i;
            if (i == held) p.totals[kCompactBelow] = rank;
        }
        before += round;
    }
    sharing_barrier(cluster);
    const int below = __ldcg(&p.totals[kCompactBelow]);
    for (int i = worker; i < entries; i += workers) {
        int r, block;
        const bool inside = held_entry(i, r, block, false);
        int id = p.tables[r * p.table_stride + block];
        if (inside && page_inside(id, p.pages) && id >= held) id = __ldcg(&p.holes[__ldcg(&p.rank[id]) - below]);
        p.tables_out[i] = id;
    }
    for (int i = worker; i < p.pages; i += workers) {
        int holders = i < held ? __ldcg(&p.holders[i]) : 1;
        if (holders == 0) holders = __ldcg(&p.holders[__ldcg(&p.movers[below + i - __ldcg(&p.rank[i])])]);
        p.shares_out[i] = holders - 1;
        p.ring_out[i] = (int)(((long long)held + i) % p.pages);
    }
    if (worker == 0) {
        p.state_out[0] = 0;
        p.state_out[1] = p.pages - held;
    }
}

struct CompactCopyParams {
    uint16_t* arrays[2 * kForkMaxCaches];
    PageStrides key_strides, value_strides;
    const int *movers, *holes, *totals;
    int kv_heads, head_dim, page_shift;
};

__global__ void __launch_bounds__(kForkThreads) paged_compact_copy_kernel(const __grid_constant__ CompactCopyParams p) {
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int held = p.totals[kCompactHeld], below = p.totals[kCompactBelow], which = blockIdx.y & 1;
    const PageStrides& strides = which ? p.value_strides : p.key_strides;
    uint16_t* pages = p.arrays[which * kForkMaxCaches + blockIdx.y / 2];
    for (int k = blockIdx.x; k < held - below; k += gridDim.x)
        copy_page_rows(pages + p.movers[below + k] * strides.page, pages + p.holes[k] * strides.page, strides, p.kv_heads, 1 << p.page_shift, p.head_dim);
}

// One CTA where that gives a thread up to eight entries, else a cluster.
template <typename Params>
inline int launch_sharing_kernel(void (*kernel)(const Params, bool), const Params& params, long long entries, cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.blockDim = dim3(kSharingThreads, 1, 1);
    config.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    config.attrs = attrs;
    int ctas = 1;
    if (entries > 8 * kSharingThreads) {
        ctas = kSharingCluster;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return MT_ERR_LAUNCH;
        attrs[1].val.clusterDim.x = ctas;
        config.gridDim = dim3(ctas, 1, 1);
        config.numAttrs = 2;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess || clusters < 1) {
            (void)cudaGetLastError();
            ctas = 8;
        }
    }
    attrs[1].val.clusterDim.x = ctas;
    config.gridDim = dim3(ctas, 1, 1);
    config.numAttrs = ctas > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, params, ctas > 1) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
}

}  // namespace mt
