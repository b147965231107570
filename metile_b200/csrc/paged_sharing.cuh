// Pages of a cache that several requests hold: requests that go on from another's tokens, requests that end, and a pool that
// is put together again.  `shares[page]` is how many requests hold a page beyond the first one; paged_resize, which knows
// nothing of it, is right for every page that has one holder.
#pragma once

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
// and array of pages.
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
// in the order of requests and blocks: the drops of every page are counted, then the CTAs, each with a range of the table
// in order, count what they give back, and then write it behind what those in front of them do.  A thread has up to sixteen entries
// of the table at once, whose loads go together, and keeps them over the passes where that is all it has.  Bound by the chain of
// dependent loads and four barriers: 500 requests of up to 213 pages, half of which end, 13 us in a graph (54 with one entry at a time,
// looked up in every pass).
struct FreeParams {
    const int* tables;             // [requests, width], rows `table_stride` apart
    const int* lengths;            // [requests]
    const unsigned char* ended;    // [requests]
    int* ring;                     // [pool]
    const int* state;              // [2]
    const int* shares;             // [pages]
    int *lengths_out, *state_out, *shares_out;  // may be lengths, state, shares
    int *drops, *earliest;         // [pages]
    int* returned;                 // [kSharingCluster]
    long long table_stride;
    int width, pool, requests, page_shift, pages;
};

__device__ __forceinline__ void sharing_barrier(bool cluster) {
    if (cluster) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    } else {
        __syncthreads();
    }
}

// kFreeKept: entries of the table that a thread has at once.
template <int kFreeKept>
__global__ void __launch_bounds__(kSharingThreads) paged_free_kernel(const FreeParams p, bool cluster) {
    __shared__ int counts[kFreeKept * 32];  // of what goes back: by round, then by warp; then what stands in front
    __shared__ int warp_counts[32];
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int ctas = gridDim.x, cta = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int worker = cta * blockDim.x + threadIdx.x, workers = ctas * blockDim.x;
    int first = p.state[0], available = p.state[1];
    if (first < 0 || first >= p.pool) first = 0;
    available = max(0, min(available, p.pool));
    const int entries = p.requests * p.width;
    const int low = (int)((long long)cta * entries / ctas), high = (int)((long long)(cta + 1) * entries / ctas);
    constexpr int kStep = kFreeKept * kSharingThreads;
    const bool kept = high - low <= kStep;
    // The pages that entries start + 1024 k + thread drop, or -1.
    int ids[kFreeKept];
    auto look = [&](int start, bool report) {
        int rows[kFreeKept];
#pragma unroll
        for (int k = 0; k < kFreeKept; ++k) {
            const int i = start + k * kSharingThreads + (int)threadIdx.x;
            rows[k] = i < high ? i / p.width : -1;
            ids[k] = -1;
        }
#pragma unroll
        for (int k = 0; k < kFreeKept; ++k) {
            const int block = start + k * kSharingThreads + (int)threadIdx.x - rows[k] * p.width;
            const bool drops = rows[k] >= 0 && p.ended[rows[k]] && block < blocks_held(p.lengths[rows[k]], p.width, p.page_shift);
            if (drops) ids[k] = p.tables[rows[k] * p.table_stride + block];
            if (drops && !page_inside(ids[k], p.pages)) {
                if (report) record_index(kPageOutside, rows[k], (unsigned int)ids[k]);
                ids[k] = -1;
            }
        }
    };
    for (int start = low; start < high; start += kStep) {
        look(start, true);
#pragma unroll
        for (int k = 0; k < kFreeKept; ++k)
            if (ids[k] >= 0) {
                p.drops[ids[k]] = 0;
                p.earliest[ids[k]] = 0x7FFFFFFF;
            }
    }
    if (p.shares_out != p.shares)
        for (int i = worker; i < p.pages; i += workers) p.shares_out[i] = p.shares[i];
    sharing_barrier(cluster);
    for (int start = low; start < high; start += kStep) {
        if (!kept) look(start, false);
#pragma unroll
        for (int k = 0; k < kFreeKept; ++k)
            if (ids[k] >= 0) {
                atomicAdd(&p.drops[ids[k]], 1);
                atomicMin(&p.earliest[ids[k]], start + k * kSharingThreads + (int)threadIdx.x);
            }
    }
    sharing_barrier(cluster);
    // Which of a thread's entries are the first to drop their page (lower half), and give it back (upper half).
    auto judge = [&](int start) {
        unsigned int bits = 0;
        int own[kFreeKept];
#pragma unroll
        for (int k = 0; k < kFreeKept; ++k) own[k] = ids[k] >= 0 ? __ldcg(&p.earliest[ids[k]]) : -1;
#pragma unroll
        for (int k = 0; k < kFreeKept; ++k)
            if (ids[k] >= 0 && own[k] == start + k * kSharingThreads + (int)threadIdx.x) bits |= (__ldcg(&p.drops[ids[k]]) > p.shares[ids[k]] ? 0x10001u : 1u) << k;
        return bits;
    };
    int mine = 0;
    unsigned int bits = 0;
    for (int start = low; start < high; start += kStep) {
        if (!kept) look(start, false);
        bits = judge(start);
        mine += __popc(bits >> 16);
    }
    mine = __reduce_add_sync(0xFFFFFFFFu, mine);
    if (lane == 0) warp_counts[warp] = mine;
    __syncthreads();
    if (warp == 0) {
        const int all = __reduce_add_sync(0xFFFFFFFFu, warp_counts[lane]);
        if (lane == 0) p.returned[cta] = all;
    }
    sharing_barrier(cluster);
    long long before = 0, total = 0;
    for (int c = 0; c < ctas; ++c) {
        const int there = __ldcg(&p.returned[c]);
        total += there;
        if (c < cta) before += there;
    }
    for (int start = low; start < high; start += kStep) {
        if (!kept) {
            look(start, false);
            bits = judge(start);
        }
#pragma unroll
        for (int k = 0; k < kFreeKept; ++k) {
            const unsigned int votes = __ballot_sync(0xFFFFFFFFu, bits >> (16 + k) & 1u);
            if (lane == 0) counts[k * 32 + warp] = __popc(votes);
        }
        __syncthreads();
        if (warp == 0) {  // kFreeKept numbers a lane
            int own[kFreeKept], sum = 0;
#pragma unroll
            for (int j = 0; j < kFreeKept; ++j) {
                own[j] = sum;
                sum += counts[lane * kFreeKept + j];
            }
            int ahead = sum;
#pragma unroll
            for (int offset = 1; offset < 32; offset <<= 1) {
                const int other = __shfl_up_sync(0xFFFFFFFFu, ahead, offset);
                if (lane >= offset) ahead += other;
            }
#pragma unroll
            for (int j = 0; j < kFreeKept; ++j) counts[lane * kFreeKept + j] = ahead - sum + own[j];
            if (lane == 31) warp_counts[0] = ahead;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kFreeKept; ++k) {
            const bool goes = bits >> (16 + k) & 1u;
            const unsigned int votes = __ballot_sync(0xFFFFFFFFu, goes);
            if (goes) p.ring[((long long)first + available + before + counts[k * 32 + warp] + __popc(votes & ((1u << lane) - 1u))) % p.pool] = ids[k];
            // The page's entry in front writes its shares; nobody else looks at them any more.
            if (bits >> k & 1u) p.shares_out[ids[k]] = max(0, p.shares[ids[k]] - __ldcg(&p.drops[ids[k]]));
        }
        before += warp_counts[0];
        __syncthreads();
    }
    sharing_barrier(cluster);
    for (int r = worker; r < p.requests; r += workers) {
        const int length = p.lengths[r];
        p.lengths_out[r] = p.ended[r] && blocks_held(length, p.width, p.page_shift) >= 0 ? 0 : length;
    }
    if (worker == 0) {
        p.state_out[0] = first;
        p.state_out[1] = (int)min((long long)p.pool, available + total);
    }
}

// ---------------------------------------------------------------------------------------------
// The pages that the block tables hold move to the lowest ids, 0 to held - 1: the n-th of those above, in ascending order, to the
// n-th free id below.  Free ids, shares and what is held are taken from the tables alone, so that pages nobody holds any
// more (of beams that were dropped) become free.  One launch for the numbers, one for the copies, none of which reads what another
// writes: sources lie above, targets below.
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
