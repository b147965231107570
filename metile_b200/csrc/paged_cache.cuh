// A key-value cache in pages: block tables and slot maps on the GPU, the rotary embedding with its append to the
// pages, and the reordering of beams.
//
// A pool holds `pages` pages of `page_size` tokens (a power of two) for every layer; row r of a block table names the
// pages of request r in order, so that token p of it lies in slot table[r][p / page_size] * page_size + p % page_size.
// The ids of the pages no request uses stand in a ring: they are taken at its head and given back at its tail, so the
// entries one call reads and the entries it writes are never the same, and a call with the same state does the same again.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"

namespace mt {

constexpr unsigned int kSlotOutside = 0x302;    // rope_kv_append_paged: word 1 = row, 2 and 3 = the slot
constexpr unsigned int kPageOutside = 0x303;    // a block table names a page outside the pool: word 1 = its row, 2 = the page
constexpr unsigned int kLengthOutside = 0x304;  // a length the block table has no room for: word 1 = its row, 2 = the length
constexpr unsigned int kParentOutside = 0x305;  // beam_reorder: word 1 = row, 2 = the parent

__device__ __forceinline__ void record_index(unsigned int code, unsigned int where, unsigned long long value) {
    if (atomicCAS(&g_device_status[0], 0u, code) == 0u) {
        g_device_status[1] = where;
        g_device_status[2] = (unsigned int)value;
        g_device_status[3] = (unsigned int)(value >> 32);
    }
}

struct PageStrides {
    long long page, head, token;  // elements
};

// ---------------------------------------------------------------------------------------------
// Requests grow and shrink: counts[r] > 0 tokens are added to request r, -counts[r] taken from its end.
struct ResizeParams {
    int* tables;              // [requests, width], rows `table_stride` apart
    const int* lengths;       // [requests]
    const int* counts;        // [requests]
    int* ring;                // [pool] free page ids
    const int* state;         // [2]: first free entry of the ring, how many there are
    long long* slots;         // [tokens]
    int* positions;           // [tokens]
    int* starts;              // [requests + 1]
    int* lengths_out;         // [requests], may be `lengths`
    int* state_out;           // [2], may be `state`
    long long table_stride;
    int width, pool, requests, page_shift, tokens;
};

constexpr int kResizeThreads = 1024;  // the most; and the requests taken at once
constexpr int kResizeCluster = 8;

// Inclusive sums over the block of kCount numbers at once.
template <int kCount>
__device__ __forceinline__ void block_scan(long long (&values)[kCount], long long (*scratch)[32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    auto warp_scan = [&](long long v) {
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const long long other = __shfl_up_sync(0xFFFFFFFFu, v, offset);
            if (lane >= offset) v += other;
        }
        return v;
    };
#pragma unroll
    for (int i = 0; i < kCount; ++i) values[i] = warp_scan(values[i]);
    if (lane == 31) {
#pragma unroll
        for (int i = 0; i < kCount; ++i) scratch[i][warp] = values[i];
    }
    __syncthreads();
    // Every warp adds up the warps in front of it.
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
        const long long v = lane < warps ? scratch[i][lane] : 0;
        const long long before = warp_scan(v) - v;
        values[i] += __shfl_sync(0xFFFFFFFFu, before, warp);
    }
    __syncthreads();
}

// The last i in [0, n) with starts[i] <= value, where starts[0] <= value and starts ascends.
__device__ __forceinline__ int last_not_above(const long long* starts, int n, long long value) {
    int low = 0, high = n;
    while (high - low > 1) {
        const int middle = (low + high) >> 1;
        if (starts[middle] <= value) low = middle; else high = middle;
    }
    return low;
}

// The requests are taken as many as threads at a time, in order.  Three sums run along them: tokens added, pages asked for, pages
// given back.  Then tokens, granted and returned pages are dealt to the threads, each of which looks its request up; a thread
// has four tokens in a row.  Bound by latency, and for long prompts by the threads: several CTAs then, which all take the
// sums and share what follows.  Where lengths and state are written in place the CTAs are one cluster, and the first of them
// writes behind a barrier.  What a decode step needs, a token and at most a page for each, the requests' own threads do at once.  64
// requests of a token each 3.2 us in a graph (5.0 with the search); 501 with 116 thousand tokens 11.0 us (one CTA 132).
// In place a cluster of eight CTAs does those 116 thousand tokens in 23 us in a graph, the separate form in 9.
// The grid follows the tokens, which the host knows, not the pages given back: 239 requests that end at once with 68 thousand
// pages 160 us beside a map of up to 1024 tokens (256 threads), 63 by 1024 threads, 35 by two CTAs of them.
__global__ void __launch_bounds__(kResizeThreads) paged_resize_kernel(const ResizeParams p, bool in_place) {
    __shared__ long long token_start[kResizeThreads], grant_start[kResizeThreads], free_start[kResizeThreads];
    __shared__ int held[kResizeThreads], added[kResizeThreads];
    __shared__ unsigned char is_served[kResizeThreads];
    __shared__ long long scratch[3][32];
    __shared__ long long totals[3];
    __shared__ int granted_shared;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int threads = blockDim.x;
    const bool leads = blockIdx.x == 0;
    const long long worker = (long long)blockIdx.x * threads + threadIdx.x, workers = (long long)gridDim.x * threads;
    const int page = 1 << p.page_shift;
    auto blocks_of = [&](long long tokens) { return (tokens + page - 1) >> p.page_shift; };
    auto all_have_read = [&] {
        if (in_place) {
            ptx::cluster_arrive();
            ptx::cluster_wait();
        }
    };
    // The ring's state as a caller may have it: kept within the ring whatever it says.
    int first = p.state[0], available = p.state[1];
    if (first < 0 || first >= p.pool) first = 0;
    available = max(0, min(available, p.pool));
    const long long room = min((long long)p.width << p.page_shift, 0x7FFFFFFFll);  // lengths are of 32 bits
    auto wrapped = [&](long long taken) {  // of fewer entries than the ring has
        const long long at = first + taken;
        return at < p.pool ? at : at - p.pool;
    };
    if (threadIdx.x == 0) granted_shared = 0;
    long long tokens_before = 0, asked_before = 0, freed_before = 0;
    for (int base = 0; base < p.requests; base += threads) {
        const int r = base + threadIdx.x, here = min(threads, p.requests - base);
        const bool exists = r < p.requests;
        const int length = exists ? p.lengths[r] : 0, count = exists ? p.counts[r] : 0;
        const long long after = (long long)length + count, added_here = max(count, 0);
        bool valid = length >= 0 && after >= 0 && length <= room && after <= room;
        long long change = valid ? blocks_of(after) - blocks_of(length) : 0;
        long long sums[3] = {added_here, max(0ll, change), max(0ll, -change)};
        block_scan(sums, scratch);
        if (threadIdx.x == threads - 1) totals[0] = sums[0] + tokens_before;
        __syncthreads();
        if (totals[0] > p.tokens) {  // whether a request's tokens fit the map decides if it asks for pages
            valid = valid && (count <= 0 || sums[0] + tokens_before <= p.tokens);
            change = valid ? change : 0;
            long long pages[2] = {max(0ll, change), max(0ll, -change)};
            block_scan(pages, scratch);
            sums[1] = pages[0];
            sums[2] = pages[1];
        }
        const long long need = max(0ll, change), back = max(0ll, -change), ends = sums[0] + tokens_before, begin = ends - added_here;
        const long long reach = sums[1] + asked_before, returned = sums[2] + freed_before;
        // In order and without overtaking: once the free pages do not reach, nobody behind is given any.
        const bool served = valid && (need == 0 || reach <= available);
        token_start[threadIdx.x] = begin;
        grant_start[threadIdx.x] = reach - need;
        free_start[threadIdx.x] = returned - back;
        held[threadIdx.x] = length;
        added[threadIdx.x] = count;
        is_served[threadIdx.x] = served;
        if (served && need > 0) atomicMax(&granted_shared, (int)reach);  // at most `available`
        if (threadIdx.x == threads - 1) {
            totals[1] = reach;
            totals[2] = returned;
        }
        const bool more = __syncthreads_or(count > 1 || need > 1 || back > 0);
        all_have_read();
        if (exists && leads) {
            // A request's own thread does its first token and page: all there is in a decode step.
            if (count > 0 && begin < p.tokens) {
                const bool fresh = (length & (page - 1)) == 0;
                int id = -1;
                if (served) id = fresh ? p.ring[wrapped(reach - need)] : p.tables[r * p.table_stride + (length >> p.page_shift)];
                if (served && need > 0) p.tables[r * p.table_stride + blocks_of(length)] = fresh ? id : p.ring[wrapped(reach - need)];
                p.slots[begin] = id < 0 ? -1 : ((long long)id << p.page_shift) + (length & (page - 1));
                p.positions[begin] = served ? length : 0;
            }
            p.starts[r] = (int)min(begin, 0x7FFFFFFFll);
            p.lengths_out[r] = served ? (int)after : length;
        }
        const long long tokens_here = more ? min((long long)p.tokens, totals[0]) : 0, asked_here = more ? min((long long)available, totals[1]) : 0;
        for (long long t0 = tokens_before + 4 * worker; t0 < tokens_here; t0 += 4 * workers) {
            int i = last_not_above(token_start, here, t0);
            int position[4], id[4];
            bool first_one[4];
            const int* named[4];  // where the id of the token's page stands
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                while (i + 1 < here && token_start[i + 1] <= t0 + k) ++i;
                position[k] = 0;
                named[k] = nullptr;
                first_one[k] = t0 + k >= tokens_here || token_start[i] == t0 + k;
                if (!first_one[k] && is_served[i]) {
                    position[k] = held[i] + (int)(t0 + k - token_start[i]);
                    const int block = position[k] >> p.page_shift, fresh = block - (int)blocks_of(held[i]);
                    named[k] = fresh < 0 ? p.tables + (base + i) * p.table_stride + block : p.ring + wrapped(grant_start[i] + fresh);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) id[k] = named[k] ? *named[k] : -1;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (first_one[k]) continue;
                p.slots[t0 + k] = id[k] < 0 ? -1 : ((long long)id[k] << p.page_shift) + (position[k] & (page - 1));
                p.positions[t0 + k] = position[k];
            }
        }
        for (long long g = asked_before + worker; g < asked_here; g += workers) {
            const int i = last_not_above(grant_start, here, g);
            if (is_served[i] && g != grant_start[i])
                p.tables[(base + i) * p.table_stride + blocks_of(held[i]) + (g - grant_start[i])] = p.ring[wrapped(g)];
        }
        for (long long f = freed_before + worker; f < totals[2]; f += workers) {
            const int i = last_not_above(free_start, here, f);
            const long long block = blocks_of((long long)held[i] + added[i]) + (f - free_start[i]);
            p.ring[((long long)first + available + f) % p.pool] = p.tables[(base + i) * p.table_stride + block];
        }
        tokens_before = totals[0];
        asked_before = totals[1];
        freed_before = totals[2];
        __syncthreads();
    }
    for (long long t = tokens_before + worker; t < p.tokens; t += workers) {
        p.slots[t] = -1;
        p.positions[t] = 0;
    }
    if (p.requests == 0) {
        __syncthreads();
        all_have_read();
    }
    if (threadIdx.x == 0 && leads) {
        p.starts[p.requests] = (int)min(tokens_before, 0x7FFFFFFFll);
        p.state_out[0] = (int)wrapped(granted_shared) % p.pool;
        p.state_out[1] = (int)min((long long)p.pool, (long long)available - granted_shared + freed_before);
    }
}

inline int launch_paged_resize(const ResizeParams& params, cudaStream_t stream) {
    const bool in_place = params.lengths_out == params.lengths || params.state_out == params.state;
    // A CTA for every four tokens of its threads; up to 64, or a cluster of eight.
    const int most = in_place ? kResizeCluster : 64;
    const long long wanted = ((long long)params.tokens + 4 * kResizeThreads - 1) / (4 * kResizeThreads);
    const int ctas = wanted <= 1 ? 1 : in_place || wanted >= most ? most : (int)wanted;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(ctas, 1, 1);
    // 256 threads where that gives every request and four tokens one.
    config.blockDim = dim3(params.requests <= 256 && params.tokens <= 1024 ? 256 : kResizeThreads, 1, 1);
    config.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = ctas;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    config.attrs = attrs;
    config.numAttrs = in_place && ctas > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, paged_resize_kernel, params, in_place && ctas > 1) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------------------------
// Rotary embedding of the rows of a ragged batch (half-split pairs (i, i + D/2)) and their append to the pages: the
// keys rotated, the values as they are, each row to its slot.  The angle position * inverse[i] is taken in 64 bits and
// reduced to a turn there: in 32 bits a position of 100000 leaves it 0.004 off.  Sine and cosine are those of 32 bits.  A CTA per
// row, whose angles serve all heads.  Bound by bytes: 4093 rows of 48 heads of 128 18.9 us, 5.3 TB/s (64 to 384 threads a CTA 18.6
// to 20.9 us, other cache hints within 3 %).
struct RopeAppendPagedParams {
    const uint16_t *q, *k, *v;            // [rows, heads, D], rows `q_stride` ... elements apart
    const float* inverse;                 // [D / 2]
    const int* positions;                 // [rows]
    const long long* slots;               // [rows]; negative: the row has none
    uint16_t* q_out;                      // [rows, Hq, D]
    uint16_t *key_pages, *value_pages;
    PageStrides key_strides, value_strides;
    long long q_stride, k_stride, v_stride, slot_count;
    int q_heads, kv_heads, head_dim, page_shift;
};

template <bool kHalf>
__device__ __forceinline__ float2 unpack_pair(uint32_t pair) {
    if constexpr (kHalf) return __half22float2(*reinterpret_cast<const __half2*>(&pair));
    else return make_float2(bf16_lo(pair), bf16_hi(pair));
}
template <bool kHalf>
__device__ __forceinline__ uint32_t pack_pair(float low, float high) {
    if constexpr (kHalf) {
        const __half2 pair = __floats2half2_rn(low, high);
        return *reinterpret_cast<const uint32_t*>(&pair);
    } else {
        return pack_bf16x2(low, high);
    }
}

constexpr int kRopePagedThreads = 128;

template <bool kHalf>
__global__ void __launch_bounds__(kRopePagedThreads) rope_kv_append_paged_kernel(const RopeAppendPagedParams p) {
    extern __shared__ float rope_angles[];  // cosines, then sines
    const int row = blockIdx.x, dim = p.head_dim, half = dim >> 1;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const double position = (double)p.positions[row];
    long long slot = p.slots[row];
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
        // In half turns: sin(pi x) has the period 2, which is taken off exactly.
        const double turns = position * (double)p.inverse[i] * 0.31830988618379067154;
        sincospif((float)(turns - 2.0 * rint(0.5 * turns)), &rope_angles[half + i], &rope_angles[i]);
    }
    if (slot >= p.slot_count) {
        if (threadIdx.x == 0) record_index(kSlotOutside, row, slot);
        slot = -1;
    }
    const long long page = slot >> p.page_shift, token = slot & ((1 << p.page_shift) - 1);
    __syncthreads();
    const int units = half / 8;  // threads of a head, eight pairs each
    for (int at = threadIdx.x; at < (p.q_heads + 2 * p.kv_heads) * units; at += blockDim.x) {
        int head = at / units;
        const int i = (at - head * units) * 8;
        const uint16_t* from;
        uint16_t* to;
        bool rotated = true;
        if (head < p.q_heads) {
            from = p.q + row * p.q_stride + (long long)head * dim;
            to = p.q_out + ((long long)row * p.q_heads + head) * dim;
        } else {
            if (slot < 0) continue;
            head -= p.q_heads;
            rotated = head < p.kv_heads;
            if (rotated) {
                from = p.k + row * p.k_stride + (long long)head * dim;
                to = p.key_pages + page * p.key_strides.page + head * p.key_strides.head + token * p.key_strides.token;
            } else {
                head -= p.kv_heads;
                from = p.v + row * p.v_stride + (long long)head * dim;
                to = p.value_pages + page * p.value_strides.page + head * p.value_strides.head + token * p.value_strides.token;
            }
        }
        const uint4 a = ptx::ld_global_dependent_u4(from + i), z = ptx::ld_global_dependent_u4(from + i + half);
        uint4 low = a, high = z;
        if (rotated) {
            const uint32_t first[4] = {a.x, a.y, a.z, a.w}, second[4] = {z.x, z.y, z.z, z.w};
            uint32_t l[4], h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 x = unpack_pair<kHalf>(first[j]), y = unpack_pair<kHalf>(second[j]);
                const float c0 = rope_angles[i + 2 * j], s0 = rope_angles[half + i + 2 * j];
                const float c1 = rope_angles[i + 2 * j + 1], s1 = rope_angles[half + i + 2 * j + 1];
                l[j] = pack_pair<kHalf>(x.x * c0 - y.x * s0, x.y * c1 - y.y * s1);
                h[j] = pack_pair<kHalf>(y.x * c0 + x.x * s0, y.y * c1 + x.y * s1);
            }
            low = make_uint4(l[0], l[1], l[2], l[3]);
            high = make_uint4(h[0], h[1], h[2], h[3]);
        }
        *reinterpret_cast<uint4*>(to + i) = low;
        *reinterpret_cast<uint4*>(to + i + half) = high;
    }
}

// ---------------------------------------------------------------------------------------------
// Block tables follow the surviving beams.  All beams of a group hold equally many tokens.  A page that is full is never
// written again, so children share it with their parent: only its id is copied.  The page in work belongs to one beam:
// the first child of a parent goes on in its page, every further child gets the page of a beam without children and a
// copy of what is in its parent's.  So as many pages are copied as there are parents missing, and none is allocated.  Bound by
// bytes: 48 pages in each of 28 layers, 85 MB read and written, 18.2 us (13.7 in a graph; a CTA per row and layer 20.9).
constexpr int kReorderMaxBeams = 32, kReorderMaxCaches = 64, kReorderThreads = 256;

struct ReorderParams {
    const int* tables;        // [groups * beams, width]
    const int* lengths;       // [groups * beams]
    const int* parents;       // [groups * beams], within the group
    int* tables_out;          // [groups * beams, width], dense
    uint16_t* pages[2 * kReorderMaxCaches];  // keys of every cache, then values
    PageStrides key_strides, value_strides;
    long long table_stride;
    int width, beams, caches, kv_heads, head_dim, page_shift, page_count, first_cache;
};

// CTA (group, y): y = 0 writes the group's tables, y = 1 + 2 c and 2 + 2 c copy the keys and the values of cache c.
__global__ void __launch_bounds__(kReorderThreads) beam_reorder_kernel(const __grid_constant__ ReorderParams p) {
    const int group = blockIdx.x, base = group * p.beams, lane = threadIdx.x & 31;
    const bool reports = threadIdx.x < 32 && blockIdx.y == 0;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    // Every warp has the group's parents, one in a lane.
    int parent = lane;
    if (lane < p.beams) {
        parent = p.parents[base + lane];
        if (parent < 0 || parent >= p.beams) {  // recorded, and taken as its own
            if (reports) record_index(kParentOutside, base + lane, (unsigned int)parent);
            parent = lane;
        }
    }
    const int length = p.lengths[base];
    const long long capacity = (long long)p.width << p.page_shift;
    if ((length < 0 || length > capacity) && reports && lane == 0) record_index(kLengthOutside, base, (unsigned int)length);
    const int held = (int)max(0ll, min((long long)length, capacity));
    const int block = held >> p.page_shift, part = held & ((1 << p.page_shift) - 1);
    // First children go on in their parent's page in work; as many are not the first of theirs as there are beams without any,
    // and the n-th of the former gets the page of the n-th of the latter.
    const unsigned int all = p.beams == 32 ? 0xFFFFFFFFu : (1u << p.beams) - 1u;
    const unsigned int firsts = __ballot_sync(0xFFFFFFFFu, __ffs(__match_any_sync(0xFFFFFFFFu, parent)) - 1 == lane) & all;
    unsigned int childless = all & ~__reduce_or_sync(0xFFFFFFFFu, lane < p.beams ? 1u << parent : 0u);
    int owner = parent;
    if (!(firsts >> lane & 1u) && lane < p.beams) {
        for (int skip = __popc(all & ~firsts & ((1u << lane) - 1u)); skip > 0; --skip) childless &= childless - 1u;
        owner = __ffs(childless) - 1;
    }
    if (blockIdx.y == 0) {
        if (p.first_cache > 0) return;
        for (int k = 0; k < p.beams; ++k) {
            const int from = __shfl_sync(0xFFFFFFFFu, parent, k), of = __shfl_sync(0xFFFFFFFFu, owner, k);
            for (int j = threadIdx.x; j < p.width; j += blockDim.x) {
                const int row = j < block ? from : j == block && part > 0 ? of : k;
                p.tables_out[(long long)(base + k) * p.width + j] = p.tables[(base + row) * p.table_stride + j];
            }
        }
        return;
    }
    if (part == 0 || firsts == all) return;
    // The pages to copy, in the lanes of the children that are not the first of theirs.
    int source = -1, target = -1;
    if (lane < p.beams && !(firsts >> lane & 1u)) {
        source = p.tables[(base + parent) * p.table_stride + block];
        target = p.tables[(base + owner) * p.table_stride + block];
        if (source < 0 || source >= p.page_count || target < 0 || target >= p.page_count) {
            if (threadIdx.x < 32 && blockIdx.y == 1)
                record_index(kPageOutside, base + lane, (unsigned int)(source < 0 || source >= p.page_count ? source : target));
            source = -1;
        }
    }
    unsigned int copies = __ballot_sync(0xFFFFFFFFu, source >= 0);
    // A thread has one 16-byte vector of a row and takes every `stride`-th row, four at a time.
    const int which = (blockIdx.y - 1) & 1, vectors = p.head_dim / 8, rows = p.kv_heads * part;
    const int stride = max(1, (int)blockDim.x / vectors), first_row = threadIdx.x / vectors;
    uint16_t* pages = p.pages[which * kReorderMaxCaches + (blockIdx.y - 1) / 2];
    const PageStrides strides = which ? p.value_strides : p.key_strides;
    for (; copies; copies &= copies - 1u) {
        const int child = __ffs(copies) - 1;
        const uint16_t* source_page = pages + __shfl_sync(0xFFFFFFFFu, source, child) * strides.page;
        uint16_t* target_page = pages + __shfl_sync(0xFFFFFFFFu, target, child) * strides.page;
        if (first_row >= stride) continue;
        for (int i = (threadIdx.x - first_row * vectors) * 8; i < p.head_dim; i += blockDim.x * 8)  // one round, but for very wide heads
            for (int at = first_row; at < rows; at += 4 * stride) {
                uint4 moved[4];
                long long offset[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int one = at + k * stride, head = one / part;
                    offset[k] = head * strides.head + (one - head * part) * strides.token + i;
                    if (one < rows) moved[k] = ptx::ld_global_dependent_u4(source_page + offset[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (at + k * stride < rows) *reinterpret_cast<uint4*>(target_page + offset[k]) = moved[k];
            }
    }
}

}  // namespace mt
