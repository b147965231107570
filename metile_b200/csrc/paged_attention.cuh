// Decode attention of one new token per request over a paged key-value cache, split over the cache's length and joined.
//
// out[b, h] = softmax(scale q[b, h] K^T) V over the tokens row b of the block table names.  Bound by the bytes of keys
// and values: 4 Hq / Hkv operations for each, far below what the tensor cores have to offer.
//
// Split.  A sequence is cut into splits of 128 tokens, twice as many for every doubling above 16384, so that there are 128
// at most, or 512 where there are fewer than four KV heads (a partial result is D + 2 numbers of 32 bits per query head: with
// eight of them a sixteenth of what 128 tokens of their KV head are).
// The cut is the sequence's own, so its bits do not depend on the others of the call.  A unit is one split of one KV head
// (its query heads, up to 16 at once) and belongs to one WARP.  The grid is one CTA per SM; the CTAs count the units of the
// lengths they find on the device and deal them out, a unit to each SM in turn: a table wide enough for
// the longest request costs nothing, and ragged lengths even out.
//
// A warp keeps a ring of chunks of 16 tokens (keys and values) of its own in flight, 16-byte asynchronous copies from
// wherever the pages lie, and never meets another warp.  What is masked (the tail behind the sequence, a page outside the
// cache) is filled with zeros by the copy itself, whatever lies there.
//
// Per chunk, on mma.sync m16n8k16 with 32-bit sums:
//   scores  S[16 tokens x 8 heads] = K[16 x D] Q^T[D x 8]
//   values  O^T[D x 8 heads] += V^T[D x 16] P^T[16 x 8], V^T by transposing matrix loads; the scores leave the first
//           product as rows of tokens and enter the second as its columns: movmatrix turns them over.
// The weights enter as two 16-bit numbers, high and low part: one alone would be off by 2^-9 (bf16).  A running maximum
// per head is moved, and the sums with it, only when a score passes it by more than 2^8: the weights stay below 256 (2^15 in
// fp16, see kPagedLift) and keep their relative precision, and a lane adds up its own tokens' weights until the end.
//
// Measured (8 KV heads of 4 x 128): 100 requests of up to 8191 tokens 337 to 349 us, 5.4 TB/s (reading alone 294); two of 100003
// 143 to 147 us, 5.6 TB/s; one of 301 7.3 us.  16 x 2048 tokens, 2 x 6 heads: 12.4 us.  Six warps with four ring slots hold what eight
// with three or four with six do (143 us against 154 and 157 for the long ones); without the arithmetic the large cases take the same.
#pragma once

#include "attention_decode.cuh"
#include "paged_cache.cuh"

namespace mt {

constexpr int kPagedChunk = 16;          // tokens
constexpr int kPagedSplitShift = 7;      // the shortest split: 128 tokens
constexpr int kPagedMostSplits = 128;    // of a sequence with four KV heads or more
constexpr int kPagedSlices = 4;          // threads of the join to one number, 128 splits each
constexpr int kPagedRowPad = 8;          // elements: rows 16 bytes longer keep matrix loads free of conflicts
constexpr int kPagedTogether = 4;        // splits that one CTA joins: a warp to each of the SM's four schedulers
constexpr float kPagedHeadroom = 8.0f;   // log2 of how far a score may pass the running maximum
// log2 of the maximum's own weight.  fp16 has nothing below 2^-24: with 1 for the maximum what is 2^-26 of it would be lost, an
// eighth of a sum over 2^23 tokens in splits of 65536.  With 2^7, 2^15 at most, the least is 2^-31 of it.
template <bool kHalf>
constexpr float kPagedLift = kHalf ? 7.0f : 0.0f;

// Most splits of a sequence: with few KV heads more of them, so that one long sequence has 512 units in any case; those beyond
// 128 are 16 tokens a query head of the group long at least (2^floor), so that partial results stay an eighth of what is read.
// One request with 1 KV head: 131072 tokens for 8 heads of 128 26 us (40 with 128 splits), 100000 for one of 64 15 (33); a
// batch of 16 with 2 x 4 heads and 32768 tokens 110 us (101): it has units enough by itself, but the cut does not know the batch.
__host__ __device__ constexpr int paged_split_limit(int kv_heads) { return kv_heads >= 4 ? kPagedMostSplits : kv_heads >= 2 ? 2 * kPagedMostSplits : 4 * kPagedMostSplits; }
static_assert(paged_split_limit(1) <= kPagedSlices * kPagedMostSplits, "the join takes 128 splits a slice");
__host__ __device__ constexpr int paged_split_floor(int group) {
    int shift = kPagedSplitShift;
    while (shift < 20 && 1 << shift < 16 * group) ++shift;
    return shift;
}
__host__ __device__ constexpr int paged_split_shift(int tokens, int limit = kPagedMostSplits, int floor = kPagedSplitShift) {
    int shift = kPagedSplitShift;
    while ((tokens - 1) >> shift >= (shift < floor ? kPagedMostSplits : limit)) ++shift;
    return shift;
}
__host__ __device__ constexpr int paged_splits(int tokens, int limit = kPagedMostSplits, int floor = kPagedSplitShift) {
    return tokens <= 1 ? 1 : ((tokens - 1) >> paged_split_shift(tokens, limit, floor)) + 1;
}
// The most splits any length up to `capacity` has.
inline int paged_most_splits(long long capacity, int limit = kPagedMostSplits) {
    const long long shortest = (capacity + (1 << kPagedSplitShift) - 1) >> kPagedSplitShift;
    return shortest < limit ? (int)shortest : limit;
}

struct PageByteStrides {
    int page, head, token;
};

struct PagedAttentionParams {
    const uint16_t* q;                 // [batch, Hq, D]
    const char *key_pages, *value_pages;
    PageByteStrides key_strides, value_strides;
    const int* tables;                 // [batch, width], rows `table_stride` apart
    const int* lengths;                // [batch]
    uint16_t* out;                     // [batch, Hq, D]
    float* partial;                    // [batch * Hq, most_splits, D]
    float2* stats;                     // [batch * Hq, most_splits]: maximum (log2) and sum
    long long table_stride;
    int width, batch, q_heads, kv_heads, page_shift, page_count, most_splits, split_limit, split_floor;
    bool together;                     // a CTA has all splits of its KV heads, one to a warp, and joins them
    float scale;
};

template <int kD>
struct PagedShape {
    static constexpr int kWarps = kD == 256 ? 4 : kD == 128 ? 6 : 8;
    static constexpr int kStages = kD == 64 ? 6 : kD == 128 ? 4 : 3;
    static constexpr int kRow = kD + kPagedRowPad;
    static constexpr int kStageElements = 2 * kPagedChunk * kRow;
    static constexpr int kSmem = kWarps * kStages * kStageElements * 2;
    static_assert(kSmem >= kWarps * 16 * (kD + 6) * 4 && kWarps >= kPagedTogether, "the rings hold the results of 16 heads from every warp");
};

// 16 bytes, or zeros where `bytes` is 0 (the address is a valid one all the same).
__device__ __forceinline__ void cp_async_16_or_zeros(void* smem_dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(smem_dst)), "l"(src), "r"(bytes) : "memory");
}

template <bool kHalf>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (kHalf)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        mma_bf16_16816(d, a, b0, b1);
}

// An 8x8 matrix of 16-bit numbers spread over the warp as an MMA fragment, turned over.
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t pair) {
    uint32_t out;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(out) : "r"(pair));
    return out;
}

__device__ __forceinline__ float power_of_two(float v) {  // 2^v to 2^-22
    float out;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(out) : "f"(v));
    return out;
}

// A length as the kernels use it: recorded and cut where the table has no room for it.
__device__ __forceinline__ int paged_length(const PagedAttentionParams& p, int b, bool report) {
    const int n = p.lengths[b];
    const long long capacity = (long long)p.width << p.page_shift;
    if (n >= 0 && n <= capacity) return n;
    if (report) record_index(kLengthOutside, b, (unsigned int)n);
    return n < 0 ? 0 : (int)capacity;
}

// kTiles: tiles of eight query heads a unit takes at once.
template <int kD, bool kHalf, int kTiles>
__global__ void __launch_bounds__(PagedShape<kD>::kWarps * 32, 1) paged_attention_kernel(const __grid_constant__ PagedAttentionParams p) {
    using Shape = PagedShape<kD>;
    constexpr int kRow = Shape::kRow, kStages = Shape::kStages, kThreads = Shape::kWarps * 32, kSlices = kD / 16;
    constexpr int kCopies = kD / 32;                 // 16-byte copies of a lane for eight rows
    constexpr int kLanesPerRow = kD / 8;             // 8, 16 or 32
    constexpr int kRowsPerCopy = 32 / kLanesPerRow;  // rows a warp's copy covers
    extern __shared__ __align__(16) uint16_t rings[];
    __shared__ int unit_start[kThreads + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = p.q_heads / p.kv_heads, parts = (group + 8 * kTiles - 1) / (8 * kTiles), per_split = p.kv_heads * parts;
    uint16_t* ring = rings + warp * (kStages * Shape::kStageElements);
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();

    // Units in front of every run of requests (a request each up to as many as there are threads).
    const int run = (p.batch + kThreads - 1) / kThreads;
    if (!p.together) {
        __shared__ int warp_units[Shape::kWarps];
        int mine = 0;
        for (int b = threadIdx.x * run; b < min((int)(threadIdx.x + 1) * run, p.batch); ++b)
            mine += paged_splits(paged_length(p, b, blockIdx.x == 0), p.split_limit, p.split_floor) * per_split;
        int sum = mine;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, sum, offset);
            if (lane >= offset) sum += other;
        }
        if (lane == 31) warp_units[warp] = sum;
        __syncthreads();
        int before = 0;
        for (int w = 0; w < warp; ++w) before += warp_units[w];
        unit_start[threadIdx.x + 1] = before + sum;
        if (threadIdx.x == 0) unit_start[0] = 0;
        __syncthreads();
    }
    const int units = p.together ? p.batch * per_split * Shape::kWarps : unit_start[kThreads];
    const float scale_log2 = p.scale * 1.4426950408889634f;
    const bool dense = p.key_strides.token == kD * 2 && p.value_strides.token == kD * 2;

    for (long long next = blockIdx.x + (long long)gridDim.x * warp; next < units; next += (long long)gridDim.x * Shape::kWarps) {
        int b, n, splits, split, rest;
        if (p.together) {
            b = blockIdx.x / per_split;
            rest = blockIdx.x - b * per_split;
            n = paged_length(p, b, rest == 0 && threadIdx.x == 0);
            splits = paged_splits(n, p.split_limit, p.split_floor);
            split = warp;
        } else {
            int unit = (int)next;
            int low = 0, high = kThreads;
            while (high - low > 1) {
                const int middle = (low + high) >> 1;
                if (unit_start[middle] <= unit) low = middle; else high = middle;
            }
            unit -= unit_start[low];
            for (b = low * run;; ++b) {
                n = paged_length(p, b, false);
                splits = paged_splits(n, p.split_limit, p.split_floor);
                if (unit < splits * per_split) break;
                unit -= splits * per_split;
            }
            split = unit / per_split;
            rest = unit - split * per_split;
        }
        const int h = rest / parts, part = rest - h * parts;
        const int shift = paged_split_shift(n, p.split_limit, p.split_floor), first = split << shift, end = max(first, min(n, first + (1 << shift)));
        const int head0 = h * group + part * 8 * kTiles, heads = min(8 * kTiles, group - part * 8 * kTiles);
        const int chunks = (end - first + kPagedChunk - 1) / kPagedChunk;

        // The pages of the unit, 32 at a time, one in a lane; the next 32 are asked for one window ahead.
        const int* table = p.tables + b * p.table_stride;
        const int page0 = first >> p.page_shift, pages = ((end - 1) >> p.page_shift) - page0 + 1;
        auto window = [&](int w) {
            const int i = 32 * w + lane;
            return end > first && i < pages ? table[page0 + i] : 0;
        };
        int in_window = 0, ids = window(0), ids_next = window(1);
        unsigned int outside = 0;  // two bits a ring slot: its first, its second eight tokens lie in a page outside the cache

        const int row0 = lane / kLanesPerRow, at = lane % kLanesPerRow * 16;
        const char* key_head = p.key_pages + (long long)h * p.key_strides.head + row0 * p.key_strides.token + at;
        const char* value_head = p.value_pages + (long long)h * p.value_strides.head + row0 * p.value_strides.token + at;
        char* ring_lane = reinterpret_cast<char*>(ring) + row0 * kRow * 2 + at;
        auto copy_chunk = [&](int c, int slot) {
            const int token0 = first + c * kPagedChunk, i0 = (token0 >> p.page_shift) - page0, i1 = ((token0 + 8) >> p.page_shift) - page0;
            if (i0 >> 5 != in_window) {
                ids = ids_next;
                ids_next = window(++in_window + 1);
            }
            int id[2] = {__shfl_sync(0xFFFFFFFFu, ids, i0 & 31), __shfl_sync(0xFFFFFFFFu, ids, i1 & 31)};
            const unsigned int bad = ((unsigned int)id[0] < (unsigned int)p.page_count ? 0u : 1u) | ((unsigned int)id[1] < (unsigned int)p.page_count ? 0u : 2u);
            outside = (outside & ~(3u << (2 * slot))) | bad << (2 * slot);
            char* keys = ring_lane + slot * (Shape::kStageElements * 2);
            char* values = keys + kPagedChunk * kRow * 2;
            const int in_page = token0 & ((1 << p.page_shift) - 1), in_second = (token0 + 8) & ((1 << p.page_shift) - 1);
            if (bad == 0 && token0 + kPagedChunk <= end && dense) {  // a whole chunk of rows that follow one another
                const char* key[2] = {key_head + (long long)id[0] * p.key_strides.page + in_page * (kD * 2),
                                      key_head + (long long)id[1] * p.key_strides.page + in_second * (kD * 2)};
                const char* value[2] = {value_head + (long long)id[0] * p.value_strides.page + in_page * (kD * 2),
                                        value_head + (long long)id[1] * p.value_strides.page + in_second * (kD * 2)};
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < kCopies; ++i) {
                        const int to = (8 * half + i * kRowsPerCopy) * kRow * 2;
                        ptx::cp_async_16(keys + to, key[half] + i * kRowsPerCopy * kD * 2);
                        ptx::cp_async_16(values + to, value[half] + i * kRowsPerCopy * kD * 2);
                    }
                return;
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int token = token0 + 8 * half, row = half ? in_second : in_page;
                const bool inside = !(bad >> half & 1u);
                if (!inside) {
                    if (lane == 0 && token < end) record_index(kPageOutside, b, (unsigned int)id[half]);
                    id[half] = 0;
                }
                const char* key = key_head + (long long)id[half] * p.key_strides.page + row * p.key_strides.token;
                const char* value = value_head + (long long)id[half] * p.value_strides.page + row * p.value_strides.token;
                const int usable = inside ? end - token - row0 : 0;  // rows from this lane's first one on
#pragma unroll
                for (int i = 0; i < kCopies; ++i) {
                    const int bytes = i * kRowsPerCopy < usable ? 16 : 0, to = (8 * half + i * kRowsPerCopy) * kRow * 2;
                    cp_async_16_or_zeros(keys + to, key, bytes);  // a row behind the end has an address inside the page all the same
                    cp_async_16_or_zeros(values + to, value, bytes);
                    key += kRowsPerCopy * p.key_strides.token;
                    value += kRowsPerCopy * p.value_strides.token;
                }
            }
        };
#pragma unroll
        for (int c = 0; c < kStages - 1; ++c) {
            if (c < chunks) copy_chunk(c, c);
            ptx::cp_async_commit();
        }

        // Query fragments: head g of each tile, dims 16 s + 2 t (+1) and + 8.
        uint32_t qf[kTiles][kSlices][2];
#pragma unroll
        for (int tile = 0; tile < kTiles; ++tile) {
            const bool real = 8 * tile + g < heads;
            const uint16_t* row = p.q + ((long long)b * p.q_heads + head0 + (real ? 8 * tile + g : 0)) * kD;
#pragma unroll
            for (int s = 0; s < kSlices; ++s) {
                uint32_t lower, upper;
                asm volatile("ld.global.u32 %0, [%1];" : "=r"(lower) : "l"(row + 16 * s + 2 * t));
                asm volatile("ld.global.u32 %0, [%1];" : "=r"(upper) : "l"(row + 16 * s + 2 * t + 8));
                qf[tile][s][0] = real ? lower : 0u;
                qf[tile][s][1] = real ? upper : 0u;
            }
        }
        float acc[kSlices][kTiles][4], top[kTiles][2], sum[kTiles][2];
#pragma unroll
        for (int tile = 0; tile < kTiles; ++tile) {
            top[tile][0] = top[tile][1] = -INFINITY;
            sum[tile][0] = sum[tile][1] = 0.0f;
#pragma unroll
            for (int s = 0; s < kSlices; ++s) acc[s][tile][0] = acc[s][tile][1] = acc[s][tile][2] = acc[s][tile][3] = 0.0f;
        }

        for (int c = 0, slot = 0; c < chunks; ++c) {
            ptx::cp_async_wait_group<kStages - 2>();
            __syncwarp();
            const uint16_t* keys = ring + slot * Shape::kStageElements;
            const uint16_t* values = keys + kPagedChunk * kRow;
            // Scores: [0], [1]: token g, heads 2 t and 2 t + 1 of the tile; [2], [3]: token g + 8.
            float score[kTiles][4], odd[kTiles][4];  // two chains of products
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
                for (int i = 0; i < 4; ++i) score[tile][i] = odd[tile][i] = 0.0f;
#pragma unroll
            for (int s = 0; s < kSlices; ++s) {
                uint32_t a[4];
                ldmatrix_x4(a, keys + (lane & 15) * kRow + 8 * (lane >> 4) + 16 * s);
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) mma_16816<kHalf>(s & 1 ? odd[tile] : score[tile], a, qf[tile][s][0], qf[tile][s][1]);
            }
            const int token = first + c * kPagedChunk + g;
            const bool there[2] = {token < end && !(outside >> (2 * slot) & 1u), token + 8 < end && !(outside >> (2 * slot + 1) & 1u)};
            bool passes = false;
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    score[tile][i] = there[i >> 1] ? (score[tile][i] + odd[tile][i]) * scale_log2 : -INFINITY;
                    passes = passes || score[tile][i] > top[tile][i & 1] + (kPagedHeadroom + kPagedLift<kHalf>);
                }
            if (__any_sync(0xFFFFFFFFu, passes)) {
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float now = fmaxf(score[tile][j], score[tile][j + 2]);
#pragma unroll
                        for (int offset = 4; offset <= 16; offset <<= 1) now = fmaxf(now, __shfl_xor_sync(0xFFFFFFFFu, now, offset));
                        now = fmaxf(now - kPagedLift<kHalf>, top[tile][j]);
                        const float factor = now == -INFINITY ? 1.0f : power_of_two(top[tile][j] - now);
                        top[tile][j] = now;
                        sum[tile][j] *= factor;
#pragma unroll
                        for (int s = 0; s < kSlices; ++s) {
                            acc[s][tile][j] *= factor;
                            acc[s][tile][j + 2] *= factor;
                        }
                    }
            }
            // Weights, high and low part, as columns of tokens.
            uint32_t high[kTiles][2], lower[kTiles][2];
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                float weight[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // Nothing for what is masked.  A NaN moves no maximum and is NaN here, also where that is -inf yet.
                    weight[i] = score[tile][i] == -INFINITY ? 0.0f : power_of_two(score[tile][i] - top[tile][i & 1]);
                    sum[tile][i & 1] += weight[i];
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t pair = pack_pair<kHalf>(weight[2 * half], weight[2 * half + 1]);
                    const float2 back = unpack_pair<kHalf>(pair);
                    high[tile][half] = transposed_8x8(pair);
                    lower[tile][half] = transposed_8x8(pack_pair<kHalf>(weight[2 * half] - back.x, weight[2 * half + 1] - back.y));
                }
            }
#pragma unroll
            for (int s = 0; s < kSlices; ++s) {
                uint32_t a[4];
                ldmatrix_x4_trans(a, values + ((lane & 7) + 8 * (lane >> 4)) * kRow + 16 * s + (lane & 8));
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) {
                    mma_16816<kHalf>(acc[s][tile], a, high[tile][0], high[tile][1]);
                    mma_16816<kHalf>(acc[s][tile], a, lower[tile][0], lower[tile][1]);
                }
            }
            __syncwarp();  // the slot read last time round is free: every lane is past its matrix loads
            if (c + kStages - 1 < chunks) copy_chunk(c + kStages - 1, slot == 0 ? kStages - 1 : slot - 1);
            ptx::cp_async_commit();
            slot = slot == kStages - 1 ? 0 : slot + 1;
        }

        ptx::cp_async_wait_group<0>();
        if (p.together) __syncthreads();  // the rings give way to the warps' results
        // acc[s][tile]: [0], [1]: dim 16 s + g, heads 2 t and 2 t + 1; [2], [3]: dim + 8.
        float* shared_partial = reinterpret_cast<float*>(rings);  // [warps][8 kTiles][D + 4], then the maxima and sums
        constexpr int kPartialRow = kD + 4;                       // the four heads of a store then lie in different banks
        float2* shared_stats = reinterpret_cast<float2*>(shared_partial + Shape::kWarps * 8 * kTiles * kPartialRow);
#pragma unroll
        for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float total = sum[tile][j];
#pragma unroll
                for (int offset = 4; offset <= 16; offset <<= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, offset);
                const int head = 8 * tile + 2 * t + j;
                if (head >= heads || split >= splits) continue;
                const long long at = (long long)b * p.q_heads + head0 + head;
                if (splits == 1) {
                    const float factor = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
                    for (int s = 0; s < kSlices; ++s) {
                        p.out[at * kD + 16 * s + g] = (uint16_t)pack_pair<kHalf>(acc[s][tile][j] * factor, 0.0f);
                        p.out[at * kD + 16 * s + g + 8] = (uint16_t)pack_pair<kHalf>(acc[s][tile][j + 2] * factor, 0.0f);
                    }
                } else {
                    float* to = p.together ? shared_partial + (warp * 8 * kTiles + head) * kPartialRow : p.partial + (at * p.most_splits + split) * kD;
#pragma unroll
                    for (int s = 0; s < kSlices; ++s) {
                        to[16 * s + g] = acc[s][tile][j];
                        to[16 * s + g + 8] = acc[s][tile][j + 2];
                    }
                    if (g == 0) *(p.together ? shared_stats + warp * 8 * kTiles + head : p.stats + at * p.most_splits + split) = make_float2(top[tile][j], total);
                }
            }
        if (p.together) {
            __syncthreads();
            if (splits > 1)
                for (int i = threadIdx.x; i < heads * (kD / 4); i += kThreads) {  // as the join kernel does it, four dims a thread
                    const int head = i / (kD / 4), d = (i - head * (kD / 4)) * 4;
                    float2 own[kPagedTogether];
                    float4 number[kPagedTogether];
                    float largest = -INFINITY, total = 0.0f;
#pragma unroll
                    for (int w = 0; w < kPagedTogether; ++w) {
                        own[w] = w < splits ? shared_stats[w * 8 * kTiles + head] : make_float2(-INFINITY, 0.0f);
                        number[w] = w < splits ? *reinterpret_cast<const float4*>(shared_partial + (w * 8 * kTiles + head) * kPartialRow + d)
                                               : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        largest = fmaxf(largest, own[w].x);
                    }
                    float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < kPagedTogether; ++w) {
                        const float factor = own[w].x == -INFINITY ? 0.0f : power_of_two(own[w].x - largest);
                        total = fmaf(own[w].y, factor, total);
                        value = make_float4(fmaf(number[w].x, factor, value.x), fmaf(number[w].y, factor, value.y), fmaf(number[w].z, factor, value.z),
                                            fmaf(number[w].w, factor, value.w));
                    }
                    uint2 packed = make_uint2(0u, 0u);
                    if (total != 0.0f) packed = make_uint2(pack_pair<kHalf>(value.x / total, value.y / total), pack_pair<kHalf>(value.z / total, value.w / total));
                    *reinterpret_cast<uint2*>(p.out + ((long long)b * p.q_heads + head0 + head) * kD + d) = packed;
                }
            return;
        }
        __syncwarp();
    }
}

// Joins the splits of one request and query head, in split order; a request of one split has its result already.  A slice of
// kD threads takes 128 splits, the first one what the slices have, in their order.
template <int kD, bool kHalf, int kSlices>
__global__ void __launch_bounds__(kD * kSlices) paged_attention_join_kernel(const __grid_constant__ PagedAttentionParams p) {
    constexpr int kAhead = 16, kRounds = kPagedMostSplits / 32;
    const long long at = blockIdx.x;                // b * Hq + query head
    const int b = (int)(at / p.q_heads), d = threadIdx.x % kD, slice = threadIdx.x / kD, lane = threadIdx.x & 31;
    __shared__ float slice_value[kSlices][kD], slice_total[kSlices];
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int all = paged_splits(paged_length(p, b, false), p.split_limit, p.split_floor), first = slice * kPagedMostSplits;
    if (all == 1) return;
    const int splits = min(all - first, kPagedMostSplits);  // of this slice
    const float* from = p.partial + (at * p.most_splits + first) * kD + d;
    const float2* stats = p.stats + at * p.most_splits + first;
    // The first results are asked for before the maxima are known, the others sixteen ahead.
    float ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = i < splits ? from[(long long)i * kD] : 0.0f;
    float2 mine[kRounds];
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        mine[r] = 32 * r + lane < splits ? stats[32 * r + lane] : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, mine[r].x);
    }
    if (kSlices > 1 && all > kPagedMostSplits)  // the maximum is that of all
        for (int i = lane; i < all; i += 32) top = fmaxf(top, p.stats[at * p.most_splits + i].x);
#pragma unroll
    for (int offset = 16; offset >= 1; offset >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, offset));
    float total = 0.0f, value = 0.0f;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        if (32 * r >= splits) break;
        const float factor = mine[r].x == -INFINITY ? 0.0f : power_of_two(mine[r].x - top);
#pragma unroll
        for (int part = 0; part < 32; part += kAhead) {
            if (32 * r + part >= splits) break;
            float numbers[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int s = 32 * r + part + kAhead + i;
                numbers[i] = ahead[i];
                ahead[i] = s < splits ? from[(long long)s * kD] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const float f = __shfl_sync(0xFFFFFFFFu, factor, part + i), sum = __shfl_sync(0xFFFFFFFFu, mine[r].y, part + i);
                total = fmaf(sum, f, total);
                value = fmaf(numbers[i], f, value);
            }
        }
    }
    if (kSlices > 1 && all > kPagedMostSplits) {
        slice_value[slice][d] = value;
        if (d == 0) slice_total[slice] = total;
        __syncthreads();
        for (int other = 1; other < kSlices && other * kPagedMostSplits < all; ++other) {
            total += slice_total[other];
            value += slice_value[other][d];
        }
    }
    if (slice > 0) return;
    p.out[at * kD + d] = (uint16_t)pack_pair<kHalf>(total == 0.0f ? 0.0f : value / total, 0.0f);
}

inline size_t paged_attention_workspace_bytes(int batch, int q_heads, int kv_heads, int head_dim, long long capacity) {
    const int splits = paged_most_splits(capacity, paged_split_limit(kv_heads));
    if (splits <= 1) return 0;
    return (size_t)batch * q_heads * splits * (head_dim + 2) * sizeof(float);
}

template <int kD, bool kHalf, int kTiles>
inline int launch_paged_attention_instance(PagedAttentionParams params, int sm_count, cudaStream_t stream) {
    using Shape = PagedShape<kD>;
    static bool configured[64] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return MT_ERR_LAUNCH;
    if (device >= 64 || !configured[device]) {
        if (cudaFuncSetAttribute(paged_attention_kernel<kD, kHalf, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem) != cudaSuccess)
            return MT_ERR_LAUNCH;
        if (device < 64) configured[device] = true;
    }
    const int group = params.q_heads / params.kv_heads;
    const long long per_split = (long long)params.kv_heads * ((group + 8 * kTiles - 1) / (8 * kTiles));
    // Short tables and few requests: one launch, a CTA for the splits of a KV head, where every CTA has an SM of its own.  The same
    // sums in the same order.  One request, 8 heads of 128, one launch and two: three splits 7.6 and 9.0 us, six 10.2 and 9.0.
    params.together = params.most_splits > 1 && params.most_splits <= kPagedTogether && params.batch * per_split <= sm_count;
    const long long most_units = params.together ? params.batch * per_split : params.batch * per_split * params.most_splits;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(most_units < sm_count ? (unsigned int)most_units : sm_count, 1, 1);
    config.blockDim = dim3(Shape::kWarps * 32, 1, 1);
    config.dynamicSmemBytes = Shape::kSmem;
    config.stream = stream;
    cudaLaunchAttribute attrs[1];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, paged_attention_kernel<kD, kHalf, kTiles>, params) != cudaSuccess) return MT_ERR_LAUNCH;
    if (params.most_splits > 1 && !params.together) {
        config.gridDim = dim3(params.batch * params.q_heads, 1, 1);
        const bool sliced = params.most_splits > kPagedMostSplits;
        config.blockDim = dim3(sliced ? kPagedSlices * kD : kD, 1, 1);
        config.dynamicSmemBytes = 0;
        if (cudaLaunchKernelEx(&config, sliced ? paged_attention_join_kernel<kD, kHalf, kPagedSlices> : paged_attention_join_kernel<kD, kHalf, 1>, params) != cudaSuccess)
            return MT_ERR_LAUNCH;
    }
    return MT_OK;
}

template <int kD, bool kHalf>
inline int launch_paged_attention(const PagedAttentionParams& params, int sm_count, cudaStream_t stream) {
    return params.q_heads / params.kv_heads <= 8 ? launch_paged_attention_instance<kD, kHalf, 1>(params, sm_count, stream)
                                                 : launch_paged_attention_instance<kD, kHalf, 2>(params, sm_count, stream);
}

}  // namespace mt
