// Attention of several new tokens per request over a paged key-value cache.
//
// Rows starts[r] .. starts[r + 1] - 1 of the queries are the last tokens of request r, which has lengths[r] tokens with them: the
// i-th of n stands at position lengths[r] - n + i and sees the tokens up to its own.
#pragma once

#include "paged_attention.cuh"

namespace mt {

constexpr unsigned int kStartOutside = 0x306;  // paged_attention_chunk: word 1 = request, 2 = its first row

struct PagedChunkParams {
    const uint16_t* q;                 // [rows, Hq, D]
    const uint16_t *key_pages, *value_pages;
    PageStrides key_strides, value_strides;
    const int* tables;                 // [requests, width], rows `table_stride` apart
    const int* lengths;                // [requests]
    const int* starts;                 // [requests + 1]
    uint16_t* out;                     // [rows, Hq, D]
    long long table_stride;
    int width, rows, requests, q_heads, kv_heads, page_shift, page_count;
    float scale;
};

// A warp for every row and query head, the head dimension over its lanes.
template <int kD, bool kHalf>
__global__ void __launch_bounds__(128) paged_chunk_kernel(const __grid_constant__ PagedChunkParams p) {
    constexpr int kPairs = kD / 64;
    const int lane = threadIdx.x & 31;
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    if (at >= (long long)p.rows * p.q_heads) return;
    const int row = (int)(at / p.q_heads), head = (int)(at - (long long)row * p.q_heads), kv_head = head / (p.q_heads / p.kv_heads);
    // The request whose rows these are.
    int request = -1, position = -1;
    for (int r = 0; r < p.requests; ++r) {
        const int first = p.starts[r], end = p.starts[r + 1];
        if (first < 0 || end < first || end > p.rows) {
            if (lane == 0) record_index(kStartOutside, r, (unsigned int)first);
            continue;
        }
        if (row >= first && row < end) {
            int n = p.lengths[r];
            const long long capacity = (long long)p.width << p.page_shift;
            if (n < 0 || n > capacity) {
                if (lane == 0) record_index(kLengthOutside, r, (unsigned int)n);
                n = n < 0 ? 0 : (int)capacity;
            }
            request = r;
            position = n - (end - row);
            break;
        }
    }
    float2 q[kPairs], acc[kPairs];
    const uint32_t* query = reinterpret_cast<const uint32_t*>(p.q + at * kD);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        q[i] = unpack_pair<kHalf>(query[i * 32 + lane]);
        acc[i] = make_float2(0.0f, 0.0f);
    }
    float top = -INFINITY, sum = 0.0f;
    for (int t = 0; t <= position; ++t) {
        const int id = p.tables[request * p.table_stride + (t >> p.page_shift)], in_page = t & ((1 << p.page_shift) - 1);
        if ((unsigned int)id >= (unsigned int)p.page_count) {
            if (lane == 0) record_index(kPageOutside, request, (unsigned int)id);
            continue;
        }
        const uint32_t* key = reinterpret_cast<const uint32_t*>(p.key_pages + id * p.key_strides.page + kv_head * p.key_strides.head + in_page * p.key_strides.token);
        const uint32_t* value = reinterpret_cast<const uint32_t*>(p.value_pages + id * p.value_strides.page + kv_head * p.value_strides.head + in_page * p.value_strides.token);
        float score = 0.0f;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const float2 k = unpack_pair<kHalf>(key[i * 32 + lane]);
            score = fmaf(q[i].x, k.x, fmaf(q[i].y, k.y, score));
        }
        score = warp_sum_xor(score) * p.scale;
        if (score == -INFINITY) continue;
        const float now = fmaxf(top, score), factor = now == -INFINITY ? 1.0f : __expf(top - now), weight = __expf(score - now);
        top = now;
        sum = fmaf(sum, factor, weight);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const float2 v = unpack_pair<kHalf>(value[i * 32 + lane]);
            acc[i] = make_float2(fmaf(acc[i].x, factor, weight * v.x), fmaf(acc[i].y, factor, weight * v.y));
        }
    }
    uint32_t* out = reinterpret_cast<uint32_t*>(p.out + at * kD);
    const float factor = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) out[i * 32 + lane] = pack_pair<kHalf>(acc[i].x * factor, acc[i].y * factor);
}

}  // namespace mt
