// Decode attention of one new token per request over a paged key-value cache.
#pragma once

#include "paged_cache.cuh"

namespace mt {

struct PagedAttentionParams {
    const uint16_t* q;                 // [batch, Hq, D]
    const uint16_t *key_pages, *value_pages;
    PageStrides key_strides, value_strides;
    const int* tables;                 // [batch, width], rows `table_stride` apart
    const int* lengths;                // [batch]
    uint16_t* out;                     // [batch, Hq, D]
    float* partial;
    long long table_stride;
    int width, batch, q_heads, kv_heads, page_shift, page_count;
    float scale;
};

// One CTA per request and query head; its four warps take the tokens in turn, a lane holds D / 32 of a row.
template <bool kHalf>
__device__ __forceinline__ float element_f32(uint16_t bits) {
    if constexpr (kHalf) return __half2float(*reinterpret_cast<const __half*>(&bits));
    else return bf16_bits_to_f32(bits);
}

template <int kD, bool kHalf>
__global__ void __launch_bounds__(128) paged_attention_kernel(const PagedAttentionParams p) {
    constexpr int kPer = kD / 32;
    __shared__ float top_of[4], sum_of[4], acc_of[4][kD];
    const int b = blockIdx.x / p.q_heads, qh = blockIdx.x - b * p.q_heads, h = qh / (p.q_heads / p.kv_heads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const long long capacity = (long long)p.width << p.page_shift;
    int n = p.lengths[b];
    if (n < 0 || n > capacity) {
        if (threadIdx.x == 0) record_index(kLengthOutside, b, (unsigned int)n);
        n = n < 0 ? 0 : (int)capacity;
    }
    float q[kPer], acc[kPer], top = -INFINITY, sum = 0.0f;
    for (int i = 0; i < kPer; ++i) {
        q[i] = element_f32<kHalf>(p.q[(long long)blockIdx.x * kD + i * 32 + lane]);
        acc[i] = 0.0f;
    }
    for (int t = warp; t < n; t += 4) {
        const int page = p.tables[b * p.table_stride + (t >> p.page_shift)];
        if (page < 0 || page >= p.page_count) {
            if (lane == 0) record_index(kPageOutside, b, (unsigned int)page);
            continue;
        }
        const int row = t & ((1 << p.page_shift) - 1);
        const uint16_t* key = p.key_pages + page * p.key_strides.page + h * p.key_strides.head + row * p.key_strides.token;
        const uint16_t* value = p.value_pages + page * p.value_strides.page + h * p.value_strides.head + row * p.value_strides.token;
        float dot = 0.0f;
        for (int i = 0; i < kPer; ++i) dot = fmaf(q[i], element_f32<kHalf>(key[i * 32 + lane]), dot);
        const float score = warp_sum_xor(dot) * p.scale, now = fmaxf(top, score);
        if (now == -INFINITY) continue;
        const float keep = __expf(top - now), weight = __expf(score - now);
        sum = sum * keep + weight;
        for (int i = 0; i < kPer; ++i) acc[i] = fmaf(weight, element_f32<kHalf>(value[i * 32 + lane]), acc[i] * keep);
        top = now;
    }
    if (lane == 0) {
        top_of[warp] = top;
        sum_of[warp] = sum;
    }
    for (int i = 0; i < kPer; ++i) acc_of[warp][i * 32 + lane] = acc[i];
    __syncthreads();
    float best = -INFINITY, total = 0.0f;
    for (int w = 0; w < 4; ++w) best = fmaxf(best, top_of[w]);
    float factor[4];
    for (int w = 0; w < 4; ++w) {
        factor[w] = top_of[w] == -INFINITY ? 0.0f : __expf(top_of[w] - best);
        total += sum_of[w] * factor[w];
    }
    for (int d = threadIdx.x; d < kD; d += blockDim.x) {
        float value = 0.0f;
        for (int w = 0; w < 4; ++w) value = fmaf(acc_of[w][d], factor[w], value);
        const uint32_t pair = pack_pair<kHalf>(total == 0.0f ? 0.0f : value / total, 0.0f);
        p.out[(long long)blockIdx.x * kD + d] = (uint16_t)pair;
    }
}

template <int kD, bool kHalf>
inline int launch_paged_attention(const PagedAttentionParams& params, cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(params.batch * params.q_heads, 1, 1);
    config.blockDim = dim3(128, 1, 1);
    config.stream = stream;
    cudaLaunchAttribute attrs[1];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, paged_attention_kernel<kD, kHalf>, params) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
}

}  // namespace mt
