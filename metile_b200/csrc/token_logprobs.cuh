// Log-probabilities of given tokens, with the entropy of their rows and the best alternatives.
//
// With m the largest logit of a row and d = x - m:  S = sum e^d,  logprob(t) = d_t - log S,  entropy = log S - sum e^d d / S.
// One pass over the logits: a CTA takes a part of a row (32 KB), keeps it in registers, and leaves its maximum, the two sums
// relative to that maximum and its `top` best entries; a second kernel joins the parts, in order and in 64 bits.  Parts
// have one size for all calls, so a row's bits do not depend on the others.
#pragma once

#include "beam_select.cuh"

namespace mt {

constexpr unsigned int kTokenOutside = 0x307;  // token_logprobs: word 1 = row, 2 and 3 = the token

constexpr int kLogprobThreads = 256, kLogprobVectors = 8, kLogprobMaxTop = 64, kLogprobJoinThreads = 128;
constexpr int kLogprobPartBytes = kLogprobThreads * kLogprobVectors * 16;
__host__ __device__ constexpr int logprob_part(int type) { return kLogprobPartBytes / beam_size(type); }  // logits
inline int logprob_parts(int vocabulary, int type) { return (vocabulary + logprob_part(type) - 1) / logprob_part(type); }

struct LogprobStats {
    float top, sum, weighted;  // maximum; sums of e^d and e^d d
};

struct LogprobParams {
    const void* logits;         // [rows, vocabulary], rows `row_stride` apart
    const long long* tokens;    // [rows]
    float *logprobs, *entropy;  // [rows]
    float* top_logprobs;        // [rows, top]
    long long* top_tokens;      // [rows, top]
    LogprobStats* stats;        // [rows, parts]
    unsigned long long* lists;  // [rows, parts, top]: keys, the largest first
    long long row_stride;
    int rows, vocabulary, parts, top;
};

// The logits of a vector, 4 of 32 bits or 8 of 16.
template <int kType>
__device__ __forceinline__ float logit_of(const uint4& v, int e) {
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
    if constexpr (kType == 2) {
        return __uint_as_float(words[e]);
    } else {
        const float2 pair = kType == 1 ? __half22float2(*reinterpret_cast<const __half2*>(&words[e >> 1]))
                                       : make_float2(bf16_lo(words[e >> 1]), bf16_hi(words[e >> 1]));
        return e & 1 ? pair.y : pair.x;
    }
}

template <int kType>
__global__ void __launch_bounds__(kLogprobThreads) token_logprobs_part_kernel(const LogprobParams p) {
    constexpr int kSize = beam_size(kType), kEach = 16 / kSize, kPart = logprob_part(kType), kWarps = kLogprobThreads / 32;
    __shared__ float warp_top[kWarps], warp_sum[kWarps], warp_weighted[kWarps];
    __shared__ unsigned long long warp_key[2][kWarps];
    const int row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = part * kPart, count = min(kPart, p.vocabulary - first);  // of this part
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const char* base = static_cast<const char*>(p.logits) + (row * p.row_stride + first) * kSize;
    const int shift = (int)(reinterpret_cast<uintptr_t>(base) & 15);
    uint4 v[kLogprobVectors];
    if (shift == 0) {
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) {
            const int at = (i * kLogprobThreads + threadIdx.x) * kEach;
            v[i] = at < count ? ptx::ld_global_dependent_u4(base + (size_t)at * kSize) : make_uint4(0u, 0u, 0u, 0u);
        }
    } else {
        // A row may start anywhere: the two aligned vectors that a vector lies in, shifted.
        const char* aligned = base - shift;
        const int bits = (shift & 3) * 8;
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) {
            const int at = (i * kLogprobThreads + threadIdx.x) * kEach;
            const uint4 a = at < count ? ptx::ld_global_dependent_u4(aligned + (size_t)at * kSize) : make_uint4(0u, 0u, 0u, 0u);
            // The second one only where it holds a logit of the part.
            const uint4 b = at + kEach - shift / kSize < count ? ptx::ld_global_dependent_u4(aligned + (size_t)at * kSize + 16) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t low = shift < 4 ? w[j] : shift < 8 ? w[j + 1] : shift < 12 ? w[j + 2] : w[j + 3];
                const uint32_t high = shift < 4 ? w[j + 1] : shift < 8 ? w[j + 2] : shift < 12 ? w[j + 3] : w[j + 4];
                out[j] = __funnelshift_r(low, high, bits);
            }
            v[i] = make_uint4(out[0], out[1], out[2], out[3]);
        }
    }
    // Logits behind the part count as -inf; a thread has element e of vector i if e < there(i).
    auto there = [&](int i) { return count - (i * kLogprobThreads + (int)threadIdx.x) * kEach; };
    auto logit = [&](int i, int e) { return e < there(i) ? logit_of<kType>(v[i], e) : -INFINITY; };
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLogprobVectors; ++i)
#pragma unroll
        for (int e = 0; e < kEach; ++e) top = fmaxf(top, logit(i, e));
    float all = top;
#pragma unroll
    for (int offset = 16; offset >= 1; offset >>= 1) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, offset));
    if (lane == 0) warp_top[warp] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all = fmaxf(all, warp_top[w]);
    // Where all are -inf their exponentials are none; a NaN is one.
    const float against = all == -INFINITY ? 0.0f : all;
    float sum = 0.0f, weighted = 0.0f;
#pragma unroll
    for (int i = 0; i < kLogprobVectors; ++i) {
        float s = 0.0f, w = 0.0f;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const float d = logit(i, e) - against;
            float power;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(power) : "f"(d * 1.4426950408889634f));
            s += power;
            w += power == 0.0f ? 0.0f : power * d;
        }
        sum += s;
        weighted += w;
    }
    sum = warp_sum_xor(sum);
    weighted = warp_sum_xor(weighted);
    if (lane == 0) {
        warp_sum[warp] = sum;
        warp_weighted[warp] = weighted;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        LogprobStats stats = {all, 0.0f, 0.0f};
        for (int w = 0; w < kWarps; ++w) {
            stats.sum += warp_sum[w];
            stats.weighted += warp_weighted[w];
        }
        p.stats[blockIdx.x] = stats;
    }
    // The best, one after the other: every thread offers the best of its own below the last one taken.
    unsigned long long last = ~0ull, best = 0;
    auto look = [&] {
        best = 0;
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i)
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (e >= there(i)) continue;
                const unsigned long long key = beam_entry_key(logit_of<kType>(v[i], e), first + (i * kLogprobThreads + (int)threadIdx.x) * kEach + e);
                if (key < last && key > best) best = key;
            }
    };
    if (p.top > 0) look();
    for (int k = 0; k < p.top; ++k) {
        unsigned int high = (unsigned int)(best >> 32), low = (unsigned int)best;
        const unsigned int highest = __reduce_max_sync(0xFFFFFFFFu, high);
        low = __reduce_max_sync(0xFFFFFFFFu, high == highest ? low : 0u);
        if (lane == 0) warp_key[k & 1][warp] = (unsigned long long)highest << 32 | low;
        __syncthreads();
        unsigned long long winner = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) winner = max(winner, warp_key[k & 1][w]);
        if (threadIdx.x == 0) p.lists[(size_t)blockIdx.x * p.top + k] = winner;
        if (best == winner && winner != 0) {
            last = winner;
            look();
        }
    }
}

// A CTA joins the parts of a row.
__global__ void __launch_bounds__(kLogprobJoinThreads) token_logprobs_join_kernel(const LogprobParams p, int type) {
    extern __shared__ unsigned long long keys[];  // [parts, top]
    __shared__ double shared_lse, shared_top;
    const int row = blockIdx.x;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const LogprobStats* stats = p.stats + (size_t)row * p.parts;
    const unsigned long long* lists = p.lists + (size_t)row * p.parts * p.top;
    for (int i = threadIdx.x; i < p.parts * p.top; i += blockDim.x) keys[i] = lists[i];
    if (threadIdx.x == 0) {
        float top = -INFINITY;
        bool usable = true;  // neither NaN nor +inf
        for (int i = 0; i < p.parts; ++i) {
            top = fmaxf(top, stats[i].top);
            usable = usable && stats[i].sum <= 3e38f;
        }
        usable = usable && top != -INFINITY && top != INFINITY;
        double sum = 0.0, weighted = 0.0;
        for (int i = 0; i < p.parts; ++i) {
            if (stats[i].top == -INFINITY) continue;
            const double d = (double)stats[i].top - top, factor = exp(d);
            sum += factor * stats[i].sum;
            weighted += factor * (stats[i].weighted + d * stats[i].sum);
        }
        const double log_sum = usable ? log(sum) : NAN;
        shared_lse = log_sum;
        shared_top = top;
        p.entropy[row] = (float)(log_sum - weighted / sum);
        const long long token = p.tokens[row];
        float logprob = token < 0 ? 0.0f : NAN;
        if (token >= p.vocabulary) {
            record_index(kTokenOutside, row, (unsigned long long)token);
        } else if (token >= 0) {
            const long long at = row * p.row_stride + token;
            const float x = type == MT_TYPE_FP32 ? static_cast<const float*>(p.logits)[at]
                            : type == MT_TYPE_FP16 ? __half2float(static_cast<const __half*>(p.logits)[at])
                                                   : bf16_bits_to_f32(static_cast<const uint16_t*>(p.logits)[at]);
            logprob = (float)((double)x - top - log_sum);
        }
        p.logprobs[row] = logprob;
    }
    __syncthreads();
    const double lse = shared_lse, largest = shared_top;
    const bool usable = lse == lse;
    for (int i = threadIdx.x; i < p.parts * p.top; i += blockDim.x) {
        // Its place: its own in its list, and in every other as many as are larger.
        const int part = i / p.top, own = i - part * p.top;
        const unsigned long long key = keys[i];
        int rank = own;
        if (usable && key == 0) continue;
        for (int other = 0; other < p.parts && rank < p.top; ++other) {
            if (other == part) continue;
            int low = 0, high = p.top;  // keys before `low` are larger, those from `high` on are not
            while (low < high) {
                const int middle = (low + high) >> 1;
                if (keys[other * p.top + middle] > key) low = middle + 1; else high = middle;
            }
            rank += low;
        }
        if (!usable) rank = i;  // the row has no distribution
        if (rank >= p.top) continue;
        const BeamEntry entry = beam_entry(key);
        p.top_logprobs[(size_t)row * p.top + rank] = usable ? (float)((double)entry.logit - largest - lse) : NAN;
        p.top_tokens[(size_t)row * p.top + rank] = usable ? entry.token : -1;
    }
}

inline size_t logprob_stats_bytes(int rows, int parts) { return ((size_t)rows * parts * sizeof(LogprobStats) + 15) / 16 * 16; }

template <int kType>
inline int launch_token_logprobs(const LogprobParams& params, cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(params.rows * params.parts, 1, 1);
    config.blockDim = dim3(kLogprobThreads, 1, 1);
    config.stream = stream;
    cudaLaunchAttribute attrs[1];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, token_logprobs_part_kernel<kType>, params) != cudaSuccess) return MT_ERR_LAUNCH;
    config.gridDim = dim3(params.rows, 1, 1);
    config.blockDim = dim3(kLogprobJoinThreads, 1, 1);
    config.dynamicSmemBytes = (size_t)params.parts * params.top * sizeof(unsigned long long);
    return cudaLaunchKernelEx(&config, token_logprobs_join_kernel, params, kType) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
}

}  // namespace mt
