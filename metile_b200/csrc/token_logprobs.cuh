// Log-probabilities of given tokens, with the entropy of their rows and the best alternatives.
//
// With m the largest logit of a row and d = x - m:  S = sum e^d,  logprob(t) = d_t - log S,  entropy = log S - sum e^d d / S.
// One pass over the logits: a CTA takes a part of a row (32 KB), keeps it in registers, and leaves its maximum, the two sums
// relative to that maximum and its `top` best entries; a second kernel joins the parts, in order and in 64 bits.  Parts
// have one size for all calls, so a row's bits do not depend on the others.
#pragma once

#include "beam_select.cuh"
#include "paged_attention.cuh"

namespace mt {

constexpr unsigned int kTokenOutside = 0x307;  // token_logprobs: word 1 = row, 2 and 3 = the token

constexpr int kLogprobThreads = 256, kLogprobVectors = 8, kLogprobMaxTop = 64, kLogprobJoinThreads = 128;
constexpr int kLogprobSlack = 16, kLogprobCollect = 512;
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

// Of a vector, NaN left out; pairs of 16 bits at once.
template <int kType>
__device__ __forceinline__ float largest_logit(const uint4& v) {
    if constexpr (kType == 2) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else {
        uint32_t a, b;
        if constexpr (kType == 1) {
            asm("max.f16x2 %0, %1, %2;" : "=r"(a) : "r"(v.x), "r"(v.y));
            asm("max.f16x2 %0, %1, %2;" : "=r"(b) : "r"(v.z), "r"(v.w));
            asm("max.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
        } else {
            asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(v.x), "r"(v.y));
            asm("max.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(v.z), "r"(v.w));
            asm("max.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
        }
        const uint4 both = make_uint4(a, 0u, 0u, 0u);
        return fmaxf(logit_of<kType>(both, 0), logit_of<kType>(both, 1));
    }
}
template <int kType>
__device__ __forceinline__ float logit_at(const char* base, int i) {
    if constexpr (kType == 2) return reinterpret_cast<const float*>(base)[i];
    else if constexpr (kType == 1) return __half2float(reinterpret_cast<const __half*>(base)[i]);
    else return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(base)[i]);
}
__device__ __forceinline__ LogprobStats share_stats(float top, const float* sums, const float* weighted) {
    LogprobStats stats = {top, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kLogprobThreads / 32; ++w) {
        stats.sum += sums[w];
        stats.weighted += weighted[w];
    }
    return stats;
}

// What has been made of the vectors is made again, rather than kept in registers until then.
__device__ __forceinline__ void forget(uint4 (&v)[kLogprobVectors]) {
#pragma unroll
    for (int i = 0; i < kLogprobVectors; ++i) asm volatile("" : "+r"(v[i].x), "+r"(v[i].y), "+r"(v[i].z), "+r"(v[i].w));
}

// kAligned: every row starts on 16 bytes.
template <int kType, bool kAligned>
__global__ void __launch_bounds__(kLogprobThreads, kAligned ? 4 : 3) token_logprobs_part_kernel(const LogprobParams p) {
    constexpr int kSize = beam_size(kType), kEach = 16 / kSize, kPart = logprob_part(kType), kWarps = kLogprobThreads / 32;
    __shared__ float warp_top[kWarps], warp_sum[kWarps], warp_weighted[kWarps];
    __shared__ unsigned long long warp_key[2][kWarps], collected[kLogprobCollect];
    __shared__ unsigned int thread_top[kLogprobThreads], bound;
    __shared__ int found;
    const int row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = part * kPart, count = min(kPart, p.vocabulary - first);  // of this part
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const char* base = static_cast<const char*>(p.logits) + (row * p.row_stride + first) * kSize;
    uint4 v[kLogprobVectors];
    if constexpr (kAligned) {
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) {
            const int at = (i * kLogprobThreads + threadIdx.x) * kEach;
            v[i] = at < count ? ptx::ld_global_dependent_u4(base + (size_t)at * kSize) : make_uint4(0u, 0u, 0u, 0u);
        }
    } else {
        // A row may start anywhere: the two aligned vectors that a vector lies in, shifted; the second one is the next lane's first.
        const int shift = (int)(reinterpret_cast<uintptr_t>(base) & 15), bits = (shift & 3) * 8;
        const char* aligned = base - shift;
        // Vectors that hold a logit of the part.
        auto load = [&](int at) { return at * kEach - shift / kSize < count ? ptx::ld_global_dependent_u4(aligned + (size_t)at * 16) : make_uint4(0u, 0u, 0u, 0u); };
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) v[i] = load(i * kLogprobThreads + threadIdx.x);
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) {
            uint4 next = {__shfl_down_sync(0xFFFFFFFFu, v[i].x, 1), __shfl_down_sync(0xFFFFFFFFu, v[i].y, 1), __shfl_down_sync(0xFFFFFFFFu, v[i].z, 1),
                          __shfl_down_sync(0xFFFFFFFFu, v[i].w, 1)};
            if (lane == 31) next = load(i * kLogprobThreads + threadIdx.x + 1);
            uint32_t w[7] = {v[i].x, v[i].y, v[i].z, v[i].w, next.x, next.y, next.z}, last = next.w;
            if (shift & 8) {
#pragma unroll
                for (int j = 0; j < 5; ++j) w[j] = w[j + 2];
                w[5] = last;
            }
            if (shift & 4) {
#pragma unroll
                for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
            }
            v[i] = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
        }
    }
    // Logits behind the part count as -inf; a thread has element e of vector i if e < there(i).
    auto there = [&](int i) { return count - (i * kLogprobThreads + (int)threadIdx.x) * kEach; };
    constexpr uint32_t kNothing = kType == 2 ? 0xFF800000u : kType == 1 ? 0xFC00u : 0xFF80u;
    if (count < kPart) {
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) {
            const int left = there(i);
            if (left >= kEach) continue;
            uint32_t words[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (kType == 2) {
                    if (left <= j) words[j] = kNothing;
                } else {
                    if (left <= 2 * j) words[j] = kNothing | kNothing << 16;
                    else if (left == 2 * j + 1) words[j] = (words[j] & 0xFFFFu) | kNothing << 16;
                }
            }
            v[i] = make_uint4(words[0], words[1], words[2], words[3]);
        }
    }
    float top = largest_logit<kType>(v[0]);
#pragma unroll
    for (int i = 1; i < kLogprobVectors; ++i) top = fmaxf(top, largest_logit<kType>(v[i]));
    forget(v);
    float all = top;
#pragma unroll
    for (int offset = 16; offset >= 1; offset >>= 1) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, offset));
    if (lane == 0) warp_top[warp] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all = fmaxf(all, warp_top[w]);
    // Where all are -inf their exponentials are none; a NaN is one.  In powers of two: e = (x - m) log2 e, sums of 2^e and of 2^e e.
    constexpr float kLog2E = 1.4426950408889634f;
    const float against = all == -INFINITY ? 0.0f : -all;
    float2 sums = make_float2(0.0f, 0.0f), weights = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kLogprobVectors; ++i) {
        float2 s = make_float2(0.0f, 0.0f), w = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < kEach / 2; ++j) {
            // The difference first: it is exact where it counts.
            const float2 d = add_f32x2(make_float2(logit_of<kType>(v[i], 2 * j), logit_of<kType>(v[i], 2 * j + 1)), make_float2(against, against));
            const float2 e = mul_f32x2(d, make_float2(kLog2E, kLog2E)), power = make_float2(power_of_two(e.x), power_of_two(e.y));
            s = add_f32x2(s, power);
            w = ptx::fma_f32x2(power, e, w);
        }
        sums = add_f32x2(sums, s);
        weights = add_f32x2(weights, w);
    }
    float sum = sums.x + sums.y, weighted = weights.x + weights.y;
    if (weighted != weighted) {  // 0 times -inf among them, which is nothing
        weighted = 0.0f;
#pragma unroll 1
        for (int i = 0; i < kLogprobVectors; ++i)
#pragma unroll 1
            for (int j = 0; j < min(kEach, there(i)); ++j) {
                const float e = (logit_at<kType>(base, (i * kLogprobThreads + (int)threadIdx.x) * kEach + j) + against) * kLog2E, power = power_of_two(e);
                weighted += power == 0.0f ? 0.0f : power * e;
            }
    }
    forget(v);
    sum = warp_sum_xor(sum);
    weighted = warp_sum_xor(weighted);
    if (lane == 0) {
        warp_sum[warp] = sum;
        warp_weighted[warp] = weighted * 0.6931471805599453f;
    }
    if (p.top == 0) {
        __syncthreads();
        if (threadIdx.x == 0) p.stats[blockIdx.x] = share_stats(all, warp_sum, warp_weighted);
        return;
    }
    // The best.  At least `top` threads have a logit at or above a bound that is found by halving; only they look for those that reach
    // it, and what they find is ranked.  The bound need not be the best one: up to kLogprobSlack threads more may reach it.
    const unsigned int own = there(0) > 0 ? beam_logit_order(top) : 0u;  // threads behind the part have none
    const int threads = min(kLogprobThreads, (count + kEach - 1) / kEach);
    thread_top[threadIdx.x] = own;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    if (warp == 0) {
        unsigned int low = 1u;
        if (threads > p.top + kLogprobSlack) {
            unsigned int tops[kWarps], least = ~0u, high = beam_logit_order(all) + 1u;  // the count reaches `top` at `low`, not at `high`
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                tops[w] = thread_top[32 * w + lane];
                least = min(least, tops[w] - 1u);  // none: the largest
            }
            low = __reduce_min_sync(0xFFFFFFFFu, least) + 1u;
            while (high - low > 1u) {
                const unsigned int middle = low + (high - low) / 2;
                int reach = 0;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) reach += tops[w] >= middle;
                reach = __reduce_add_sync(0xFFFFFFFFu, reach);
                if (reach >= p.top) low = middle; else high = middle;
                if (reach >= p.top && reach <= p.top + kLogprobSlack) break;
            }
        }
        if (lane == 0) bound = low;
    }
    __syncthreads();
    const unsigned int low = bound;
    if (threadIdx.x == 0) p.stats[blockIdx.x] = share_stats(all, warp_sum, warp_weighted);
    if (own >= low) {
        const float least = low <= 1u ? -INFINITY : beam_ordered_logit(low);
        unsigned int vectors = 0;  // with a logit that reaches it
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) vectors |= (largest_logit<kType>(v[i]) >= least ? 1u : 0u) << i;
        for (; vectors; vectors &= vectors - 1u) {  // read again: an index into the registers would move them, and eight copies of this do not fit the cache
            const int at = ((__ffs(vectors) - 1) * kLogprobThreads + (int)threadIdx.x) * kEach, here = min(kEach, count - at);
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (e >= here) break;
                const float x = logit_at<kType>(base, at + e);
                if (!(x >= least)) continue;
                const int to = atomicAdd(&found, 1);
                if (to < kLogprobCollect) collected[to] = beam_entry_key(x, first + at + e);
            }
        }
    }
    __syncthreads();
    const int many = found;
    unsigned long long* list = p.lists + (size_t)blockIdx.x * p.top;
    if (many <= kLogprobCollect) {
        for (int i = threadIdx.x; i < many; i += kLogprobThreads) {
            const unsigned long long key = collected[i];
            int rank = 0;
            for (int j = 0; j < many; ++j) rank += collected[j] > key;
            if (rank < p.top) list[rank] = key;
        }
        for (int i = many + threadIdx.x; i < p.top; i += kLogprobThreads) list[i] = 0;  // the part has fewer
        return;
    }
    // More than are collected reach the bound (equal ones, or all of them one thread's): one after the other, every thread offering
    // the best of its own below the last one taken.
    unsigned long long last = ~0ull, best = 0;
    auto look = [&] {
        best = 0;
#pragma unroll 1
        for (int i = 0; i < kLogprobVectors; ++i)
#pragma unroll 1
            for (int e = 0; e < kEach; ++e) {
                if (e >= there(i)) continue;
                const int token = (i * kLogprobThreads + (int)threadIdx.x) * kEach + e;  // read again: an index into the registers would move them
                const unsigned long long key = beam_entry_key(logit_at<kType>(base, token), first + token);
                if (key < last && key > best) best = key;
            }
    };
    look();
    for (int k = 0; k < p.top; ++k) {
        unsigned int upper = (unsigned int)(best >> 32), lower = (unsigned int)best;
        const unsigned int highest = __reduce_max_sync(0xFFFFFFFFu, upper);
        lower = __reduce_max_sync(0xFFFFFFFFu, upper == highest ? lower : 0u);
        if (lane == 0) warp_key[k & 1][warp] = (unsigned long long)highest << 32 | lower;
        __syncthreads();
        unsigned long long winner = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) winner = max(winner, warp_key[k & 1][w]);
        if (threadIdx.x == 0) list[k] = winner;
        if (best == winner && winner != 0) {
            last = winner;
            look();
        }
    }
}

__device__ __forceinline__ double warp_sum_double(double v) {
#pragma unroll
    for (int offset = 16; offset >= 1; offset >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, offset);
    return v;
}

// A CTA joins the parts of a row: its first warp the sums, a part a lane, while the others fetch the lists.
__global__ void __launch_bounds__(kLogprobJoinThreads) token_logprobs_join_kernel(const LogprobParams p, int type) {
    extern __shared__ unsigned long long keys[];  // [parts, top]
    __shared__ double shared_lse, shared_top;
    const int row = blockIdx.x, entries = p.parts * p.top;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    if (threadIdx.x < 32) {
        const LogprobStats* stats = p.stats + (size_t)row * p.parts;
        const long long token = threadIdx.x == 0 ? p.tokens[row] : -1;
        float chosen = 0.0f;
        if (token >= 0 && token < p.vocabulary) {
            const char* at = static_cast<const char*>(p.logits) + (row * p.row_stride + token) * beam_size(type);
            chosen = type == MT_TYPE_FP32 ? logit_at<2>(at, 0) : type == MT_TYPE_FP16 ? logit_at<1>(at, 0) : logit_at<0>(at, 0);
        }
        float top = -INFINITY;
        bool usable = true;  // neither NaN nor +inf
        for (int i = threadIdx.x; i < p.parts; i += 32) {
            top = fmaxf(top, stats[i].top);
            usable = usable && stats[i].sum <= 3e38f;
        }
#pragma unroll
        for (int offset = 16; offset >= 1; offset >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, offset));
        usable = __all_sync(0xFFFFFFFFu, usable) && top != -INFINITY && top != INFINITY;
        double sum = 0.0, weighted = 0.0;
        for (int i = threadIdx.x; i < p.parts; i += 32) {
            const LogprobStats part = stats[i];
            if (part.top == -INFINITY) continue;
            const double d = (double)part.top - top, factor = exp(d);
            sum += factor * part.sum;
            weighted += factor * (part.weighted + d * part.sum);
        }
        sum = warp_sum_double(sum);
        weighted = warp_sum_double(weighted);
        if (threadIdx.x == 0) {
            const double log_sum = usable ? log(sum) : NAN;
            shared_lse = log_sum;
            shared_top = top;
            p.entropy[row] = (float)(log_sum - weighted / sum);
            if (token >= p.vocabulary) record_index(kTokenOutside, row, (unsigned long long)token);
            p.logprobs[row] = token < 0 ? 0.0f : token >= p.vocabulary ? NAN : (float)((double)chosen - top - log_sum);
        }
    } else {
        const unsigned long long* lists = p.lists + (size_t)row * entries;
        for (int i = threadIdx.x - 32; i < entries; i += blockDim.x - 32) keys[i] = lists[i];
    }
    if (p.top == 0) return;
    __syncthreads();
    const double lse = shared_lse, largest = shared_top;
    const bool usable = lse == lse;
    for (int i = threadIdx.x; i < entries; i += blockDim.x) {
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
    const bool aligned = aligned_to(params.logits, 16) && (params.rows == 1 || params.row_stride * beam_size(kType) % 16 == 0);
    if (cudaLaunchKernelEx(&config, aligned ? token_logprobs_part_kernel<kType, true> : token_logprobs_part_kernel<kType, false>, params) != cudaSuccess) return MT_ERR_LAUNCH;
    config.gridDim = dim3(params.rows, 1, 1);
    config.blockDim = dim3(kLogprobJoinThreads, 1, 1);
    config.dynamicSmemBytes = (size_t)params.parts * params.top * sizeof(unsigned long long);
    return cudaLaunchKernelEx(&config, token_logprobs_join_kernel, params, kType) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
}

}  // namespace mt
