// Log-probabilities of given tokens, with the entropy of their rows and the best alternatives.
//
// With m the largest logit of a row and d = x - m:  S = sum e^d,  logprob(t) = d_t - log S,  entropy = log S - sum e^d d / S.
// One pass over the logits: a warp takes 2 KB of a row, keeps it in registers, and leaves its maximum, the two sums relative to
// that maximum, and the maxima of its stretches of 512 bytes; warps do not meet.  A second kernel joins the shares, in order and in 64
// bits, and looks for the best entries in the stretches with the largest maxima alone.  Shares have one size for all calls, so a row's
// bits do not depend on the others.
//
// What bounds it: 2001 rows of 128256 in bf16 106 us without alternatives, 4.9 TB/s (reading alone would take 78, the exponentials 57, and
// a warp does one after the other), 126 with 20, 144 with 64, in a graph; 8 rows of 32001 with 5 9.5 us, two launches and a chain of some eight
// loads that wait for one another.  Blocks that took 32 KB, met for the maximum and sorted their own best took 117, 195 and 261.
#pragma once

#include "beam_select.cuh"
#include "paged_attention.cuh"

namespace mt {

constexpr unsigned int kTokenOutside = 0x307;  // token_logprobs: word 1 = row, 2 and 3 = the token

constexpr int kLogprobThreads = 256, kLogprobVectors = 4, kLogprobMaxTop = 64;
constexpr int kLogprobSlack = 16;      // stretches that may be looked at beside the `top` ones with the largest maxima
constexpr int kLogprobChosen = kLogprobMaxTop + kLogprobSlack;
constexpr int kLogprobCollect = 512;
// A warp's share of a row: stretches of 512 bytes, a vector a lane.
__host__ __device__ constexpr int logprob_stretch(int type) { return 512 / beam_size(type); }  // logits
__host__ __device__ constexpr int logprob_share(int type) { return kLogprobVectors * logprob_stretch(type); }
inline int logprob_shares(int vocabulary, int type) { return (vocabulary + logprob_share(type) - 1) / logprob_share(type); }

struct LogprobStats {
    float top, sum, weighted;  // maximum; sums of e^d and e^d d
};

struct LogprobParams {
    const void* logits;         // [rows, vocabulary], rows `row_stride` apart
    const long long* tokens;    // [rows]
    float *logprobs, *entropy;  // [rows]
    float* top_logprobs;        // [rows, top]
    long long* top_tokens;      // [rows, top]
    LogprobStats* stats;        // [rows, shares]
    float* tops;                // [rows, shares, kLogprobVectors]: maxima of the stretches, where `top` asks for them
    long long row_stride;
    int rows, vocabulary, shares, top;
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
// The largest of a warp's numbers, NaN left out; -inf where there are none.
__device__ __forceinline__ float largest_of_warp(float x) {
    float out;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(out) : "f"(x));
    return fmaxf(out, -INFINITY);
}

// What has been made of the vectors is made again, rather than kept in registers until then.
__device__ __forceinline__ void forget(uint4 (&v)[kLogprobVectors]) {
#pragma unroll
    for (int i = 0; i < kLogprobVectors; ++i) asm volatile("" : "+r"(v[i].x), "+r"(v[i].y), "+r"(v[i].z), "+r"(v[i].w));
}

// kAligned: every row starts on 16 bytes.
template <int kType, bool kAligned>
__global__ void __launch_bounds__(kLogprobThreads, kAligned ? 6 : 5) token_logprobs_part_kernel(const LogprobParams p) {
    constexpr int kSize = beam_size(kType), kEach = 16 / kSize, kShare = logprob_share(kType);
    const int lane = threadIdx.x & 31, item = blockIdx.x * (kLogprobThreads / 32) + (int)(threadIdx.x >> 5);
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    if (item >= p.rows * p.shares) return;
    const int row = item / p.shares, first = (item - row * p.shares) * kShare, count = min(kShare, p.vocabulary - first);
    const char* base = static_cast<const char*>(p.logits) + (row * p.row_stride + first) * kSize;
    uint4 v[kLogprobVectors];
    if constexpr (kAligned) {
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) {
            const int at = (i * 32 + lane) * kEach;
            v[i] = at < count ? ptx::ld_global_dependent_u4(base + (size_t)at * kSize) : make_uint4(0u, 0u, 0u, 0u);
        }
    } else {
        // A row may start anywhere: the two aligned vectors that a vector lies in, shifted; the second one is the next lane's first.
        const int shift = (int)(reinterpret_cast<uintptr_t>(base) & 15), bits = (shift & 3) * 8;
        const char* aligned = base - shift;
        // Vectors that hold a logit of the share.
        auto load = [&](int at) { return at * kEach - shift / kSize < count ? ptx::ld_global_dependent_u4(aligned + (size_t)at * 16) : make_uint4(0u, 0u, 0u, 0u); };
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) v[i] = load(i * 32 + lane);
#pragma unroll
        for (int i = 0; i < kLogprobVectors; ++i) {
            uint4 next = {__shfl_down_sync(0xFFFFFFFFu, v[i].x, 1), __shfl_down_sync(0xFFFFFFFFu, v[i].y, 1), __shfl_down_sync(0xFFFFFFFFu, v[i].z, 1),
                          __shfl_down_sync(0xFFFFFFFFu, v[i].w, 1)};
            if (lane == 31) next = load(i * 32 + 32);
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
    // Logits behind the row count as -inf; a thread has element e of vector i if e < there(i).
    auto there = [&](int i) { return count - (i * 32 + lane) * kEach; };
    constexpr uint32_t kNothing = kType == 2 ? 0xFF800000u : kType == 1 ? 0xFC00u : 0xFF80u;
    if (count < kShare) {
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
    float tops[kLogprobVectors], all = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLogprobVectors; ++i) {
        tops[i] = largest_of_warp(largest_logit<kType>(v[i]));
        all = fmaxf(all, tops[i]);
    }
    if (p.top > 0) {
        float own = tops[0];
#pragma unroll
        for (int i = 1; i < kLogprobVectors; ++i) own = lane == i ? tops[i] : own;
        if (lane < kLogprobVectors) p.tops[(size_t)item * kLogprobVectors + lane] = own;
    }
    forget(v);
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
                const float e = (logit_at<kType>(base, (i * 32 + lane) * kEach + j) + against) * kLog2E, power = power_of_two(e);
                weighted += power == 0.0f ? 0.0f : power * e;
            }
    }
    sum = warp_sum_xor(sum);
    weighted = warp_sum_xor(weighted);
    if (lane == 0) p.stats[item] = {all, sum, weighted * 0.6931471805599453f};
}

__device__ __forceinline__ double warp_sum_double(double v) {
#pragma unroll
    for (int offset = 16; offset >= 1; offset >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, offset);
    return v;
}

// A CTA joins the shares of a row and finds its best entries: its first warp the sums, a share a lane, while the second one chooses
// the stretches that the best lie in.  `top` stretches reach the `top`-th largest of their maxima, and so do `top` logits: only what
// reaches it is collected and ranked.  Of stretches with just that maximum the first ones will do.
template <int kType, int kThreads>
__global__ void __launch_bounds__(kThreads) token_logprobs_join_kernel(const LogprobParams p) {
    constexpr int kSize = beam_size(kType), kStretch = logprob_stretch(kType), kWarps = kThreads / 32, kEach = kStretch / 32;
    // Logits are looked for by their order, without the bits that those of the type have all alike: fewer halvings.
    constexpr int kShift = kType == 2 ? 0 : kType == 1 ? 13 : 16;
    extern __shared__ unsigned int orders[];  // of the maxima of the stretches
    __shared__ double shared_lse, shared_top;
    __shared__ unsigned long long collected[kLogprobCollect];
    __shared__ unsigned int bound;
    __shared__ int chosen_stretch[kLogprobChosen], chosen_count, found, counted[2][kWarps];
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, stretches = (p.vocabulary + kStretch - 1) / kStretch;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const char* base = static_cast<const char*>(p.logits) + row * p.row_stride * beam_size(kType);
    // The aligned vectors of stretches, dealt to the threads, four of them on their way at once: use(stretch, token, hits) learns which of
    // the logits from `token` on reach(logit).  Some of them may lie beside the stretch.
    const int shift = (int)(reinterpret_cast<uintptr_t>(base) & 15), before = shift / kSize, vectors = shift ? 33 : 32;
    auto visit = [&](int count, auto stretch_of, auto reach, auto use) {
        constexpr int kAtOnce = 4;
        for (int j = threadIdx.x; j < count * vectors; j += kAtOnce * kThreads) {
            uint4 v[kAtOnce];
            int stretch[kAtOnce], token[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const int at = j + i * kThreads, k = at / vectors;
                v[i] = make_uint4(~0u, ~0u, ~0u, ~0u);  // NaN
                if (at >= count * vectors) continue;
                stretch[i] = stretch_of(k);
                token[i] = stretch[i] * kStretch + (at - k * vectors) * kEach - before;
                if (token[i] < p.vocabulary) v[i] = ptx::ld_global_dependent_u4(base + (long long)token[i] * kSize);
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                unsigned int hits = 0;
#pragma unroll
                for (int e = 0; e < kEach; ++e) hits |= (reach(logit_of<kType>(v[i], e)) ? 1u : 0u) << e;
                if (hits) use(stretch[i], token[i], hits);
            }
        }
    };
    auto within = [&](int stretch, int token) { return token >= stretch * kStretch && token < min(p.vocabulary, (stretch + 1) * kStretch); };
    // Where there are few stretches, all of them are looked at, and the bound is that of the threads' maxima.
    const bool few = stretches <= p.top + kLogprobSlack;
    const int maxima = few ? kThreads : stretches;
    if (p.top > 0) {
        if (few) {
            unsigned int most = 0u;  // of a thread that has none
#pragma unroll 4
            for (int token = (int)threadIdx.x * kEach - before; token < p.vocabulary; token += kThreads * kEach) {
                const uint4 v = ptx::ld_global_dependent_u4(base + (long long)token * kSize);
                float x = largest_logit<kType>(v);
                if (token < 0 || token + kEach > p.vocabulary) {
                    x = NAN;
#pragma unroll
                    for (int e = 0; e < kEach; ++e)
                        if (token + e >= 0 && token + e < p.vocabulary) x = fmaxf(x, logit_of<kType>(v, e));
                }
                if (x == x) most = max(most, beam_logit_order(x) >> kShift);
            }
            orders[threadIdx.x] = most;
        } else {
            const float* tops = p.tops + (size_t)row * p.shares * kLogprobVectors;
            for (int i = threadIdx.x; i < stretches; i += kThreads) orders[i] = beam_logit_order(tops[i]) >> kShift;
        }
        if (threadIdx.x == 0) found = 0;
        __syncthreads();
    }
    if (warp == 0) {
        const LogprobStats* stats = p.stats + (size_t)row * p.shares;
        const long long token = threadIdx.x == 0 ? p.tokens[row] : -1;
        float chosen = 0.0f;
        if (token >= 0 && token < p.vocabulary) chosen = logit_at<kType>(base + token * kSize, 0);
        float top = -INFINITY;
        bool usable = true;  // neither NaN nor +inf
        for (int i = threadIdx.x; i < p.shares; i += 32) {
            top = fmaxf(top, stats[i].top);
            usable = usable && stats[i].sum <= 3e38f;
        }
#pragma unroll
        for (int offset = 16; offset >= 1; offset >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, offset));
        usable = __all_sync(0xFFFFFFFFu, usable) && top != -INFINITY && top != INFINITY;
        double sum = 0.0, weighted = 0.0;
        for (int i = threadIdx.x; i < p.shares; i += 32) {
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
    } else if (warp == 1 && p.top > 0) {
        unsigned int low = ~0u, high = 0u;  // as many as are wanted reach `low`, fewer reach `high`
        int reach = maxima, beyond = 0;
        for (int i = lane; i < maxima; i += 32) {
            low = min(low, orders[i]);
            high = max(high, orders[i]);
        }
        low = __reduce_min_sync(0xFFFFFFFFu, low);
        high = __reduce_max_sync(0xFFFFFFFFu, high) + 1u;
        while (high - low > 1u && reach > p.top + kLogprobSlack) {
            const unsigned int middle = low + (high - low) / 2;
            int here = 0;
            for (int i = lane; i < maxima; i += 32) here += orders[i] >= middle;
            here = __reduce_add_sync(0xFFFFFFFFu, here);
            if (here >= p.top) {
                low = middle;
                reach = here;
            } else {
                high = middle;
                beyond = here;
            }
        }
        // All that reach it, or, where they are too many, those beyond it and the first others.
        int others = reach > p.top + kLogprobSlack ? p.top - beyond : kLogprobChosen, taken = 0;
        for (int start = 0; start < stretches; start += 32) {
            const int i = start + lane;
            const bool reaches = i < stretches && (few || orders[i] >= low), equal = reaches && !few && orders[i] == low;
            const unsigned int equals = __ballot_sync(0xFFFFFFFFu, equal);
            const bool takes = reaches && (!equal || __popc(equals & ((1u << lane) - 1u)) < others);
            others -= __popc(equals);
            const unsigned int votes = __ballot_sync(0xFFFFFFFFu, takes);
            if (takes) chosen_stretch[taken + __popc(votes & ((1u << lane) - 1u))] = i;
            taken += __popc(votes);
        }
        if (lane == 0) {
            chosen_count = taken;
            bound = low;
        }
    }
    if (p.top == 0) return;
    __syncthreads();
    const double lse = shared_lse, largest = shared_top;
    float* logprobs = p.top_logprobs + (size_t)row * p.top;
    long long* tokens = p.top_tokens + (size_t)row * p.top;
    if (lse != lse) {  // the row has no distribution
        for (int i = threadIdx.x; i < p.top; i += kThreads) {
            logprobs[i] = NAN;
            tokens[i] = -1;
        }
        return;
    }
    const int chosen = chosen_count;
    unsigned int low = bound;
    auto least_of = [&](unsigned int order) { return order << kShift <= beam_logit_order(-INFINITY) ? -INFINITY : beam_ordered_logit(order << kShift); };
    auto collect = [&](unsigned int order) {
        const float least = least_of(order);
        visit(chosen, [&](int k) { return chosen_stretch[k]; }, [&](float x) { return x >= least; }, [&](int stretch, int token, unsigned int hits) {
            for (; hits; hits &= hits - 1u) {
                const int at = token + __ffs(hits) - 1;
                if (!within(stretch, at)) continue;
                const int to = atomicAdd(&found, 1);
                if (to < kLogprobCollect) collected[to] = beam_entry_key(logit_at<kType>(base, at), at);
            }
        });
    };
    collect(low);
    __syncthreads();
    int many = found;
    if (many > kLogprobCollect) {
        // More than are collected reach it.  `top` at least reach `low`, fewer reach `high`.
        __syncthreads();
        unsigned int high = (beam_logit_order((float)largest) >> kShift) + 1u;
        for (int round = 0; high - low > 1u && many > kLogprobCollect; ++round) {
            const unsigned int middle = low + (high - low) / 2;
            const float least = least_of(middle);
            int here = 0;
            visit(chosen, [&](int k) { return chosen_stretch[k]; }, [&](float x) { return x >= least; }, [&](int stretch, int token, unsigned int hits) {
                for (; hits; hits &= hits - 1u) here += within(stretch, token + __ffs(hits) - 1);
            });
            here = __reduce_add_sync(0xFFFFFFFFu, here);
            if (lane == 0) counted[round & 1][warp] = here;
            __syncthreads();
            here = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) here += counted[round & 1][w];
            if (here >= p.top) {
                low = middle;
                many = here;
            } else {
                high = middle;
            }
        }
        if (threadIdx.x == 0) found = 0;
        __syncthreads();
        const bool equals = many > kLogprobCollect;  // hundreds are equal: those beyond them, and of them the first
        collect(equals ? high : low);
        __syncthreads();
        many = found;
        if (equals) {
            if (warp == 0)
                for (int k = 0, have = many; k < chosen && have < p.top; ++k) {
                    float x[kEach];
                    const int first = chosen_stretch[k] * kStretch + lane;
#pragma unroll
                    for (int e = 0; e < kEach; ++e) x[e] = first + 32 * e < p.vocabulary ? logit_at<kType>(base, first + 32 * e) : NAN;
#pragma unroll
                    for (int e = 0; e < kEach; ++e) {
                        const bool equal = x[e] == x[e] && beam_logit_order(x[e]) >> kShift == low;
                        const unsigned int votes = __ballot_sync(0xFFFFFFFFu, equal);
                        const int to = have + __popc(votes & ((1u << lane) - 1u));
                        if (equal && to < p.top) collected[to] = beam_entry_key(x[e], first + 32 * e);
                        have += __popc(votes);
                    }
                }
            many = p.top;
            __syncthreads();
        }
    }
    for (int i = threadIdx.x; i < many; i += kThreads) {
        const unsigned long long key = collected[i];
        int rank = 0;
        for (int j = 0; j < many; ++j) rank += collected[j] > key;
        if (rank >= p.top) continue;
        const BeamEntry entry = beam_entry(key);
        logprobs[rank] = (float)((double)entry.logit - largest - lse);
        tokens[rank] = entry.token;
    }
}

inline size_t logprob_stats_bytes(int rows, int shares) { return ((size_t)rows * shares * sizeof(LogprobStats) + 15) / 16 * 16; }
inline size_t logprob_bytes(int rows, int shares, int top) {
    return logprob_stats_bytes(rows, shares) + (top > 0 ? (size_t)rows * shares * kLogprobVectors * sizeof(float) : 0);
}

template <int kType>
inline int launch_token_logprobs(const LogprobParams& params, cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((params.rows * params.shares + kLogprobThreads / 32 - 1) / (kLogprobThreads / 32), 1, 1);
    config.blockDim = dim3(kLogprobThreads, 1, 1);
    config.stream = stream;
    cudaLaunchAttribute attrs[1];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = 1;
    const bool aligned = aligned_to(params.logits, 16) && (params.rows == 1 || params.row_stride * beam_size(kType) % 16 == 0);
    if (cudaLaunchKernelEx(&config, aligned ? token_logprobs_part_kernel<kType, true> : token_logprobs_part_kernel<kType, false>, params) != cudaSuccess) return MT_ERR_LAUNCH;
    // Rows enough to fill the chip have smaller CTAs: 2001 rows of 128256 with 20 alternatives 124 us (127 with 256 threads), 8 rows of 32001
    // with 5 12.7 (12.2), of 16000 with 64 17.4 (13.5).
    const bool many = params.rows >= 1024;
    const int threads = many ? 128 : 256, stretches = (params.vocabulary + logprob_stretch(kType) - 1) / logprob_stretch(kType);
    config.gridDim = dim3(params.rows, 1, 1);
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = params.top > 0 ? (stretches > threads ? stretches : threads) * sizeof(unsigned int) : 0;
    return cudaLaunchKernelEx(&config, many ? token_logprobs_join_kernel<kType, 128> : token_logprobs_join_kernel<kType, 256>, params) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
}

}  // namespace mt
