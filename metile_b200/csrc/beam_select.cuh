// Beam search's selection: the best continuations over a group's beams and the vocabulary.
//
// A candidate is (beam, token) with the value score[beam] + ((logit - max) - log sum exp(logit - max)), in 64 bits; equal
// ones go by the lower beam, then the lower token.  What has no value (a row with a NaN, with +inf or with nothing above
// -inf; a score that is a mask) counts as -inf.  Bound by the bytes of the logits, and near to it by the exponentials (an
// SM takes 16 a cycle: 9 TB/s of 16-bit logits on 148 of them).
//
// One pass.  A CTA holds a span of 16384 logits of a row in registers, 64 a thread, and leaves its maximum, the sum of
// its exponentials and its `keep` best.  Within a beam candidates are ordered as their logits are, so no sum is needed for
// that.  Of 64 bucket maxima (four threads each) the keep-th largest bounds the keep-th best from below; only the few
// logits that reach it are collected and ranked.  Spans have one size for all calls: a row's bits do not depend on the others.
//
// Then a CTA per group joins spans and beams.  The sums are of 32-bit exponentials, each beam's log-sum off by up to
// kBeamError; where two beams' candidates are closer than twice that, the sums of the two are taken again, in 64 bits, so
// that beams and tokens are those of the exact values.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"

namespace mt {

constexpr double kDeadScore = -1e9;  // no sum of log-probabilities but the mask of a beam that is out; above it 64 bits keep logits apart
// |d| 2^-24 for the rounding of the argument d log2 e (the weighted mean of |d| is at most the log of the row's
// length, 13, and e^d |d| is small beyond it), 2^-22 for ex2.approx, six roundings of 2^-24 in a thread's
// sum (the rest is added in 64 bits): 1.4e-6.
constexpr double kBeamError = 0x1p-19;

constexpr int kBeamMaxBeams = 32, kBeamMaxKeep = 64;
constexpr int kBeamThreads = 256, kBeamPerThread = 64, kBeamSpan = kBeamThreads * kBeamPerThread;
constexpr int kBeamMaxVocabulary = 32 * kBeamSpan;           // of the join: at most 1024 lists
constexpr int kBeamBuckets = 64, kBeamCollect = 1024;        // of a span
constexpr int kBeamJoinCollect = kBeamMaxKeep * kBeamMaxKeep;
static_assert(kBeamBuckets >= kBeamMaxKeep && kBeamMaxVocabulary == MT_BEAM_MAX_VOCABULARY, "bounds of the selection");

struct BeamSpanStats {
    double sum;   // of exp(logit - top); NaN: the span has a NaN or +inf
    float top;
};

struct BeamEntry {
    float logit;
    int token;    // -1: there is none
};

struct BeamSelectParams {
    const void* logits;             // [groups * beams, vocabulary], rows `row_stride` apart
    const float* scores;            // [groups, beams]
    const unsigned char* finished;  // [groups, beams] or null
    float* scores_out;              // [groups, keep]
    int* parents_out;
    long long* tokens_out;
    unsigned char* finished_out;
    BeamSpanStats* stats;           // [groups * beams, spans]
    BeamEntry* lists;               // [groups * beams, spans, keep]
    long long row_stride, end_token;  // no end token: -1
    int groups, beams, vocabulary, keep, spans;
};

inline int beam_spans(int vocabulary) { return (vocabulary + kBeamSpan - 1) / kBeamSpan; }
inline size_t beam_workspace_bytes(int groups, int beams, int vocabulary, int keep) {
    return (size_t)groups * beams * beam_spans(vocabulary) * (sizeof(BeamSpanStats) + (size_t)keep * sizeof(BeamEntry));
}

// kType: 0 bf16, 1 fp16, 2 fp32.
template <int kType>
__device__ __forceinline__ float beam_logit(const uint32_t (&words)[4], int e) {
    if constexpr (kType == 2) return __uint_as_float(words[e]);
    else if constexpr (kType == 1) {
        const __half2 pair = *reinterpret_cast<const __half2*>(&words[e >> 1]);
        return e & 1 ? __high2float(pair) : __low2float(pair);
    } else return e & 1 ? bf16_hi(words[e >> 1]) : bf16_lo(words[e >> 1]);
}

template <int kType>
__device__ __forceinline__ float beam_logit_at(const void* row, long long i) {
    if constexpr (kType == 0) return bf16_bits_to_f32(static_cast<const uint16_t*>(row)[i]);
    else if constexpr (kType == 1) return __half2float(static_cast<const __half*>(row)[i]);
    else return static_cast<const float*>(row)[i];
}

// 16 bytes from an address that is `skew` bytes behind a boundary, by aligned loads; of the second only if `more`.
__device__ __forceinline__ uint4 load_skewed(const char* address, int skew, bool more) {
    const uint4 a = ptx::ld_global_dependent_u4(address - skew);
    if (skew == 0) return a;
    const uint4 b = more ? ptx::ld_global_dependent_u4(address - skew + 16) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t words[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const int first = skew >> 2, bits = (skew & 3) * 8;
    uint32_t shifted[5];
#pragma unroll
    for (int i = 0; i < 5; ++i)
        shifted[i] = first == 0 ? words[i] : first == 1 ? words[i + 1] : first == 2 ? words[i + 2] : words[i + 3];
    return make_uint4(__funnelshift_r(shifted[0], shifted[1], bits), __funnelshift_r(shifted[1], shifted[2], bits),
                      __funnelshift_r(shifted[2], shifted[3], bits), __funnelshift_r(shifted[3], shifted[4], bits));
}

__device__ __forceinline__ float warp_max_f32(float v) {
#pragma unroll
    for (int offset = 16; offset >= 1; offset >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, offset));
    return v;
}

template <int kType>
__global__ void __launch_bounds__(kBeamThreads) beam_span_kernel(const BeamSelectParams p) {
    constexpr int kPer = kType == 2 ? 4 : 8, kVectors = kBeamPerThread / kPer, kSize = kType == 2 ? 4 : 2, kWarps = kBeamThreads / 32;
    __shared__ float warp_top[kWarps], bucket[kBeamBuckets];
    __shared__ double warp_sum[kWarps];
    __shared__ float collected[kBeamCollect], bound_shared;
    __shared__ int collected_token[kBeamCollect], count, above;
    const int span = blockIdx.x % p.spans, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = blockIdx.x / p.spans;
    const int first = span * kBeamSpan, here = min(kBeamSpan, p.vocabulary - first);
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const char* from = static_cast<const char*>(p.logits) + (row * p.row_stride + first) * kSize;
    const int skew = (int)(reinterpret_cast<uintptr_t>(from) & 15);
    // Element e of vector v: the span's (v * 256 + thread) * kPer + e; those behind the row are -inf and left out below.
    uint32_t raw[kVectors][4];
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = (v * kBeamThreads + threadIdx.x) * kPer;
        uint4 vector = make_uint4(0u, 0u, 0u, 0u);
        if (at < here) vector = load_skewed(from + (long long)at * kSize, skew, at + (16 - skew) / kSize < here);
        raw[v][0] = vector.x; raw[v][1] = vector.y; raw[v][2] = vector.z; raw[v][3] = vector.w;
    }
    if (here < kBeamSpan) {
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if ((v * kBeamThreads + (int)threadIdx.x) * kPer + e >= here) {
                    if constexpr (kType == 2) raw[v][e] = 0xFF800000u;
                    else {
                        const uint32_t least = kType == 1 ? 0xFC00u : 0xFF80u;
                        raw[v][e >> 1] = e & 1 ? (raw[v][e >> 1] & 0xFFFFu) | least << 16 : (raw[v][e >> 1] & 0xFFFF0000u) | least;
                    }
                }
    }
    float mine = -INFINITY;
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
#pragma unroll
        for (int e = 0; e < kPer; ++e) mine = fmaxf(mine, beam_logit<kType>(raw[v], e));
    float top = fmaxf(mine, __shfl_xor_sync(0xFFFFFFFFu, mine, 1));
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    if ((lane & 3) == 0) bucket[threadIdx.x >> 2] = top;
#pragma unroll
    for (int offset = 4; offset <= 16; offset <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, offset));
    if (lane == 0) warp_top[warp] = top;
    if (threadIdx.x == 0) count = above = 0;
    __syncthreads();
    top = warp_top[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, warp_top[w]);
    // The keep-th largest bucket: at least `keep` logits of the span are not below it.
    if (threadIdx.x < kBeamBuckets) {
        const float own = bucket[threadIdx.x];
        int rank = 0;
#pragma unroll 16
        for (int j = 0; j < kBeamBuckets; ++j) {
            const float other = bucket[j];
            rank += other > own || (other == own && j < (int)threadIdx.x);
        }
        if (rank == p.keep - 1) bound_shared = own;
    }
    // Exponentials of the differences to the span's maximum; a vector's sums as a tree.
    double total = 0.0;
    if (top == -INFINITY) {
        bool bad = false;
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
#pragma unroll
            for (int e = 0; e < kPer; ++e) bad = bad || beam_logit<kType>(raw[v], e) != beam_logit<kType>(raw[v], e);
        total = bad ? NAN : 0.0;
    } else {
        float sums[kVectors];
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            float weight[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const float d = beam_logit<kType>(raw[v], e) - top;  // log2 e in two parts
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(weight[e]) : "f"(fmaf(d, 1.44269502162933349609f, d * 1.92596299112661484e-8f)));
            }
#pragma unroll
            for (int width = kPer / 2; width >= 1; width >>= 1)
#pragma unroll
                for (int e = 0; e < width; ++e) weight[e] += weight[e + width];
            sums[v] = weight[0];
        }
#pragma unroll
        for (int width = kVectors / 2; width >= 1; width >>= 1)
#pragma unroll
            for (int v = 0; v < width; ++v) sums[v] += sums[v + width];
        total = sums[0];
    }
#pragma unroll
    for (int offset = 16; offset >= 1; offset >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, offset);
    if (lane == 0) warp_sum[warp] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        total = warp_sum[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) total += warp_sum[w];
        p.stats[blockIdx.x] = {total, top};
    }
    const float bound = bound_shared;
    // What each element's thread does with it where it qualifies.
    auto collect = [&](auto qualifies) {
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const float logit = beam_logit<kType>(raw[v], e);
                const int at = (v * kBeamThreads + threadIdx.x) * kPer + e;
                if (qualifies(logit, at) && at < here) {
                    const int place = atomicAdd(&count, 1);
                    if (place < kBeamCollect) {
                        collected[place] = logit;
                        collected_token[place] = first + at;
                    }
                }
            }
    };
    if (mine >= bound) collect([&](float logit, int) { return logit >= bound; });
    __syncthreads();
    BeamEntry* list = p.lists + (long long)blockIdx.x * p.keep;
    int found = count;
    if (found > kBeamCollect) {
        // More equal ones than the buffer takes.  Where they are the span's least (masked tokens, a constant row) and
        // few lie above, the first `keep` of them are among its first keep + above elements.
        int greater = 0;
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
#pragma unroll
            for (int e = 0; e < kPer; ++e) greater += beam_logit<kType>(raw[v], e) > bound;
        atomicAdd(&above, greater);
        __syncthreads();
        greater = above;
        const bool least = found == here && 2 * greater + p.keep <= kBeamCollect;
        __syncthreads();
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        if (!least) {
            // `keep` rounds: the best behind the last one.
            float last = INFINITY;
            int last_token = -1;
            for (int r = 0; r < p.keep; ++r) {
                float best = -INFINITY;
                int token = 0x7FFFFFFF;
#pragma unroll
                for (int v = 0; v < kVectors; ++v)
#pragma unroll
                    for (int e = 0; e < kPer; ++e) {
                        const float logit = beam_logit<kType>(raw[v], e);
                        const int at = (v * kBeamThreads + threadIdx.x) * kPer + e;
                        const bool behind = logit < last || (logit == last && first + at > last_token);
                        if (at < here && behind && (logit > best || (logit == best && first + at < token))) {
                            best = logit;
                            token = first + at;
                        }
                    }
#pragma unroll
                for (int offset = 16; offset >= 1; offset >>= 1) {
                    const float other = __shfl_xor_sync(0xFFFFFFFFu, best, offset);
                    const int other_token = __shfl_xor_sync(0xFFFFFFFFu, token, offset);
                    if (other > best || (other == best && other_token < token)) { best = other; token = other_token; }
                }
                if (lane == 0) {
                    collected[warp] = best;
                    collected_token[warp] = token;
                }
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kWarps; ++w)
                    if (collected[w] > best || (collected[w] == best && collected_token[w] < token)) { best = collected[w]; token = collected_token[w]; }
                if (threadIdx.x == 0) list[r] = {best, token == 0x7FFFFFFF ? -1 : token};
                last = best;
                last_token = token;
                __syncthreads();
            }
            return;
        }
        collect([&](float logit, int at) { return logit > bound || (logit == bound && at < p.keep + greater); });
        __syncthreads();
        found = count;
    }
    for (int i = threadIdx.x; i < found; i += kBeamThreads) {
        const float logit = collected[i];
        const int token = collected_token[i];
        int rank = 0;
        for (int j = 0; j < found; ++j) rank += collected[j] > logit || (collected[j] == logit && collected_token[j] < token);
        if (rank < p.keep) list[rank] = {logit, token};
    }
    for (int i = found + threadIdx.x; i < p.keep; i += kBeamThreads) list[i] = {-INFINITY, -1};
}

struct BeamCandidate {
    double value;
    long long flat;  // beam * vocabulary + token; -1: there is none
};
__device__ __forceinline__ bool beam_before(const BeamCandidate& a, const BeamCandidate& b) {
    return a.value > b.value || (a.value == b.value && a.flat < b.flat);
}

// One CTA per group; a list of sorted candidates for every span of every beam.
template <int kType>
__global__ void __launch_bounds__(1024) beam_join_kernel(const BeamSelectParams p) {
    extern __shared__ __align__(16) unsigned char join_smem[];
    BeamCandidate* collected = reinterpret_cast<BeamCandidate*>(join_smem);          // [kBeamJoinCollect]
    BeamCandidate* sample = collected + kBeamJoinCollect;                            // [lists + keep]
    int* order = reinterpret_cast<int*>(sample + p.beams * p.spans + kBeamMaxKeep);  // [kBeamJoinCollect]
    __shared__ double top[kBeamMaxBeams], log_sum[kBeamMaxBeams], score[kBeamMaxBeams], scratch[32];
    __shared__ unsigned char kind[kBeamMaxBeams];  // 0: a beam's own lists, 1: it has finished, 2: it has no candidate
    __shared__ BeamCandidate bound;
    __shared__ int count;
    __shared__ unsigned int close;
    const int group = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int lists = p.beams * p.spans;
    const long long row0 = (long long)group * p.beams;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    for (int beam = warp; beam < p.beams; beam += warps) {
        const float given = p.scores[row0 + beam];
        const bool ended = p.finished && p.finished[row0 + beam];
        float best = -INFINITY;
        double sum = 0.0;
        const BeamSpanStats* stats = p.stats + (row0 + beam) * p.spans;
        BeamSpanStats own = {0.0, -INFINITY};
        if (lane < p.spans) own = stats[lane];  // 32 spans at most
        best = warp_max_f32(own.top);
        if (lane < p.spans) sum = own.sum == 0.0 ? 0.0 : own.sum * exp((double)own.top - (double)best);
#pragma unroll
        for (int offset = 16; offset >= 1; offset >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, offset);
        if (lane == 0) {
            top[beam] = best;
            log_sum[beam] = log(sum);
            score[beam] = given;
            kind[beam] = !(given > kDeadScore) ? 2 : ended ? 1 : !(sum > 0.0 && sum < INFINITY && best < INFINITY) ? 2 : 0;
        }
    }
    if (threadIdx.x == 0) close = 0;
    __syncthreads();
    // Candidate `depth` of a list.
    auto candidate = [&](int list, int depth) -> BeamCandidate {
        const int beam = list / p.spans, span = list - beam * p.spans;
        const long long base = (long long)beam * p.vocabulary;
        if (kind[beam] == 0) {
            const BeamEntry entry = p.lists[((row0 + beam) * p.spans + span) * p.keep + depth];
            if (entry.token < 0) return {-INFINITY, -1};
            return {score[beam] + (((double)entry.logit - top[beam]) - log_sum[beam]), base + entry.token};
        }
        long long token = depth;  // no candidate: the first tokens, at -inf
        if (kind[beam] == 1) {
            if (depth == 0) return span == 0 ? BeamCandidate{score[beam], base + p.end_token} : BeamCandidate{-INFINITY, -1};
            token = depth - 1 < p.end_token ? depth - 1 : depth;
        }
        if (span > 0 || token >= p.vocabulary) return {-INFINITY, -1};
        return {-INFINITY, base + token};
    };
    // Samples enough for `keep`, the first ones of every list; the keep-th best of them is not above the keep-th best of all.
    const int depths = min(p.keep, (p.keep + lists - 1) / lists), samples = lists * depths;
    for (int phase = 0;; ++phase) {
        const double margin = phase == 0 && p.beams > 1 ? 2.0 * kBeamError : 0.0;
        if (threadIdx.x == 0) {
            bound = {-INFINITY, 0x7FFFFFFFFFFFFFFFll};
            count = 0;
        }
        for (int i = threadIdx.x; i < samples; i += blockDim.x) sample[i] = candidate(i / depths, i % depths);
        __syncthreads();
        for (int i = threadIdx.x; i < samples; i += blockDim.x) {
            const BeamCandidate own = sample[i];
            if (own.flat < 0) continue;
            int rank = 0;
            for (int j = 0; j < samples; ++j) rank += sample[j].flat >= 0 && beam_before(sample[j], own);
            if (rank == p.keep - 1) bound = own;
        }
        __syncthreads();
        const BeamCandidate limit = bound;
        for (int list = threadIdx.x; list < lists; list += blockDim.x)
            for (int depth = 0; depth < p.keep; ++depth) {
                const BeamCandidate own = candidate(list, depth);
                if (own.flat < 0) break;
                if (own.value == -INFINITY ? beam_before(limit, own) : own.value < limit.value - margin || (margin == 0.0 && beam_before(limit, own))) break;
                const int place = atomicAdd(&count, 1);
                if (place < kBeamJoinCollect) collected[place] = own;
            }
        __syncthreads();
        const int found = count;
        const bool overflow = found > kBeamJoinCollect;  // of the margin only: without it there are keep lists of keep
        if (!overflow) {
            for (int i = threadIdx.x; i < found; i += blockDim.x) {
                int rank = 0;
                for (int j = 0; j < found; ++j) rank += beam_before(collected[j], collected[i]);
                order[rank] = i;
            }
            __syncthreads();
        }
        if (margin > 0.0) {
            if (overflow) {
                if (threadIdx.x == 0) close = 0xFFFFFFFFu;
            } else {
                for (int i = threadIdx.x; i + 1 < found; i += blockDim.x) {
                    const BeamCandidate upper = collected[order[i]], lower = collected[order[i + 1]];
                    const int a = (int)(upper.flat / p.vocabulary), b = (int)(lower.flat / p.vocabulary);
                    if (a != b && lower.value > -INFINITY && upper.value - lower.value <= margin)
                        atomicOr(&close, 1u << a | 1u << b);
                }
            }
            __syncthreads();
            if (close) {
                for (int beam = 0; beam < p.beams; ++beam) {
                    if (!(close >> beam & 1u) || kind[beam] != 0) continue;
                    const char* row = static_cast<const char*>(p.logits) + (row0 + beam) * p.row_stride * (kType == 2 ? 4 : 2);
                    double sum = 0.0;
                    for (int i = threadIdx.x; i < p.vocabulary; i += blockDim.x) sum += exp((double)beam_logit_at<kType>(row, i) - top[beam]);
#pragma unroll
                    for (int offset = 16; offset >= 1; offset >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, offset);
                    if (lane == 0) scratch[warp] = sum;
                    __syncthreads();
                    if (threadIdx.x == 0) {
                        sum = scratch[0];
                        for (int w = 1; w < warps; ++w) sum += scratch[w];
                        log_sum[beam] = log(sum);
                    }
                    __syncthreads();
                }
                continue;
            }
        }
        for (int r = threadIdx.x; r < p.keep; r += blockDim.x) {
            const BeamCandidate best = collected[order[r]];
            const int parent = (int)(best.flat / p.vocabulary);
            const long long token = best.flat - (long long)parent * p.vocabulary, at = (long long)group * p.keep + r;
            p.scores_out[at] = (float)best.value;
            p.parents_out[at] = parent;
            p.tokens_out[at] = token;
            p.finished_out[at] = kind[parent] == 1 || (p.finished && p.finished[row0 + parent]) || token == p.end_token;
        }
        return;
    }
}

template <int kType>
inline int launch_beam_select(const BeamSelectParams& params, cudaStream_t stream) {
    const int lists = params.beams * params.spans;
    int threads = (lists + 31) / 32 * 32;
    threads = threads < 128 ? 128 : threads;
    auto smem_of = [](int lists) { return (kBeamJoinCollect + lists + kBeamMaxKeep) * sizeof(BeamCandidate) + kBeamJoinCollect * sizeof(int); };
    static bool configured[64] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return MT_ERR_LAUNCH;
    if (device >= 64 || !configured[device]) {
        if (cudaFuncSetAttribute(beam_join_kernel<kType>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(1024)) != cudaSuccess)
            return MT_ERR_LAUNCH;
        if (device < 64) configured[device] = true;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(params.groups * lists, 1, 1);
    config.blockDim = dim3(kBeamThreads, 1, 1);
    config.stream = stream;
    cudaLaunchAttribute attrs[1];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, beam_span_kernel<kType>, params) != cudaSuccess) return MT_ERR_LAUNCH;
    config.gridDim = dim3(params.groups, 1, 1);
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = smem_of(lists);
    return cudaLaunchKernelEx(&config, beam_join_kernel<kType>, params) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
}

}  // namespace mt
