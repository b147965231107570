// Beam search's selection: the best continuations over a group's beams and the vocabulary.
//
// A candidate is (beam, token) with the value score[beam] + ((logit - max) - log sum exp(logit - max)), in 64 bits; equal
// ones go by the lower beam, then the larger logit (64 bits may round the values of two to one), then the lower token.  So
// a beam's candidates are always in the order of their logits, which its sorted lists rest on.  What has no value (a row
// with a NaN, with +inf or with nothing above -inf; a score that is a mask) counts as -inf.  Bound by the bytes of the logits,
// and near to it by the exponentials (an SM takes 16 a cycle: 9 TB/s of 16-bit logits on 148 of them).
//
// One pass.  Rows are cut into spans of 16 KB, 64 bytes a thread, and a row's spans dealt out to CTAs; a CTA's share of a row is a
// part.  Every warp leaves the maximum and the sum of exponentials of its share of a span, and the CTA the `keep` best of its
// part.  Within a beam candidates are ordered as their logits are, so no sum is needed for that.  Of 64 bucket maxima (four
// threads each) the keep-th largest bounds the keep-th best from below; the few threads that reach it look at their logits
// again, and what they find is ranked.  (Short rows and ends of rows, and the most kept, take 256 maxima: with 64 kept of
// 128256 in 128 rows 37 us, by the buckets alone 458; 14 rows of 524 with 28 kept 14 us, 34.)  The shares of a row have one
// size for all calls: its bits do not depend on the others.
//
// Then a CTA per group joins parts and beams.  The sums are of 32-bit exponentials, each beam's log-sum off by up to
// kBeamError; where two beams' candidates are closer than twice that, the sums of the two are taken again, in 64 bits, so
// that beams and tokens are those of sums in 64 bits.  One CTA does that, beam after beam: 8 beams of one row of 128256 388 us.
//
// Measured: 32 groups of 8 beams over 128256 (bf16, 65.7 MB, 16 kept) 23.1 to 23.6 us, 2.8 TB/s; of that reading with the exponentials 13, the
// end of the parts 4 and the join 5, both chains of short steps.  4 beams over 32001: 8.1 us.  Spans of all rows dealt out evenly,
// so that a CTA may have the end of one row and the start of another: 27 us; three CTAs to an SM with three ring slots instead of four
// with two: 5 % more.
#pragma once

#include <cuda_fp16.h>
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace mt {

constexpr double kDeadScore = -1e9;  // no sum of log-probabilities but the mask of a beam that is out; above it 64 bits keep logits apart
// d = logit - top rounded, then d log2 e: |d| 2^-24 each and |d| 1.4e-8 for log2 e itself, 2^-22 for ex2.approx, within a share
// and once more for the share in the row, where the two |d| add up to the one to the row's maximum; fourteen roundings of 2^-24
// in sums (the rest is added in 64 bits).  The mean of |d| by the weights is at most the log of the row's length, 13.2: 3.1e-6.
constexpr double kBeamError = 0x1p-18;

constexpr int kBeamMaxBeams = 32, kBeamMaxKeep = 64;
constexpr int kBeamThreads = 256, kBeamVectors = 4, kBeamSpanBytes = kBeamThreads * kBeamVectors * 16, kBeamShares = kBeamThreads / 32;
constexpr int kBeamMaxParts = 32, kBeamMostPerPart = 16;     // parts of a row (at most 1024 lists to join), spans of a part
constexpr int kBeamAtOnce = 4, kBeamStages = 2;              // CTAs of an SM, spans each has in flight or in work
constexpr int kBeamShareBytes = kBeamVectors * 512, kBeamBlock = kBeamShareBytes + 16;  // a warp's share of a span, in the ring with the vector behind it
constexpr int kBeamRing = kBeamStages * kBeamShares * kBeamBlock;
constexpr int kBeamBuckets = 64, kBeamCollect = 512;         // of a part
static_assert(kBeamCollect >= kBeamMaxKeep + kBeamThreads, "equal ones are collected a step of all threads at a time");
constexpr int kBeamSlack = 8, kBeamKeys = 256, kBeamMany = 256, kBeamStage = 4096;              // entries of the lists that the join has in shared memory
static_assert(kBeamBuckets >= kBeamMaxKeep, "the bound of a part comes from its buckets");

__host__ __device__ constexpr int beam_size(int type) { return type == 2 ? 4 : 2; }               // bytes of a logit
__host__ __device__ constexpr int beam_span(int type) { return kBeamSpanBytes / beam_size(type); }  // logits

struct BeamShareStats {
    float top, sum;  // of exp(logit - top); NaN: there is a NaN or +inf
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
    BeamShareStats* stats;          // [groups * beams, spans * 8]
    BeamEntry* lists;               // [groups * beams, parts, keep]
    long long row_stride, end_token;  // no end token: -1
    int groups, beams, vocabulary, keep, spans;
    int parts;                      // of a row
    // Of the join: entries of a list in shared memory and among the samples; 2^32 / n rounded up, for whole quotients of
    // numbers up to 65536 (0 where n is 1).
    int staged, depths;
    unsigned int per_keep, per_staged, per_depths, per_parts;
};

__host__ __device__ inline unsigned int beam_reciprocal(unsigned int n) { return n == 1 ? 0u : (unsigned int)((0x100000000ull + n - 1) / n); }
__device__ __forceinline__ int beam_divided(int i, unsigned int reciprocal) { return reciprocal ? (int)__umulhi((unsigned int)i, reciprocal) : i; }

// Part `part` of a row: from its first span to the next one's.
__host__ __device__ inline int beam_part_start(int part, int spans, int parts) { return (int)((long long)part * spans / parts); }

inline int beam_spans(int vocabulary, int type) { return (vocabulary + beam_span(type) - 1) / beam_span(type); }

// The most candidates the join collects without a margin: from keep + slack lists, `keep` of each.  (No more first entries
// reach the bound, and what reaches it in a list stands behind a first entry that does: lists are sorted by value and place.)
__host__ __device__ inline int beam_join_most(int keep) { return (keep + kBeamSlack) * keep; }

// Parts of a row: as many as let all CTAs run at once, but none longer than a part may be, and no more than the join takes.
inline int beam_parts(int rows, int spans, int sm_count) {
    const int shortest = (spans + kBeamMostPerPart - 1) / kBeamMostPerPart, at_once = sm_count * kBeamAtOnce / rows;
    int parts = at_once < shortest ? shortest : at_once;
    if (parts > kBeamMaxParts) parts = kBeamMaxParts;
    return parts < spans ? parts : spans;
}

inline size_t beam_workspace_bytes(int groups, int beams, int vocabulary, int keep, int type) {
    const int spans = beam_spans(vocabulary, type);  // parts at most
    return (size_t)groups * beams * ((size_t)spans * kBeamShares * sizeof(BeamShareStats) + (size_t)(spans < kBeamMaxParts ? spans : kBeamMaxParts) * keep * sizeof(BeamEntry));
}

// A logit as a whole number of the same order (one zero, never 0 itself), and back.
__device__ __forceinline__ unsigned int beam_logit_order(float logit) {
    const unsigned int bits = __float_as_uint(logit + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float beam_ordered_logit(unsigned int order) { return __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order); }
// An entry as one number: the larger logit, among equals the lower token first.
__device__ __forceinline__ unsigned long long beam_entry_key(float logit, int token) {
    return (unsigned long long)beam_logit_order(logit) << 32 | (0xFFFFFFFFu - (unsigned int)token);
}
__device__ __forceinline__ BeamEntry beam_entry(unsigned long long key) {
    if (key == 0) return {-INFINITY, -1};
    return {beam_ordered_logit((unsigned int)(key >> 32)), (int)(0xFFFFFFFFu - (unsigned int)key)};
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

// Bytes skew ... skew + 15 of two 16-byte vectors that follow one another.
__device__ __forceinline__ void take_skewed(uint32_t (&out)[4], const uint4& a, const uint4& b, int skew) {
    const uint32_t words[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const int first = skew >> 2, bits = (skew & 3) * 8;
    uint32_t shifted[5];
#pragma unroll
    for (int i = 0; i < 5; ++i)
        shifted[i] = first == 0 ? words[i] : first == 1 ? words[i + 1] : first == 2 ? words[i + 2] : words[i + 3];
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __funnelshift_r(shifted[i], shifted[i + 1], bits);
}

// The larger of two words of logits, pair by pair.
template <int kType>
__device__ __forceinline__ uint32_t beam_word_max(uint32_t a, uint32_t b) {
    if constexpr (kType == 2) return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    uint32_t out = 0;
    if constexpr (kType == 1) asm("max.f16x2 %0, %1, %2;" : "=r"(out) : "r"(a), "r"(b));
    if constexpr (kType == 0) asm("max.bf16x2 %0, %1, %2;" : "=r"(out) : "r"(a), "r"(b));
    return out;
}
template <int kType>
__device__ __forceinline__ float beam_word_top(uint32_t word) {
    const uint32_t words[4] = {word, 0u, 0u, 0u};
    if constexpr (kType == 2) return __uint_as_float(word);
    else return fmaxf(beam_logit<kType>(words, 0), beam_logit<kType>(words, 1));
}

__device__ __forceinline__ float2 add_f32x2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul_f32x2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// A warp's shares of the spans of a part, copied ahead into its part of the ring.  A share is 2 KB in one piece: element e of a
// lane's vector v is its (32 v + lane) * kPer + e.
template <int kType>
struct BeamCopies {
    static constexpr int kPer = 16 / beam_size(kType), kShare = kBeamShareBytes / beam_size(kType);
    const char* vector;  // this lane's first one of the next share, aligned
    int left, skew;      // logits of the row from the share on, counted from the boundary in front; bytes behind that

    __device__ __forceinline__ BeamCopies(const char* row, int vocabulary, int span) {
        const int share = span * beam_span(kType) + (int)(threadIdx.x >> 5) * kShare;
        const char* from = row + (long long)share * beam_size(kType);
        skew = (int)(reinterpret_cast<uintptr_t>(from) & 15);
        vector = from - skew + (threadIdx.x & 31) * 16;
        left = vocabulary - share + skew / beam_size(kType);
    }
    __device__ __forceinline__ void next(char* ring) {
        const int lane = threadIdx.x & 31;
        char* to = ring + lane * 16;
        if (left >= kShare + kPer) {
#pragma unroll
            for (int v = 0; v < kBeamVectors; ++v) ptx::cp_async_16(to + v * 512, vector + v * 512);
            if (skew && lane == 0) ptx::cp_async_16(to + kBeamShareBytes, vector + kBeamShareBytes);
        } else {
#pragma unroll
            for (int v = 0; v < kBeamVectors; ++v)
                if ((32 * v + lane) * kPer < left) ptx::cp_async_16(to + v * 512, vector + v * 512);
            if (skew && lane == 0 && kShare < left) ptx::cp_async_16(to + kBeamShareBytes, vector + kBeamShareBytes);
        }
        vector += kBeamSpanBytes;
        left -= beam_span(kType);
    }
};

template <int kType>
__global__ void __launch_bounds__(kBeamThreads, kBeamAtOnce) beam_span_kernel(const BeamSelectParams p) {
    using Copies = BeamCopies<kType>;
    constexpr int kPer = Copies::kPer, kShare = Copies::kShare, kVectors = kBeamVectors, kWarps = kBeamShares;
    extern __shared__ __align__(16) char beam_ring[];  // [warps][stages][block]
    __shared__ float span_top[kBeamMostPerPart][kBeamThreads];
    __shared__ __align__(16) unsigned int bucket[kBeamBuckets];
    __shared__ __align__(16) unsigned long long collected[kBeamCollect];
    __shared__ unsigned int bound_order, finer_order;
    __shared__ int count;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = blockIdx.x / p.parts;
    const int part = (int)(blockIdx.x - row * p.parts);
    const int span0 = beam_part_start(part, p.spans, p.parts), span1 = beam_part_start(part + 1, p.spans, p.parts);
    char* ring = beam_ring + warp * (kBeamStages * kBeamBlock);
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const char* from = static_cast<const char*>(p.logits) + row * p.row_stride * beam_size(kType);
    Copies copies(from, p.vocabulary, span0);
    int to_copy = span1 - span0;
    auto copy_next = [&](int slot) {
        if (to_copy-- > 0) copies.next(ring + slot * kBeamBlock);
        ptx::cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kBeamStages - 1; ++i) copy_next(i);
    int slot = 0;
    if (threadIdx.x == 0) {
        count = 0;
        bound_order = finer_order = 0xFFFFFFFFu;
    }
    float mine = -INFINITY;
    uint32_t raw[kVectors][4];
    const int skew = copies.skew;
    BeamShareStats* stats = p.stats + (row * p.spans + span0) * kWarps + warp;
    float last_top = 0.0f, last_total = 0.0f;
    for (int span = span0; span < span1; ++span) {
        ptx::cp_async_wait_group<kBeamStages - 2>();
        __syncwarp();
        const char* share = ring + slot * kBeamBlock + lane * 16;
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const uint4 own = *reinterpret_cast<const uint4*>(share + v * 512);
            if (skew) {
                take_skewed(raw[v], own, *reinterpret_cast<const uint4*>(share + v * 512 + 16), skew);
            } else {
                raw[v][0] = own.x; raw[v][1] = own.y; raw[v][2] = own.z; raw[v][3] = own.w;
            }
        }
        const int left = p.vocabulary - span * beam_span(kType) - warp * kShare;  // behind the row: -inf, and left out below
        if (left < kShare) {
#pragma unroll
            for (int v = 0; v < kVectors; ++v)
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if ((32 * v + lane) * kPer + e >= left) {
                        if constexpr (kType == 2) raw[v][e] = 0xFF800000u;
                        else {
                            const uint32_t least = kType == 1 ? 0xFC00u : 0xFF80u;
                            raw[v][e >> 1] = e & 1 ? (raw[v][e >> 1] & 0xFFFFu) | least << 16 : (raw[v][e >> 1] & 0xFFFF0000u) | least;
                        }
                    }
        }
        __syncwarp();
        copy_next(slot == 0 ? kBeamStages - 1 : slot - 1);
        slot = slot == kBeamStages - 1 ? 0 : slot + 1;
        uint32_t largest = raw[0][0];
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) largest = beam_word_max<kType>(largest, raw[v][i]);
        float top = beam_word_top<kType>(largest);
        if (top != top) top = -INFINITY;  // nothing but NaN
        span_top[span - span0][threadIdx.x] = top;
        mine = fmaxf(mine, top);
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(top));
        // The exponentials of the differences to the share's maximum, added as a tree.  (With nothing above -inf the sum is
        // zero, or NaN where there is one.)  What the warp's lanes have is added one span later, beside the next exponentials.
        float2 sums[kVectors];
        const float away = top == -INFINITY ? 0.0f : -top;
        const float2 shift = make_float2(away, away), log2_e = make_float2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            float2 weight[kPer / 2];
#pragma unroll
            for (int e = 0; e < kPer / 2; ++e) {
                const float2 d = add_f32x2(make_float2(beam_logit<kType>(raw[v], 2 * e), beam_logit<kType>(raw[v], 2 * e + 1)), shift);
                const float2 power = mul_f32x2(d, log2_e);
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(weight[e].x) : "f"(power.x));
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(weight[e].y) : "f"(power.y));
            }
#pragma unroll
            for (int width = kPer / 4; width >= 1; width >>= 1)
#pragma unroll
                for (int e = 0; e < width; ++e) weight[e] = add_f32x2(weight[e], weight[e + width]);
            sums[v] = weight[0];
        }
#pragma unroll
        for (int width = kVectors / 2; width >= 1; width >>= 1)
#pragma unroll
            for (int v = 0; v < width; ++v) sums[v] = add_f32x2(sums[v], sums[v + width]);
        const float total = warp_sum_xor(last_total);
        if (lane == 0 && span > span0) *(stats - kWarps) = {last_top, total};
        stats += kWarps;
        last_top = top;
        last_total = sums[0].x + sums[0].y;
    }
    last_total = warp_sum_xor(last_total);
    if (lane == 0) *(stats - kWarps) = {last_top, last_total};
    // Four threads to a bucket: of the `keep` largest of 64 the least bounds `keep` logits of the CTA from below.  They are
    // ranked as whole numbers that differ in their last bits (which rounds those of 32-bit logits, for the ranks alone).
    float top = fmaxf(mine, __shfl_xor_sync(0xFFFFFFFFu, mine, 1));
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    const unsigned int top_order = beam_logit_order(top), own_bucket = (top_order & ~(kBeamBuckets - 1u)) | threadIdx.x >> 2;
    if ((lane & 3) == 0) bucket[threadIdx.x >> 2] = own_bucket;
    __syncthreads();
    {
        int rank = 0;
#pragma unroll
        for (int i = 0; i < kBeamBuckets / 16; ++i) {
            const uint4 others = *reinterpret_cast<const uint4*>(&bucket[16 * i + 4 * (lane & 3)]);
            rank += (others.x > own_bucket) + (others.y > own_bucket) + (others.z > own_bucket) + (others.w > own_bucket);
        }
        rank += __shfl_xor_sync(0xFFFFFFFFu, rank, 1);
        rank += __shfl_xor_sync(0xFFFFFFFFu, rank, 2);
        const unsigned int least = __reduce_min_sync(0xFFFFFFFFu, rank < p.keep ? top_order : 0xFFFFFFFFu);
        if (lane == 0) atomicMin(&bound_order, least);
    }
    __syncthreads();
    float bound = beam_ordered_logit(bound_order);
    const bool single = span1 - span0 == 1;  // span: it is in the ring yet
    const int n = single ? min(p.vocabulary - span0 * beam_span(kType), beam_span(kType)) : beam_span(kType);
    if (n / (beam_span(kType) / kBeamBuckets) < p.keep + p.keep / 16) {
        // The least of all buckets of many, or of one with few logits in a short row or end of one, bounds badly: 256 maxima
        // then, one to a thread (1.4 us); of every 256th logit where they are in the ring, so that as many threads as can have
        // some.  Where the buckets can bound the search they do, with some 17 logits found for eight and 110 for 32 of them.
        float sample = single ? -INFINITY : mine;
        if (single)
            for (int i = threadIdx.x; i < n; i += kBeamThreads) sample = fmaxf(sample, beam_logit_at<kType>(beam_ring + i / kShare * (kBeamStages * kBeamBlock) + skew, i % kShare));
        const unsigned int order = beam_logit_order(sample), own = (order & ~(kBeamThreads - 1u)) | threadIdx.x;
        unsigned int* samples = reinterpret_cast<unsigned int*>(collected);  // which is empty yet
        samples[threadIdx.x] = own;
        __syncthreads();
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < kBeamThreads; i += 4) {
            const uint4 others = *reinterpret_cast<const uint4*>(&samples[i]);
            rank += (others.x > own) + (others.y > own) + (others.z > own) + (others.w > own);
        }
        const unsigned int least = __reduce_min_sync(0xFFFFFFFFu, rank < p.keep ? order : 0xFFFFFFFFu);
        if (lane == 0) atomicMin(&finer_order, least);
        __syncthreads();
        bound = beam_ordered_logit(finer_order);
    }
    // The logits of the threads whose maximum of a span qualifies, by their warp: a lane each, with their tokens; read again
    // from the ring or from memory, those of four threads together.
    const char* source = single ? ring + skew : from;
    const int source0 = single ? span0 * beam_span(kType) + warp * kShare : 0;
    auto reach = [&](auto qualifies, auto visit) {
        unsigned int spans_left = 0;  // of this thread's that qualify
        for (int span = span0; span < span1; ++span) spans_left |= (qualifies(span_top[span - span0][threadIdx.x]) ? 1u : 0u) << (span - span0);
        unsigned int lanes = __ballot_sync(0xFFFFFFFFu, spans_left != 0);
        while (lanes && !__any_sync(0xFFFFFFFFu, count > kBeamCollect)) {
            float logit[4];
            int token[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int of = __ffs(lanes) - 1, span = span0 + __ffs(__shfl_sync(0xFFFFFFFFu, spans_left, max(of, 0))) - 1;
                token[i] = span * beam_span(kType) + warp * kShare + (lane / kPer * 32 + of) * kPer + lane % kPer;
                if (!lanes || lane >= kVectors * kPer || token[i] >= p.vocabulary) token[i] = -1;
                logit[i] = token[i] >= 0 ? beam_logit_at<kType>(source, token[i] - source0) : 0.0f;
                if (lane == of) spans_left &= spans_left - 1u;
                lanes = __ballot_sync(0xFFFFFFFFu, spans_left != 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (token[i] >= 0) visit(logit[i], token[i]);
        }
    };
    auto collect = [&](float logit, int token) {
        const int place = atomicAdd(&count, 1);
        if (place < kBeamCollect) collected[place] = beam_entry_key(logit, token);
    };
    reach([&](float top) { return top >= bound; }, [&](float logit, int token) { if (logit >= bound) collect(logit, token); });
    __syncthreads();
    BeamEntry* list = p.lists + (row * p.parts + part) * p.keep;
    int found = count;
    if (found > kBeamCollect) {
        // Very many equal ones (masked tokens, a constant row).  What lies above them, then the first of themselves.
        const int first = span0 * beam_span(kType), last = min(p.vocabulary, span1 * beam_span(kType));
        __syncthreads();
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        reach([&](float top) { return top > bound; }, [&](float logit, int token) { if (logit > bound) collect(logit, token); });
        __syncthreads();
        found = count;
        if (found > kBeamCollect) {
            // The large ones lie in few buckets: `keep` rounds over everything, each for the best behind the last.
            unsigned long long before = ~0ull;
            for (int r = 0; r < p.keep; ++r) {
                unsigned long long best = 0;  // none
                for (int token = first + threadIdx.x; token < last; token += kBeamThreads) {
                    const float logit = beam_logit_at<kType>(from, token);
                    const unsigned long long key = logit == logit ? beam_entry_key(logit, token) : 0ull;
                    if (key < before && key > best) best = key;
                }
#pragma unroll
                for (int offset = 16; offset >= 1; offset >>= 1) best = max(best, __shfl_xor_sync(0xFFFFFFFFu, best, offset));
                if (lane == 0) collected[warp] = best;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kWarps; ++w) best = max(best, collected[w]);
                if (threadIdx.x == 0) list[r] = beam_entry(best);
                before = best;
                __syncthreads();
            }
            return;
        }
        for (int at = first; at < last && found < p.keep; at += kBeamThreads) {  // room for all of a step: keep + 256
            const int token = at + threadIdx.x;
            if (token < last && beam_logit_at<kType>(from, token) == bound) collect(bound, token);
            __syncthreads();
            found = count;
            __syncthreads();
        }
    }
    // Eight threads rank an entry.
    for (int i = threadIdx.x >> 3; i < (found + 3) / 4 * 4; i += kBeamThreads / 8) {
        const unsigned long long own = collected[min(i, found - 1)];
        int rank = 0;
        for (int j = threadIdx.x & 7; j < found; j += 8) rank += collected[j] > own;
#pragma unroll
        for (int offset = 1; offset <= 4; offset <<= 1) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, offset);
        if (i < found && (lane & 7) == 0 && rank < p.keep) list[rank] = beam_entry(own);
    }
    for (int i = found + threadIdx.x; i < p.keep; i += kBeamThreads) list[i] = {-INFINITY, -1};
}

struct __align__(16) BeamCandidate {
    long long value;  // the 64-bit number as a whole one of the same order
    long long place;  // beam, logit (the larger first) and token from the top bit down; -1: there is none
};
constexpr int kBeamTokenBits = 19, kBeamPlaceShift = kBeamTokenBits + 32;
static_assert(MT_BEAM_MAX_VOCABULARY <= 1 << kBeamTokenBits && (long long)kBeamMaxBeams << kBeamPlaceShift > 0, "a place is a positive number");
__device__ __forceinline__ bool beam_before(const BeamCandidate& a, const BeamCandidate& b) {
    return a.value > b.value || (a.value == b.value && a.place < b.place);
}
__device__ __forceinline__ long long beam_order(double value) {
    const long long bits = __double_as_longlong(value + 0.0);  // one zero
    return bits ^ (bits >> 63 & 0x7FFFFFFFFFFFFFFFll);
}
__device__ __forceinline__ double beam_value(long long order) {
    return __longlong_as_double(order ^ (order >> 63 & 0x7FFFFFFFFFFFFFFFll));
}

// The order's 64-bit value rounded down to a 32-bit number, as a whole one of the same order (never 0); and the least
// value with that key, with its top bit turned over.
__device__ __forceinline__ unsigned int beam_key(long long order) { return beam_logit_order(__double2float_rd(beam_value(order))); }
__device__ __forceinline__ unsigned long long beam_key_floor(unsigned int key) {
    return (unsigned long long)beam_order((double)beam_ordered_logit(key)) ^ 0x8000000000000000ull;
}

// How many of n candidates come before `own`, eight neighbouring threads together; those without a place do not count.
__device__ __forceinline__ int beam_rank(const BeamCandidate* candidates, int n, const BeamCandidate& own) {
    int rank = 0;
#pragma unroll 4
    for (int j = threadIdx.x & 7; j < n; j += 8) {
        const BeamCandidate other = candidates[j];
        rank += other.place >= 0 && beam_before(other, own);
    }
#pragma unroll
    for (int offset = 1; offset <= 4; offset <<= 1) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, offset);
    return rank;
}

// e^d for d <= 0 in 64 bits, after Tang's table method (ACM TOMS 15, 1989): with t = d / ln 2 = n / 64 + f, |f| <= 1/128,
// e^d = 2^(n / 64) e^(f ln 2), the power of the last six bits of n from a table and the rest by its series, whose sixth term is
// below 2^-54.  t is off by 2^-53 |t| at most and is taken in one product: weighted by e^d in a softmax's sum, |d| is 13.2 at
// most in the mean, so that the sum is off by some 2^-48 of itself.  What lies below 2^-1000 is taken as that, the masked too.
__device__ __forceinline__ double beam_exp(double d, const double* powers) {
    constexpr double kLn2 = 0.693147180559945309417;
    const double t = fmax(d * (1.0 / kLn2), -1000.0);
    const int n = __double2int_rn(64.0 * t);
    const double y = fma((double)n, -1.0 / 64, t) * kLn2;
    const double rest = fma(fma(fma(fma(y, 1.0 / 120, 1.0 / 24), y, 1.0 / 6), y, 0.5), y, 1.0);
    const double power = powers[n & 63], product = fma(power * y, rest, power);
    return __hiloint2double(__double2hiint(product) + ((n >> 6) << 20), __double2loint(product));
}

// A thread's share of the sum of e^(logit - top) over a row, in 64 bits.  Vectors of 16 bytes of the row go round the threads,
// four of them asked for together; a row that is not on 16 bytes is read by the elements, in the same order of sums.  48 us for a
// row of 128256 in bf16, 15 us for 32001 (element by element with the library's exp: 150 and 34 us); with the conversions from and
// to 64 bits done by 32-bit instructions, 42 and 13 us.
template <int kType>
__device__ __forceinline__ double beam_exact_share(const char* row, int vocabulary, double top, const double* powers) {
    using Bits = std::conditional_t<kType == 2, uint32_t, uint16_t>;
    constexpr int kEach = 16 / sizeof(Bits), kTogether = 4;
    constexpr Bits kMasked = kType == 0 ? 0xFF80 : kType == 1 ? 0xFC00 : (Bits)0xFF800000;  // -inf: adds 2^-1000
    const bool whole = reinterpret_cast<uintptr_t>(row) % 16 == 0;
    const Bits* from = reinterpret_cast<const Bits*>(row);
    double sum = 0.0;
    for (long long first = (long long)threadIdx.x * kEach; first < vocabulary; first += (long long)blockDim.x * kEach * kTogether) {
        alignas(16) Bits bits[kTogether][kEach];
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            const long long at = first + (long long)k * blockDim.x * kEach;
            if (whole && at + kEach <= vocabulary) {
                *reinterpret_cast<uint4*>(bits[k]) = *reinterpret_cast<const uint4*>(from + at);
            } else {
#pragma unroll
                for (int i = 0; i < kEach; ++i) bits[k][i] = at + i < vocabulary ? from[at + i] : kMasked;
            }
        }
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            double part = 0.0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) part += beam_exp((double)beam_logit_at<kType>(bits[k], i) - top, powers);
            sum += part;
        }
    }
    return sum;
}

// One CTA per group; a list of sorted candidates for every part of every beam.  Bound by the latency of its steps: what it
// reads is asked for at once, the first `staged` entries of every list among it.  Where a beam or two have most of the best
// candidates, a second search among those collected keeps the ranks short (32 beams over 32001, 64 kept, with the kernel
// before: 23 us; 480 more without it).
template <int kType>
__global__ void __launch_bounds__(1024) beam_join_kernel(const BeamSelectParams p) {
    extern __shared__ __align__(16) unsigned char join_smem[];
    const int lists = p.beams * p.parts, staged = p.staged, most = beam_join_most(p.keep);
    unsigned int* keys = reinterpret_cast<unsigned int*>(join_smem);                    // [kBeamKeys]
    BeamCandidate* collected = reinterpret_cast<BeamCandidate*>(keys + kBeamKeys);      // [most]
    BeamEntry* stage = reinterpret_cast<BeamEntry*>(collected + most);                  // [lists, staged]
    int* order = reinterpret_cast<int*>(stage + lists * staged);                        // [most]
    __shared__ double top[kBeamMaxBeams], log_sum[kBeamMaxBeams], score[kBeamMaxBeams], scratch[32], powers[64];
    __shared__ unsigned char kind[kBeamMaxBeams];  // 0: a beam's own lists, 1: it has finished, 2: it has no candidate
    __shared__ int count, reaching, tally[32];
    __shared__ unsigned int close, reached, key_bound;
    const int group = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const long long row0 = (long long)group * p.beams;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const BeamEntry* entries = p.lists + row0 * p.parts * p.keep;
    for (int i = threadIdx.x; i < lists * staged; i += blockDim.x) {
        const int list = beam_divided(i, p.per_staged);
        ptx::cp_async_8(stage + i, entries + (long long)list * p.keep + (i - list * staged));
    }
    ptx::cp_async_commit();
    for (int beam = warp; beam < p.beams; beam += warps) {
        const float given = p.scores[row0 + beam];
        const bool ended = p.finished && p.finished[row0 + beam];
        const BeamShareStats* stats = p.stats + (row0 + beam) * p.spans * kBeamShares;
        const int shares = p.spans * kBeamShares;
        // 128 shares at a time: a lane's four of them are asked for together.  The row's maximum first, so that every share is
        // weighted once; what does not fit the first 128 is read twice.
        BeamShareStats own[4];
        auto take = [&](int first) {
            float most = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = first + 32 * k + lane;
                own[k] = i < shares ? stats[i] : BeamShareStats{-INFINITY, 0.0f};
                most = fmaxf(most, own[k].top);
            }
            return most;
        };
        float best = -INFINITY;
#pragma unroll 1
        for (int first = 128; first < shares; first += 128) best = fmaxf(best, take(first));
        best = fmaxf(best, take(0));
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(best) : "f"(best));
        auto weighted = [&] {
            float part = 0.0f;  // of the same error as within a share
#pragma unroll
            for (int k = 0; k < 4; ++k) part += own[k].sum == 0.0f ? 0.0f : own[k].sum * __expf(own[k].top - best);
            return (double)part;
        };
        double sum = weighted();
#pragma unroll 1
        for (int first = 128; first < shares; first += 128) {
            take(first);
            sum += weighted();
        }
#pragma unroll
        for (int offset = 16; offset >= 1; offset >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, offset);
        if (lane == 0) {
            top[beam] = best;
            log_sum[beam] = log(sum);
            score[beam] = given;
            kind[beam] = !(given > kDeadScore) ? 2 : ended ? 1 : !(sum > 0.0 && sum < INFINITY && best < INFINITY) ? 2 : 0;
        }
    }
    if (threadIdx.x == 0) close = reached = 0;
    ptx::cp_async_wait_group<0>();
    __syncthreads();
    const long long nothing = beam_order(-INFINITY);
    // Candidate `depth` of a list of a beam.
    auto candidate = [&](int list, int beam, int depth) -> BeamCandidate {
        const long long base = (long long)beam << kBeamPlaceShift;
        if (kind[beam] == 0) {
            const BeamEntry entry = depth < staged ? stage[list * staged + depth] : entries[(long long)list * p.keep + depth];
            if (entry.token < 0) return {nothing, -1};
            return {beam_order(score[beam] + (((double)entry.logit - top[beam]) - log_sum[beam])),
                    base + ((long long)(0xFFFFFFFFu - beam_logit_order(entry.logit)) << kBeamTokenBits) + entry.token};
        }
        const int part = list - beam * p.parts;
        long long token = depth;  // no candidate: the first tokens, at -inf
        if (kind[beam] == 1) {
            if (depth == 0) return part == 0 ? BeamCandidate{beam_order(score[beam]), base + p.end_token} : BeamCandidate{nothing, -1};
            token = depth - 1 < p.end_token ? depth - 1 : depth;
        }
        if (part > 0 || token >= p.vocabulary) return {nothing, -1};
        return {nothing, base + token};
    };
    // The first entries of every list, one to a thread and `keep` at least: what the keep-th best of them reaches bounds the
    // keep-th best of all from below.  It is found among the values rounded to 32 bits, which keeps their order; where too many
    // are equal there, bit by bit, by value and among equals by place.
    const int samples = lists * p.depths;
    constexpr unsigned long long kTopBit = 0x8000000000000000ull;
    for (int phase = 0;; ++phase) {
        const double margin = phase == 0 && p.beams > 1 ? 2.0 * kBeamError : 0.0;
        if (threadIdx.x == 0) {
            count = 0;
            key_bound = 0;
            reaching = 0;
        }
        BeamCandidate sample = {0, -1};
        if (threadIdx.x < samples) {
            const int list = beam_divided(threadIdx.x, p.per_depths);
            sample = candidate(list, beam_divided(list, p.per_parts), threadIdx.x - list * p.depths);
        }
        const unsigned int key = sample.place < 0 ? 0u : beam_key(sample.value);
        if (threadIdx.x < kBeamKeys) keys[threadIdx.x] = key;
        __syncthreads();
        if (warp == 0 && samples <= kBeamKeys) {  // from the first bit in which they differ
            unsigned int own[kBeamKeys / 32], highest = 0, lowest = 0xFFFFFFFFu;
            int now = 0;
#pragma unroll
            for (int k = 0; k < kBeamKeys / 32; ++k) {
                own[k] = keys[32 * k + lane];
                highest = max(highest, own[k]);
                lowest = min(lowest, own[k] - 1u);  // none is the largest so
                now += own[k] != 0;
            }
            highest = __reduce_max_sync(0xFFFFFFFFu, highest);
            lowest = __reduce_min_sync(0xFFFFFFFFu, lowest) + 1u;
            now = __reduce_add_sync(0xFFFFFFFFu, now);
            if (now >= p.keep) {
                unsigned int found_key = lowest, bit = highest ^ lowest;
                for (bit = bit ? 0x80000000u >> __clz(bit) : 0u; bit && now > p.keep + kBeamSlack; bit >>= 1) {
                    const unsigned int tried = (found_key & ~(bit - 1u)) | bit;
                    int reach_it = 0;
#pragma unroll
                    for (int k = 0; k < kBeamKeys / 32; ++k) reach_it += own[k] >= tried;
                    reach_it = __reduce_add_sync(0xFFFFFFFFu, reach_it);
                    if (reach_it >= p.keep) {
                        found_key = tried;
                        now = reach_it;
                    } else {
                        found_key &= ~bit;
                    }
                }
                if (lane == 0) {
                    key_bound = max(found_key, lowest);
                    reaching = now;
                }
            }
        }
        __syncthreads();
        unsigned long long value_bound = 0, place_bound = 0;
        if (reaching > p.keep + kBeamSlack || samples > kBeamKeys) {
            const unsigned long long value = (unsigned long long)sample.value ^ kTopBit, place = ~(unsigned long long)sample.place;
            int now_reaching = 0x7FFFFFFF;
            for (unsigned long long bit = kTopBit; bit && now_reaching > p.keep + kBeamSlack; bit >>= 1) {
                const int now = __syncthreads_count(sample.place >= 0 && value >= (value_bound | bit));
                if (now >= p.keep) {
                    value_bound |= bit;
                    now_reaching = now;
                }
            }
            for (unsigned long long bit = kTopBit; bit && now_reaching > p.keep + kBeamSlack; bit >>= 1) {
                const int now = __syncthreads_count(sample.place >= 0 && (value > value_bound || (value == value_bound && place >= (place_bound | bit))));
                if (now >= p.keep) {
                    place_bound |= bit;
                    now_reaching = now;
                }
            }
        } else if (key_bound) {
            value_bound = beam_key_floor(key_bound);
        }
        const unsigned long long least = (unsigned long long)nothing ^ kTopBit;
        bool wider = margin > 0.0 && value_bound > least, again = true, dropped = false;
        int found;
        for (;;) {
            const unsigned long long reach = wider ? (unsigned long long)beam_order(beam_value((long long)(value_bound ^ kTopBit)) - margin) ^ kTopBit : value_bound;
            for (int i = threadIdx.x; i < lists * p.keep; i += blockDim.x) {
                const int list = beam_divided(i, p.per_keep);
                const BeamCandidate own = candidate(list, beam_divided(list, p.per_parts), i - list * p.keep);
                const unsigned long long value = (unsigned long long)own.value ^ kTopBit;
                if (own.place < 0 || value < reach || (!wider && value == reach && ~(unsigned long long)own.place < place_bound)) continue;
                const int at = atomicAdd(&count, 1);
                if (at < most) collected[at] = own;
            }
            if (threadIdx.x < 32) tally[threadIdx.x] = 0;
            __syncthreads();
            found = min(count, wider ? count : most);  // only the margin can let in more than `most`
            const bool full = found > most;            // without it then, and what lies within it is looked at below
            if (!full && (!again || found <= kBeamMany)) break;
            __syncthreads();
            if (threadIdx.x == 0) count = 0;
            if (full) {
                wider = false;
                dropped = true;
                __syncthreads();
                continue;
            }
            // Few lists hold most of the best, and the first entries of all bounded them badly: the keep-th best of what was
            // collected, by the values rounded to 32 bits.
            again = false;
            unsigned int* rounded = reinterpret_cast<unsigned int*>(order);
            for (int i = threadIdx.x; i < found; i += blockDim.x) rounded[i] = beam_key(collected[i].value);
            unsigned int bound_key = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned int tried = bound_key | 1u << bit;
                int reach_it = 0;
                for (int i = threadIdx.x; i < found; i += blockDim.x) reach_it += rounded[i] >= tried;
                reach_it = __reduce_add_sync(0xFFFFFFFFu, reach_it);
                if (lane == 0) atomicAdd(&tally[bit], reach_it);
                __syncthreads();
                reach_it = tally[bit];
                if (reach_it >= p.keep) bound_key = tried;
                if (reach_it >= p.keep && reach_it <= p.keep + kBeamSlack) break;
            }
            const unsigned long long raised = bound_key ? beam_key_floor(bound_key) : 0ull;
            if (raised > value_bound) {
                value_bound = raised;
                place_bound = 0;
            }
            wider = margin > 0.0 && value_bound > least;
            dropped = dropped && !wider;
            __syncthreads();
        }
        for (int i = threadIdx.x >> 3; i < (found + 3) / 4 * 4; i += blockDim.x >> 3) {
            const int rank = beam_rank(collected, found, collected[min(i, found - 1)]);
            if (i < found && (lane & 7) == 0) order[rank] = i;
        }
        __syncthreads();
        if (margin > 0.0) {
            const BeamCandidate last = collected[order[p.keep - 1]];  // nobody further below it than the margin can rise
            for (int i = threadIdx.x; i + 1 < found; i += blockDim.x) {
                const BeamCandidate upper = collected[order[i]], lower = collected[order[i + 1]];
                if (i + 1 >= p.keep && beam_value(last.value) - beam_value(lower.value) > margin) break;
                const int a = (int)(upper.place >> kBeamPlaceShift), b = (int)(lower.place >> kBeamPlaceShift);
                if (a != b && lower.value > nothing && beam_value(upper.value) - beam_value(lower.value) <= margin) atomicOr(&close, 1u << a | 1u << b);
            }
            if (dropped) {
                // What was too many to collect and rank: all beams with a candidate from the last one down to the margin below it, if
                // those are two or more.  A ranking of all finds the same beams, so a group's bits do not depend on how many there
                // were, which follows the cut of the rows.
                for (int i = threadIdx.x; i < lists * p.keep; i += blockDim.x) {
                    const int list = beam_divided(i, p.per_keep), beam = beam_divided(list, p.per_parts);
                    const BeamCandidate own = candidate(list, beam, i - list * p.keep);
                    if (own.place >= 0 && own.value > nothing && !beam_before(own, last) && beam_value(last.value) - beam_value(own.value) <= margin)
                        atomicOr(&reached, 1u << beam);
                }
                __syncthreads();
                if (threadIdx.x == 0 && __popc(reached) > 1) close |= reached;
            }
            __syncthreads();
            if (close) {
                if (threadIdx.x < 64) powers[threadIdx.x] = exp2(threadIdx.x / 64.0);
                __syncthreads();
                for (int beam = 0; beam < p.beams; ++beam) {
                    if (!(close >> beam & 1u) || kind[beam] != 0) continue;
                    const char* row = static_cast<const char*>(p.logits) + (row0 + beam) * p.row_stride * (kType == 2 ? 4 : 2);
                    double sum = beam_exact_share<kType>(row, p.vocabulary, top[beam], powers);
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
            const int parent = (int)(best.place >> kBeamPlaceShift);
            const long long token = best.place & ((1ll << kBeamTokenBits) - 1), at = (long long)group * p.keep + r;
            p.scores_out[at] = (float)beam_value(best.value);
            p.parents_out[at] = parent;
            p.tokens_out[at] = token;
            p.finished_out[at] = (p.finished && p.finished[row0 + parent]) || token == p.end_token;
        }
        return;
    }
}

template <int kType>
inline int launch_beam_select(BeamSelectParams params, int sm_count, cudaStream_t stream) {
    params.spans = beam_spans(params.vocabulary, kType);
    params.parts = beam_parts(params.groups * params.beams, params.spans, sm_count);
    const int lists = params.beams * params.parts;
    // A list or more of each, and a beam of each warp (16 beams over 12626: 14 us, with two to a warp 16).
    const int threads = lists > 512 || params.beams > 16 ? 1024 : lists > 256 || params.beams > 8 ? 512 : 256;
    params.staged = params.keep < kBeamStage / lists ? params.keep : kBeamStage / lists;
    const int covering = (params.keep + lists - 1) / lists, filling = threads / lists;
    params.depths = covering > filling ? covering : filling;
    params.depths = params.depths < params.keep ? params.depths : params.keep;
    params.per_keep = beam_reciprocal(params.keep);
    params.per_staged = beam_reciprocal(params.staged);
    params.per_depths = beam_reciprocal(params.depths);
    params.per_parts = beam_reciprocal(params.parts);
    auto smem_of = [](int keep, int entries) {
        return beam_join_most(keep) * (sizeof(BeamCandidate) + sizeof(int)) + entries * sizeof(BeamEntry) + kBeamKeys * sizeof(int);
    };
    static bool configured[64] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return MT_ERR_LAUNCH;
    if (device >= 64 || !configured[device]) {
        if (cudaFuncSetAttribute(beam_join_kernel<kType>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(kBeamMaxKeep, kBeamStage)) != cudaSuccess)
            return MT_ERR_LAUNCH;
        if (cudaFuncSetAttribute(beam_span_kernel<kType>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBeamRing) != cudaSuccess) return MT_ERR_LAUNCH;
        if (device < 64) configured[device] = true;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(params.groups * params.beams * params.parts, 1, 1);
    config.blockDim = dim3(kBeamThreads, 1, 1);
    config.dynamicSmemBytes = kBeamRing;
    config.stream = stream;
    cudaLaunchAttribute attrs[1];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, beam_span_kernel<kType>, params) != cudaSuccess) return MT_ERR_LAUNCH;
    config.gridDim = dim3(params.groups, 1, 1);
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = smem_of(params.keep, lists * params.staged);
    return cudaLaunchKernelEx(&config, beam_join_kernel<kType>, params) == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
}

}  // namespace mt
