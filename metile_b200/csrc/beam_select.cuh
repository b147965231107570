// Beam search's selection: the best continuations over a group's beams and the vocabulary.
//
// A candidate is (beam, token) with the value score[beam] + (logit - max) - log sum exp(logit - max), in 64 bits; equal
// ones go by the lower beam, then the lower token.  What has no value (a row with a NaN, with +inf or with nothing above
// -inf; a score that is a mask) counts as -inf.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"

namespace mt {

constexpr double kDeadScore = -1e15;  // no sum of log-probabilities: the mask of a beam that is out

struct BeamSelectParams {
    const void* logits;             // [groups * beams, vocabulary], rows `row_stride` apart
    const float* scores;            // [groups, beams]
    const unsigned char* finished;  // [groups, beams] or null
    float* scores_out;              // [groups, keep]
    int* parents_out;
    long long* tokens_out;
    unsigned char* finished_out;
    long long row_stride, end_token;   // no end token: -1
    int groups, beams, vocabulary, keep, type;
};

constexpr int kBeamMaxBeams = 32, kBeamMaxKeep = 64;

__device__ __forceinline__ float logit_at(const void* row, int type, long long i) {
    if (type == 0) return bf16_bits_to_f32(static_cast<const uint16_t*>(row)[i]);
    if (type == 1) return __half2float(static_cast<const __half*>(row)[i]);
    return static_cast<const float*>(row)[i];
}

struct BeamBest {
    double value;
    long long flat;
};
__device__ __forceinline__ bool beam_before(const BeamBest& a, const BeamBest& b) {
    return a.value > b.value || (a.value == b.value && a.flat < b.flat);
}

// One CTA per group: the rows' maxima and sums, then `keep` walks over all candidates, each for the best behind the last.
__global__ void __launch_bounds__(1024) beam_select_kernel(const BeamSelectParams p) {
    __shared__ double top[kBeamMaxBeams], log_sum[kBeamMaxBeams], scratch[32];
    __shared__ BeamBest found[32];
    __shared__ BeamBest last;
    const int group = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const size_t size = p.type == 2 ? 4 : 2;
    auto row_of = [&](int beam) {
        return static_cast<const char*>(p.logits) + ((long long)group * p.beams + beam) * p.row_stride * size;
    };
    for (int beam = 0; beam < p.beams; ++beam) {
        const void* row = row_of(beam);
        float m = -INFINITY;
        bool bad = false;
        for (long long i = threadIdx.x; i < p.vocabulary; i += blockDim.x) {
            const float v = logit_at(row, p.type, i);
            bad = bad || v != v;
            m = fmaxf(m, v);
        }
        if (bad) m = INFINITY;
        for (int offset = 16; offset >= 1; offset >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, offset));
        if (lane == 0) scratch[warp] = m;
        __syncthreads();
        double best = scratch[0];
        for (int w = 1; w < 32; ++w) best = fmax(best, scratch[w]);
        __syncthreads();
        double sum = 0.0;
        for (long long i = threadIdx.x; i < p.vocabulary; i += blockDim.x) sum += exp((double)logit_at(row, p.type, i) - best);
        for (int offset = 16; offset >= 1; offset >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, offset);
        if (lane == 0) scratch[warp] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            double total = 0.0;
            for (int w = 0; w < 32; ++w) total += scratch[w];
            top[beam] = best;
            log_sum[beam] = log(total);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) last = {INFINITY, -1};
    __syncthreads();
    for (int r = 0; r < p.keep; ++r) {
        const BeamBest before = last;
        BeamBest best = {-INFINITY, 0x7FFFFFFFFFFFFFFFll};
        for (int beam = 0; beam < p.beams; ++beam) {
            const void* row = row_of(beam);
            const float score = p.scores[group * p.beams + beam];
            const bool ended = p.finished && p.finished[group * p.beams + beam];
            const bool dead = !(score > kDeadScore) || (!ended && !(top[beam] > -INFINITY && top[beam] < INFINITY));
            for (long long i = threadIdx.x; i < p.vocabulary; i += blockDim.x) {
                BeamBest mine = {-INFINITY, (long long)beam * p.vocabulary + i};
                if (!dead && ended) mine.value = i == p.end_token ? (double)score : -INFINITY;
                else if (!dead) mine.value = (double)score + ((double)logit_at(row, p.type, i) - top[beam] - log_sum[beam]);
                if (beam_before(before, mine) && beam_before(mine, best)) best = mine;
            }
        }
        for (int offset = 16; offset >= 1; offset >>= 1) {
            const BeamBest other = {__shfl_xor_sync(0xFFFFFFFFu, best.value, offset), __shfl_xor_sync(0xFFFFFFFFu, best.flat, offset)};
            if (beam_before(other, best)) best = other;
        }
        if (lane == 0) found[warp] = best;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 32; ++w)
                if (beam_before(found[w], best)) best = found[w];
            const int parent = (int)(best.flat / p.vocabulary);
            const long long token = best.flat - (long long)parent * p.vocabulary, at = (long long)group * p.keep + r;
            p.scores_out[at] = (float)best.value;
            p.parents_out[at] = parent;
            p.tokens_out[at] = token;
            p.finished_out[at] = (p.finished && p.finished[group * p.beams + parent]) || token == p.end_token;
            last = best;
        }
        __syncthreads();
    }
}

}  // namespace mt
