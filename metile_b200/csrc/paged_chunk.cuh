// Attention of several new tokens per request over a paged key-value cache, on the tcgen05 tensor cores.
//
// Rows starts[r] .. starts[r + 1] - 1 of the queries are the last tokens of request r, which has lengths[r] tokens with them: the
// i-th of n stands at position lengths[r] - n + i and sees the tokens up to its own:
//   out[i, h] = sum over t <= position of softmax_t(scale q[i, h] k[t]) v[t]
// 4 D operations per query head, row and token it sees; keys and values are read once for every 256 rows of a KV head's queries.
//
// A query tile is 128 rows: the query heads of one KV head for as many tokens as fit, so that a group of heads shares what it
// reads.  A unit of work is two tiles (one for D = 256, whose results fill tensor memory) against a range of the request's tokens.
// The tokens come in tiles of 128 (64), keys and values by TMA from wherever their pages lie, into a ring.  Per token tile and query
// tile, in tensor memory:
//   S[128 x tile] = Q K^T                  both operands in shared memory
//   O[128 x D]   += P V                    P, the 16-bit weights, in the place of S; V as it lies in memory (rows of D)
// A warpgroup per query tile, a row a thread, turns S into P: while it works on one tile the tensor cores have the other's.  Scores come in
// steps of 64 tokens, two of them ahead, so a row's scores stay in registers.  A row's maximum moves, and its O with it, only when a
// score passes it by more than 2^8.  The other warps: one asks for the tiles, one mends values that some rows do not see, and for each
// query tile a thread issues the products.
//
// The CTAs, one per SM, share the work of all units equally, counted in tokens; a unit that is cut between two of them is joined by a
// second kernel.  Where shares come out short, or the bits must not depend on the call, units stay whole.
//
// What bounds it.  Long prompts: the exponentials and the moves between registers and tensor memory, about 1650 cycles per 64 tokens of a
// pair of tiles, for which the products take 1240: 4093 tokens behind 11000, 32 heads of 128, 770 us in a graph, 1.14 PFLOP/s, and 873 one
// call behind the other, where the clock follows the power.  Few rows: the chain of one tile, some 1300 cycles per 64 tokens, which one SM's
// share of the reads just covers: 17 tokens behind 100003 96 us, 4.3 TB/s with the join.  Short calls: the start, 11 us of 17 for
// four drafts of five tokens behind 700.
// Tried: a quarter of the exponentials as polynomials (long prompt 791 us against 767), 13 warps and more (128 registers a thread: 15 %
// slower), two sets of scores in registers (they spill).
//
// P is rounded once to 16 bits: a weight is off by half a step of the type, and an output, an average by these weights, by less
// than its own rounding for all but the shortest rows.  (In fp16 weights are lifted by 2^7, see kPagedLift.)  Sums are of the
// unrounded weights, in 32 bits.
//
// What a row does not see must weigh nothing whatever lies there.  Scores are masked by position.  Values behind the unit's last
// position are overwritten by zeros in shared memory; among those that some rows see and others do not, infinities and NaN are
// taken out and noted, by column, with the first position that has one, and put into the results of the rows that see them.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "affine_umma.cuh"
#include "beam_select.cuh"
#include "paged_attention.cuh"

namespace mt {

constexpr unsigned int kStartOutside = 0x306;  // paged_attention_chunk: word 1 = request, 2 = its first row
constexpr unsigned int kChunkWait = 0x9D0;     // a wait that gave up: + the role

constexpr int kChunkRows = 128;                // of a query tile
constexpr int kChunkStep = 64;                 // tokens whose scores are taken at once
constexpr int kChunkRuns = 64;                 // runs of requests whose work is counted
constexpr int kChunkUnitCost = 256;            // what a unit costs beside its tokens, in tokens
constexpr int kChunkShare = 512;               // the least work of a CTA, in tokens: at least two tiles between two cuts
constexpr int kChunkCutGain = 1024;            // units are cut where that takes more than this off the longest share, in tokens
constexpr int kChunkNotes = 2;                 // units whose noted columns may be needed at once: the one begun and the one that ends

template <int kD>
struct ChunkShape {
    static constexpr int kGroups = kD == 256 ? 1 : 2;               // query tiles of a unit
    static constexpr int kTile = kD == 256 ? 64 : 128;              // tokens that come together
    static constexpr int kSteps = kTile / kChunkStep;
    static constexpr int kSlots = kD == 256 ? 4 : kD == 128 ? 5 : 6;  // tiles of keys or values
    static constexpr int kQBytes = kChunkRows * kD * 2, kSlotBytes = kTile * kD * 2;
    static constexpr int kSoftmaxWarps = 4 * kGroups, kWarps = kSoftmaxWarps + 2 + kGroups, kThreads = 32 * kWarps;
    static constexpr int kOColumn = 256;                            // in tensor memory; scores of tile g at 128 g and 128 g + 64
    static constexpr int kTiles = kGroups * kQBytes + kSlots * kSlotBytes;
    static constexpr int kSlotRows = kGroups * kChunkRows;          // of a partial result
    static_assert(kOColumn + kGroups * kD <= 512 && kGroups * 2 * kChunkStep <= kOColumn && kSlots <= 6);
};

struct PagedChunkParams {
    CUtensorMap q_map;                 // (D, Hq, rows): boxes of 64 x heads of a part x tokens of a tile
    CUtensorMap key_map, value_map;    // (64, 8 rows, D / 64, rows of a page / 8, places of heads and pages): boxes of up to a tile's rows of a page
    int key_head, key_page, value_head, value_page;  // steps of the last dimension for a head and a page
    int key_none, value_none;          // behind its end: zeros
    const int* tables;                 // [requests, width], rows `table_stride` apart
    const int* lengths;                // [requests]
    const int* starts;                 // [requests + 1]
    uint16_t* out;                     // [rows, Hq, D]
    float* partial;                    // [CTAs, 2, rows of a unit, D]: of the first unit, begun before, and of the last one, which goes on
    float2* stats;                     // [CTAs, 2, rows of a unit]: maximum (log2) and sum
    struct ChunkCut* cuts;             // [CTAs]
    long long table_stride;
    int width, rows, requests, q_heads, kv_heads, page_shift, page_count;
    int part_heads, parts;             // query heads of a KV head that share a tile; tiles that takes
    int tile_tokens;                   // of a query tile
    bool whole;                        // units are not cut
    float scale;
};

// What a CTA leaves to be joined.
struct ChunkCut {
    int row0, tokens, head0, heads;    // the unit that begins here and goes on elsewhere; no tokens: there is none
    int continues, through;            // the first unit was begun before; and goes on behind this CTA
};

// What a unit is, for all warps of a CTA.
struct ChunkUnit {
    int request, kv_head, head0;       // head0: the first query head
    int heads;                         // of the tile
    int row0, tokens;                  // rows of the query: the first, how many (both tiles)
    int position0;                     // of the first row, may be negative
    int first_tile, tiles;             // token tiles of this part of it; -1: there are no more units
    int end;                           // tokens from here on are seen by no row or belong to another part
    int slot;                          // of the partial results: 0 or 1, or -1 where this is all of it
};

struct ChunkRequest {
    int first, n, length;
};

__device__ __forceinline__ ChunkRequest chunk_request(const PagedChunkParams& p, int r, bool report) {
    ChunkRequest q = {p.starts[r], 0, p.lengths[r]};
    const int end = p.starts[r + 1];
    if (q.first < 0 || end < q.first || end > p.rows) {
        if (report) record_index(kStartOutside, r, (unsigned int)q.first);
        return q;
    }
    q.n = end - q.first;
    const long long capacity = (long long)p.width << p.page_shift;
    if (q.length < 0 || q.length > capacity) {
        if (report) record_index(kLengthOutside, r, (unsigned int)q.length);
        q.length = q.length < 0 ? 0 : (int)capacity;
    }
    return q;
}

// A request's queries in blocks of `unit` rows; a block is a unit for every KV head and part.  The work of a unit is counted as the
// tokens that its last row sees and kChunkUnitCost.  chunk_work: of the first b blocks, for one head.
__host__ __device__ __forceinline__ int chunk_blocks(int n, int unit) { return (n + unit - 1) / unit; }
__host__ __device__ __forceinline__ int chunk_seen(int length, int n, int unit, int b) {
    const int rows = (b + 1) * unit < n ? (b + 1) * unit : n, seen = length - n + rows;
    return seen > 0 ? seen : 0;
}
__host__ __device__ __forceinline__ long long chunk_work(int length, int n, int unit, int b) {
    long long work = (long long)b * kChunkUnitCost;
    const int whole = b < n / unit ? b : n / unit;       // blocks of `unit` rows, which see before + unit, before + 2 unit, ...
    const long long before = (long long)length - n;
    const long long blind = before >= 0 ? 0 : (-before / unit < whole ? -before / unit : whole);  // of them see nothing
    const long long count = whole - blind;
    work += count * before + (long long)unit * ((long long)whole * (whole + 1) / 2 - blind * (blind + 1) / 2);
    if (b > whole) work += length > 0 ? length : 0;      // and the last one, of fewer rows
    return work;
}

// A place in the work of all units: a unit and a token tile of it.
struct ChunkPlace {
    int request, block, head, tile;
};
__device__ __forceinline__ bool same_unit(const ChunkPlace& a, const ChunkPlace& b) { return a.request == b.request && a.block == b.block && a.head == b.head; }

// Two numbers rounded to 16 bits in one instruction.  (Single conversions run in the pipe of the exponentials, which bounds this
// kernel as much as the tensor cores do.)
template <bool kHalf>
__device__ __forceinline__ uint32_t rounded_pair(float low, float high) {
    uint32_t pair;
    if constexpr (kHalf) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pair) : "f"(high), "f"(low));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(pair) : "f"(high), "f"(low));
    return pair;
}

__device__ __forceinline__ float largest_of(float a, float b, float c) {
    float out;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(out) : "f"(a), "f"(b), "f"(c));
    return out;
}
// The largest of 32 numbers, NaN left out.
__device__ __forceinline__ float most_of(const float* x) {
    float most[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        most[i] = fmaxf(x[i], x[4 + i]);
#pragma unroll
        for (int c = 8; c < 32; c += 8) most[i] = largest_of(most[i], x[c + i], x[c + 4 + i]);
    }
    return largest_of(fmaxf(most[0], most[1]), most[2], most[3]);
}
namespace ptx {

// 32 bytes by a thread: half the instructions where every thread has a row of its own.
__device__ __forceinline__ void st_global_32(void* to, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ void tma_load_5d(void* smem_dst, const void* tensor_map, int c0, int c1, int c2, int c3, int c4, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(smem_u32(smem_dst)), "l"(tensor_map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar))
        : "memory");
}

// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

// D[tmem] (+)= A[smem desc] * B[smem desc].
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 lanes x 32 consecutive 32-bit columns; thread i of the warp has lane (base lane + i).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]),
          "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]),
          "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}
// Waits for this thread's tcgen05.ld and names the registers as in/out operands, so that nothing on them moves above the wait.
__device__ __forceinline__ void tc_wait_ld32(float* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                   "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]),
                   "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]),
                   "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
                 :
                 : "memory");
}

// Shared-memory matrix descriptor of keys or values as they lie in the ring: groups of eight rows, of each D / 64 blocks of
// 8 x 128 bytes with 128-byte swizzle.  Keys: rows along N, and a block of 64 dims after the other along K.  Values: rows along K, the
// blocks along N.
__device__ __forceinline__ uint64_t smem_desc_grouped_sw128(uint32_t smem_addr, int blocks) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)(1024 >> 4) << 16 | (uint64_t)(blocks * 1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// Instruction descriptor for kind::f16: 16-bit x 16-bit -> fp32; bit 16 turns B over (rows along N).
__host__ __device__ constexpr uint32_t umma_idesc_half(int m, int n, bool half, bool b_mn_major) {
    return (1u << 4) | (half ? 0u : 1u << 7 | 1u << 10) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

}  // namespace ptx

// The barriers and small arrays behind the tiles.
template <int kD>
struct ChunkShared {
    using Shape = ChunkShape<kD>;
    uint32_t notes[kChunkNotes][kD];   // of a column: the first positions with a NaN, +inf, -inf, 10 bits each, from the unit's first on
    long long work[kChunkRuns + 1];    // in front of every run of requests
    int longest[kChunkRuns / 32];      // unit
    uint64_t q_full, q_empty, drained;
    uint64_t full[6], empty[6];        // of the ring
    uint64_t turn[2];                  // of the issuers
    uint64_t to_fix, fixed;            // tiles of values that some rows do not see, one after the other
    uint64_t s_full[2][2], p_full[2][2], o_done[2][2];  // of a query tile, and of its two places for scores
    ChunkUnit unit;
    unsigned int bad_rows[8];          // of a token tile: groups of eight tokens whose page lies outside the cache
    int noted[kChunkNotes];            // whether a unit has notes
    uint32_t tmem;
    int abort;
};

// The tiles start on 1024 bytes, which the kernel sees to: an alignment of the dynamic array would be that of every kernel's.
template <int kD>
constexpr int chunk_smem() { return 1024 + ChunkShape<kD>::kTiles + (int)sizeof(ChunkShared<kD>); }
static_assert(chunk_smem<64>() <= 232448 && chunk_smem<128>() <= 232448 && chunk_smem<256>() <= 232448);

template <int kD, bool kHalf>
__global__ void __launch_bounds__(ChunkShape<kD>::kThreads, 1) paged_chunk_kernel(const __grid_constant__ PagedChunkParams p) {
    using Shape = ChunkShape<kD>;
    using Shared = ChunkShared<kD>;
    constexpr int kTile = Shape::kTile, kGroups = Shape::kGroups, kSlots = Shape::kSlots, kChunks = kD / 64;
    extern __shared__ __align__(16) uint8_t chunk_dynamic[];
    uint8_t* q_tiles = chunk_dynamic + (-ptx::smem_u32(chunk_dynamic) & 1023u);
    uint8_t* ring = q_tiles + kGroups * Shape::kQBytes;
    Shared& s = *reinterpret_cast<Shared*>(q_tiles + Shape::kTiles);
    volatile int* abort_flag = &s.abort;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    constexpr int kLoader = Shape::kSoftmaxWarps, kFixer = kLoader + 1, kIssuer = kLoader + 2;  // an issuer for each query tile

    if (threadIdx.x == 0) {
        ptx::mbar_init(&s.q_full, 1);
        ptx::mbar_init(&s.q_empty, kGroups + Shape::kSoftmaxWarps + 1);  // the last products of keys; the other warps have read the unit
        ptx::mbar_init(&s.drained, kGroups);
        ptx::mbar_init(&s.to_fix, kGroups);  // both issuers: neither is more than a tile that was mended behind
        ptx::mbar_init(&s.fixed, 1);
        for (int i = 0; i < kSlots; ++i) {
            ptx::mbar_init(&s.full[i], 1);
            ptx::mbar_init(&s.empty[i], kGroups);
        }
        for (int g = 0; g < kGroups; ++g) {
            for (int i = 0; i < 2; ++i) {
                ptx::mbar_init(&s.s_full[g][i], 1);
                ptx::mbar_init(&s.p_full[g][i], 4);
                ptx::mbar_init(&s.o_done[g][i], 1);
            }
            ptx::mbar_init(&s.turn[g], 1);
        }
        s.abort = 0;
        ptx::mbar_fence_init();
    }
    if (warp == kIssuer) {
        ptx::tmem_alloc(&s.tmem, 512);
        ptx::tmem_relinquish();
    }
    if (warp == kLoader && lane == 0) {
        ptx::prefetch_tensor_map(&p.q_map);
        ptx::prefetch_tensor_map(&p.key_map);
        ptx::prefetch_tensor_map(&p.value_map);
    }
    ptx::griddep_wait();

    // Work in front of every run of requests.
    const int run = (p.requests + kChunkRuns - 1) / kChunkRuns, unit_tokens = kGroups * p.tile_tokens, unit_heads = p.kv_heads * p.parts;
    if (threadIdx.x < kChunkRuns) {
        long long mine = 0;
        int longest = 0;
        for (int r = threadIdx.x * run; r < min((int)(threadIdx.x + 1) * run, p.requests); ++r) {
            const ChunkRequest q = chunk_request(p, r, blockIdx.x == 0);
            mine += unit_heads * chunk_work(q.length, q.n, unit_tokens, chunk_blocks(q.n, unit_tokens));
            if (q.n > 0) longest = max(longest, min(q.length, 0x7FFFFFFF - kChunkUnitCost) + kChunkUnitCost);
        }
        s.work[threadIdx.x + 1] = mine;
        longest = __reduce_max_sync(0xFFFFFFFFu, longest);
        if (lane == 0) s.longest[warp] = longest;
    }
    __syncthreads();
    // Not before this CTA has its tensor memory: the next kernel's could take it and then wait for this one's end.
    ptx::griddep_launch_dependents();
    if (warp == 0) {
        constexpr int kEach = kChunkRuns / 32;
        long long own[kEach], sum = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) own[i] = sum += s.work[lane * kEach + i + 1];
        long long before = sum;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const long long other = __shfl_up_sync(0xFFFFFFFFu, before, offset);
            if (lane >= offset) before += other;
        }
        before -= sum;
#pragma unroll
        for (int i = 0; i < kEach; ++i) s.work[lane * kEach + i + 1] = before + own[i];
        if (lane == 0) s.work[0] = 0;
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = s.tmem;

    if (warp == kLoader) {
        // ---- units, queries, keys and values ------------------------------------------------------------------
        // The work of all units, one behind the other, is cut into equal shares.  A cut within a unit falls between two token tiles, and
        // not beside its ends; where units are to stay whole it goes to the nearer end.
        const long long all = s.work[kChunkRuns];
        const int ctas = (int)max(1ll, min((long long)gridDim.x, all / kChunkShare));
        const long long share = all / ctas, rest = all - share * ctas;
        // Left whole, the units make the longest share half a unit longer than the others, or one unit where shares are shorter than that.
        // Whole and cut, us: 4 x 512 tokens behind 512 (2 x 6 heads) 39 and 49, 16 x 6 behind 2000 44 and 50, 256 x 2 behind 300 115 and 145;
        // 4096 from the start 209 and 174, 512 behind 8192 162 and 108, 8 behind 3000 53 and 31 (8 x 4 heads).
        int longest = 0;
        for (int i = 0; i < kChunkRuns / 32; ++i) longest = max(longest, s.longest[i]);
        const bool whole = p.whole || (longest >= share ? longest - share : longest / 2) <= kChunkCutGain;
        auto tiles_of = [&](int seen) { return (seen + kTile - 1) / kTile; };
        ChunkRequest now = {0, 0, 0};  // the request of `at`
        auto next_unit = [&](ChunkPlace& at, ChunkRequest& q) {
            at.tile = 0;
            if (++at.head < unit_heads) return;
            at.head = 0;
            ++at.block;
            while (at.request < p.requests && at.block >= chunk_blocks(q.n, unit_tokens)) {
                at.block = 0;
                if (++at.request < p.requests) q = chunk_request(p, at.request, false);
            }
        };
        auto cut_at = [&](long long x, ChunkRequest& q) {
            ChunkPlace at = {p.requests, 0, 0, 0};
            if (x >= all) return at;
            const bool first = x == 0;
            int low = 0, high = kChunkRuns;
            while (high - low > 1) {
                const int middle = (low + high) >> 1;
                if (s.work[middle] <= x) low = middle; else high = middle;
            }
            x -= s.work[low];
            for (at.request = low * run;; ++at.request) {
                q = chunk_request(p, at.request, false);
                const long long here = unit_heads * chunk_work(q.length, q.n, unit_tokens, chunk_blocks(q.n, unit_tokens));
                if (x < here) break;
                x -= here;
            }
            int block = 0, above = chunk_blocks(q.n, unit_tokens);
            while (above - block > 1) {
                const int middle = (block + above) >> 1;
                if (unit_heads * chunk_work(q.length, q.n, unit_tokens, middle) <= x) block = middle; else above = middle;
            }
            at.block = block;
            if (block > 0) x -= unit_heads * chunk_work(q.length, q.n, unit_tokens, block);
            const int seen = chunk_seen(q.length, q.n, unit_tokens, block), tiles = tiles_of(seen);
            const long long work = (long long)seen + kChunkUnitCost;
            for (above = unit_heads; above - at.head > 1;) {
                const int middle = (at.head + above) >> 1;
                if (middle * work <= x) at.head = middle; else above = middle;
            }
            x -= at.head * work;
            const int tile = (int)min((x + kTile / 2) / kTile, (long long)tiles);
            if (!first && (whole ? 2 * x >= work : tile >= tiles)) next_unit(at, q);  // the first unit is somebody's, if it has no tile
            else at.tile = whole ? 0 : tile;
            return at;
        };
        const int box_rows = min(1 << p.page_shift, kTile), boxes = kTile / box_rows, group = p.q_heads / p.kv_heads;
        int item = 0, count = 0;  // tiles of keys and values so far, units so far
        bool alive = true;
        ChunkPlace at = {p.requests, 0, 0, 0}, stop = at;
        if (blockIdx.x < ctas) {
            // The cuts in front and behind, by two lanes at once.
            const long long cta = blockIdx.x + (lane == 1);
            const ChunkPlace own = cut_at(share * cta + min(cta, rest), now);
            auto of = [&](int v, int from) { return __shfl_sync(0xFFFFFFFFu, v, from); };
            __syncwarp();
            at = {of(own.request, 0), of(own.block, 0), of(own.head, 0), of(own.tile, 0)};
            stop = {of(own.request, 1), of(own.block, 1), of(own.head, 1), of(own.tile, 1)};
            now = {of(now.first, 0), of(now.n, 0), of(now.length, 0)};
        }
        ChunkCut cut = {0, 0, 0, 0, 0, 0};
        auto describe = [&] {  // the next unit
            ChunkUnit u = {};
            u.tiles = -1;
            if (at.request >= p.requests || (same_unit(at, stop) && at.tile == stop.tile)) return u;
            const ChunkRequest q = now;
            const int head = p.parts == 1 ? at.head : at.head / p.parts, part = at.head - head * p.parts, token = at.block * unit_tokens;
            u.request = at.request;
            u.kv_head = head;
            u.head0 = u.kv_head * group + part * p.part_heads;
            u.heads = min(p.part_heads, group - part * p.part_heads);
            u.row0 = q.first + token;
            u.tokens = min(unit_tokens, q.n - token);
            u.position0 = q.length - q.n + token;
            const int seen = max(0, u.position0 + u.tokens), tiles = tiles_of(seen), to = same_unit(at, stop) ? stop.tile : tiles;
            u.first_tile = at.tile;
            u.tiles = to - at.tile;
            u.end = min(seen, to * kTile);
            u.slot = at.tile > 0 ? 0 : to < tiles ? 1 : -1;
            if (at.tile > 0) {
                cut.continues = 1;
                cut.through = to < tiles;
            } else if (to < tiles) {
                cut.row0 = u.row0;
                cut.tokens = u.tokens;
                cut.head0 = u.head0;
                cut.heads = u.heads;
            }
            if (same_unit(at, stop)) at = stop;
            else next_unit(at, now);
            return u;
        };
        // The page that this lane's box of a tile lies in.
        auto page_of = [&](const ChunkUnit& u, int tile) {
            const int token = (u.first_tile + tile) * kTile + lane * box_rows;
            return tile < u.tiles && lane < boxes && token < u.end ? p.tables[u.request * p.table_stride + (token >> p.page_shift)] : 0;
        };
        auto load = [&](const ChunkUnit& u, int tile, int id, bool values) {
            const int token = (u.first_tile + tile) * kTile + lane * box_rows;
            const bool wanted = lane < boxes && token < u.end, inside = (unsigned int)id < (unsigned int)p.page_count;
            const unsigned int wants = __ballot_sync(0xFFFFFFFFu, wanted);
            unsigned int bad = __ballot_sync(0xFFFFFFFFu, wanted && !inside);
            if (bad) {
                if (wanted && !inside && !values) record_index(kPageOutside, u.request, (unsigned int)id);
                unsigned int spread = 0;
                for (int i = 0; i < kTile / 8; ++i) spread |= (bad >> (8 * i / box_rows) & 1u) << i;
                bad = spread;
            }
            const int slot = item % kSlots, round = item / kSlots;
            if (round > 0 && !ptx::mbar_wait_spin(&s.empty[slot], (round - 1) & 1, abort_flag, kChunkWait + 1)) {
                alive = false;
                return;
            }
            if (lane == 0) {
                if (!values) s.bad_rows[(item >> 1) & 7] = bad;
                ptx::mbar_expect_tx(&s.full[slot], __popc(wants) * box_rows * kD * 2);
            }
            __syncwarp();
            if (wanted) {
                const int place = values ? (inside ? id * p.value_page + u.kv_head * p.value_head : p.value_none) : inside ? id * p.key_page + u.kv_head * p.key_head : p.key_none;
                ptx::tma_load_5d(ring + slot * Shape::kSlotBytes + lane * box_rows * (kD * 2), values ? &p.value_map : &p.key_map, 0, 0, 0,
                                 (token & ((1 << p.page_shift) - 1)) >> 3, place, &s.full[slot]);
            }
            ++item;
        };
        ChunkUnit u = describe();
        int id = page_of(u, 0);
        for (; alive; ++count) {
            // The first keys and values are asked for before the unit in front is done with the queries' place.
            // (The first unit's come behind its queries: nobody is waited for.)
            auto start = [&] {
                const int here = id;
                id = page_of(u, 1);
                load(u, 0, here, false);
                if (alive) load(u, 0, here, true);
            };
            if (count > 0 && u.tiles > 0) start();
            if (!alive) break;
            if (count > 0 && !ptx::mbar_wait_spin(&s.q_empty, (count - 1) & 1, abort_flag, kChunkWait)) break;
            if (lane == 0) s.unit = u;
            const int groups_here = u.tokens > p.tile_tokens ? kGroups : 1;
            if (lane == 0) {
                if (u.tiles > 0) ptx::mbar_expect_tx(&s.q_full, groups_here * kChunks * 128 * p.part_heads * p.tile_tokens);
                else ptx::mbar_arrive(&s.q_full);
            }
            __syncwarp();
            if (u.tiles < 0) break;
            if (u.tiles > 0 && lane < groups_here * kChunks) {
                const int g = lane / kChunks, c = lane - g * kChunks;
                ptx::tma_load_3d(q_tiles + g * Shape::kQBytes + c * (kChunkRows * 128), &p.q_map, c * 64, u.head0, u.row0 + g * p.tile_tokens, &s.q_full);
            }
            if (count == 0 && u.tiles > 0) start();
            ChunkUnit next = {};
            int next_id = 0;
            for (int tile = 1; tile < max(2, u.tiles) && alive; ++tile) {
                if (tile < u.tiles) {
                    const int here = id;
                    id = page_of(u, tile + 1);
                    load(u, tile, here, false);
                    if (alive) load(u, tile, here, true);
                }
                if (tile == 1) {  // what the ring has room for is on its way
                    next = describe();
                    next_id = page_of(next, 0);
                }
            }
            u = next;
            id = next_id;
        }
        if (p.cuts && lane == 0) p.cuts[blockIdx.x] = cut;
    } else if (warp >= kIssuer) {
        // ---- the products of query tile g, by one thread -----------------------------------------------------------------
        // A thread for each: the tensor cores take but a few products ahead, and what a thread does between two steps would leave them
        // idle.  They take turns, so that the two warpgroups are half a step apart: one makes exponentials while the other looks for its
        // maximum.
        constexpr uint32_t kScores = ptx::umma_idesc_half(kChunkRows, kChunkStep, kHalf, false), kResults = ptx::umma_idesc_half(kChunkRows, kD, kHalf, true);
        const int g = warp - kIssuer;
        const uint32_t ring_base = ptx::smem_u32(ring), s_columns = tmem + g * 128, o_columns = tmem + Shape::kOColumn + g * kD;
        const uint64_t queries = ptx::smem_desc_k_major_sw128(ptx::smem_u32(q_tiles) + g * Shape::kQBytes);
        if (ptx::elect_one()) {
            int item = 0, fixed = 0;
            uint32_t p_phase = 0;  // a bit for either place
            uint32_t turns = g == 0 ? 1 : 0;  // the parity to wait for: the first turn is the first one's
            bool alive = true;
            for (int count = 0; alive; ++count) {
                if (!ptx::mbar_wait(&s.q_full, count & 1, abort_flag, kChunkWait + 2)) break;
                const int unit_tiles = s.unit.tiles, position0 = s.unit.position0, first_tile = s.unit.first_tile;
                const int steps = (s.unit.end - first_tile * kTile + kChunkStep - 1) / kChunkStep;
                const bool works = g * p.tile_tokens < s.unit.tokens, both = kGroups == 2 && p.tile_tokens < s.unit.tokens;
                if (unit_tiles < 0) break;
                if (unit_tiles == 0) {
                    ptx::mbar_arrive(&s.q_empty);
                    continue;
                }
                const int fix_from = max(0, min(unit_tiles - 1, max(0, position0 + 1) / kTile - first_tile));
                // Every phase of the ring's barriers is waited for here, in order: whoever looked at some of them only could take an
                // older phase for the one it wants.  So the values are handed on to be looked at, while the weights are made.
                auto arrived = [&](int it) { return ptx::mbar_wait_spin(&s.full[it % kSlots], it / kSlots & 1, abort_flag, kChunkWait + 3); };
                auto scores = [&](int step) {
                    const int key_item = item + 2 * (step / Shape::kSteps), part = step % Shape::kSteps;
                    if (works) {
                        const uint64_t keys = ptx::smem_desc_grouped_sw128(ring_base + key_item % kSlots * Shape::kSlotBytes + part * (kChunkStep * kD * 2), kChunks);
#pragma unroll
                        for (int k = 0; k < kD / 16; ++k)
                            ptx::umma_ss(s_columns + (step & 1) * kChunkStep, queries + (k >> 2) * (kChunkRows * 128 >> 4) + (k & 3) * 2,
                                         keys + (k >> 2) * (1024 >> 4) + (k & 3) * 2, kScores, k > 0);
                        ptx::umma_commit(&s.s_full[g][step & 1]);
                    }
                    if (part == Shape::kSteps - 1 || step == steps - 1) ptx::umma_commit(&s.empty[key_item % kSlots]);
                    if (step == steps - 1) ptx::umma_commit(&s.q_empty);
                };
                // The scores of two steps are ahead of the weights.
                for (int step = 0; step < min(2, steps) && alive; ++step) {
                    if (step % Shape::kSteps == 0) alive = arrived(item + 2 * (step / Shape::kSteps));
                    ptx::tc_fence_after_sync();
                    if (alive) scores(step);
                }
                for (int step = 0; step < steps && alive; ++step) {
                    const int tile = step / Shape::kSteps, part = step % Shape::kSteps, value_item = item + 2 * tile + 1, ahead = step + 2;
                    if (part == 0) {
                        alive = arrived(value_item);
                        if (alive && tile >= fix_from) ptx::mbar_arrive(&s.to_fix);
                        if (alive && ahead < steps) alive = arrived(item + 2 * (ahead / Shape::kSteps));
                        if (alive && tile >= fix_from) alive = ptx::mbar_wait_spin(&s.fixed, fixed++ & 1, abort_flag, kChunkWait + 4);
                        if (!alive) break;
                    }
                    if (works) {
                        alive = ptx::mbar_wait_spin(&s.p_full[g][step & 1], p_phase >> (step & 1) & 1u, abort_flag, kChunkWait + 5);
                        if (!alive) break;
                        p_phase ^= 1u << (step & 1);
                        if (both) {
                            alive = ptx::mbar_wait_spin(&s.turn[g], turns, abort_flag, kChunkWait + 6);
                            if (!alive) break;
                            turns ^= 1u;
                        }
                        ptx::tc_fence_after_sync();
                        const uint64_t values = ptx::smem_desc_grouped_sw128(ring_base + value_item % kSlots * Shape::kSlotBytes + part * (kChunkStep * kD * 2), kChunks);
#pragma unroll
                        for (int k = 0; k < kChunkStep / 16; ++k)
                            ptx::umma_ts(o_columns, s_columns + (step & 1) * kChunkStep + k * 8, values + k * (16 * kD * 2 >> 4), kResults, step > 0 || k > 0);
                        ptx::umma_commit(&s.o_done[g][step & 1]);
                    }
                    if (part == Shape::kSteps - 1 || step == steps - 1) ptx::umma_commit(&s.empty[value_item % kSlots]);
                    if (ahead < steps) scores(ahead);
                    if (both) ptx::mbar_arrive(&s.turn[g ^ 1]);
                }
                item += 2 * unit_tiles;
            }
            // Whatever was committed has arrived before the CTA may end.
            ptx::umma_commit(&s.drained);
        }
        __syncwarp();
        ptx::mbar_wait(&s.drained, 0, abort_flag, kChunkWait + 8);
    } else if (warp == kFixer) {
        // ---- values that some rows of the unit do not see -------------------------------------------------------------
        constexpr int kUnits = kD / 8, kRowsAtOnce = 32 / kUnits;              // 16-byte units of a row
        const uint32_t exponent = kHalf ? 0x7C007C00u : 0x7F807F80u, carry = kHalf ? 0x04000400u : 0x00800080u;
        int fixed = 0, items = 0;
        for (int count = 0;; ++count) {
            if (!ptx::mbar_wait(&s.q_full, count & 1, abort_flag, kChunkWait + 9)) break;
            const ChunkUnit u = s.unit;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&s.q_empty);
            if (u.tiles < 0) break;
            const int buffer = count & (kChunkNotes - 1);
            bool noted = false, alive = true;
            if (lane == 0) s.noted[buffer] = 0;
            const int seen_by_all = max(0, u.position0 + 1), fix_from = max(0, min(u.tiles - 1, seen_by_all / kTile - u.first_tile));
            for (int tile = fix_from; tile < u.tiles; ++tile) {
                alive = ptx::mbar_wait_spin(&s.to_fix, fixed++ & 1, abort_flag, kChunkWait + 10);
                if (!alive) break;
                uint8_t* values = ring + (items + 2 * tile + 1) % kSlots * Shape::kSlotBytes;
                const int first = (u.first_tile + tile) * kTile, some = max(0, seen_by_all - first), none = min(kTile, u.end - first);
                // Where row r has its logical 16-byte unit `at`.
                auto place = [&](int r, int at) { return values + ((r >> 3) * kChunks + (at >> 3)) * 1024 + (r & 7) * 128 + (((at & 7) ^ (r & 7)) << 4); };
                bool strange = false;
#pragma unroll 4
                for (int r = some + lane / kUnits; r < none; r += kRowsAtOnce) {
                    const uint4 v = *reinterpret_cast<const uint4*>(place(r, lane % kUnits));
                    const uint32_t found = (((v.x & exponent) + carry) | ((v.y & exponent) + carry) | ((v.z & exponent) + carry) | ((v.w & exponent) + carry)) & 0x80008000u;
                    strange = strange || found;
                }
                for (int r = none + lane / kUnits; r < kTile; r += kRowsAtOnce) *reinterpret_cast<uint4*>(place(r, lane % kUnits)) = make_uint4(0u, 0u, 0u, 0u);
                if (__any_sync(0xFFFFFFFFu, strange)) {
                    if (!noted)
                        for (int d = lane; d < kD; d += 32) s.notes[buffer][d] = 0x3FFFFFFFu;
                    noted = true;
#pragma unroll 1
                    for (int d = lane; d < kD; d += 32) {
                        uint32_t note = s.notes[buffer][d];
#pragma unroll 1
                        for (int r = some; r < none; ++r) {
                            uint16_t* at = reinterpret_cast<uint16_t*>(place(r, d >> 3)) + (d & 7);
                            const uint32_t v = *at, infinite = kHalf ? 0x7C00u : 0x7F80u;
                            if ((v & infinite) != infinite) continue;
                            const uint32_t shift = (v & 0x7FFFu) != infinite ? 0 : v & 0x8000u ? 20 : 10, position = first + r - u.position0;
                            if ((note >> shift & 1023u) > position) note = (note & ~(1023u << shift)) | position << shift;
                            *at = 0;
                        }
                        s.notes[buffer][d] = note;
                    }
                    if (lane == 0) s.noted[buffer] = 1;
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&s.fixed);
            }
            if (!alive) break;
            if (u.tiles > 0) items += 2 * u.tiles;
        }
    } else {
        // ---- a row a thread: the softmax and the results ----------------------------------------------------------------
        const int g = warp >> 2, row = threadIdx.x & (kChunkRows - 1);
        const uint32_t lanes = (uint32_t)(warp & 3) * 32 << 16, s_columns = tmem + lanes + g * 128, o_columns = tmem + lanes + Shape::kOColumn + g * kD;
        const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
        // (A factor of 0 would make NaN of what is masked.)
        const float factor = p.scale != p.scale ? p.scale : fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-37f);
        const int tile_token = row / p.part_heads, tile_head = row - tile_token * p.part_heads;
        uint32_t s_phase = 0;  // a bit for either place; the products of a place go through the same phases
        int tiles_before = 0;
        bool alive = true;
        for (int count = 0; alive; ++count) {
            if (!ptx::mbar_wait(&s.q_full, count & 1, abort_flag, kChunkWait + 11)) break;
            const ChunkUnit u = s.unit;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&s.q_empty);
            if (u.tiles < 0) break;
            const int token = g * p.tile_tokens + tile_token;
            const bool real = tile_token < p.tile_tokens && token < u.tokens && tile_head < u.heads;
            const int position = real ? u.position0 + token : 0x7FFFFFFF;  // a row of nobody needs no mask
            const bool works = __any_sync(0xFFFFFFFFu, real);
            float top = -INFINITY, sum = 0.0f;
            const int steps = g * p.tile_tokens < u.tokens ? (u.end - u.first_tile * kTile + kChunkStep - 1) / kChunkStep : 0;
            float x[kChunkStep];
            auto arrived = [&](int step) {
                const int place = step & 1;
                const bool here = ptx::mbar_wait_spin(&s.s_full[g][place], s_phase >> place & 1u, abort_flag, kChunkWait + 12);
                s_phase ^= 1u << place;
                ptx::tc_fence_after_sync();
                __syncwarp();
                return here;
            };
            // Scores are masked, and the row's maximum, with what there is of its results, moves where they ask for it.
            auto take = [&](int step) {
                float correction = 1.0f;
                if (works) {
#pragma unroll
                    for (int c = 0; c < kChunkStep; c += 32) ptx::tc_wait_ld32(x + c);
                    const int last = position - (u.first_tile * kTile + step * kChunkStep);  // columns behind it are not seen
                    const unsigned int bad = s.bad_rows[(tiles_before + step / Shape::kSteps) & 7] >> (step % Shape::kSteps * (kChunkStep / 8));
                    if (__any_sync(0xFFFFFFFFu, last < kChunkStep - 1) || bad || sign < 0.0f) {
#pragma unroll
                        for (int c = 0; c < kChunkStep; ++c) x[c] = c <= last && !(bad >> (c >> 3) & 1u) ? x[c] * sign : -INFINITY;
                    }
                    const float highest = fmaxf(most_of(x), most_of(x + 32)) * factor;
                    if (highest > top + (kPagedHeadroom + kPagedLift<kHalf>)) {
                        const float now = highest - kPagedLift<kHalf>;
                        if (top != -INFINITY) correction = power_of_two(top - now);
                        top = now;
                        sum *= correction;
                    }
                }
                if (__any_sync(0xFFFFFFFFu, correction != 1.0f)) {  // never in the first step
                    // The results of the step before.  (A wait must be one phase behind at most and not ahead.  The scores of this step were
                    // taken behind the results of the one before the last, and a place's next product waits for this step.)
                    const int before = (step & 1) ^ 1;
                    alive = ptx::mbar_wait_spin(&s.o_done[g][before], s_phase >> before & 1u ^ 1u, abort_flag, kChunkWait + 14);
                    ptx::tc_fence_after_sync();
                    __syncwarp();
#pragma unroll 1
                    for (int c = 0; c < kD; c += 16) {
                        uint32_t o[16];
                        ptx::tmem_ld16(o_columns + c, o);
                        ptx::tc_wait_ld16(o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * correction);
                        ptx::tmem_st16(o_columns + c, o);
                    }
                }
            };
            if (steps > 0) {
                alive = arrived(0);
                if (alive && works) {
#pragma unroll
                    for (int c = 0; c < kChunkStep; c += 32) ptx::tmem_ld32(s_columns + c, x + c);
                }
                if (alive) take(0);
            }
            for (int step = 0; step < steps && alive; ++step) {
                const uint32_t columns = s_columns + (step & 1) * kChunkStep, other_columns = s_columns + ((step & 1) ^ 1) * kChunkStep;
                const bool more = step + 1 < steps;
                bool early = false;  // the next step's scores are there already
                if (works) {  // (the weights of rows that nobody has may be anything)
                    const float2 against = make_float2(top == -INFINITY ? 0.0f : -top, top == -INFINITY ? 0.0f : -top), factors = make_float2(factor, factor);
                    float2 sums[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                    for (int c = 0; c < kChunkStep; c += 32) {
                        uint32_t packed[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 e = ptx::fma_f32x2(make_float2(x[c + i], x[c + i + 1]), factors, against);
                            const float2 weights = make_float2(power_of_two(e.x), power_of_two(e.y));
                            sums[i / 2 & 1] = add_f32x2(sums[i / 2 & 1], weights);
                            packed[i / 2] = rounded_pair<kHalf>(weights.x, weights.y);
                        }
                        ptx::tmem_st16(columns + c / 2, packed);
                        // The next step's scores take the place of those that are done with, half by half, if they are there.
                        if (more && c == 0) {
                            const int other = (step & 1) ^ 1;
                            early = __all_sync(0xFFFFFFFFu, ptx::mbar_test(&s.s_full[g][other], s_phase >> other & 1u));
                            ptx::tc_fence_after_sync();
                        }
                        if (early) ptx::tmem_ld32(other_columns + c, x + c);
                    }
                    sum += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
                }
                ptx::tc_wait_st();
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&s.p_full[g][step & 1]);
                if (!more) break;
                if (early) {
                    s_phase ^= 1u << ((step & 1) ^ 1);
                } else {
                    alive = arrived(step + 1);
                    if (!alive) break;
                    if (works) {
#pragma unroll
                        for (int c = 0; c < kChunkStep; c += 32) ptx::tmem_ld32(other_columns + c, x + c);
                    }
                }
                take(step + 1);
            }
            if (!alive) break;
            if (steps > 0) {
                const int place = steps - 1 & 1;
                alive = ptx::mbar_wait_spin(&s.o_done[g][place], s_phase >> place & 1u ^ 1u, abort_flag, kChunkWait + 13);
                if (!alive) break;
                ptx::tc_fence_after_sync();
                __syncwarp();
            }
            tiles_before += u.tiles;
            const int buffer = count & (kChunkNotes - 1);
            const bool notes = steps > 0 && s.noted[buffer] != 0;
            const long long at = (long long)(u.row0 + token) * p.q_heads + u.head0 + tile_head;
            const bool whole = u.slot < 0;
            const long long place = (blockIdx.x * 2ll + u.slot) * Shape::kSlotRows + threadIdx.x;
            const float share = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
            if (g * p.tile_tokens >= u.tokens) continue;
#pragma unroll 1
            for (int c = 0; c < kD; c += 32) {
                float o[32];
                if (steps > 0) {
                    ptx::tmem_ld32(o_columns + c, o);
                    ptx::tc_wait_ld32(o);
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = sum == 0.0f ? 0.0f : o[i] * share;
                if (notes && sum != 0.0f) {
                    const uint32_t own = position - u.position0;
#pragma unroll 1
                    for (int i = 0; i < 32; ++i) {
                        const uint32_t note = s.notes[buffer][c + i];
                        const bool nan = (note & 1023u) <= own, up = (note >> 10 & 1023u) <= own, down = (note >> 20) <= own;
                        if (!(nan || up || down)) continue;
                        const float value = nan || (up && down) ? NAN : up ? INFINITY : -INFINITY;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (j == i) o[j] = o[j] + value;
                    }
                }
                if (real && whole) {
#pragma unroll
                    for (int i = 0; i < 32; i += 16) {
                        uint32_t packed[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) packed[j] = rounded_pair<kHalf>(o[i + 2 * j], o[i + 2 * j + 1]);
                        ptx::st_global_32(p.out + at * kD + c + i, packed);
                    }
                } else if (real) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t words[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) words[j] = __float_as_uint(o[i + j]);
                        ptx::st_global_32(p.partial + place * kD + c + i, words);
                    }
                }
                __syncwarp();
            }
            if (real && !whole) p.stats[place] = make_float2(top, sum);
            ptx::tc_fence_before_sync();
        }
    }
    // Rows that no request has are zeros.
    if (warp == kFixer && !*abort_flag) {
        for (long long base = (long long)blockIdx.x * 32; base < p.rows; base += (long long)gridDim.x * 32) {
            const int r = (int)base + lane;
            bool nobody = false;
            if (r < p.rows) {
                int low = 0, high = p.requests + 1;  // the last start at or before r
                while (high - low > 1) {
                    const int middle = (low + high) >> 1;
                    if (p.starts[middle] <= r) low = middle; else high = middle;
                }
                nobody = p.requests == 0 || low >= p.requests || p.starts[low] > r || r >= p.starts[low] + chunk_request(p, low, false).n;
            }
            for (unsigned int rest = __ballot_sync(0xFFFFFFFFu, nobody); rest; rest &= rest - 1u) {
                uint4* to = reinterpret_cast<uint4*>(p.out + (base + __ffs(rest) - 1) * p.q_heads * kD);
                for (int i = lane; i < p.q_heads * (kD / 8); i += 32) to[i] = make_uint4(0u, 0u, 0u, 0u);
            }
        }
    }
    __syncwarp();
    if (*abort_flag) ptx::drain_copies();
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == kIssuer) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem, 512);
    }
}

// Joins the parts of the units that were cut, in their order.  The rows of the unit that CTA b began are dealt to the CTAs (b, y) up to
// (b', y), where b' begins the next one, at most 32 on; a row a warp, several of them or of their parts on their way at once.  Bound by
// its start and three loads that wait for one another: 17 tokens behind 100003 in 148 shares 98 us in all (108 when CTA b alone joined), 8
// behind 3000 26.6 (30.7); a serving batch whose units have two parts loses, 257 (253).
constexpr int kChunkJoinWarps = 8, kChunkJoinColumns = 4, kChunkJoinReach = 32;

template <int kD, bool kHalf>
__global__ void __launch_bounds__(kChunkJoinWarps * 32) paged_chunk_join_kernel(const __grid_constant__ PagedChunkParams p, int ctas) {
    using Shape = ChunkShape<kD>;
    using Numbers = typename std::conditional<kD == 64, float2, float4>::type;
    constexpr int kEach = kD / 32, kLoads = kEach * 4 / (int)sizeof(Numbers);  // numbers of a row that a lane has
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, x = blockIdx.x;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const unsigned int began = __ballot_sync(0xFFFFFFFFu, lane <= x && p.cuts[x - lane].tokens > 0);
    if (began == 0) return;
    const int b = x - (__ffs(began) - 1);
    const ChunkCut cut = p.cuts[b];
    // Part 0 is that CTA's second slot, part i the first slot of the i-th CTA behind it.
    int parts = 2, helpers = 0;
    for (bool more = true; more;) {
        const int cta = b + parts - 1 + lane;
        const bool there = cta < ctas;
        const unsigned int ends = __ballot_sync(0xFFFFFFFFu, !there || !p.cuts[cta].through);
        if (helpers == 0) {
            const unsigned int begins = __ballot_sync(0xFFFFFFFFu, !there || p.cuts[cta].tokens > 0);
            helpers = begins ? __ffs(begins) : kChunkJoinReach;
        }
        more = ends == 0;
        parts += more ? 32 : __ffs(ends) - 1;
    }
    parts = min(parts, ctas - b);
    if (x - b >= helpers) return;
    const int workers = helpers * kChunkJoinColumns * kChunkJoinWarps;
    auto join = [&](int first, auto rows_tag, auto parts_tag) {
        constexpr int kRows = decltype(rows_tag)::value, kParts = decltype(parts_tag)::value;
        int slot_row[kRows];
        long long to[kRows];  // row and head of the result, or -1
        float top[kRows], total[kRows], value[kRows][kEach];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            slot_row[k] = first + k * workers;
            const int g = slot_row[k] / kChunkRows, in_tile = slot_row[k] - g * kChunkRows, tile_token = in_tile / p.part_heads, head = in_tile - tile_token * p.part_heads;
            const int token = g * p.tile_tokens + tile_token;
            const bool real = slot_row[k] < Shape::kSlotRows && tile_token < p.tile_tokens && token < cut.tokens && head < cut.heads;
            to[k] = real ? (long long)(cut.row0 + token) * p.q_heads + cut.head0 + head : -1;
            top[k] = -INFINITY;
            total[k] = 0.0f;
#pragma unroll
            for (int e = 0; e < kEach; ++e) value[k][e] = 0.0f;
        }
        for (int part = 0; part < parts; part += kParts) {
            float2 own[kParts][kRows];
            Numbers numbers[kParts][kRows][kLoads];
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                const long long slot = ((long long)(b + part + i) * 2 + (part + i == 0)) * Shape::kSlotRows;
#pragma unroll
                for (int k = 0; k < kRows; ++k) {
                    own[i][k] = make_float2(-INFINITY, 0.0f);
                    if (to[k] < 0 || part + i >= parts) continue;
                    own[i][k] = p.stats[slot + slot_row[k]];
#pragma unroll
                    for (int l = 0; l < kLoads; ++l) numbers[i][k][l] = reinterpret_cast<const Numbers*>(p.partial + (slot + slot_row[k]) * kD)[l * 32 + lane];
                }
            }
#pragma unroll
            for (int i = 0; i < kParts; ++i)
#pragma unroll
                for (int k = 0; k < kRows; ++k) {
                    if (own[i][k].x == -INFINITY) continue;  // nothing in this part
                    const float now = fmaxf(top[k], own[i][k].x), before = power_of_two(top[k] - now), factor = power_of_two(own[i][k].x - now);
                    top[k] = now;
                    total[k] = fmaf(total[k], before, own[i][k].y * factor);
                    const float* there = reinterpret_cast<const float*>(&numbers[i][k]);
#pragma unroll
                    for (int e = 0; e < kEach; ++e) value[k][e] = fmaf(value[k][e], before, there[e] * factor);
                }
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            if (to[k] < 0) continue;
            constexpr int kWords = (int)sizeof(Numbers) / 8;  // of the result, that lie side by side
#pragma unroll
            for (int l = 0; l < kLoads; ++l) {
                uint32_t words[kWords];
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    const int e = (l * kWords + w) * 2;
                    words[w] = total[k] == 0.0f ? 0u : rounded_pair<kHalf>(value[k][e] / total[k], value[k][e + 1] / total[k]);
                }
                uint32_t* out = reinterpret_cast<uint32_t*>(p.out + to[k] * kD) + (l * 32 + lane) * kWords;
                if constexpr (kWords == 2) *reinterpret_cast<uint2*>(out) = make_uint2(words[0], words[1]);
                else out[0] = words[0];
            }
        }
    };
    constexpr int kAtOnce = kD == 256 ? 4 : 8;
    int row = ((x - b) * kChunkJoinColumns + (int)blockIdx.y) * kChunkJoinWarps + warp;
    auto all = [&](auto rows_tag, auto parts_tag) {
        for (; row < Shape::kSlotRows; row += workers * decltype(rows_tag)::value) join(row, rows_tag, parts_tag);
    };
    if (parts == 2) all(std::integral_constant<int, kAtOnce / 2>{}, std::integral_constant<int, 2>{});
    else if (parts <= 4) all(std::integral_constant<int, kAtOnce / 4>{}, std::integral_constant<int, 4>{});
    else all(std::integral_constant<int, 1>{}, std::integral_constant<int, kAtOnce>{});
}

// CTAs of a call: one per SM, or as many as the work can be shared by at most.
inline int chunk_ctas(int rows, int requests, int kv_heads, int group, int head_dim, long long capacity, int sm_count) {
    const int parts = (group + kChunkRows - 1) / kChunkRows, part_heads = (group + parts - 1) / parts;
    const int unit_tokens = (head_dim == 256 ? 1 : 2) * (kChunkRows / part_heads);
    const long long units = ((long long)rows / unit_tokens + (requests < rows ? requests : rows)) * kv_heads * parts;
    const long long most = units > sm_count ? sm_count : units * (capacity + kChunkUnitCost) / kChunkShare;
    return most < 1 ? 1 : most < sm_count ? (int)most : sm_count;
}
// Where no unit can be long enough for a cut to pay, nothing is left to be joined.
inline size_t chunk_partial_bytes(int head_dim, int ctas, long long capacity, bool whole) {
    if (whole || ctas <= 1 || capacity + kChunkUnitCost - kChunkShare <= kChunkCutGain) return 0;
    return (size_t)ctas * (2 * (head_dim == 256 ? 1 : 2) * kChunkRows * (head_dim + 2) * sizeof(float) + sizeof(ChunkCut));
}

// A map of 16-bit numbers; strides in bytes, of all dimensions but the first.
inline bool chunk_map(CUtensorMap& map, bool half, const void* base, int rank, const cuuint64_t* sizes, const cuuint64_t* strides, const cuuint32_t* box) {
    const EncodeTiledFn encode = encode_tiled_fn();
    const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
    return encode && encode(&map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), sizes, strides,
                            box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kD, bool kHalf>
inline int launch_paged_chunk(PagedChunkParams& params, const void* q, const void* keys, const PageStrides& key_strides, const void* values,
                              const PageStrides& value_strides, void* workspace, int ctas, cudaStream_t stream) {
    using Shape = ChunkShape<kD>;
    const int group = params.q_heads / params.kv_heads, page = 1 << params.page_shift;
    const size_t slots = (size_t)ctas * 2 * Shape::kSlotRows;
    params.whole = workspace == nullptr;
    params.partial = static_cast<float*>(workspace);
    params.stats = workspace ? reinterpret_cast<float2*>(params.partial + slots * kD) : nullptr;
    params.cuts = workspace ? reinterpret_cast<ChunkCut*>(params.stats + slots) : nullptr;
    params.parts = (group + kChunkRows - 1) / kChunkRows;
    params.part_heads = (group + params.parts - 1) / params.parts;
    params.tile_tokens = kChunkRows / params.part_heads;
    const cuuint64_t q_sizes[3] = {kD, (cuuint64_t)params.q_heads, (cuuint64_t)params.rows}, q_strides[2] = {kD * 2, (cuuint64_t)params.q_heads * kD * 2};
    const cuuint32_t q_box[3] = {64, (cuuint32_t)params.part_heads, (cuuint32_t)params.tile_tokens};
    if (!chunk_map(params.q_map, kHalf, q, 3, q_sizes, q_strides, q_box)) return MT_ERR_LAUNCH;
    const cuuint32_t box[5] = {64, 8, kD / 64, (cuuint32_t)(page < Shape::kTile ? page : Shape::kTile) / 8, 1};
    for (int which = 0; which < 2; ++which) {
        // A map has five dimensions at most: heads and pages share one, in steps of what divides the strides of both.  (Dimensions of one
        // element come with a stride of 0.)
        const PageStrides& given = which ? value_strides : key_strides;
        const long long token = given.token ? given.token : kD;
        long long unit = given.head, rest = given.page;
        while (rest) {
            const long long next = unit % rest;
            unit = rest;
            rest = next;
        }
        if (unit == 0) unit = 8;
        const long long head = given.head / unit, page_step = given.page / unit, places = (params.kv_heads - 1) * head + (params.page_count - 1) * page_step + 1;
        if (places > 0x7FFFFFFF) return MT_ERR_SHAPE;
        (which ? params.value_head : params.key_head) = (int)head;
        (which ? params.value_page : params.key_page) = (int)page_step;
        (which ? params.value_none : params.key_none) = (int)places;
        const cuuint64_t sizes[5] = {64, 8, kD / 64, (cuuint64_t)page / 8, (cuuint64_t)places};
        const cuuint64_t strides[4] = {(cuuint64_t)token * 2, 128, (cuuint64_t)token * 16, (cuuint64_t)unit * 2};
        if (!chunk_map(which ? params.value_map : params.key_map, kHalf, which ? values : keys, 5, sizes, strides, box)) return MT_ERR_LAUNCH;
    }
    static bool configured[64] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return MT_ERR_LAUNCH;
    if (device >= 64 || !configured[device]) {
        if (cudaFuncSetAttribute(paged_chunk_kernel<kD, kHalf>, cudaFuncAttributeMaxDynamicSharedMemorySize, chunk_smem<kD>()) != cudaSuccess) return MT_ERR_LAUNCH;
        if (device < 64) configured[device] = true;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(ctas, 1, 1);
    config.blockDim = dim3(Shape::kThreads, 1, 1);
    config.dynamicSmemBytes = chunk_smem<kD>();
    config.stream = stream;
    cudaLaunchAttribute attrs[1];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, paged_chunk_kernel<kD, kHalf>, params) != cudaSuccess) return MT_ERR_LAUNCH;
    if (params.cuts) {
        config.gridDim = dim3(ctas, kChunkJoinColumns, 1);
        config.blockDim = dim3(kChunkJoinWarps * 32, 1, 1);
        config.dynamicSmemBytes = 0;
        if (cudaLaunchKernelEx(&config, paged_chunk_join_kernel<kD, kHalf>, params, ctas) != cudaSuccess) return MT_ERR_LAUNCH;
    }
    return MT_OK;
}

}  // namespace mt
