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
// A warpgroup per query tile, a row a thread, turns S into P: while it works on one tile the tensor cores have the other's.  A row's
// maximum moves, and its O with it, only when a score passes it by more than 2^8.
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

#include "affine_umma.cuh"
#include "paged_attention.cuh"

namespace mt {

constexpr unsigned int kStartOutside = 0x306;  // paged_attention_chunk: word 1 = request, 2 = its first row
constexpr unsigned int kChunkWait = 0x9D0;     // a wait that gave up: + the role

constexpr int kChunkRows = 128;                // of a query tile
constexpr int kChunkRuns = 128;                // runs of requests whose units are counted
constexpr int kChunkMinTiles = 4;              // token tiles of a split
constexpr int kChunkUnitsWanted = 2;           // units an SM should have before long requests are not split
constexpr int kChunkNotes = 2;                 // units whose noted columns may be needed at once: the one begun and the one that ends

template <int kD>
struct ChunkShape {
    static constexpr int kGroups = kD == 256 ? 1 : 2;               // query tiles of a unit
    static constexpr int kTile = kD == 256 ? 64 : 128;              // tokens
    static constexpr int kSlots = kD == 256 ? 4 : kD == 128 ? 5 : 6;  // tiles of keys or values
    static constexpr int kQBytes = kChunkRows * kD * 2, kSlotBytes = kTile * kD * 2;
    static constexpr int kSoftmaxWarps = 4 * kGroups, kWarps = kSoftmaxWarps + 4, kThreads = 32 * kWarps;
    static constexpr int kOColumn = 256;                            // in tensor memory; the scores of tile g at g * kTile
    static constexpr int kTiles = kGroups * kQBytes + kSlots * kSlotBytes;
    static constexpr int kSmem = kTiles + kChunkNotes * kD * 4 + (kChunkRuns + 1) * 4 + 500;
    static_assert(kSmem <= 232448 && kOColumn + kGroups * kD <= 512 && kGroups * kTile <= kOColumn && kSlots <= 6);
};

struct PagedChunkParams {
    CUtensorMap q_map;                 // (D, Hq, rows): boxes of 64 x heads of a part x tokens of a tile
    CUtensorMap key_map, value_map;    // (D, page size, KV heads, pages): boxes of 64 x up to a tile's rows of a page
    const int* tables;                 // [requests, width], rows `table_stride` apart
    const int* lengths;                // [requests]
    const int* starts;                 // [requests + 1]
    uint16_t* out;                     // [rows, Hq, D]
    float* partial;                    // [rows * Hq, split_limit, D]
    float2* stats;                     // [rows * Hq, split_limit]: maximum (log2) and sum
    long long table_stride;
    int width, rows, requests, q_heads, kv_heads, page_shift, page_count, split_limit;
    int part_heads, parts;             // query heads of a KV head that share a tile; tiles that takes
    int tile_tokens;                   // of a query tile
    float scale;
};

// What a unit is, for all warps of a CTA.
struct ChunkUnit {
    int request, kv_head, head0;       // head0: the first query head
    int heads;                         // of the tile
    int row0, tokens;                  // rows of the query: the first, how many (both tiles)
    int position0;                     // of the first row, may be negative
    int first_tile, tiles;             // token tiles; -1: there are no more units
    int end;                           // tokens from here on are seen by no row or belong to the next split
    int split, splits;
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

template <int kD>
__device__ __forceinline__ int chunk_splits(const PagedChunkParams& p, int length) {
    if (p.split_limit == 1) return 1;
    const int tiles = (int)(((long long)length + ChunkShape<kD>::kTile - 1) / ChunkShape<kD>::kTile);
    return max(1, min(p.split_limit, tiles / kChunkMinTiles));
}
template <int kD>
__device__ __forceinline__ int chunk_units(const PagedChunkParams& p, const ChunkRequest& q) {
    const int unit_tokens = ChunkShape<kD>::kGroups * p.tile_tokens;
    return (q.n + unit_tokens - 1) / unit_tokens * chunk_splits<kD>(p, q.length) * p.kv_heads * p.parts;
}

namespace ptx {

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const void* tensor_map, int c0, int c1, int c2, int c3, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(smem_u32(smem_dst)), "l"(tensor_map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
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

// Shared-memory matrix descriptor of an operand whose rows run along M or N (here: values, rows of the head dimension): 128-byte
// swizzle, blocks of 64 columns `column_bytes` apart, groups of 8 rows (of K) 1024 B apart.
__device__ __forceinline__ uint64_t smem_desc_mn_major_sw128(uint32_t smem_addr, uint32_t column_bytes) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)(column_bytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
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
    int unit_start[kChunkRuns + 1];
    uint64_t q_full, q_empty, drained;
    uint64_t full[6], empty[6];        // of the ring
    uint64_t to_fix, fixed;            // tiles of values that some rows do not see, one after the other
    uint64_t s_full[2], p_full[2], o_full[2];
    ChunkUnit unit;
    unsigned int bad_rows[8];          // of a token tile: groups of eight tokens whose page lies outside the cache
    int noted[kChunkNotes][2];         // whether a unit has notes, by the two warps that make them
    uint32_t tmem;
    int abort;
};

template <int kD, bool kHalf>
__global__ void __launch_bounds__(ChunkShape<kD>::kThreads, 1) paged_chunk_kernel(const __grid_constant__ PagedChunkParams p) {
    using Shape = ChunkShape<kD>;
    using Shared = ChunkShared<kD>;
    static_assert(Shape::kTiles + sizeof(Shared) <= Shape::kSmem);
    constexpr int kTile = Shape::kTile, kGroups = Shape::kGroups, kSlots = Shape::kSlots, kChunks = kD / 64;
    extern __shared__ __align__(1024) uint8_t chunk_tiles[];
    uint8_t* q_tiles = chunk_tiles;
    uint8_t* ring = chunk_tiles + kGroups * Shape::kQBytes;
    Shared& s = *reinterpret_cast<Shared*>(chunk_tiles + Shape::kTiles);
    volatile int* abort_flag = &s.abort;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    constexpr int kLoader = Shape::kSoftmaxWarps, kIssuer = kLoader + 1, kFixer = kLoader + 2;

    if (threadIdx.x == 0) {
        ptx::mbar_init(&s.q_full, 1);
        ptx::mbar_init(&s.q_empty, 1 + Shape::kSoftmaxWarps + 2);  // the last product of keys; the warps that have read the unit
        ptx::mbar_init(&s.drained, 1);
        ptx::mbar_init(&s.to_fix, 1);
        ptx::mbar_init(&s.fixed, 2);
        for (int i = 0; i < kSlots; ++i) {
            ptx::mbar_init(&s.full[i], 1);
            ptx::mbar_init(&s.empty[i], 1);
        }
        for (int g = 0; g < kGroups; ++g) {
            ptx::mbar_init(&s.s_full[g], 1);
            ptx::mbar_init(&s.p_full[g], kChunkRows);
            ptx::mbar_init(&s.o_full[g], 1);
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
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();

    // Units in front of every run of requests.
    const int run = (p.requests + kChunkRuns - 1) / kChunkRuns;
    if (threadIdx.x < kChunkRuns) {
        int mine = 0;
        for (int r = threadIdx.x * run; r < min((int)(threadIdx.x + 1) * run, p.requests); ++r)
            mine += chunk_units<kD>(p, chunk_request(p, r, blockIdx.x == 0));
        s.unit_start[threadIdx.x + 1] = mine;
    }
    __syncthreads();
    if (warp == 0) {
        constexpr int kEach = kChunkRuns / 32;
        int own[kEach], sum = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) own[i] = sum += s.unit_start[lane * kEach + i + 1];
        int before = sum;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, before, offset);
            if (lane >= offset) before += other;
        }
        before -= sum;
#pragma unroll
        for (int i = 0; i < kEach; ++i) s.unit_start[lane * kEach + i + 1] = before + own[i];
        if (lane == 0) s.unit_start[0] = 0;
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = s.tmem;

    if (warp == kLoader) {
        // ---- units, queries, keys and values ------------------------------------------------------------------
        const int units = s.unit_start[kChunkRuns];
        const int box_rows = min(1 << p.page_shift, kTile), boxes = kTile / box_rows;
        int item = 0, count = 0;  // tiles of keys and values so far, units so far
        bool alive = true;
        for (int next = blockIdx.x; alive; next += gridDim.x, ++count) {
            ChunkUnit u = {};
            u.tiles = -1;
            if (next < units) {
                int low = 0, high = kChunkRuns;
                while (high - low > 1) {
                    const int middle = (low + high) >> 1;
                    if (s.unit_start[middle] <= next) low = middle; else high = middle;
                }
                int unit = next - s.unit_start[low];
                ChunkRequest q;
                for (u.request = low * run;; ++u.request) {
                    q = chunk_request(p, u.request, false);
                    const int here = chunk_units<kD>(p, q);
                    if (unit < here) break;
                    unit -= here;
                }
                // The last rows, which see most, come first.
                const int unit_tokens = kGroups * p.tile_tokens, blocks = (q.n + unit_tokens - 1) / unit_tokens;
                u.splits = chunk_splits<kD>(p, q.length);
                const int per_block = u.splits * p.kv_heads * p.parts, from_end = unit / per_block, rest = unit - from_end * per_block;
                const int head = rest / u.splits, part = head % p.parts, group = p.q_heads / p.kv_heads;
                const int token = (blocks - 1 - from_end) * unit_tokens;
                u.split = rest - head * u.splits;
                u.kv_head = head / p.parts;
                u.head0 = u.kv_head * group + part * p.part_heads;
                u.heads = min(p.part_heads, group - part * p.part_heads);
                u.row0 = q.first + token;
                u.tokens = min(unit_tokens, q.n - token);
                u.position0 = q.length - q.n + token;
                const int seen = max(0, u.position0 + u.tokens), all = (seen + kTile - 1) / kTile, per = (all + u.splits - 1) / u.splits;
                u.first_tile = min(all, u.split * per);
                u.tiles = min(all, u.first_tile + per) - u.first_tile;
                u.end = min(seen, (u.first_tile + u.tiles) * kTile);
            }
            if (count > 0 && !ptx::mbar_wait(&s.q_empty, (count - 1) & 1, abort_flag, kChunkWait)) break;
            if (lane == 0) s.unit = u;
            const int groups_here = u.tokens > p.tile_tokens ? kGroups : 1;
            if (lane == 0) {
                if (u.tiles > 0) ptx::mbar_expect_tx(&s.q_full, groups_here * kChunks * 128 * p.part_heads * p.tile_tokens);
                else ptx::mbar_arrive(&s.q_full);
            }
            __syncwarp();
            if (u.tiles < 0) break;
            if (u.tiles == 0) continue;
            if (lane < groups_here * kChunks) {
                const int g = lane / kChunks, c = lane - g * kChunks;
                ptx::tma_load_3d(q_tiles + g * Shape::kQBytes + c * (kChunkRows * 128), &p.q_map, c * 64, u.head0, u.row0 + g * p.tile_tokens, &s.q_full);
            }
            const int* table = p.tables + u.request * p.table_stride;
            auto page_of = [&](int tile) {
                const int token = (u.first_tile + tile) * kTile + lane * box_rows;
                return tile < u.tiles && lane < boxes && token < u.end ? table[token >> p.page_shift] : 0;
            };
            int id_next = page_of(0);
            for (int tile = 0; tile < u.tiles && alive; ++tile) {
                const int id = id_next, token = (u.first_tile + tile) * kTile + lane * box_rows;
                id_next = page_of(tile + 1);
                const bool wanted = lane < boxes && token < u.end, inside = (unsigned int)id < (unsigned int)p.page_count;
                if (wanted && !inside) record_index(kPageOutside, u.request, (unsigned int)id);
                const unsigned int wants = __ballot_sync(0xFFFFFFFFu, wanted);
                unsigned int bad = __ballot_sync(0xFFFFFFFFu, wanted && !inside);
                const uint32_t bytes = __popc(wants) * box_rows * 128 * kChunks;
                const int page = inside ? id : p.page_count, in_page = token & ((1 << p.page_shift) - 1);  // behind the last page: zeros
                if (bad) {
                    unsigned int spread = 0;
                    for (int i = 0; i < kTile / 8; ++i) spread |= (bad >> (8 * i / box_rows) & 1u) << i;
                    bad = spread;
                }
                for (int values = 0; values < 2; ++values, ++item) {
                    const int slot = item % kSlots, round = item / kSlots;
                    if (round > 0 && !ptx::mbar_wait(&s.empty[slot], (round - 1) & 1, abort_flag, kChunkWait + 1)) {
                        alive = false;
                        break;
                    }
                    if (lane == 0) {
                        if (!values) s.bad_rows[(item >> 1) & 7] = bad;
                        ptx::mbar_expect_tx(&s.full[slot], bytes);
                    }
                    __syncwarp();
                    if (wanted) {
                        uint8_t* to = ring + slot * Shape::kSlotBytes + lane * box_rows * 128;
#pragma unroll
                        for (int c = 0; c < kChunks; ++c)
                            ptx::tma_load_4d(to + c * (kTile * 128), values ? &p.value_map : &p.key_map, c * 64, in_page, u.kv_head, page, &s.full[slot]);
                    }
                }
            }
        }
    } else if (warp == kIssuer) {
        // ---- the products ---------------------------------------------------------------------------------------
        constexpr uint32_t kScores = ptx::umma_idesc_half(kChunkRows, kTile, kHalf, false), kResults = ptx::umma_idesc_half(kChunkRows, kD, kHalf, true);
        const uint32_t q_base = ptx::smem_u32(q_tiles), ring_base = ptx::smem_u32(ring);
        const bool leader = ptx::elect_one();
        uint32_t p_phase[2] = {0, 0};
        int item = 0, fixed = 0;
        for (int count = 0;; ++count) {
            if (!ptx::mbar_wait(&s.q_full, count & 1, abort_flag, kChunkWait + 2)) break;
            const int unit_tiles = s.unit.tiles, tokens = s.unit.tokens, position0 = s.unit.position0, first_tile = s.unit.first_tile;
            if (unit_tiles < 0) break;
            if (unit_tiles == 0) {
                __syncwarp();
                if (leader) ptx::mbar_arrive(&s.q_empty);
                continue;
            }
            const int groups_here = tokens > p.tile_tokens ? kGroups : 1;
            const int fix_from = max(0, min(unit_tiles - 1, max(0, position0 + 1) / kTile - first_tile));
            auto scores = [&](int g, uint32_t keys) {
                const uint64_t a = ptx::smem_desc_k_major_sw128(q_base + g * Shape::kQBytes), b = ptx::smem_desc_k_major_sw128(keys);
#pragma unroll
                for (int k = 0; k < kD / 16; ++k)
                    ptx::umma_ss(tmem + g * kTile, a + (k >> 2) * (kChunkRows * 128 >> 4) + (k & 3) * 2, b + (k >> 2) * (kTile * 128 >> 4) + (k & 3) * 2, kScores, k > 0);
                ptx::umma_commit(&s.s_full[g]);
            };
            bool alive = ptx::mbar_wait(&s.full[item % kSlots], item / kSlots & 1, abort_flag, kChunkWait + 3);
            if (!alive) break;
            ptx::tc_fence_after_sync();
            __syncwarp();
            if (leader) {
                for (int g = 0; g < groups_here; ++g) scores(g, ring_base + item % kSlots * Shape::kSlotBytes);
                if (unit_tiles == 1) ptx::umma_commit(&s.q_empty);
                ptx::umma_commit(&s.empty[item % kSlots]);
            }
            for (int tile = 0; tile < unit_tiles && alive; ++tile, item += 2) {
                const int value_item = item + 1, key_item = item + 2;
                const bool more = tile + 1 < unit_tiles;
                // Every phase of the ring's barriers is waited for here, in order: whoever looked at some of them only could take an
                // older phase for the one it wants.  So the values are handed on to be looked at, while the weights are made.
                alive = ptx::mbar_wait(&s.full[value_item % kSlots], value_item / kSlots & 1, abort_flag, kChunkWait + 5);
                if (alive && tile >= fix_from) {
                    __syncwarp();
                    if (leader) ptx::mbar_arrive(&s.to_fix);
                }
                if (alive && more) alive = ptx::mbar_wait(&s.full[key_item % kSlots], key_item / kSlots & 1, abort_flag, kChunkWait + 6);
                if (alive && tile >= fix_from) alive = ptx::mbar_wait(&s.fixed, fixed++ & 1, abort_flag, kChunkWait + 4);
                if (!alive) break;
                for (int g = 0; g < groups_here; ++g) {
                    alive = ptx::mbar_wait(&s.p_full[g], p_phase[g], abort_flag, kChunkWait + 7);
                    if (!alive) break;
                    p_phase[g] ^= 1;
                    ptx::tc_fence_after_sync();
                    __syncwarp();
                    if (leader) {
                        const uint64_t b = ptx::smem_desc_mn_major_sw128(ring_base + value_item % kSlots * Shape::kSlotBytes, kTile * 128);
#pragma unroll
                        for (int k = 0; k < kTile / 16; ++k)
                            ptx::umma_ts(tmem + Shape::kOColumn + g * kD, tmem + g * kTile + k * 8, b + k * (16 * 128 >> 4), kResults, tile > 0 || k > 0);
                        if (more) scores(g, ring_base + key_item % kSlots * Shape::kSlotBytes);
                        else ptx::umma_commit(&s.o_full[g]);
                    }
                }
                if (alive && leader) {
                    ptx::umma_commit(&s.empty[value_item % kSlots]);
                    if (more) ptx::umma_commit(&s.empty[key_item % kSlots]);
                    if (tile + 2 == unit_tiles) ptx::umma_commit(&s.q_empty);
                }
                __syncwarp();
            }
            if (!alive) break;
        }
        // Whatever was committed has arrived before the CTA may end.
        if (leader) ptx::umma_commit(&s.drained);
        __syncwarp();
        ptx::mbar_wait(&s.drained, 0, abort_flag, kChunkWait + 8);
    } else if (warp >= kFixer) {
        // ---- values that some rows of the unit do not see -------------------------------------------------------------
        const int half = warp - kFixer;                                        // of the head dimension
        constexpr int kUnits = kD / 16, kRowsAtOnce = 32 / kUnits;             // 16-byte units of a row's half
        const uint32_t exponent = kHalf ? 0x7C007C00u : 0x7F807F80u, carry = kHalf ? 0x04000400u : 0x00800080u;
        int item = 0, fixed = 0;
        for (int count = 0;; ++count) {
            if (!ptx::mbar_wait(&s.q_full, count & 1, abort_flag, kChunkWait + 9)) break;
            const ChunkUnit u = s.unit;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&s.q_empty);
            if (u.tiles < 0) break;
            const int buffer = count & (kChunkNotes - 1);
            bool noted = false, alive = true;
            if (lane == 0) s.noted[buffer][half] = 0;
            const int seen_by_all = max(0, u.position0 + 1), fix_from = max(0, min(u.tiles - 1, seen_by_all / kTile - u.first_tile));
            for (int tile = fix_from; tile < u.tiles; ++tile) {
                const int value_item = item + 2 * tile + 1, slot = value_item % kSlots;
                alive = ptx::mbar_wait(&s.to_fix, fixed++ & 1, abort_flag, kChunkWait + 10);
                if (!alive) break;
                uint8_t* values = ring + slot * Shape::kSlotBytes;
                const int first = (u.first_tile + tile) * kTile, some = max(0, seen_by_all - first), none = min(kTile, u.end - first);
                // Logical 16-byte unit of this lane, and where row r has it.
                const int unit = half * kUnits + lane % kUnits, row0 = lane / kUnits;
                auto place = [&](int r, int at) { return values + (at >> 3) * (kTile * 128) + r * 128 + (((at & 7) ^ (r & 7)) << 4); };
                bool strange = false;
                for (int r = some + row0; r < none; r += kRowsAtOnce) {
                    const uint4 v = *reinterpret_cast<const uint4*>(place(r, unit));
                    const uint32_t found = (((v.x & exponent) + carry) | ((v.y & exponent) + carry) | ((v.z & exponent) + carry) | ((v.w & exponent) + carry)) & 0x80008000u;
                    strange = strange || found;
                }
                for (int r = none + row0; r < kTile; r += kRowsAtOnce) *reinterpret_cast<uint4*>(place(r, unit)) = make_uint4(0u, 0u, 0u, 0u);
                if (__any_sync(0xFFFFFFFFu, strange)) {
                    if (!noted)
                        for (int d = half * (kD / 2) + lane; d < (half + 1) * (kD / 2); d += 32) s.notes[buffer][d] = 0x3FFFFFFFu;
                    noted = true;
                    __syncwarp();
                    for (int d = half * (kD / 2) + lane; d < (half + 1) * (kD / 2); d += 32) {
                        uint32_t note = s.notes[buffer][d];
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
                    if (lane == 0) s.noted[buffer][half] = 1;
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&s.fixed);
            }
            if (!alive) break;
            if (u.tiles > 0) item += 2 * u.tiles;
        }
    } else {
        // ---- a row a thread: the softmax and the results ----------------------------------------------------------------
        const int g = warp >> 2, row = threadIdx.x & (kChunkRows - 1);
        const uint32_t lanes = (uint32_t)(warp & 3) * 32 << 16, s_columns = tmem + lanes + g * kTile, o_columns = tmem + lanes + Shape::kOColumn + g * kD;
        const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
        // (A factor of 0 would make NaN of what is masked.)
        const float factor = p.scale != p.scale ? p.scale : fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-37f);
        const int tile_token = row / p.part_heads, tile_head = row - tile_token * p.part_heads;
        uint32_t s_phase = 0, o_phase = 0;
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
            const int tiles_here = g * p.tile_tokens < u.tokens ? u.tiles : 0;
            for (int tile = 0; tile < tiles_here; ++tile) {
                alive = ptx::mbar_wait(&s.s_full[g], s_phase, abort_flag, kChunkWait + 12);
                if (!alive) break;
                s_phase ^= 1;
                ptx::tc_fence_after_sync();
                __syncwarp();
                if (!works) {  // the weights of rows that nobody has may be anything
                    ptx::mbar_arrive(&s.p_full[g]);
                    continue;
                }
                float x[kTile];
#pragma unroll
                for (int c = 0; c < kTile; c += 32) ptx::tmem_ld32(s_columns + c, x + c);
#pragma unroll
                for (int c = 0; c < kTile; c += 32) ptx::tc_wait_ld32(x + c);
                if (sign < 0.0f)
#pragma unroll
                    for (int c = 0; c < kTile; ++c) x[c] = -x[c];
                const int last = position - (u.first_tile + tile) * kTile;  // columns behind it are not seen
                if (__any_sync(0xFFFFFFFFu, last < kTile - 1)) {
#pragma unroll
                    for (int c = 0; c < kTile; ++c) x[c] = c <= last ? x[c] : -INFINITY;
                }
                const unsigned int bad = s.bad_rows[(tiles_before + tile) & 7];
                if (bad) {
#pragma unroll
                    for (int c = 0; c < kTile; ++c) x[c] = bad >> (c >> 3) & 1u ? -INFINITY : x[c];
                }
                float most[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int c = 4; c < kTile; ++c) most[c & 3] = fmaxf(most[c & 3], x[c]);
                const float highest = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * factor;
                float correction = 1.0f;
                if (highest > top + (kPagedHeadroom + kPagedLift<kHalf>)) {
                    const float now = highest - kPagedLift<kHalf>;
                    if (top != -INFINITY) correction = power_of_two(top - now);
                    top = now;
                    sum *= correction;
                }
                if (__any_sync(0xFFFFFFFFu, correction != 1.0f)) {  // never in the first tile
#pragma unroll
                    for (int c = 0; c < kD; c += 32) {
                        float o[32];
                        ptx::tmem_ld32(o_columns + c, o);
                        ptx::tc_wait_ld32(o);
#pragma unroll
                        for (int i = 0; i < 32; i += 16) {
                            uint32_t scaled[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) scaled[j] = __float_as_uint(o[i + j] * correction);
                            ptx::tmem_st16(o_columns + c + i, scaled);
                        }
                    }
                }
                const float against = top == -INFINITY ? 0.0f : top;
                float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < kTile; c += 32) {
                    uint32_t packed[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float a = power_of_two(fmaf(x[c + i], factor, -against)), b = power_of_two(fmaf(x[c + i + 1], factor, -against));
                        sums[i & 2] += a;
                        sums[(i & 2) + 1] += b;
                        packed[i / 2] = pack_pair<kHalf>(a, b);
                    }
                    ptx::tmem_st16(s_columns + c / 2, packed);
                }
                sum += (sums[0] + sums[1]) + (sums[2] + sums[3]);
                ptx::tc_wait_st();
                ptx::tc_fence_before_sync();
                ptx::mbar_arrive(&s.p_full[g]);
            }
            if (!alive) break;
            if (tiles_here > 0) {
                alive = ptx::mbar_wait(&s.o_full[g], o_phase, abort_flag, kChunkWait + 13);
                if (!alive) break;
                o_phase ^= 1;
                ptx::tc_fence_after_sync();
                __syncwarp();
            }
            tiles_before += u.tiles;
            const int buffer = count & (kChunkNotes - 1);
            const bool notes[2] = {tiles_here > 0 && s.noted[buffer][0] != 0, tiles_here > 0 && s.noted[buffer][1] != 0};
            const long long at = (long long)(u.row0 + token) * p.q_heads + u.head0 + tile_head;
            const bool whole = u.splits == 1;
            const float share = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
            if (g * p.tile_tokens >= u.tokens) continue;
#pragma unroll
            for (int c = 0; c < kD; c += 32) {
                float o[32];
                if (tiles_here > 0) {
                    ptx::tmem_ld32(o_columns + c, o);
                    ptx::tc_wait_ld32(o);
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = sum == 0.0f ? 0.0f : o[i] * share;
                if (notes[c / 32 >= kD / 64] && sum != 0.0f) {
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
                    uint4* to = reinterpret_cast<uint4*>(p.out + at * kD + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        to[i] = make_uint4(pack_pair<kHalf>(o[8 * i], o[8 * i + 1]), pack_pair<kHalf>(o[8 * i + 2], o[8 * i + 3]),
                                           pack_pair<kHalf>(o[8 * i + 4], o[8 * i + 5]), pack_pair<kHalf>(o[8 * i + 6], o[8 * i + 7]));
                } else if (real) {
                    float4* to = reinterpret_cast<float4*>(p.partial + (at * p.split_limit + u.split) * kD + c);
#pragma unroll
                    for (int i = 0; i < 8; ++i) to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
                __syncwarp();
            }
            if (real && !whole) p.stats[at * p.split_limit + u.split] = make_float2(top, sum);
            ptx::tc_fence_before_sync();
        }
    }
    // Rows that no request has are zeros.
    if (warp >= kFixer && !*abort_flag) {
        for (long long base = ((long long)blockIdx.x * 2 + warp - kFixer) * 32; base < p.rows; base += (long long)gridDim.x * 64) {
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

// Joins the splits of a row's heads, in split order, a warp a head.
constexpr int kChunkJoinWarps = 4;

template <int kD, bool kHalf>
__global__ void __launch_bounds__(kChunkJoinWarps * 32) paged_chunk_join_kernel(const __grid_constant__ PagedChunkParams p) {
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    int low = 0, high = p.requests + 1;
    while (high - low > 1) {
        const int middle = (low + high) >> 1;
        if (p.starts[middle] <= row) low = middle; else high = middle;
    }
    if (low >= p.requests || p.starts[low] > row) return;
    const ChunkRequest q = chunk_request(p, low, false);
    if (row >= q.first + q.n) return;
    const int splits = chunk_splits<kD>(p, q.length);
    if (splits == 1) return;
    constexpr int kEach = kD / 32;
    for (int head = warp; head < p.q_heads; head += kChunkJoinWarps) {
        const long long at = (long long)row * p.q_heads + head;
        const float2* stats = p.stats + at * p.split_limit;
        const float* from = p.partial + at * p.split_limit * kD + lane * kEach;
        float top = -INFINITY;
        for (int i = lane; i < splits; i += 32) top = fmaxf(top, stats[i].x);
#pragma unroll
        for (int offset = 16; offset >= 1; offset >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, offset));
        float value[kEach], total = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) value[i] = 0.0f;
#pragma unroll 4
        for (int split = 0; split < splits; ++split) {
            const float2 own = stats[split];
            const float factor = own.x == -INFINITY ? 0.0f : power_of_two(own.x - top);
            total = fmaf(own.y, factor, total);
#pragma unroll
            for (int i = 0; i < kEach; i += 2) {
                const float2 pair = *reinterpret_cast<const float2*>(from + (long long)split * kD + i);
                value[i] = fmaf(pair.x, factor, value[i]);
                value[i + 1] = fmaf(pair.y, factor, value[i + 1]);
            }
        }
        uint32_t* to = reinterpret_cast<uint32_t*>(p.out + at * kD + lane * kEach);
#pragma unroll
        for (int i = 0; i < kEach; i += 2)
            to[i / 2] = total == 0.0f ? 0u : pack_pair<kHalf>(value[i] / total, value[i + 1] / total);
    }
}

// How requests are cut: into up to this many splits, where the call has fewer units than the chip asks for.
inline int chunk_split_limit(int rows, int requests, int kv_heads, int group, int head_dim, long long capacity, bool own_order, int sm_count) {
    if (own_order) return 1;
    const int parts = (group + kChunkRows - 1) / kChunkRows, part_heads = (group + parts - 1) / parts;
    const int tile = head_dim == 256 ? 64 : 128, unit_tokens = (head_dim == 256 ? 1 : 2) * (kChunkRows / part_heads);
    const long long units = ((long long)rows / unit_tokens + (requests < rows ? requests : rows)) * kv_heads * parts;
    if (units < 1) return 1;
    const long long wanted = ((long long)kChunkUnitsWanted * sm_count + units - 1) / units, most = (capacity + tile - 1) / tile / kChunkMinTiles;
    const long long limit = wanted < most ? wanted : most;
    return limit < 1 ? 1 : (int)limit;
}
inline size_t chunk_partial_bytes(int rows, int q_heads, int head_dim, int limit) {
    return limit <= 1 ? 0 : (size_t)rows * q_heads * limit * (head_dim + 2) * sizeof(float);
}

// A map of 16-bit numbers; strides in bytes, of all dimensions but the first.
inline bool chunk_map(CUtensorMap& map, bool half, const void* base, int rank, const cuuint64_t* sizes, const cuuint64_t* strides, const cuuint32_t* box) {
    const EncodeTiledFn encode = encode_tiled_fn();
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    return encode && encode(&map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), sizes, strides,
                            box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kD, bool kHalf>
inline int launch_paged_chunk(PagedChunkParams& params, const void* q, const void* keys, const PageStrides& key_strides, const void* values,
                              const PageStrides& value_strides, int sm_count, cudaStream_t stream) {
    using Shape = ChunkShape<kD>;
    const int group = params.q_heads / params.kv_heads, page = 1 << params.page_shift;
    params.parts = (group + kChunkRows - 1) / kChunkRows;
    params.part_heads = (group + params.parts - 1) / params.parts;
    params.tile_tokens = kChunkRows / params.part_heads;
    const cuuint64_t q_sizes[3] = {kD, (cuuint64_t)params.q_heads, (cuuint64_t)params.rows}, q_strides[2] = {kD * 2, (cuuint64_t)params.q_heads * kD * 2};
    const cuuint32_t q_box[3] = {64, (cuuint32_t)params.part_heads, (cuuint32_t)params.tile_tokens};
    if (!chunk_map(params.q_map, kHalf, q, 3, q_sizes, q_strides, q_box)) return MT_ERR_LAUNCH;
    const cuuint64_t sizes[4] = {kD, (cuuint64_t)page, (cuuint64_t)params.kv_heads, (cuuint64_t)params.page_count};
    const cuuint32_t box[4] = {64, (cuuint32_t)(page < Shape::kTile ? page : Shape::kTile), 1, 1};
    for (int which = 0; which < 2; ++which) {
        const PageStrides& given = which ? value_strides : key_strides;
        // (Dimensions of one element come with a stride of 0.)
        const cuuint64_t strides[3] = {(cuuint64_t)(given.token ? given.token : kD) * 2, (cuuint64_t)(given.head ? given.head : kD) * 2,
                                       (cuuint64_t)(given.page ? given.page : kD) * 2};
        if (!chunk_map(which ? params.value_map : params.key_map, kHalf, which ? values : keys, 4, sizes, strides, box)) return MT_ERR_LAUNCH;
    }
    static bool configured[64] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return MT_ERR_LAUNCH;
    if (device >= 64 || !configured[device]) {
        if (cudaFuncSetAttribute(paged_chunk_kernel<kD, kHalf>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem) != cudaSuccess) return MT_ERR_LAUNCH;
        if (device < 64) configured[device] = true;
    }
    const int unit_tokens = Shape::kGroups * params.tile_tokens;
    const long long units = ((long long)params.rows / unit_tokens + (params.requests < params.rows ? params.requests : params.rows)) * params.kv_heads *
                            params.parts * params.split_limit;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(units < 1 ? 1 : units < sm_count ? (unsigned int)units : sm_count, 1, 1);
    config.blockDim = dim3(Shape::kThreads, 1, 1);
    config.dynamicSmemBytes = Shape::kSmem;
    config.stream = stream;
    cudaLaunchAttribute attrs[1];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, paged_chunk_kernel<kD, kHalf>, params) != cudaSuccess) return MT_ERR_LAUNCH;
    if (params.split_limit > 1) {
        config.gridDim = dim3(params.rows, 1, 1);
        config.blockDim = dim3(kChunkJoinWarps * 32, 1, 1);
        config.dynamicSmemBytes = 0;
        if (cudaLaunchKernelEx(&config, paged_chunk_join_kernel<kD, kHalf>, params) != cudaSuccess) return MT_ERR_LAUNCH;
    }
    return MT_OK;
}

}  // namespace mt
