// Scores of given tokens (iomb_token_logprobs): log probability of one token per row of logits,
// the entropy of the row, and its K best tokens with their log probabilities.
//
//   lse = m + log z,  m = max x,  z = sum exp(x - m)
//   logprob = (x_token - m) - log z
//   entropy = log z - t / z,  t = sum exp(x - m) (x - m), a term of weight zero counting zero
//
// Sums in binary32. A row with a NaN, with +inf or with nothing but -inf has NaN results (what
// the formula gives); its best tokens are still the K largest, NaN above everything, -0 equal
// to +0, equal values by the lower index.
//
// The logits are read once. A band of 16 rows is one contiguous run of tiles; a cluster of one
// to eight CTAs takes a band, its warps take tiles in turn, and a lane owns eight columns of one
// row of a tile (bands with fewer rows spread the lanes over several tiles). Each lane keeps a
// running (m, z, t) and four running maxima, one per load slot. The cluster's warps hand these
// to the row's owner, which joins them. The best tokens take no second pass: of the maxima of G
// disjoint groups of columns at least K reach the K-th largest, tau, so every one of the K best
// reaches it too, and only the slots whose own maximum does (about K of them) are read again for
// their elements. The owner ranks these candidates. Rows where that breaks down are
// ranked by one warp that walks the row: with NaN, or with more than 256 candidates. tau has 16 leading
// bits, so those are values by the hundred that tie or lie within one part in 128 of the K-th best, or
// fewer than K tokens beside a finite mask. It costs about 160 us a walk of 32000 columns (64 rows of F32
// 11 us, 161 with one such row and 185 with 64; 2045 rows of 50021 92 us, 1117 when all are such).
//
// Bound by HBM where there are many rows: 2045 rows of 50021 F32 logits take 73 us per call on a B200
// (5.6 TB/s). 64 rows of 32000 BF16 take 9.3 us, bound by the chain load, cluster
// barrier, candidates, ranking; clusters of eight put 32 CTAs on them instead of four.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "host.hpp"

namespace iomb {

namespace cg = cooperative_groups;

constexpr int kScoreThreads = 256;
constexpr uint32_t kScoreWarps = kScoreThreads / 32;
constexpr uint32_t kMaxTop = 32;
constexpr uint32_t kSlots = 4;              // loads in flight per lane, and maxima it keeps
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kMaxGroups = 128;        // maxima per row that the owner sees
constexpr uint32_t kCandidates = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct ScoreParams {
    Operand logits, tokens, logprob, entropy, top_value, top_token;
    Leading leading;
    uint32_t rows, vocab, top;
    uint32_t bands;                         // row groups per plane
    uint32_t group_log;                     // log2 of the rows of a group (at most a tile's 16)
    uint32_t has_entropy;
    uint32_t token_bits, token_signed;
    uint32_t* status;
};

struct ScoreBf16 {
    static constexpr uint32_t kBytes = 2;
    static __device__ __forceinline__ float load(const unsigned char* at) {
        return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at)) << 16);
    }
    static __device__ __forceinline__ void unpack(uint32_t word, float& lo, float& hi) {
        lo = bf16_lo(word);
        hi = bf16_hi(word);
    }
};
struct ScoreF16 {
    static constexpr uint32_t kBytes = 2;
    static __device__ __forceinline__ float load(const unsigned char* at) {
        return __half2float(*reinterpret_cast<const __half*>(at));
    }
    static __device__ __forceinline__ void unpack(uint32_t word, float& lo, float& hi) {
        const float2 both = __half22float2(*reinterpret_cast<const __half2*>(&word));
        lo = both.x;
        hi = both.y;
    }
};
struct ScoreF32 {
    static constexpr uint32_t kBytes = 4;
    static __device__ __forceinline__ float load(const unsigned char* at) {
        return *reinterpret_cast<const float*>(at);
    }
};

// Eight columns of one row of a tile: 16 or 32 bytes. (Volatile and without a condition, so that a
// group of loads stays in front of the first use: sunk into their uses they would wait one by one.)
template <class Leaf>
struct Chunk {
    uint4 lo, hi;
    __device__ __forceinline__ void load(const unsigned char* at) {
        if constexpr (Leaf::kBytes == 4) {
            asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w), "=r"(hi.x), "=r"(hi.y), "=r"(hi.z), "=r"(hi.w)
                         : "l"(at));
        } else {
            asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w) : "l"(at));
        }
    }
    __device__ __forceinline__ void values(float (&x)[8]) const {
        if constexpr (Leaf::kBytes == 4) {
            const uint32_t words[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(words[i]);
        } else {
            Leaf::unpack(lo.x, x[0], x[1]);
            Leaf::unpack(lo.y, x[2], x[3]);
            Leaf::unpack(lo.z, x[4], x[5]);
            Leaf::unpack(lo.w, x[6], x[7]);
        }
    }
};

__device__ __forceinline__ uint64_t score_slot(const Operand& o, uint64_t plane, uint32_t row, uint32_t col) {
    return ((plane * o.tile_rows + row / kTile) * o.tile_cols + col / kTile) * kTileSlots
            + (row % kTile) * kTile + col % kTile;
}

// The order of the best tokens: larger value first (NaN above all, -0 as +0), then lower index.
__device__ __forceinline__ uint64_t score_key(float x, uint32_t index) {
    uint32_t bits = x == 0.0f ? 0u : __float_as_uint(x);
    uint32_t order = (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
    if (x != x) order = 0xFFFFFFFEu;     // (no key is all ones)
    return (static_cast<uint64_t>(order) << 32) | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t order = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((order & 0x80000000u) ? order & 0x7FFFFFFFu : ~order);
}

// The token of row r; false when it is negative or not in the vocabulary.
__device__ __forceinline__ bool score_token(const ScoreParams& p, uint64_t plane, uint32_t r, uint32_t* token) {
    const uint64_t slot = score_slot(p.tokens, plane, 0, r);
    uint64_t id;
    if (p.token_bits == 32) id = *reinterpret_cast<const uint32_t*>(p.tokens.base + slot * 4);
    else id = *reinterpret_cast<const uint64_t*>(p.tokens.base + slot * 8);
    *token = static_cast<uint32_t>(id);
    return !(p.token_signed && ((id >> (p.token_bits - 1)) & 1u)) && id < p.vocab;
}

__device__ __forceinline__ void report_tokens(const ScoreParams& p) {
    bool bad = false;
    const uint64_t all = p.leading.planes * p.rows;
    for (uint64_t i = threadIdx.x; i < all; i += blockDim.x) {
        uint32_t token;
        bad = bad || !score_token(p, operand_plane(p.tokens, p.leading, i / p.rows),
                                  static_cast<uint32_t>(i % p.rows), &token);
    }
    const int any = __syncthreads_or(bad ? 1 : 0);
    if (threadIdx.x == 0) *p.status = any ? 1u : 0u;
}

__device__ __forceinline__ float score_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint64_t score_pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}

// A running maximum m, z = sum exp(x - m), t = sum exp(x - m) (x - m). m = -inf: nothing but
// -inf so far, z and t are zero (or NaN, which stays).
struct RunningSum {
    float m, z, t;
};
// How far a sum is moved to a new maximum. Beyond 10^4 its weights are zero all the same, and z times
// the distance stays finite: logits may lie at the end of binary32 (masks of the leaf's lowest value),
// and an infinite product would turn NaN under the weight of zero.
__device__ __forceinline__ float score_step(float from, float to) { return fmaxf(from - to, -1e4f); }
__device__ __forceinline__ RunningSum join_sums(const RunningSum& a, const RunningSum& b) {
    const float kNone = __int_as_float(0xFF800000);
    RunningSum r{fmaxf(a.m, b.m), 0.0f, 0.0f};
    float z = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const RunningSum& s = i == 0 ? a : b;
        if (s.m == kNone) {
            z += s.z;
        } else {
            const float d = score_step(s.m, r.m), f = score_exp2(d * kLog2e);
            z = __fmaf_rn(s.z, f, z);
            t = __fmaf_rn(__fmaf_rn(s.z, d, s.t), f, t);
        }
    }
    r.z = z;
    r.t = t;
    return r;
}
__device__ __forceinline__ RunningSum shuffle_sum(const RunningSum& s, int distance) {
    return RunningSum{__shfl_xor_sync(0xffffffffu, s.m, distance), __shfl_xor_sync(0xffffffffu, s.z, distance),
                      __shfl_xor_sync(0xffffffffu, s.t, distance)};
}

// log2 of the rows of a tile a warp's lanes are spread over: as many as there are, so that they
// load 16 / rows tiles side by side; for short rows more (lanes without a row idle), so that
// there are at least 16 spans and with them more groups of columns than best tokens.
__host__ __device__ __forceinline__ uint32_t lane_spread(uint32_t live, uint32_t tile_cols) {
    uint32_t log = live > 8 ? 4 : live > 4 ? 3 : live > 2 ? 2 : live > 1 ? 1 : 0;
    while (log < 4 && (tile_cols >> (4 - log)) < 16) ++log;
    return log;
}

// The owner's side: rows rank, rank + cluster, ... of the band, row i / cluster in these arrays.
struct ScoreShared {
    RunningSum sums[kTile * kScoreWarps];       // [rows here][warps of the cluster]
    float groups[kTile * 64];                   // [rows here][groups]: 16 x 64, 8 x 128, 4 x 64, 2 x 128
    float top[kTile], log_z[kTile];
    uint32_t odd[kTile], count[kTile];
    float tau[kTile];                           // of every row of the group, from the rows' owners
    uint8_t hot[kScoreWarps][32 * kSlots];      // a warp's (slot, lane) pairs that reach tau
    unsigned long long candidates[kTile][kCandidates];
};

// One warp walks a row in the order of its columns with the K best so far in its lanes, lane 0
// the best. Any row; hundreds of instructions per insertion, so for rare rows.
template <class Leaf>
__device__ __noinline__ uint64_t walk_row(const ScoreParams& p, uint64_t plane, uint32_t row) {
    const uint32_t lane = threadIdx.x & 31u;
    uint64_t mine = 0;                          // (every key is above zero)
    uint64_t last = 0;                          // the K-th best so far
    for (uint32_t first = 0; first < p.vocab; first += 32 * kSlots) {
        float x[kSlots];
#pragma unroll
        for (uint32_t u = 0; u < kSlots; ++u) {
            const uint32_t c = first + u * 32 + lane;
            x[u] = c < p.vocab ? Leaf::load(p.logits.base + score_slot(p.logits, plane, row, c) * Leaf::kBytes) : 0.0f;
        }
#pragma unroll
        for (uint32_t u = 0; u < kSlots; ++u) {
            const uint32_t c = first + u * 32 + lane;
            const uint64_t key = c < p.vocab ? score_key(x[u], c) : 0;
            uint32_t hits = __ballot_sync(0xffffffffu, key > last);
            while (hits != 0) {
                const int who = __ffs(hits) - 1;
                hits &= hits - 1;
                const uint64_t one = __shfl_sync(0xffffffffu, key, who);
                if (one <= last) continue;
                const uint64_t before = __shfl_up_sync(0xffffffffu, mine, 1);
                const bool above = mine > one;
                if (!above) mine = lane == 0 || before > one ? one : before;
                last = __shfl_sync(0xffffffffu, mine, p.top - 1);
            }
        }
    }
    return mine;
}

template <class Leaf>
__global__ void __launch_bounds__(kScoreThreads)
score_kernel(const __grid_constant__ ScoreParams p) {
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t unit = blockIdx.x / ctas;
    if (unit == p.leading.planes * p.bands) {       // the last cluster checks the tokens
        if (rank == 0) report_tokens(p);
        return;
    }
    __shared__ ScoreShared sh;
    const float kNone = __int_as_float(0xFF800000), kInf = __int_as_float(0x7F800000);
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    if (threadIdx.x < kTile) sh.count[threadIdx.x] = 0;
    // Nobody writes into a neighbour before all have started and zeroed their counts.
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const uint64_t index = unit / p.bands;
    const uint32_t first_row = (unit % p.bands) << p.group_log;
    const uint32_t live = min(1u << p.group_log, p.rows - first_row);
    const uint64_t plane = operand_plane(p.logits, p.leading, index);
    // Lanes: half a tile row each; `spread` rows of a tile, 16 / spread tiles side by side.
    const uint32_t spread_log = lane_spread(live, p.logits.tile_cols);
    const uint32_t row = (lane >> 1) & ((1u << spread_log) - 1u);
    const uint32_t side = lane >> (1 + spread_log), sides_log = 4 - spread_log;
    const uint32_t half = lane & 1u;
    const uint32_t warps = ctas * kScoreWarps, my_warp = rank * kScoreWarps + warp;
    const uint32_t tile_cols = p.logits.tile_cols;
    const unsigned char* const row_base = p.logits.base
            + (plane * p.logits.tile_rows + first_row / kTile) * tile_cols * static_cast<uint64_t>(kTileSlots * Leaf::kBytes)
            + first_row % kTile * (kTile * Leaf::kBytes);
    const unsigned char* const base = row_base + min(row, live - 1) * (kTile * Leaf::kBytes) + half * (8 * Leaf::kBytes);
    const uint32_t spans = (tile_cols + (1u << sides_log) - 1) >> sides_log;    // a warp's loads side by side
    const bool mine = row < live;              // (lanes of rows that are not there read the last one)

    float m = kNone, less = 0.0f;               // running maximum, and what is subtracted (0 while -inf)
    uint64_t z2 = 0, t2 = 0;                    // sums over even and odd columns
    float best[kSlots];
#pragma unroll
    for (uint32_t u = 0; u < kSlots; ++u) best[u] = kNone;
    const uint64_t scale2 = score_pair(kLog2e, kLog2e);
    for (uint32_t first = my_warp; first < spans; first += kSlots * warps) {
        Chunk<Leaf> chunk[kSlots];
#pragma unroll
        for (uint32_t u = 0; u < kSlots; ++u) {
            const uint32_t tile = ((first + u * warps) << sides_log) + side;
            chunk[u].load(base + static_cast<uint64_t>(min(tile, tile_cols - 1)) * (kTileSlots * Leaf::kBytes));
        }
#pragma unroll
        for (uint32_t u = 0; u < kSlots; ++u) {
            const uint32_t tile = ((first + u * warps) << sides_log) + side;
            if (tile >= tile_cols) continue;
            float x[8];
            chunk[u].values(x);
            const uint32_t column = tile * kTile + half * 8;
            if (column + 8 > p.vocab) {
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    if (column + i >= p.vocab) x[i] = kNone;
                }
            }
            const float high = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            best[u] = fmaxf(best[u], high);
            if (high > m) {
                if (m != kNone) {
                    // exp(x - high) = exp(x - m) f and (x - high) = (x - m) + d
                    const float d = score_step(m, high), f = score_exp2(d * kLog2e);
                    const uint64_t f2 = score_pair(f, f), d2 = score_pair(d, d);
                    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(t2) : "l"(z2), "l"(d2));
                    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(t2) : "l"(f2));
                    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(z2) : "l"(f2));
                }
                m = high;
                less = -high;
            }
            const uint64_t less2 = score_pair(less, less);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                uint64_t d2 = score_pair(x[i], x[i + 1]), y2;
                asm("add.rn.f32x2 %0, %0, %1;" : "+l"(d2) : "l"(less2));
                asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y2) : "l"(d2), "l"(scale2));
                float d0, d1, y0, y1;
                asm("mov.b64 {%0, %1}, %2;" : "=f"(d0), "=f"(d1) : "l"(d2));
                asm("mov.b64 {%0, %1}, %2;" : "=f"(y0), "=f"(y1) : "l"(y2));
                const uint64_t e2 = score_pair(score_exp2(y0), score_exp2(y1));
                // A term of weight zero counts zero, whatever its logarithm.
                d2 = score_pair(fmaxf(d0, -1e30f), fmaxf(d1, -1e30f));
                asm("add.rn.f32x2 %0, %0, %1;" : "+l"(z2) : "l"(e2));
                asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(t2) : "l"(e2), "l"(d2));
            }
        }
    }
    RunningSum sum;
    {
        float z0, z1, t0, t1;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(z0), "=f"(z1) : "l"(z2));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(t0), "=f"(t1) : "l"(t2));
        sum = RunningSum{m, z0 + z1, t0 + t1};
    }
    // Join the lanes of a row: the half, then the tiles side by side.
    sum = join_sums(sum, shuffle_sum(sum, 1));
    for (uint32_t d = 2u << spread_log; d < 32; d <<= 1) sum = join_sums(sum, shuffle_sum(sum, static_cast<int>(d)));
    // Hand over: sums, and the slots' maxima as eight groups per warp (two where four or more
    // CTAs share the row: 64 or 128 groups a row either way).
    const uint32_t owner = row % ctas, place = row / ctas;
    const uint32_t per_warp = ctas >= 4 ? 2 : 8, groups = per_warp * warps;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    {
        ScoreShared* const there = cluster.map_shared_rank(&sh, owner);
        if (mine && half == 0 && side == 0) there->sums[place * warps + my_warp] = sum;
        if (p.top != 0) {
            float fold[kSlots];
#pragma unroll
            for (uint32_t u = 0; u < kSlots; ++u) fold[u] = best[u];
            // Values per lane and lanes per row after folding: 4 x 2, 2 x 4, 1 x 8, or 1 x 2.
            uint32_t values = kSlots, lanes = 2u << sides_log;
            if (per_warp == 2 || lanes > 2) {
                fold[0] = fmaxf(fold[0], fold[1]);
                fold[1] = fmaxf(fold[2], fold[3]);
                values = 2;
            }
            if (per_warp == 2 || lanes > 4) {
                fold[0] = fmaxf(fold[0], fold[1]);
                values = 1;
            }
            for (uint32_t d = 16; lanes * values > per_warp; d >>= 1) {      // the highest lane bits are the tiles
                fold[0] = fmaxf(fold[0], __shfl_xor_sync(0xffffffffu, fold[0], static_cast<int>(d)));
                lanes >>= 1;
            }
            const uint32_t lane_in_row = half | (side << 1);
            if (mine && lane_in_row < lanes) {
                float* to = there->groups + place * groups + my_warp * per_warp + lane_in_row * values;
#pragma unroll
                for (uint32_t u = 0; u < kSlots; ++u) {
                    if (u < values) to[u] = fold[u];
                }
            }
        }
    }
    cluster.sync();
    // ---- the owners' rows ---------------------------------------------------------------------------
    for (uint32_t at = warp; rank + at * ctas < live; at += kScoreWarps) {
        const uint32_t r = rank + at * ctas, logical = first_row + r;
        RunningSum all{kNone, 0.0f, 0.0f};
        for (uint32_t w = lane; w < warps; w += 32) all = join_sums(all, sh.sums[at * warps + w]);
        for (int d = 16; d > 0; d >>= 1) all = join_sums(all, shuffle_sum(all, d));
        const bool odd = all.m == kNone || all.z != all.z || all.m == kInf;
        const float log_z = logf(all.z);
        if (p.top != 0) {
            // tau: the K-th largest group maximum, or a little less: the largest value of 16 leading
            // bits (in the order of the keys) that at least K of them reach.
            const float* g = sh.groups + at * groups;
            uint32_t order[kMaxGroups / 32];
#pragma unroll
            for (uint32_t i = 0; i < kMaxGroups / 32; ++i) {
                order[i] = i * 32 < groups ? static_cast<uint32_t>(score_key(g[i * 32 + lane], 0) >> 32) : 0;
            }
            uint32_t reached = 0;
            for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
                uint32_t n = 0;
#pragma unroll
                for (uint32_t i = 0; i < kMaxGroups / 32; ++i) n += __popc(__ballot_sync(0xffffffffu, order[i] >= (reached | bit)));
                if (n >= p.top) reached |= bit;
            }
            // (the smallest orders are NaN's as a float: nothing is ruled out by it)
            float tau = key_value(static_cast<uint64_t>(reached) << 32);
            if (tau != tau) tau = kNone;
            if (odd) tau = kInf;                        // (no candidates: the row is walked)
            if (lane < ctas) cluster.map_shared_rank(&sh, lane)->tau[r] = tau;
            if (lane == 0) {
                sh.top[at] = all.m;
                sh.log_z[at] = log_z;
                sh.odd[at] = odd;
            }
        }
        if (lane == 0) {
            const float kNan = __int_as_float(0x7FC00000);
            uint32_t token;
            if (score_token(p, operand_plane(p.tokens, p.leading, index), logical, &token)) {
                const float x = Leaf::load(p.logits.base + score_slot(p.logits, plane, logical, token) * Leaf::kBytes);
                const uint64_t slot = score_slot(p.logprob, operand_plane(p.logprob, p.leading, index), 0, logical);
                reinterpret_cast<float*>(p.logprob.base)[slot] = odd ? kNan : (x - all.m) - log_z;
            }
            if (p.has_entropy) {
                const uint64_t slot = score_slot(p.entropy, operand_plane(p.entropy, p.leading, index), 0, logical);
                reinterpret_cast<float*>(p.entropy.base)[slot] = odd ? kNan : log_z - all.t / all.z;
            }
        }
    }
    if (p.top == 0) return;                             // (nobody reads a neighbour any more)
    cluster.sync();
    // ---- candidates: the slots that reach tau, once more ---------------------------------------------
    {
        const float tau = sh.tau[row];
        uint32_t hot = 0;
#pragma unroll
        for (uint32_t u = 0; u < kSlots; ++u) {
            const bool reaches = mine && best[u] >= tau && best[u] != kNone;
            const uint32_t who = __ballot_sync(0xffffffffu, reaches);
            if (reaches) sh.hot[warp][hot + __popc(who & ((1u << lane) - 1u))] = static_cast<uint8_t>(u * 32 + lane);
            hot += __popc(who);
        }
        __syncwarp();
        // Eight lanes per pair: each takes every eighth of the pair's chunks, so that a pair costs
        // one wait for memory and not one per chunk.
        for (uint32_t first = 0; first < hot; first += 4) {
            const uint32_t at = first + lane / 8;
            const uint32_t pair = sh.hot[warp][min(at, hot - 1)];
            const uint32_t its_lane = pair % 32, u = pair / 32;
            const uint32_t its_row = (its_lane >> 1) & ((1u << spread_log) - 1u), its_side = its_lane >> (1 + spread_log);
            const float its_tau = sh.tau[its_row];
            ScoreShared* const there = cluster.map_shared_rank(&sh, its_row % ctas);
            const uint32_t its_place = its_row / ctas;
            const unsigned char* const from = row_base + its_row * (kTile * Leaf::kBytes) + (its_lane & 1u) * (8 * Leaf::kBytes);
            const uint32_t step = kSlots * warps;
            for (uint32_t span = my_warp + u * warps + (lane % 8) * step; ; span += 8 * step) {
                const uint32_t tile = (span << sides_log) + its_side;
                const bool there_is = at < hot && span < spans && tile < tile_cols;
                if (!__any_sync(0xffffffffu, there_is)) break;
                if (!there_is) continue;
                Chunk<Leaf> chunk;
                chunk.load(from + static_cast<uint64_t>(tile) * (kTileSlots * Leaf::kBytes));
                float x[8];
                chunk.values(x);
                const uint32_t column = tile * kTile + (its_lane & 1u) * 8;
                uint32_t reach = 0;
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    reach |= (x[i] >= its_tau && x[i] > kNone && column + i < p.vocab ? 1u : 0u) << i;
                }
                if (reach == 0) continue;
                uint32_t n = atomicAdd(&there->count[its_place], static_cast<uint32_t>(__popc(reach)));
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    if (!((reach >> i) & 1u)) continue;
                    if (n < kCandidates) there->candidates[its_place][n] = score_key(x[i], column + i);
                    ++n;
                }
            }
        }
    }
    cluster.sync();
    for (uint32_t at = warp; rank + at * ctas < live; at += kScoreWarps) {
        const uint32_t r = rank + at * ctas, logical = first_row + r;
        const bool odd = sh.odd[at] != 0;
        const uint32_t n = sh.count[at];
        const uint64_t value_plane = operand_plane(p.top_value, p.leading, index);
        const uint64_t token_plane = operand_plane(p.top_token, p.leading, index);
        const float top = sh.top[at], log_z = sh.log_z[at];
        auto store = [&](uint32_t k, uint64_t key) {
            const float value = odd ? __int_as_float(0x7FC00000) : (key_value(key) - top) - log_z;
            reinterpret_cast<float*>(p.top_value.base)[score_slot(p.top_value, value_plane, logical, k)] = value;
            reinterpret_cast<uint32_t*>(p.top_token.base)[score_slot(p.top_token, token_plane, logical, k)] =
                    0xFFFFFFFFu - static_cast<uint32_t>(key);
        };
        if (odd || n > kCandidates) {
            const uint64_t key = walk_row<Leaf>(p, plane, logical);
            if (lane < p.top) store(lane, key);
            continue;
        }
        for (uint32_t first = 0; first < n; first += 32) {
            const uint64_t key = first + lane < n ? sh.candidates[at][first + lane] : 0;
            uint32_t above = 0;
            for (uint32_t j = 0; j < n; ++j) above += sh.candidates[at][j] > key ? 1u : 0u;
            if (first + lane < n && above < p.top) store(above, key);
        }
        // Fewer than K tokens that are not ruled out: the lowest ruled-out ones follow.
        for (uint32_t k = n, c = 0; k < p.top; c += 32) {
            const bool out = c + lane < p.vocab
                    && Leaf::load(p.logits.base + score_slot(p.logits, plane, logical, c + lane) * Leaf::kBytes) == kNone;
            const uint32_t found = __ballot_sync(0xffffffffu, out);
            const uint32_t mine_at = k + __popc(found & ((1u << lane) - 1u));
            if (out && mine_at < p.top) store(mine_at, score_key(kNone, c + lane));
            k += __popc(found);
        }
    }
}

}  // namespace iomb

extern "C" int iomb_token_logprobs(const iomb_view* logits, const iomb_view* tokens, const iomb_view* logprob,
                                   const iomb_view* entropy, const iomb_view* top_logprobs,
                                   const iomb_view* top_tokens, uint32_t* status, void* stream) {
    using namespace iomb;
    const iomb_view* views[6] = {logits, tokens, logprob, entropy, top_logprobs, top_tokens};
    static const char* const names[6] = {"token_logprobs logits", "token_logprobs tokens", "token_logprobs logprob",
                                         "token_logprobs entropy", "token_logprobs top_logprobs",
                                         "token_logprobs top_tokens"};
    ViewFacts facts[6] = {};
    for (int i = 0; i < 6; ++i) {
        if (i >= 3 && views[i] == nullptr) continue;
        const int rc = check_view(views[i], names[i], &facts[i]);
        if (rc != IOMB_OK) return rc;
    }
    if ((top_logprobs == nullptr) != (top_tokens == nullptr)) {
        return fail(IOMB_ERR_INVALID_ARGUMENT, "token_logprobs: top_logprobs and top_tokens come together");
    }
    const uint64_t rows = facts[0].rows, vocab = facts[0].cols;
    for (int i = 1; i < 6; ++i) {
        if (views[i] == nullptr) continue;
        bool same = views[i]->rank == logits->rank;
        for (uint32_t a = 0; a < facts[0].leading && same; ++a) same = views[i]->dims[a] == logits->dims[a];
        if (!same) return fail(IOMB_ERR_INVALID_ARGUMENT, "token_logprobs: leading extents differ");
        if (i <= 3 ? (facts[i].rows != 1 || facts[i].cols != rows) : facts[i].rows != rows) {
            return fail(IOMB_ERR_INVALID_ARGUMENT,
                        "token_logprobs: shapes must be X[...,R,V], T[...,1,R], L[...,1,R], best [...,R,K]");
        }
    }
    if (logits->dtype != IOMB_BF16 && logits->dtype != IOMB_F16 && logits->dtype != IOMB_F32) {
        return fail(IOMB_ERR_UNSUPPORTED, "token_logprobs: logits must be BF16, F16 or F32");
    }
    if (tokens->dtype != IOMB_I32 && tokens->dtype != IOMB_U32 && tokens->dtype != IOMB_I64 && tokens->dtype != IOMB_U64) {
        return fail(IOMB_ERR_UNSUPPORTED, "token_logprobs: tokens must be I32, U32, I64 or U64");
    }
    if (logprob->dtype != IOMB_F32 || (entropy != nullptr && entropy->dtype != IOMB_F32)
            || (top_logprobs != nullptr && (top_logprobs->dtype != IOMB_F32
                                            || (top_tokens->dtype != IOMB_U32 && top_tokens->dtype != IOMB_I32)))) {
        return fail(IOMB_ERR_INVALID_ARGUMENT, "token_logprobs: results are F32, best tokens U32 or I32");
    }
    if (top_logprobs != nullptr) {
        if (facts[4].cols != facts[5].cols || facts[4].cols > vocab) {
            return fail(IOMB_ERR_INVALID_ARGUMENT, "token_logprobs: K best of V values need equal K <= V");
        }
        if (facts[4].cols > kMaxTop) return fail(IOMB_ERR_UNSUPPORTED, "token_logprobs: at most 32 best tokens");
    }
    if (status == nullptr || reinterpret_cast<uintptr_t>(status) % 4 != 0) {
        return fail(IOMB_ERR_INVALID_ARGUMENT, "token_logprobs: status must be a device word");
    }
    for (int i = 2; i < 6; ++i) {
        if (views[i] == nullptr) continue;
        for (int j = 0; j < i; ++j) {
            if (views[j] != nullptr && storage_overlaps(*views[i], facts[i], *views[j], facts[j])) {
                return fail(IOMB_ERR_INVALID_ARGUMENT, "token_logprobs: a result overlaps another operand");
            }
        }
    }
    if (rows > (1ull << 30) || vocab > (1ull << 30) || facts[0].planes > (1ull << 30) / rows) {
        return fail(IOMB_ERR_UNSUPPORTED, "token_logprobs: an extent exceeds the kernel limit");
    }
    ScoreParams p{};
    uint64_t strides[6][kMaxLead] = {};
    for (int i = 0; i < 6; ++i) {
        const iomb_view* view = views[i] != nullptr ? views[i] : logits;
        for (uint32_t a = 0; a < facts[0].leading; ++a) strides[i][a] = view->plane_strides[a];
    }
    collapse_leading(facts[0].leading, logits->dims, strides, 6, &p.leading);
    Operand* const operands[6] = {&p.logits, &p.tokens, &p.logprob, &p.entropy, &p.top_value, &p.top_token};
    for (int i = 0; i < 6; ++i) {
        if (views[i] != nullptr) *operands[i] = make_operand(*views[i], facts[i], strides[i], p.leading, false, false);
    }
    p.rows = static_cast<uint32_t>(rows);
    p.vocab = static_cast<uint32_t>(vocab);
    p.top = top_logprobs != nullptr ? static_cast<uint32_t>(facts[4].cols) : 0;
    p.has_entropy = entropy != nullptr ? 1u : 0u;
    p.token_bits = facts[1].bits;
    p.token_signed = tokens->dtype == IOMB_I32 || tokens->dtype == IOMB_I64;
    p.status = status;
    // Rows per cluster: a tile's 16 (whole tiles in one read), fewer while the clusters would leave
    // SMs idle: 64 rows of 32000 BF16 take 18 us in groups of 16 and 9.7 in groups of two. CTAs
    // per cluster: up to eight while each warp still has two loads to do (a row is then read at the
    // rate of several SMs, and the more groups of columns, the less of it is read twice).
    uint32_t group_log = 4, ctas = 1;
    for (;; --group_log) {
        const uint32_t most = rows < (1ull << group_log) ? static_cast<uint32_t>(rows) : 1u << group_log;
        const uint64_t spans = (facts[0].tile_cols << lane_spread(most, p.logits.tile_cols)) / kTile;
        ctas = 1;
        while (ctas < kMaxCluster && spans >= static_cast<uint64_t>(ctas) * 2 * kScoreWarps * 2) ctas *= 2;
        p.bands = static_cast<uint32_t>((rows + (1u << group_log) - 1) >> group_log);
        if (group_log == 0 || facts[0].planes * p.bands * ctas >= static_cast<uint64_t>(sm_count())) break;
    }
    p.group_log = group_log;
    const uint64_t grid = (facts[0].planes * p.bands + 1) * ctas;
    if (grid > 0x7FFFFFFFull) return fail(IOMB_ERR_UNSUPPORTED, "token_logprobs: too many rows for one launch");
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(grid));
    config.blockDim = dim3(kScoreThreads);
    config.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute shape{};
    shape.id = cudaLaunchAttributeClusterDimension;
    shape.val.clusterDim.x = ctas;
    shape.val.clusterDim.y = shape.val.clusterDim.z = 1;
    config.attrs = &shape;
    config.numAttrs = 1;
    cudaError_t error;
    switch (logits->dtype) {
        case IOMB_BF16: error = cudaLaunchKernelEx(&config, score_kernel<ScoreBf16>, p); break;
        case IOMB_F16: error = cudaLaunchKernelEx(&config, score_kernel<ScoreF16>, p); break;
        default: error = cudaLaunchKernelEx(&config, score_kernel<ScoreF32>, p); break;
    }
    return error == cudaSuccess ? IOMB_OK : check_launch("token_logprobs launch");
}
