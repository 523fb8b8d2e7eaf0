// Shared pieces of the attention operators (sdpa_packed, sdpa_tree): operand addressing, the
// rule which tokens a row sees, and the row-at-a-time form both kernels fall back on.
//
//   out[row, h*D + d] = sum_t w_t v[t, d],   w = softmax over the visible t of scale * q.k_t
//
// on heads h of one key/value head h / group. Special rows follow the attention stages
// (iomb_sdpa_softmax): a NaN among the visible scores, or only -inf, makes the row NaN; +inf
// scores share the weight; a row that sees nothing is +0. Stored results are canonical as
// iomb_sdpa_canonicalize_output leaves them: -0 becomes +0, every NaN the positive quiet NaN.
#pragma once

#include <cuda_fp16.h>

#include "host.hpp"

namespace iomb {

constexpr uint32_t kMaxHeadWidth = 256;     // row-at-a-time form: eight values per lane
constexpr uint32_t kMaxTreeNodes = 256;
constexpr uint64_t kMaxAttnRows = 1ull << 30, kMaxAttnExtent = 1ull << 20;     // tokens; heads, sequences
constexpr uint32_t kKvBlock = 128;          // tokens per block of the tensor-core kernel

// One operand [b, h, rows, columns]: its planes by two strides (0 where the axis is absent).
struct AttnOperand {
    unsigned char* base;
    uint64_t plane0, stride_b, stride_h;
    uint64_t planes;            // planes of the owner up to the view's last
    uint32_t tile_rows, tile_cols;
};

struct AttnParams {
    AttnOperand q, k, v, out;
    uint32_t hq, hkv, group, width;     // heads, heads per key/value head, D
    uint32_t rows;                      // T (packed) or N (tree): rows of q per head
    uint32_t cache_rows;                // T (packed) or C (tree): rows of k and v
    uint32_t batch;                     // sequences (packed) or B (tree)
    float scale;
    const uint32_t* offsets;            // packed: batch + 1 borders
    const uint32_t* lengths;            // tree: rows before the tree
    const int32_t* parents;             // tree: [B, N] or null (a chain)
    const uint32_t* counts;             // tree: nodes in use, or null (all)
    uint32_t* status;
};

__host__ __device__ __forceinline__ uint64_t attn_plane(const AttnOperand& o, uint32_t b, uint32_t h) {
    return o.plane0 + b * o.stride_b + h * o.stride_h;
}

// First byte of the 16-column piece `piece` of a row (16-bit leaves: 32 bytes).
__device__ __forceinline__ const unsigned char* attn_piece(const AttnOperand& o, uint64_t plane,
                                                           uint32_t row, uint32_t piece) {
    const uint64_t tile = (plane * o.tile_rows + row / kTile) * o.tile_cols + piece;
    return o.base + tile * (kTileSlots * 2) + (row % kTile) * (kTile * 2);
}
__device__ __forceinline__ unsigned char* attn_out_piece(const AttnOperand& o, uint64_t plane,
                                                         uint32_t row, uint32_t piece) {
    return const_cast<unsigned char*>(attn_piece(o, plane, row, piece));
}

// ---- 16-bit leaves ---------------------------------------------------------------------------

struct LeafBf16 {
    static constexpr uint32_t kFormat = 1;      // operand format of the matrix instructions
    static constexpr float kWeightLog = 0.0f;   // log2 of the weight that a row's maximum gets in them
    static __device__ __forceinline__ float decode(uint16_t code) {
        return __uint_as_float(static_cast<uint32_t>(code) << 16);
    }
    // Two binary32 values to a packed pair, round to nearest even.
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
    // x + (+0): -0 becomes +0, every finite value and infinity stays.
    static __device__ __forceinline__ uint32_t plus_zero(uint32_t word) {
        uint32_t r;
        asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(word), "r"(0u));
        return r;
    }
    static constexpr uint32_t kNan = 0x7FC0u;
    static constexpr uint32_t kInf = 0x7F80u;
};
struct LeafF16 {
    static constexpr uint32_t kFormat = 0;
    static constexpr float kWeightLog = 7.0f;
    static __device__ __forceinline__ float decode(uint16_t code) {
        return __half2float(__ushort_as_half(code));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 packed = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&packed);
    }
    static __device__ __forceinline__ uint32_t plus_zero(uint32_t word) {
        uint32_t r;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(word), "r"(0u));
        return r;
    }
    static constexpr uint32_t kNan = 0x7E00u;
    static constexpr uint32_t kInf = 0x7C00u;
};

// -0 to +0 and every NaN to the leaf's positive quiet NaN, both halves.
template <class Leaf>
__device__ __forceinline__ uint32_t canonical_pair(uint32_t word) {
    const uint32_t lo = word & 0x7FFFu, hi = (word >> 16) & 0x7FFFu;
    uint32_t out = word;
    if (lo == 0) out &= 0xFFFF0000u;
    if (hi == 0) out &= 0x0000FFFFu;
    if (lo > Leaf::kInf) out = (out & 0xFFFF0000u) | Leaf::kNan;
    if (hi > Leaf::kInf) out = (out & 0x0000FFFFu) | (Leaf::kNan << 16);
    return out;
}

// ---- which tokens a row sees -------------------------------------------------------------------

// Rows [first, row] of a packed sequence.
struct CausalRows {
    uint32_t first, row;
    __device__ __forceinline__ uint32_t begin() const { return first; }
    __device__ __forceinline__ uint32_t end() const { return row + 1; }
    __device__ __forceinline__ bool sees(uint32_t) const { return true; }    // of [begin, end)
};

// A parent that does not lie before its node (or is negative) makes the node a root: walks end.
__device__ __forceinline__ int32_t tree_parent(const int32_t* parents, int32_t node) {
    const int32_t parent = parents[node];
    return parent < node ? parent : -1;
}

// The prefix [0, length) and the node's ancestors at length + index.
struct TreeRow {
    uint32_t length, node;
    const int32_t* parents;     // of this sequence, or null (a chain)
    __device__ __forceinline__ uint32_t begin() const { return 0; }
    __device__ __forceinline__ uint32_t end() const { return length + node + 1; }
    __device__ __forceinline__ bool sees(uint32_t token) const {
        if (token < length || parents == nullptr) return true;
        int32_t at = static_cast<int32_t>(node);
        const int32_t wanted = static_cast<int32_t>(token - length);
        while (at > wanted) at = tree_parent(parents, at);
        return at == wanted;
    }
};

// Live rows and nodes of one sequence of a tree call; a sequence whose arguments do not fit its
// cache has no nodes (and is reported).
struct TreeExtent {
    uint32_t length, nodes;
    bool bad;
};
__device__ __forceinline__ TreeExtent tree_extent(const AttnParams& p, uint32_t b) {
    TreeExtent e;
    e.length = p.lengths[b];
    e.nodes = p.counts != nullptr ? p.counts[b] : p.rows;
    e.bad = e.nodes > p.rows || e.length > p.cache_rows || e.nodes > p.cache_rows - e.length;
    if (e.bad) { e.length = 0; e.nodes = 0; }
    return e;
}

// ---- one row by one warp -------------------------------------------------------------------------

// q.k over the head's columns in order, binary32.
template <class Leaf>
__device__ __forceinline__ float row_score(const AttnParams& p, uint64_t q_plane, uint32_t row,
                                           uint64_t k_plane, uint32_t token) {
    float sum = 0.0f;
    for (uint32_t piece = 0; piece * kTile < p.width; ++piece) {
        const uint4* a = reinterpret_cast<const uint4*>(attn_piece(p.q, q_plane, row, piece));
        const uint4* b = reinterpret_cast<const uint4*>(attn_piece(p.k, k_plane, token, piece));
        const uint4 qa[2] = {a[0], a[1]}, kb[2] = {b[0], b[1]};
        const uint32_t* qw = reinterpret_cast<const uint32_t*>(qa);
        const uint32_t* kw = reinterpret_cast<const uint32_t*>(kb);
        const uint32_t live = min(kTile, p.width - piece * kTile);   // padding is not read into sums
#pragma unroll
        for (uint32_t c = 0; c < kTile; ++c) {
            const uint16_t x = static_cast<uint16_t>(qw[c / 2] >> (16 * (c & 1u)));
            const uint16_t y = static_cast<uint16_t>(kw[c / 2] >> (16 * (c & 1u)));
            if (c < live) sum = __fmaf_rn(Leaf::decode(x), Leaf::decode(y), sum);
        }
    }
    return sum;
}

// One output row by one warp: a pass for the maximum and the sum, a pass for the weighted
// values. Reads the visible tokens only, so whatever masked places hold has no influence. The
// kernel for head widths the tensor cores do not take, and the way out for special rows (NaN,
// infinities, garbage under the mask) of the kernel that runs on them.
template <class Leaf, class Rule>
__device__ void attend_row(const AttnParams& p, uint32_t b, uint32_t h, uint32_t row, const Rule& rule) {
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t q_plane = attn_plane(p.q, b, h);
    const uint64_t k_plane = attn_plane(p.k, b, h / p.group), v_plane = attn_plane(p.v, b, h / p.group);
    const float kInf = __int_as_float(0x7F800000);
    float m = -kInf, l = 0.0f;
    uint32_t infinite = 0;
    bool nan = false;
    for (uint32_t t = rule.begin() + lane; t < rule.end(); t += 32) {
        if (!rule.sees(t)) continue;
        const float s = row_score<Leaf>(p, q_plane, row, k_plane, t) * p.scale;
        if (s != s) { nan = true; continue; }
        if (s == kInf) { ++infinite; continue; }
        if (s > m) {
            l = m == -kInf ? 0.0f : l * expf(m - s);
            m = s;
        }
        if (s != -kInf) l += expf(s - m);
    }
    float top = m;
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    l = m == -kInf ? 0.0f : l * expf(m - top);
    for (int d = 16; d > 0; d >>= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, d);
        infinite += __shfl_xor_sync(0xffffffffu, infinite, d);
    }
    nan = __any_sync(0xffffffffu, nan);
    const bool nothing = rule.begin() >= rule.end();
    // (a visible row always holds at least one score: itself)
    if (!nothing && infinite == 0 && l == 0.0f) nan = true;      // every visible score is -inf
    float o[kMaxHeadWidth / 32];
#pragma unroll
    for (uint32_t i = 0; i < kMaxHeadWidth / 32; ++i) o[i] = 0.0f;
    if (!nan && !nothing) {
        for (uint32_t first = rule.begin(); first < rule.end(); first += 32) {
            const uint32_t t = first + lane;
            bool seen = t < rule.end() && rule.sees(t);
            float w = 0.0f;
            if (seen) {
                const float s = row_score<Leaf>(p, q_plane, row, k_plane, t) * p.scale;
                w = infinite ? (s == kInf ? 1.0f / static_cast<float>(infinite) : 0.0f) : expf(s - top) / l;
            }
            uint32_t left = __ballot_sync(0xffffffffu, seen);
            while (left != 0) {
                const int i = __ffs(left) - 1;
                left &= left - 1;
                const float wi = __shfl_sync(0xffffffffu, w, i);
#pragma unroll
                for (uint32_t k = 0; k < kMaxHeadWidth / 32; ++k) {
                    const uint32_t d = lane + 32 * k;
                    if (d >= p.width) break;
                    const uint16_t code = *(reinterpret_cast<const uint16_t*>(
                            attn_piece(p.v, v_plane, first + i, d / kTile)) + d % kTile);
                    o[k] = __fmaf_rn(wi, Leaf::decode(code), o[k]);
                }
            }
        }
    }
    const uint64_t out_plane = attn_plane(p.out, b, 0);
#pragma unroll
    for (uint32_t k = 0; k < kMaxHeadWidth / 32; ++k) {
        const uint32_t d = lane + 32 * k;
        if (d >= p.width) break;
        const uint32_t column = h * p.width + d;
        const float value = nan ? __int_as_float(0x7FC00000) : o[k];
        *(reinterpret_cast<uint16_t*>(attn_out_piece(p.out, out_plane, row, column / kTile)) + column % kTile) =
                static_cast<uint16_t>(canonical_pair<Leaf>(Leaf::pack(value, 0.0f)));
    }
}

// ---- checks of the index arrays ----------------------------------------------------------------

// Packed borders: ascending, none beyond the tensor. Every warp of a launch comes to the same
// answer, so a call with wrong borders writes nothing at all.
__device__ __forceinline__ bool warp_borders_ok(const AttnParams& p) {
    bool ok = true;
    for (uint32_t s = threadIdx.x & 31u; s < p.batch; s += 32) {
        const uint32_t a = p.offsets[s], e = p.offsets[s + 1];
        ok = ok && a <= e && e <= p.rows;
    }
    return __all_sync(0xffffffffu, ok);
}

// One warp looks through a tree call's arguments: extents that do not fit, parents not before their nodes.
// (One element a lane and round, so many large trees over short caches wait for it: 64 of 256 nodes, 32
// heads on 8, D 64, caches of 456 take 466 us with parents and 174 as chains; 8 of 64 nodes over caches of
// 8192 57 and 55.)
__device__ __forceinline__ bool warp_tree_bad(const AttnParams& p) {
    bool bad = false;
    const uint32_t lane = threadIdx.x & 31u;
    for (uint32_t b = lane; b < p.batch; b += 32) bad = bad || tree_extent(p, b).bad;
    if (p.parents != nullptr) {
        const uint64_t all = static_cast<uint64_t>(p.batch) * p.rows;
        for (uint64_t i = lane; i < all; i += 32) {
            const uint32_t node = static_cast<uint32_t>(i % p.rows);
            const uint32_t nodes = p.counts != nullptr ? p.counts[i / p.rows] : p.rows;
            const int32_t parent = p.parents[i];
            bad = bad || (node < nodes && (parent >= static_cast<int32_t>(node) || parent < -1));
        }
    }
    return __any_sync(0xffffffffu, bad);
}

// The tensor-core kernel (attention_tc.cu). The workspace is the partial sums of a tree call.
bool attention_tc_takes(const AttnParams& p);
uint64_t attention_tc_workspace(const AttnParams& p);
int launch_attention_tc(const AttnParams& p, bool tree, bool bf16, void* workspace, cudaStream_t stream);

}  // namespace iomb
