// Attention on the tensor cores: the kernel behind iomb_sdpa_packed and iomb_sdpa_tree for head
// widths that are multiples of 16 up to 128.
//
// One CTA works on two tiles, A and B, of 128 score rows each. Per block of 128 tokens and tile
//   S = Q K^T          tcgen05.mma, both operands in shared memory, S in tensor memory (FP32)
//   P = exp2(c S - c m) softmax warpgroup of the tile: one thread per row, S read back from
//                      tensor memory, P (16-bit) written over S
//   O += P V           tcgen05.mma, P from tensor memory, V from shared memory, O in tensor memory
// with the running maximum m and sum l of each row in its thread. O is rescaled only when a
// row's maximum grows by more than 2^8 (P then stays below 2^8, far from any overflow); the sum
// takes the unrounded exponentials. F16 holds P times 2^7 (below 2^15), so that weights down to 2^-32 of
// the maximum's count: times one, those below 2^-25 vanished beside the sum that held them (60000 weights
// of 2^-26.5 against one large weight are 6e-4 of the result). While one tile's softmax runs, the other
// tile's products do.
// P is handed over in two halves, so that its product with V begins while the second half's
// exponentials are still computed.
//
// The library's 16x16 tiles feed the matrix instructions without any re-layout: a tile row is 32
// bytes, so a column of tiles is a K-major operand with 32-byte swizzle and K = 16 (one
// instruction) for Q and K, and the same bytes are the MN-major operand of V. One tensor-map
// copy per block fetches 128 tokens x D as [D/16][8 tiles][16][32 B], the tokens in an order of
// their own (block_order).
//
// What a tile's 128 rows are:
//   packed   `pack` heads of one key/value head x 128/pack consecutive rows, so that short
//            sequences share a tile between heads; A and B are neighbouring row blocks
//   shared   a tree call with more than 128 (head, node) pairs per key/value head: A and B hold
//            128 pairs each and share the token blocks
//   workers  a tree call with up to 128 pairs: A and B are two workers, each with row sets, queries,
//            ring of blocks and issuing warp of its own, so that one's change from a row set to the
//            next (5000 clocks) runs beside the other's work. B's rows sit 32 or 64 lanes higher where
//            they are few enough: the two then compute on different schedulers
// A tree call cuts the token blocks of all sequences and heads into equal ranges, one per CTA or
// worker. A row whose blocks lie in several ranges leaves partial (m, l, O) in the workspace and a
// second kernel joins them, in the order of the ranges.
//
// Special rows: a row with a result that is not finite (NaN or infinities among its operands or
// under its mask, where the matrix instruction multiplies them by zero) is computed again by
// attend_row, which reads visible tokens only. Tiles of tokens that no row sees take no part, and
// values beside the sequence in its first and last tile are zeroed as they arrive.
//
// What bounds it (one B200; rates by the algorithm's bytes and products):
//   packed 8192 rows       32 heads on 8, D 128: 508 us, 1080 TFLOP/s. Per step of 128 x 128 scores the
//                          exponentials take 1024 clocks of the SM's special-function units, the two
//                          products 1024 of the tensor cores, and neither reaches beyond 53 % of the
//                          time: what is left is the softmax's other instructions between two handovers.
//   tree, long caches      2 trees of 5 nodes, caches of 100001 rows (427 MB): 88 us, 4.9 TB/s
//   tree, single tokens    64 decodes: 28 us, 2.4 TB/s; the changes between row sets and the second kernel
//
// Warps: 0-3 softmax of A, 4-7 softmax of B, 8 issues the matrix instructions, 9 the copies, 10
// and 11 bring the queries of a tree call's next row set while the last one is worked on; with
// workers 8 and 9 issue A's and B's matrix instructions, 10 and 11 their copies and queries. The
// last four hand registers to the softmax (2 x 128 x 208 + 128 x 80 of the 384 x 168 a CTA starts
// with).
// Every wait is bounded; one that gives up ends all roles, is counted and makes the status 2.
#include <cuda.h>

#include <stdio.h>

#include "attention.cuh"

namespace iomb {
namespace {

constexpr uint32_t kThreads = 384;
constexpr uint32_t kSoftmaxWarps = 8;
constexpr uint32_t kQueryThreads = 64;
constexpr uint32_t kTileRows = 128;
constexpr uint32_t kMaxWidth = 128;
constexpr uint32_t kMaxStages = 12;
constexpr uint32_t kDynamicBytes = 227 * 1024 - 20 * 1024;        // beside the static part
constexpr uint32_t kTmemColumns = 512;          // S of A and B: 0, 128; O of A and B: 256, 384
constexpr uint32_t kMaskWords = kMaxTreeNodes / 32;
constexpr float kRescale = 8.0f;                // in powers of two
// Bounds of the waits: about a second, and a quarter of a minute where the other side may be
// computing special rows again.
constexpr long long kWaitCycles = 1ll << 31, kLongWaitCycles = 1ll << 35;

__device__ unsigned int g_attention_timeouts;

struct TcParams {
    AttnParams a;
    float scale_log2;           // scale * log2(e)
    uint32_t stages;
    // packed
    uint32_t pack, tile_rows;   // heads per tile, rows per head of a tile
    uint32_t head_tiles;        // tiles side by side: Hq / pack
    // tree
    uint32_t members;           // (head, node) pairs per key/value head
    uint32_t lane_shift;        // workers: lanes B's rows sit higher
    uint32_t ranges;            // of token blocks: one per CTA, or two
    uint32_t query_buffers;     // one, or two where they fit
    uint32_t pairs;             // tile pairs per key/value head
    uint32_t row_cap;           // rows of one partial
    uint32_t set_cost, cut;     // see set_length
    uint64_t slot_floats;       // floats of one partial: row_cap * (D + 2), a multiple of eight
    float* partial;             // [ranges * 2][slot_floats]: O [row_cap][D], m, l
};

// ---- barriers, copies, tensor memory ---------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_address(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ bool bar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(shared_address(bar)), "r"(parity) : "memory");
    return done != 0;
}
// True when the phase completed; false when this wait or another of the CTA gave up.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* stop,
                                         long long limit = kWaitCycles) {
    if (bar_test(bar, parity)) return true;
    const long long start = clock64();
    do {
        if (bar_test(bar, parity)) return true;
        if (*stop != 0) return false;
    } while (clock64() - start < limit);
    *stop = 1;
    return false;
}
// Whether any of the query warps' threads says so; a barrier for them.
__device__ __forceinline__ bool any_query_thread(bool mine) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred mine, any;\n\tsetp.ne.u32 mine, %2, 0;\n\t"
                 "barrier.cta.red.or.pred any, 1, %1, mine;\n\tselp.u32 %0, 1, 0, any;\n\t}"
                 : "=r"(any) : "n"(kQueryThreads), "r"(mine ? 1u : 0u) : "memory");
    return any != 0;
}
__device__ __forceinline__ void copy16(uint32_t shared, const void* global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
}
__device__ __forceinline__ void copies_done() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// 128 tokens x D of one plane: tile rows [tile_row, tile_row + 8), every tile column.
__device__ __forceinline__ void copy_block(uint32_t dst, const CUtensorMap* map, uint64_t* bar, uint32_t tile_row,
                                           uint32_t plane) {
    asm volatile(
            "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %3, %4, %3, %5}], [%2];"
            ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(shared_address(bar)), "r"(0u), "r"(tile_row), "r"(plane)
            : "memory");
}

__device__ __forceinline__ void tmem_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_load32(uint32_t address, uint32_t* r) {
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
            "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
              "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
              "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(address));
}
__device__ __forceinline__ void tmem_store32(uint32_t address, const uint32_t* r) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
            "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
            ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
              "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
              "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
              "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
              "r"(address)
            : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t address, uint32_t* r) {
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(address));
}
__device__ __forceinline__ void tmem_store16(uint32_t address, const uint32_t* r) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
            ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
              "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
              "r"(address)
            : "memory");
}

// Shared-memory operand with 32-byte swizzle. Groups of eight 32-byte rows lie 256 bytes apart
// (stride offset); the leading offset is the distance of neighbouring 16-column pieces and only
// the MN-major operand (V) uses it.
__device__ __forceinline__ uint64_t operand_descriptor(uint32_t address, uint32_t leading_bytes) {
    return static_cast<uint64_t>((address & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(leading_bytes >> 4) << 16)
            | (static_cast<uint64_t>(256u >> 4) << 32) | (1ull << 46) | (6ull << 61);
}
// FP32 accumulators, A and B of one 16-bit format, M = 128, N = n; b_mn: B is MN-major.
__device__ __forceinline__ uint32_t product_descriptor(uint32_t format, uint32_t n, bool b_mn) {
    return (1u << 4) | (format << 7) | (format << 10) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17)
            | ((kTileRows >> 4) << 24);
}
// The warp that issues runs as a whole, on values that are the same in every lane, and one lane's
// predicate guards each instruction: their operands then stay in uniform registers. (Issued inside
// a one-lane branch an instruction took 85 cycles, more than many of them compute.)
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t mine;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(mine));
    return mine;
}
__device__ __forceinline__ void mma_shared(uint32_t lane, uint32_t d, uint64_t a, uint64_t b, uint32_t kind, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(kind), "r"(accumulate), "r"(lane) : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t lane, uint32_t d, uint32_t a, uint64_t b, uint32_t kind, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(kind), "r"(accumulate), "r"(lane) : "memory");
}
// The barrier is reached when every matrix instruction issued so far has completed.
__device__ __forceinline__ void mma_commit(uint32_t lane, uint64_t* bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                 ::"r"(shared_address(bar)), "r"(lane) : "memory");
}

// Packed binary32 pairs: one instruction per two values.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

enum Mode : int { kPacked, kShared, kWorkers };

// ---- the work of one CTA -----------------------------------------------------------------------------

// A run of token blocks of one row set (a tile pair).
struct Piece {
    uint32_t b, kv_head, pair;  // sequence, key/value head, tile pair
    uint32_t first_token;       // multiple of 16: the first block's first row of k and v
    uint32_t blocks;            // blocks of 128 tokens; none: there are no more pieces
    uint32_t steps[2];          // blocks per tile
    uint32_t seen[2];           // tokens from first_token on, beyond which no row of the tile sees
    uint32_t end;               // rows of the sequence end here (packed), live rows (tree)
    uint32_t row0;              // packed: first row of tile A
    uint32_t start;             // packed: first row of the sequence; tree: rows before the tree
    uint32_t nodes;
    uint32_t whole;             // tree: every block of the row set lies in this piece
    uint32_t slot;              // tree: which of the CTA's partials
};

__device__ __forceinline__ uint32_t tree_blocks(const TreeExtent& e) {
    return e.nodes == 0 ? 0 : (e.length + e.nodes + kKvBlock - 1) / kKvBlock;
}
// Length of a row set when ranges are cut: its blocks, behind `set_cost` more that stand for the change
// to it from another set (queries, first scores, results). Where sets stay whole it is one place.
__device__ __forceinline__ uint32_t set_length(const TcParams& p, const TreeExtent& e) {
    const uint32_t blocks = tree_blocks(e);
    return blocks == 0 ? 0 : p.cut ? blocks + p.set_cost : 1;
}

// Walks the pieces of a range: sequences, then (head, pair), then places of the set.
struct Walk {
    uint32_t b, set, place;     // next piece begins here
    uint64_t left;              // places of the range not walked yet
};

__device__ __forceinline__ bool next_piece(const TcParams& p, Walk& w, Piece& out) {
    while (w.left != 0 && w.b < p.a.batch) {
        const TreeExtent e = tree_extent(p.a, w.b);
        const uint32_t blocks = tree_blocks(e), length = set_length(p, e);
        if (blocks == 0) {
            ++w.b;
            continue;
        }
        const uint32_t rest = length - w.place;
        const uint32_t take = w.left < rest ? static_cast<uint32_t>(w.left) : rest;
        const uint32_t begin = p.cut ? max(w.place, p.set_cost) - p.set_cost : 0;
        const uint32_t end = p.cut ? max(w.place + take, p.set_cost) - p.set_cost : blocks;
        out.b = w.b;
        out.kv_head = w.set / p.pairs;
        out.pair = w.set % p.pairs;
        w.left -= take;
        w.place += take;
        if (w.place == length) {
            w.place = 0;
            if (++w.set == p.a.hkv * p.pairs) {
                w.set = 0;
                ++w.b;
            }
        }
        if (begin == end) continue;
        out.first_token = begin * kKvBlock;
        out.blocks = out.steps[0] = out.steps[1] = end - begin;
        out.end = e.length + e.nodes;
        out.seen[0] = out.seen[1] = out.end - out.first_token;
        out.row0 = 0;
        out.start = e.length;
        out.nodes = e.nodes;
        out.whole = begin == 0 && end == blocks ? 1u : 0u;
        out.slot = begin != 0 ? 0u : 1u;
        return true;
    }
    return false;
}

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// Range [total * cta / ctas, total * (cta + 1) / ctas) of places.
__device__ __forceinline__ uint64_t range_begin(uint64_t total, uint32_t cta, uint32_t ctas) {
    if (total < (1u << 22) && ctas < 1024) return static_cast<uint32_t>(total) * cta / ctas;   // (short division)
    return total * cta / ctas;
}

// One warp: where range `cta` of `ctas` begins.
__device__ __forceinline__ Walk plan_walk(const TcParams& p, uint32_t cta, uint32_t ctas) {
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t sets = p.a.hkv * p.pairs;
    // (the first 32 sequences, often all, are read once)
    const uint32_t first_length = lane < p.a.batch ? set_length(p, tree_extent(p.a, lane)) : 0;
    uint64_t total = first_length;
    for (uint32_t b = lane + 32; b < p.a.batch; b += 32) total += set_length(p, tree_extent(p.a, b));
    total = warp_sum64(total) * sets;
    const uint64_t begin = range_begin(total, cta, ctas), end = range_begin(total, cta + 1, ctas);
    Walk w{0, 0, 0, end - begin};
    if (w.left == 0) return w;
    uint64_t before = 0;
    for (uint32_t base = 0; base < p.a.batch; base += 32) {
        const uint32_t b = base + lane;
        const uint32_t length = base == 0 ? first_length : b < p.a.batch ? set_length(p, tree_extent(p.a, b)) : 0;
        uint64_t run = static_cast<uint64_t>(length) * sets;
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t up = __shfl_up_sync(0xffffffffu, run, d);
            if (lane >= static_cast<uint32_t>(d)) run += up;
        }
        const uint64_t mine_end = before + run, mine_begin = mine_end - static_cast<uint64_t>(length) * sets;
        const uint32_t found = __ballot_sync(0xffffffffu, begin >= mine_begin && begin < mine_end);
        if (found != 0) {
            const int who = __ffs(found) - 1;
            const uint64_t first = __shfl_sync(0xffffffffu, mine_begin, who);
            const uint32_t n = __shfl_sync(0xffffffffu, length, who);
            w.b = base + who;
            w.set = static_cast<uint32_t>((begin - first) / n);
            w.place = static_cast<uint32_t>((begin - first) % n);
            return w;
        }
        before = __shfl_sync(0xffffffffu, mine_end, 31);
    }
    w.left = 0;     // not reached
    return w;
}

// One warp: the tile pair of this CTA in a packed call. Units run over the sequences, each one's
// row blocks from the last (the longest) to the first, heads innermost. False: nothing to do.
__device__ __forceinline__ bool plan_packed(const TcParams& p, uint32_t unit, Piece& out, bool& ok) {
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t step = 2 * p.tile_rows;
    const uint32_t head_tile = unit % p.head_tiles, wanted = unit / p.head_tiles;
    constexpr uint32_t kChunks = 4;
    uint32_t before = 0;
    bool have = false;
    ok = true;
    for (uint32_t base = 0; base < p.a.batch; base += 32 * kChunks) {
        uint32_t first[kChunks], last[kChunks];
#pragma unroll
        for (uint32_t c = 0; c < kChunks; ++c) {
            const uint32_t s = base + c * 32 + lane;
            first[c] = s < p.a.batch ? p.a.offsets[s] : 0;
            last[c] = s < p.a.batch ? p.a.offsets[s + 1] : 0;
        }
#pragma unroll
        for (uint32_t c = 0; c < kChunks; ++c) {
            ok = ok && first[c] <= last[c] && last[c] <= p.a.rows;
            const uint32_t rows = last[c] >= first[c] ? last[c] - first[c] : 0;
            const uint32_t blocks = rows / step + (rows % step != 0 ? 1u : 0u);
            uint32_t run = blocks;
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, run, d);
                if (lane >= static_cast<uint32_t>(d)) run += up;
            }
            const uint32_t mine_end = before + run, mine_begin = mine_end - blocks;
            const uint32_t found = __ballot_sync(0xffffffffu, wanted >= mine_begin && wanted < mine_end);
            if (found != 0 && !have) {
                const int who = __ffs(found) - 1;
                have = true;
                out.start = __shfl_sync(0xffffffffu, first[c], who);
                out.end = __shfl_sync(0xffffffffu, last[c], who);
                out.row0 = out.start + __shfl_sync(0xffffffffu, mine_end - 1 - wanted, who) * step;
            }
            before = __shfl_sync(0xffffffffu, mine_end, 31);
        }
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok || !have) return false;
    out.b = 0;
    out.kv_head = head_tile * p.pack / p.a.group;
    out.pair = head_tile;
    out.first_token = out.start / kTile * kTile;
    for (uint32_t x = 0; x < 2; ++x) {
        const uint32_t row = out.row0 + x * p.tile_rows;
        const uint32_t last = min(out.end, row + p.tile_rows);      // one behind the tile's last row
        out.seen[x] = row < out.end ? last - out.first_token : 0;
        out.steps[x] = (out.seen[x] + kKvBlock - 1) / kKvBlock;
    }
    out.blocks = max(out.steps[0], out.steps[1]);
    out.nodes = 0;
    out.whole = 1;
    out.slot = 0;
    return true;
}

// Bits c of a word with low <= c <= high.
__device__ __forceinline__ uint32_t range_word(int32_t low, int32_t high) {
    const uint32_t up = high >= 31 ? 0xFFFFFFFFu : high < 0 ? 0u : (2u << high) - 1u;
    const uint32_t down = low <= 0 ? 0xFFFFFFFFu : low > 31 ? 0u : 0xFFFFFFFFu << low;
    return up & down;
}

// Bits of 32 tokens in the order in which the operands hold them. The copy's 128-byte swizzle is an
// exclusive-or of address bits 4, 5, 6 with bits 7, 8, 9; inside [tile row][16 rows][32 bytes] these are
// the 16-byte half and bits 0, 1 of the row with bits 2, 3 of the row and bit 0 of the tile row. The
// first is the 32-byte swizzle the matrix instruction undoes. The other two permute the rows of a
// tile, for K and V alike: products and sums do not change, but the token of a column of S does.
__device__ __forceinline__ uint32_t block_order(uint32_t tokens) {
    // rows 8-15 of each tile: bit 0 of the row flips
    uint32_t w = (tokens & 0x00FF00FFu) | ((tokens & 0x55005500u) << 1) | ((tokens >> 1) & 0x55005500u);
    // odd tile rows: bit 1 flips
    return (w & 0x0000FFFFu) | ((w & 0x33330000u) << 2) | ((w >> 2) & 0x33330000u);
}

// attend_row for one row of a tree or packed call, out of line: rare.
template <class Leaf, bool TREE>
__device__ __noinline__ void redo_row(const AttnParams& p, uint32_t b, uint32_t h, uint32_t row, uint32_t start) {
    if constexpr (TREE) {
        const int32_t* parents = p.parents != nullptr ? p.parents + static_cast<uint64_t>(b) * p.rows : nullptr;
        attend_row<Leaf>(p, b, h, row, TreeRow{start, row, parents});
    } else {
        attend_row<Leaf>(p, b, h, row, CausalRows{start, row});
    }
}

struct Shared {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t scores[2], weights[2][2], done[2]; // per tile: S written, P written (halves), O complete
    uint64_t landed[2];                         // per copying warp: values to be cleaned are there
    // Per worker and buffer (one worker but with kWorkers):
    uint64_t queries[2][2], queries_free[2][2]; // a piece's queries are there; its scores are computed
    uint64_t piece_free[2][2];                  // nobody reads the piece any more
    uint64_t drain[2];
    uint32_t tmem, stop, run;
    Piece pieces[2][2];
    Walk walk[2];
    uint32_t mask[2][kMaxTreeNodes * kMaskWords];       // per buffer (workers: the first or second half of it):
                                                        // a node's ancestors and itself
    int16_t parent[2][kMaxTreeNodes];
};

template <class Leaf, Mode MODE>
__global__ void __launch_bounds__(kThreads, 1)
attention_tc_kernel(const __grid_constant__ TcParams p, const __grid_constant__ CUtensorMap k_map,
                    const __grid_constant__ CUtensorMap v_map) {
    constexpr bool TREE = MODE != kPacked, WORKERS = MODE == kWorkers;
    extern __shared__ __align__(1024) unsigned char dynamic[];
    __shared__ Shared sh;
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u;     // (the warp: a uniform value)
    const uint32_t width = p.a.width, slices = width / kTile;
    const uint32_t block_bytes = width * kTileRows * 2;         // a Q tile, a K block, a V block
    // Queries [buffer][tile], then the ring. The dynamic part starts behind the static one: round up
    // to the swizzle's alignment.
    const uint32_t q_base = (shared_address(dynamic) + 1023u) & ~1023u;
    const uint32_t ring = q_base + p.query_buffers * 2 * block_bytes;
    volatile uint32_t* const stop = &sh.stop;

    if (warp == 0) {
        if constexpr (TREE) {
            const uint32_t range = WORKERS ? blockIdx.x * 2 : blockIdx.x;
            const Walk w = plan_walk(p, range, p.ranges);
            if (lane == 0) {
                sh.walk[0] = w;
                sh.run = 1;
            }
        } else {
            Piece piece;
            bool ok;
            const bool run = plan_packed(p, blockIdx.x, piece, ok);
            if (lane == 0) {
                sh.pieces[0][0] = piece;
                sh.run = run;
                if (blockIdx.x == 0) *p.a.status = ok ? 0u : 1u;
            }
        }
    } else if (WORKERS && warp == 4) {
        const Walk w = plan_walk(p, blockIdx.x * 2 + 1, p.ranges);
        if (lane == 0) sh.walk[1] = w;
    } else if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(shared_address(&sh.tmem)), "r"(kTmemColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else if (warp == 9 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&k_map)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&v_map)) : "memory");
        for (uint32_t i = 0; i < kMaxStages; ++i) {
            bar_init(&sh.full[i], 1);
            bar_init(&sh.empty[i], 1);
        }
        for (uint32_t x = 0; x < 2; ++x) {
            bar_init(&sh.scores[x], 1);
            bar_init(&sh.weights[x][0], 4);
            bar_init(&sh.weights[x][1], 4);
            bar_init(&sh.done[x], 1);
            for (uint32_t i = 0; i < 2; ++i) {
                bar_init(&sh.queries[x][i], MODE == kPacked ? kSoftmaxWarps : MODE == kShared ? 2 : 1);
                bar_init(&sh.queries_free[x][i], 1);
                bar_init(&sh.piece_free[x][i], WORKERS ? 4 : kSoftmaxWarps);
            }
            bar_init(&sh.drain[x], 1);
            bar_init(&sh.landed[x], 1);
        }
        sh.stop = 0;
        // The status begins at zero and only grows: 1 from this CTA's check of the arguments, 2 from a CTA
        // in which a wait gave up (a second after its start at the least, and the first CTA starts first).
        if (TREE && blockIdx.x == 0) *p.a.status = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tmem_before_sync();
    __syncthreads();
    tmem_after_sync();
    if constexpr (TREE) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = sh.tmem;
    const bool run = sh.run != 0;
    if (warp < kSoftmaxWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");

    // A node's ancestor words. With workers a tree has at most 128 nodes: half the room each.
    constexpr uint32_t mask_words = WORKERS ? kMaskWords / 2 : kMaskWords;
    auto tree_mask = [&](uint32_t buffer, uint32_t worker) {
        return sh.mask[buffer] + (WORKERS ? worker * (kMaxTreeNodes / 2) * mask_words : 0u);
    };
    // Publishes a piece (none: the end) with its queries and ancestor masks; `threads` threads.
    auto bring_queries = [&](uint32_t turn, bool go, Piece& piece, uint32_t worker, uint32_t thread, uint32_t threads, bool& alive) {
        if constexpr (TREE) {
            auto meet = [&] {
                if constexpr (WORKERS) __syncwarp();
                else asm volatile("bar.sync 1, 64;" ::: "memory");
            };
            const uint32_t buffer = turn & 1u;
            if (!go) piece.blocks = 0;
            // The piece two turns back is out of use, and the queries that lie where these go.
            if (turn >= 2) alive = bar_wait(&sh.piece_free[worker][buffer], (turn / 2 - 1) & 1u, stop, kLongWaitCycles);
            const uint32_t place = p.query_buffers == 2 ? buffer : 0u;
            const uint32_t used = p.query_buffers == 2 ? turn / 2 : turn;      // times the place was filled
            if (go && used > 0) {
                alive = alive && bar_wait(&sh.queries_free[worker][place], (used - 1) & 1u, stop, kLongWaitCycles);
            }
            // (all threads go on or all give up)
            if constexpr (WORKERS) alive = __all_sync(0xffffffffu, alive);
            else alive = !any_query_thread(!alive);
            if (!alive) return;
            if (thread == 0) sh.pieces[worker][buffer] = piece;
            if (go) {
                if (p.a.parents != nullptr && piece.first_token + piece.blocks * kKvBlock > piece.start) {
                    const int32_t* parents = p.a.parents + static_cast<uint64_t>(piece.b) * p.a.rows;
                    for (uint32_t i = thread; i < piece.nodes; i += threads) {
                        sh.parent[worker][i] = static_cast<int16_t>(max(-1, tree_parent(parents, static_cast<int32_t>(i))));
                    }
                    meet();
                    for (uint32_t i = thread; i < piece.nodes; i += threads) {
                        uint32_t* words = tree_mask(buffer, worker) + i * mask_words;
                        for (uint32_t w = 0; w < mask_words; ++w) words[w] = 0;
                        for (int32_t at = static_cast<int32_t>(i); at >= 0; at = sh.parent[worker][at]) {
                            words[at / 32] |= 1u << (at % 32);
                        }
                    }
                }
                // Rows of the set, 32 bytes of a tile row at a time; what the rows beside them hold
                // reaches only results nobody stores.
                const uint32_t offset = piece.pair * 256;
                const uint32_t rows = min(WORKERS ? kTileRows : 2 * kTileRows, p.members - offset);
                const uint32_t base = q_base + (place * 2 + worker) * block_bytes;
                for (uint32_t r = thread; r < rows; r += threads) {
                    const uint32_t of_head = offset + r, q_head = piece.kv_head * p.a.group + of_head / p.a.rows;
                    const unsigned char* src = attn_piece(p.a.q, attn_plane(p.a.q, piece.b, q_head), of_head % p.a.rows, 0);
                    const uint32_t at = WORKERS ? r + worker * p.lane_shift : r;
                    const uint32_t m = at % kTileRows, flip = ((m >> 2) & 1u) * 16;
                    uint32_t to = base + (at / kTileRows) * block_bytes + m * 32;
                    for (uint32_t c = 0; c < slices; ++c, to += 4096, src += kTileSlots * 2) {
                        copy16(to + flip, src);
                        copy16(to + (16 - flip), src + 16);
                    }
                }
                copies_done();
            }
            meet();
            if (lane == 0) bar_arrive(&sh.queries[worker][buffer]);
        }
    };

    if (run && warp < kSoftmaxWarps) {
        // ---- softmax, one thread per row ---------------------------------------------------------------
        const uint32_t x = warp / 4, m = (warp & 3u) * 32 + lane;
        const uint32_t lanes = (warp & 3u) << 21;               // this warp's 32 tensor memory lanes
        const uint32_t s_at = tmem + lanes + x * 128, o_at = tmem + lanes + 256 + x * 128;
        const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
        const uint32_t me = WORKERS ? x : 0, shift_lanes = WORKERS ? x * p.lane_shift : 0u;
        uint32_t steps_done = 0, pieces_done = 0;               // of this tile, over all pieces
        uint32_t head = 0, row = 0, member = m - shift_lanes;   // (lanes below the shift: a huge number, no row)
        if constexpr (WORKERS) {
            head = member / p.a.rows;
            row = member % p.a.rows;
        }
        bool alive = true;
        for (uint32_t turn = 0; ; ++turn) {
            const uint32_t buffer = TREE ? turn & 1u : 0u;
            if constexpr (TREE) {
                alive = __all_sync(0xffffffffu, bar_wait(&sh.queries[me][buffer], (turn / 2) & 1u, stop, kLongWaitCycles));
                if (!alive) break;
            }
            const Piece& piece = sh.pieces[me][buffer];
            if (piece.blocks == 0) break;
            const uint32_t n = piece.steps[x], start = piece.start;
            // This thread's row.
            uint32_t q_head;
            bool valid;
            if constexpr (TREE) {
                if constexpr (!WORKERS) {
                    member = piece.pair * 256 + x * 128 + m;
                    head = member / p.a.rows;
                    row = member % p.a.rows;
                }
                q_head = piece.kv_head * p.a.group + head;
                valid = member < p.members && row < piece.nodes;
            } else {
                q_head = piece.pair * p.pack + m / p.tile_rows;
                row = piece.row0 + x * p.tile_rows + m % p.tile_rows;
                valid = row < piece.end;
            }
            const bool busy = __any_sync(0xffffffffu, valid) && n != 0;
            if constexpr (!TREE) {
                // Q, 32 bytes of a tile row at a time, into the swizzled K-major operand. (What the rows
                // that are not there hold reaches only results nobody stores.)
                if (valid && n != 0) {
                    const uint64_t plane = attn_plane(p.a.q, piece.b, q_head);
                    const unsigned char* src = attn_piece(p.a.q, plane, row, 0);
                    uint32_t to = q_base + x * block_bytes + m * 32;
                    const uint32_t flip = ((m >> 2) & 1u) * 16;
                    for (uint32_t c = 0; c < slices; ++c, to += 4096, src += kTileSlots * 2) {
                        copy16(to + flip, src);
                        copy16(to + (16 - flip), src + 16);
                    }
                }
                copies_done();
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.queries[0][0]);
            }

            const float kNone = __int_as_float(0xFF800000);
            // Running maximum (of S), what is added to scaled scores, and sum. Maxima are compared scaled: the
            // difference of two scores may overflow where that of the scaled ones does not.
            float top = kNone, shift = 0.0f, sum = 0.0f;
            const uint32_t first = piece.first_token;
            // Tokens from here on may be hidden from some row of the tile.
            const uint32_t clear = TREE ? start : piece.row0 + x * p.tile_rows + 1;
            for (uint32_t step = 0; step < n; ++step, ++steps_done) {
                // (one answer per warp)
                alive = __all_sync(0xffffffffu, bar_wait(&sh.scores[x], steps_done & 1u, stop, kLongWaitCycles));
                if (!alive) break;
                tmem_after_sync();
                if (busy) {
                    uint32_t s[kKvBlock];
#pragma unroll
                    for (int c = 0; c < static_cast<int>(kKvBlock); c += 32) tmem_load32(s_at + c, s + c);
                    const uint32_t token = first + step * kKvBlock;
                    tmem_wait_load();
                    if (token + kKvBlock > clear || (!TREE && token < start)) {
                        uint32_t see[kKvBlock / 32];
#pragma unroll
                        for (int w = 0; w < static_cast<int>(kKvBlock / 32); ++w) {
                            const int32_t from = static_cast<int32_t>(token) + 32 * w;
                            if constexpr (!TREE) {
                                see[w] = range_word(static_cast<int32_t>(start) - from, static_cast<int32_t>(row) - from);
                            } else if (p.a.parents == nullptr) {
                                see[w] = range_word(0, static_cast<int32_t>(start + row) - from);
                            } else {
                                see[w] = range_word(0, static_cast<int32_t>(start) - 1 - from);
                                const int32_t rel = from - static_cast<int32_t>(start);
                                if (valid && rel > -32 && rel < static_cast<int32_t>(mask_words * 32)) {
                                    const uint32_t* words = tree_mask(buffer, x) + row * mask_words;
                                    if (rel < 0) {
                                        see[w] |= words[0] << -rel;
                                    } else {
                                        const uint32_t i = rel / 32;
                                        see[w] |= __funnelshift_r(words[i], i + 1 < mask_words ? words[i + 1] : 0u, rel % 32);
                                    }
                                }
                            }
                            see[w] = valid ? block_order(see[w]) : 0u;
                        }
#pragma unroll
                        for (int c = 0; c < static_cast<int>(kKvBlock); ++c) {
                            if (!((see[c / 32] >> (c % 32)) & 1u)) s[c] = 0xFF800000u;
                        }
                    }
                    float best[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) best[i] = fmaxf(__uint_as_float(s[i]), __uint_as_float(s[i + 4]));
#pragma unroll
                    for (int c = 8; c < static_cast<int>(kKvBlock); c += 8) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            best[i] = fmaxf(fmaxf(best[i], __uint_as_float(s[c + i])), __uint_as_float(s[c + i + 4]));
                        }
                    }
                    const float high = fmaxf(top, fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3])));
                    // The first tokens seen, or a maximum that grew beyond what P may: a new reference.
                    const bool fresh = top == kNone;
                    const float next = Leaf::kWeightLog - high * p.scale_log2, rise = shift - next;
                    const bool grow = !fresh && rise > kRescale;
                    if (__any_sync(0xffffffffu, grow)) {
                        // (not the first step; these scores came behind the products of the steps before)
                        const float factor = grow ? exp2_fast(-rise) : 1.0f;
                        sum *= factor;
                        for (uint32_t c = 0; c < slices; ++c) {
                            uint32_t o[16];
                            tmem_load16(o_at + c * 16, o);
                            tmem_wait_load();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                            tmem_store16(o_at + c * 16, o);
                        }
                    }
                    if (fresh || grow) {
                        top = high;
                        shift = high == kNone ? 0.0f : next;
                    }
                    const uint64_t shift2 = pair(shift, shift);
                    uint64_t sums[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t* const from = s + half * 64;
#pragma unroll
                        for (int c = 0; c < 64; c += 2) {
                            float e0, e1;
                            unpair(fma2(pair(__uint_as_float(from[c]), __uint_as_float(from[c + 1])), scale2, shift2), e0, e1);
                            e0 = exp2_fast(e0);
                            e1 = exp2_fast(e1);
                            sums[(c / 2) % 4] = add2(sums[(c / 2) % 4], pair(e0, e1));
                            from[c / 2] = Leaf::pack(e0, e1);
                        }
                        tmem_store32(s_at + half * 32, from);
                        if (half == 1) {
                            float a, b;
                            unpair(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])), a, b);
                            sum += a + b;
                        }
                        tmem_wait_store();
                        tmem_before_sync();
                        __syncwarp();
                        if (lane == 0) bar_arrive(&sh.weights[x][half]);
                    }
                } else {
                    tmem_before_sync();
                    if (lane == 0) {
                        bar_arrive(&sh.weights[x][0]);
                        bar_arrive(&sh.weights[x][1]);
                    }
                }
            }
            if (alive && n != 0) {
                alive = __all_sync(0xffffffffu, bar_wait(&sh.done[x], pieces_done & 1u, stop, kLongWaitCycles));
                ++pieces_done;
                tmem_after_sync();
            }
            // ---- results ---------------------------------------------------------------------------
            if (alive && busy) {
                const bool whole = !TREE || piece.whole;
                const float inverse = whole ? 1.0f / sum : 1.0f;
                const uint64_t plane = attn_plane(p.a.out, piece.b, 0);
                const uint32_t column = q_head * slices, local = WORKERS ? member : x * 128 + m;
                float* const slot = p.partial + static_cast<uint64_t>((WORKERS ? blockIdx.x * 2 + x : blockIdx.x) * 2 + piece.slot) * p.slot_floats;
                const uint64_t inverse2 = pair(inverse, inverse);
                uint64_t zero = 0;                  // turns NaN when a result is not finite
                for (uint32_t c = 0; c < slices; c += 2) {
                    // (32 columns at a time; those behind the head's width are not used)
                    uint32_t o[32];
                    tmem_load32(o_at + c * 16, o);
                    tmem_wait_load();
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (c + half >= slices) break;
                        uint32_t* const part = o + 16 * half;
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const uint64_t v = mul2(pair(__uint_as_float(part[i]), __uint_as_float(part[i + 1])), inverse2);
                            zero = fma2(v, 0, zero);
                            float lo, hi;
                            unpair(v, lo, hi);
                            part[i] = __float_as_uint(lo);
                            part[i + 1] = __float_as_uint(hi);
                        }
                        if (!valid) continue;
                        if (whole) {
                            uint32_t packed[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                packed[i] = Leaf::plus_zero(Leaf::pack(__uint_as_float(part[2 * i]), __uint_as_float(part[2 * i + 1])));
                            }
                            store_u8_stream(attn_out_piece(p.a.out, plane, row, column + c + half),
                                            make_uint4(packed[0], packed[1], packed[2], packed[3]),
                                            make_uint4(packed[4], packed[5], packed[6], packed[7]));
                        } else {
                            uint4* to = reinterpret_cast<uint4*>(slot + static_cast<uint64_t>(local) * width + (c + half) * 16);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                to[i] = make_uint4(part[4 * i], part[4 * i + 1], part[4 * i + 2], part[4 * i + 3]);
                            }
                        }
                    }
                }
                float zero_lo, zero_hi;
                unpair(zero, zero_lo, zero_hi);
                const bool bad = !(sum > 0.0f && sum <= 3.0e38f) || zero_lo != 0.0f || zero_hi != 0.0f;
                if (whole) {
                    // Rows with a result that is not finite: once more, behind the stores.
                    uint32_t again = __ballot_sync(0xffffffffu, bad && valid);
                    while (again != 0) {
                        const int who = __ffs(again) - 1;
                        again &= again - 1;
                        __syncwarp();
                        redo_row<Leaf, TREE>(p.a, piece.b, __shfl_sync(0xffffffffu, q_head, who),
                                             __shfl_sync(0xffffffffu, row, who), start);
                    }
                } else if (valid) {
                    slot[static_cast<uint64_t>(p.row_cap) * width + local] = top;
                    slot[static_cast<uint64_t>(p.row_cap) * (width + 1) + local] = sum;
                }
            }
            if constexpr (!TREE) break;
            tmem_before_sync();
            if (!alive) break;
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.piece_free[me][buffer]);
        }
    } else if (run && (warp == 8 || (WORKERS && warp == 9))) {
        // ---- matrix instructions ---------------------------------------------------------------------
        const uint32_t me = WORKERS ? warp - 8 : 0u;        // (workers: also the tile)
        const uint32_t leader = elect_lane();
        const uint32_t kind_s = product_descriptor(Leaf::kFormat, kKvBlock, false);
        const uint32_t kind_o = product_descriptor(Leaf::kFormat, width, true);
        const uint32_t columns = __shfl_sync(0xffffffffu, tmem, 0);
        const uint32_t stages = WORKERS ? p.stages / 2 : p.stages, stage0 = WORKERS ? me * stages : 0u;
        uint32_t slot = 0, round = 0;               // next ring slot, and its phase
        uint32_t weighed[2] = {0, 0};               // steps of each tile, over all pieces
        bool alive = true;
        auto reach = [&](uint64_t* bar, uint32_t phase, long long limit) {
            alive = __all_sync(0xffffffffu, bar_wait(bar, phase & 1u, stop, limit));
        };
        for (uint32_t turn = 0; ; ++turn) {
            const uint32_t buffer = TREE ? turn & 1u : 0u;
            reach(&sh.queries[me][buffer], turn / 2, kLongWaitCycles);
            if (!alive) break;
            tmem_after_sync();
            const uint32_t blocks = __shfl_sync(0xffffffffu, sh.pieces[me][buffer].blocks, 0);
            if (blocks == 0) break;
            const uint32_t steps0 = __shfl_sync(0xffffffffu, sh.pieces[me][buffer].steps[0], 0);
            const uint32_t steps1 = __shfl_sync(0xffffffffu, sh.pieces[me][buffer].steps[1], 0);
            const uint32_t seen0 = __shfl_sync(0xffffffffu, sh.pieces[me][buffer].seen[0], 0);
            const uint32_t seen1 = __shfl_sync(0xffffffffu, sh.pieces[me][buffer].seen[1], 0);
            const uint32_t place = TREE && p.query_buffers == 2 ? buffer : 0u;
            const uint64_t queries = operand_descriptor(q_base + place * 2 * block_bytes, 0);
            uint32_t k_slot = 0, v_slot = 0;
            auto take = [&](uint32_t& at) {
                at = stage0 + slot;
                reach(&sh.full[at], round, kWaitCycles);
                if (++slot == stages) { slot = 0; ++round; }
            };
            // S of tile x = Q K^T
            auto score = [&](uint32_t x) {
                uint64_t k = operand_descriptor(ring + k_slot * block_bytes, 0);
                uint64_t rows = queries + x * (block_bytes >> 4);
                for (uint32_t c = 0; c < slices; ++c) {
                    mma_shared(leader, columns + x * 128, rows, k, kind_s, c);
                    rows += 4096 >> 4;
                    k += 4096 >> 4;
                }
                mma_commit(leader, &sh.scores[x]);
            };
            // O of tile x += P V, each half of P as it comes; not the tiles of 16 tokens that no row sees
            auto weigh = [&](uint32_t x, uint32_t phase, uint32_t step, bool last) {
                const uint64_t v = operand_descriptor(ring + v_slot * block_bytes, 4096);
                const uint32_t seen = (x == 0 ? seen0 : seen1) - step * kKvBlock;
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half) {
                    reach(&sh.weights[x][half], phase, kLongWaitCycles);
                    if (!alive) return;
                    tmem_after_sync();
                    auto product = [&](uint32_t t) {
                        mma_tensor(leader, columns + 256 + x * 128, columns + x * 128 + t * 8, v + t * (512 >> 4), kind_o, step + t);
                    };
                    if (seen >= (half + 1) * 64) {
#pragma unroll
                        for (uint32_t t = 0; t < 4; ++t) product(half * 4 + t);
                    } else {
                        for (uint32_t t = half * 4; t * kTile < seen; ++t) product(t);
                    }
                }
                if (last) mma_commit(leader, &sh.done[x]);
            };
            take(k_slot);
            if (!alive) break;
            if constexpr (WORKERS) {
                score(me);
                mma_commit(leader, &sh.empty[k_slot]);
                if (blocks == 1) mma_commit(leader, &sh.queries_free[me][place]);
                for (uint32_t i = 0; i < blocks; ++i) {
                    take(v_slot);
                    if (!alive) break;
                    weigh(me, weighed[0]++, i, i + 1 == blocks);
                    if (!alive) break;
                    mma_commit(leader, &sh.empty[v_slot]);
                    if (i + 1 == blocks) break;
                    take(k_slot);
                    if (!alive) break;
                    score(me);
                    mma_commit(leader, &sh.empty[k_slot]);
                    if (i + 2 == blocks) mma_commit(leader, &sh.queries_free[me][place]);
                }
            } else {
                const uint32_t most = max(steps0, steps1);
                if (steps0 != 0) score(0);
                if (steps1 != 0) score(1);
                mma_commit(leader, &sh.empty[k_slot]);
                if (TREE && most == 1) mma_commit(leader, &sh.queries_free[0][place]);
                for (uint32_t i = 0; i < most && alive; ++i) {
                    take(v_slot);
                    bool keys = false;          // (the next keys come behind these values: the order of the copies)
#pragma unroll
                    for (uint32_t x = 0; x < 2; ++x) {
                        const uint32_t steps = x == 0 ? steps0 : steps1;
                        if (i >= steps || !alive) continue;
                        weigh(x, weighed[x]++, i, i + 1 == steps);
                        if (!alive || i + 1 == steps) continue;
                        if (!keys) take(k_slot);
                        keys = true;
                        if (alive) score(x);
                    }
                    if (!alive) break;
                    mma_commit(leader, &sh.empty[v_slot]);
                    if (keys) mma_commit(leader, &sh.empty[k_slot]);
                    if (TREE && i + 2 == most) mma_commit(leader, &sh.queries_free[0][place]);
                }
            }
            if (!TREE || !alive) break;
        }
        if (!alive) {
            // Instructions still in flight end before the tensor memory is given back.
            mma_commit(leader, &sh.drain[me]);
            const long long start = clock64();
            while (!bar_test(&sh.drain[me], 0) && clock64() - start < kWaitCycles) {}
        }
        __syncwarp();
    } else if (run && ((!WORKERS && warp == 9) || (WORKERS && warp >= 10))) {
        // ---- copies of keys and values (workers: and the queries) -----------------------------------------
        const uint32_t me = WORKERS ? warp - 10 : 0u;
        const uint32_t stages = WORKERS ? p.stages / 2 : p.stages, stage0 = WORKERS ? me * stages : 0u;
        uint32_t issued = 0, filled = 0, cleaned = 0;   // (filled: lane 0, copies under way or done)
        bool alive = true;
        Walk walk = sh.walk[me];
        Piece piece = sh.pieces[0][0];
        for (uint32_t turn = 0; alive; ++turn) {
            bool go = TREE ? next_piece(p, walk, piece) : turn == 0;
            if (!WORKERS && !go) break;
            const uint32_t k_plane = go ? static_cast<uint32_t>(attn_plane(p.a.k, piece.b, piece.kv_head)) : 0u;
            const uint32_t v_plane = go ? static_cast<uint32_t>(attn_plane(p.a.v, piece.b, piece.kv_head)) : 0u;
            const uint32_t first = piece.first_token / kTile;
            // Values beside the sequence, in a tile of 16 tokens that it begins or ends in, become zeros: what
            // such rows hold (a cache is rarely set up before use) would make every result NaN, by way of
            // 0 x NaN, and every row be computed again, one at a time: 32 single-token decodes over caches
            // with NaN behind the live rows took 5065 us instead of 25, and take 26 with the zeros.
            const uint32_t lead = TREE ? 0u : piece.start - piece.first_token, live = piece.end - piece.first_token;
            auto fetch = [&](bool keys, uint32_t block) {
                const uint32_t slot = stage0 + issued % stages, to = ring + slot * block_bytes;
                const uint32_t low = block == 0 ? lead : 0u, high = min(kKvBlock, live - block * kKvBlock);
                const bool clean = !keys && (low != 0 || high % kTile != 0);
                if (lane == 0) {
                    if (issued >= stages) {
                        alive = alive && bar_wait(&sh.empty[slot], (issued / stages - 1) & 1u, stop, kLongWaitCycles);
                    }
                    if (alive) {
                        uint64_t* const bar = clean ? &sh.landed[me] : &sh.full[slot];
                        bar_expect(bar, block_bytes);
                        copy_block(to, keys ? &k_map : &v_map, bar, first + block * (kKvBlock / kTile), keys ? k_plane : v_plane);
                        filled = issued + 1;
                    }
                }
                ++issued;
                if (!clean) return;
                alive = __all_sync(0xffffffffu, alive);
                if (!alive) return;
                alive = __all_sync(0xffffffffu, bar_wait(&sh.landed[me], cleaned++ & 1u, stop));
                if (!alive) return;
                // A lane per 16 bytes of a tile row's 32: of rows [0, low) and [high, the tile's end).
                const uint32_t row = lane / 2, last = high / kTile;
                for (uint32_t side = 0; side < 2; ++side) {
                    if (side == 0 ? row >= low : high % kTile == 0 || row < high % kTile) continue;
                    const uint32_t at = (side == 0 ? 0u : last * 512) + lane * 16, place = at ^ (at >> 7 & 7u) << 4;
                    for (uint32_t c = 0; c < slices; ++c) {
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to + c * 4096 + place), "r"(0u) : "memory");
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.full[slot]);
            };
            // In the order the products take them: the keys one block ahead of the values.
            if (go) fetch(true, 0);
            if constexpr (WORKERS) {
                alive = __all_sync(0xffffffffu, alive);
                if (!alive) break;
                bring_queries(turn, go, piece, me, lane, 32u, alive);
                if (!alive || !go) break;
            }
            // (all lanes to the end, also where lane 0 gave up)
            for (uint32_t i = 0; i < piece.blocks; ++i) {
                fetch(false, i);
                if (i + 1 < piece.blocks) fetch(true, i + 1);
            }
            alive = __all_sync(0xffffffffu, alive);
        }
        // No copy and no barrier arrival outlives the CTA.
        if (lane == 0) {
            const uint32_t tail = filled < stages ? filled : stages;
            for (uint32_t i = filled - tail; i < filled; ++i) {
                const uint32_t slot = stage0 + i % stages;
                const long long start = clock64();
                bool normal = alive;
                while (!bar_test(normal ? &sh.empty[slot] : &sh.full[slot], (i / stages) & 1u) && clock64() - start < kWaitCycles) {
                    if (*stop != 0) normal = false;
                }
            }
        }
        __syncwarp();
    } else if (MODE == kShared && run && warp >= 10) {
        // ---- queries, pieces and ancestor masks, two warps -----------------------------------------------
        Walk walk = sh.walk[0];
        Piece piece;
        bool alive = true;
        for (uint32_t turn = 0; alive; ++turn) {
            const bool go = next_piece(p, walk, piece);
            bring_queries(turn, go, piece, 0, threadIdx.x - 320, kQueryThreads, alive);
            if (!go) break;
        }
    }
    if constexpr (TREE) {
        // (behind the copies, beside the last products)
        if (warp == 9 && blockIdx.x == 0) {
            const bool bad = warp_tree_bad(p.a);
            if (bad && lane == 0) atomicMax(p.a.status, 1u);
        }
    }
    tmem_before_sync();
    __syncthreads();
    tmem_after_sync();
    if (warp == 8) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
        if (lane == 0 && sh.stop != 0) {
            atomicAdd(&g_attention_timeouts, 1u);
            atomicMax(p.a.status, 2u);
        }
    }
}

// Joins the partial sums of row sets whose blocks lie in several ranges: a warp per row, the
// ranges in order. Reads a few KB per row; bound by the latency of two dependent reads.
constexpr uint32_t kJoinWarps = 4, kJoinRows = kJoinWarps;     // rows per CTA: one per warp

template <class Leaf>
__global__ void __launch_bounds__(kJoinWarps * 32)
attention_join_kernel(const __grid_constant__ TcParams p) {
    const uint32_t ctas = p.ranges;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t sets = p.a.hkv * p.pairs;
    const uint32_t b = blockIdx.x / sets, set = blockIdx.x % sets;
    __shared__ uint64_t shared_total[kJoinWarps], shared_before[kJoinWarps];
    uint64_t total = 0, before = 0;
    for (uint32_t i = threadIdx.x; i < p.a.batch; i += kJoinWarps * 32) {
        const uint32_t n = set_length(p, tree_extent(p.a, i));
        total += n;
        if (i < b) before += n;
    }
    total = warp_sum64(total);
    before = warp_sum64(before);
    if (lane == 0) {
        shared_total[warp] = total;
        shared_before[warp] = before;
    }
    __syncthreads();
    total = before = 0;
    for (uint32_t w = 0; w < kJoinWarps; ++w) {
        total += shared_total[w];
        before += shared_before[w];
    }
    const TreeExtent e = tree_extent(p.a, b);
    const uint32_t length = set_length(p, e);
    total *= sets;
    const uint64_t begin = before * sets + static_cast<uint64_t>(set) * length;
    // The range that holds a place: the last one that begins at or before it,
    // total * c / ctas < place + 1.
    auto owner = [&](uint64_t place) {
        if (total < (1u << 22) && ctas < 1024) {        // (short division)
            const uint32_t n = static_cast<uint32_t>(total);
            return ((static_cast<uint32_t>(place) + 1) * ctas + n - 1) / n - 1;
        }
        return static_cast<uint32_t>(((place + 1) * ctas + total - 1) / total - 1);
    };
    const uint32_t c0 = length != 0 ? owner(begin + p.set_cost) : 0, c1 = length != 0 ? owner(begin + length - 1) : 0;
    // With fewer places than ranges (short lengths in a large cache) some ranges between the two hold
    // nothing and left their partials unwritten; those that hold something then hold one block each.
    // (`places`: their number, or zero where there are enough; the owner's formula, in 32 bits)
    const uint32_t places = total < ctas ? static_cast<uint32_t>(total) : 0u;
    const uint32_t behind = static_cast<uint32_t>(begin) + p.set_cost + 1;
    const uint32_t ranges = places != 0 && length != 0 ? length - p.set_cost : c1 - c0 + 1;
    // The partial of the set's i-th range. (The row set began in range c0, behind its first block or
    // at it: the second partial; the others began with it.)
    auto partial = [&](uint32_t i) {
        const uint32_t c = places != 0 ? ((behind + i) * ctas + places - 1) / places - 1 : c0 + i;
        return c * 2 + (i == 0 ? 1u : 0u);
    };
    const uint32_t first_ready = partial(min(lane, ranges - 1));
    // (every CTA waits, also one with nothing to do: the join ends after the ranges)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (c0 == c1) return;                       // no blocks, or one range wrote the result itself
    const uint32_t width = p.a.width;
    const uint32_t kv_head = set / p.pairs, offset = (set % p.pairs) * 256;
    const uint32_t rows = min(p.row_cap, p.members - offset);
    for (uint32_t r = blockIdx.y * kJoinRows + warp; r < min(rows, (blockIdx.y + 1) * kJoinRows); r += kJoinWarps) {
        const uint32_t member = offset + r, node = member % p.a.rows;
        const uint32_t head = kv_head * p.a.group + member / p.a.rows;
        if (node >= e.nodes) continue;
        auto slot = [&](uint32_t which) { return p.partial + which * p.slot_floats; };
        uint32_t ready = first_ready;           // every lane one of 32 ranges
        // The first ranges' values are asked for before anything else: all waits run together.
        constexpr uint32_t kAhead = 8;
        float v[kAhead][kMaxWidth / 32];
        auto ask = [&](uint32_t from) {
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) {
                const uint32_t which = __shfl_sync(0xffffffffu, ready, min(from + i, ranges - 1) & 31u);
                const float* at = slot(which) + static_cast<uint64_t>(r) * width;
#pragma unroll
                for (uint32_t k = 0; k < kMaxWidth / 32; ++k) v[i][k] = lane + 32 * k < width ? at[lane + 32 * k] : 0.0f;
            }
        };
        ask(0);
        // A row is also bad when a score was seen and yet no weight was left (a score so large that its
        // product with log2(e) overflowed): that range may hold all of the row's weight.
        const float kNone = __int_as_float(0xFF800000);
        float top = kNone;
        bool bad = false;
        for (uint32_t c = lane; c < ranges; c += 32) {
            const float* at = slot(c == lane ? ready : partial(c));
            const float part = at[static_cast<uint64_t>(p.row_cap) * (width + 1) + r];
            const float high = at[static_cast<uint64_t>(p.row_cap) * width + r];
            top = fmaxf(top, high);             // (-inf: nothing seen in that range, or only scores of -inf)
            bad = bad || (part == 0.0f && high != kNone);
        }
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        float sum = 0.0f, o[kMaxWidth / 32] = {};
        for (uint32_t base = 0; base < ranges; base += 32) {
            // Every lane has one range's factor ready; all lanes then add the ranges up in order.
            if (base != 0) ready = partial(min(base + lane, ranges - 1));
            float factor = 0.0f, part = 0.0f;
            if (base + lane < ranges) {
                const float* at = slot(ready);
                part = at[static_cast<uint64_t>(p.row_cap) * (width + 1) + r];
                const float high = at[static_cast<uint64_t>(p.row_cap) * width + r];
                // (each range's weights were taken against its maximum as rounded here)
                if (high != kNone) factor = exp2_fast((Leaf::kWeightLog - top * p.scale_log2) - (Leaf::kWeightLog - high * p.scale_log2));
            }
            const uint32_t count = min(32u, ranges - base);
            for (uint32_t i0 = 0; i0 < count; i0 += kAhead) {
                if (base + i0 != 0) ask(base + i0);
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i) {
                    const float f = __shfl_sync(0xffffffffu, factor, (i0 + i) & 31u);
                    const float l = __shfl_sync(0xffffffffu, part, (i0 + i) & 31u);
                    if (i0 + i >= count) continue;
                    // (nothing seen in that range: zeros, or NaN from infinite values under weights of zero,
                    // which may be those of visible tokens)
                    sum = __fmaf_rn(l, f, sum);
#pragma unroll
                    for (uint32_t k = 0; k < kMaxWidth / 32; ++k) o[k] = __fmaf_rn(v[i][k], f, o[k]);
                }
            }
        }
        const float inverse = 1.0f / sum;
        bad = bad || !(sum > 0.0f && sum <= 3.0e38f);
#pragma unroll
        for (uint32_t k = 0; k < kMaxWidth / 32; ++k) {
            o[k] *= inverse;
            bad = bad || !(fabsf(o[k]) <= 3.4028234e38f);
        }
        if (__any_sync(0xffffffffu, bad)) {
            redo_row<Leaf, true>(p.a, b, head, node, e.length);
            continue;
        }
        const uint64_t plane = attn_plane(p.a.out, b, 0);
#pragma unroll
        for (uint32_t k = 0; k < kMaxWidth / 32; ++k) {
            const uint32_t d = lane + 32 * k;
            if (d >= width) break;
            const uint32_t column = head * width + d;
            *(reinterpret_cast<uint16_t*>(attn_out_piece(p.a.out, plane, node, column / kTile)) + column % kTile) =
                    static_cast<uint16_t>(canonical_pair<Leaf>(Leaf::pack(o[k], 0.0f)));
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled entry = [] {
        void* symbol = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &symbol, cudaEnableDefault, &found) != cudaSuccess
                || found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            return static_cast<EncodeTiled>(nullptr);
        }
        return reinterpret_cast<EncodeTiled>(symbol);
    }();
    return entry;
}

// The owner's storage as (64 values of a tile, its four such lines, tile row, tile column, plane): a
// box of eight tile rows and every tile column lands as [tile column][tile row][512 bytes] with the
// 128-byte swizzle (see block_order). Lines of 128 bytes because the copy engine works line by line:
// with the 32-byte lines that the operands' own swizzle allows it brought 20 bytes a clock and SM,
// and head widths of 128 waited for it.
bool make_block_map(CUtensorMap* map, const AttnOperand& o) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    const uint64_t tile_bytes = kTileSlots * 2, band_bytes = o.tile_cols * tile_bytes;
    const cuuint64_t dims[5] = {64, 4, o.tile_rows, o.tile_cols, o.planes};
    const cuuint64_t strides[4] = {128, band_bytes, tile_bytes, o.tile_rows * band_bytes};
    const cuuint32_t box[5] = {64, 4, kKvBlock / kTile, o.tile_cols, 1};
    const cuuint32_t element_strides[5] = {1, 1, 1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, o.base, dims, strides, box, element_strides,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The tree call's shape: which rows share a tile, how many ranges.
struct TreeShape {
    uint32_t members, workers, pairs, row_cap, ctas, ranges;
    bool cut;               // a row set's blocks may lie in several ranges
    uint64_t slot_floats;
};
TreeShape tree_shape(const AttnParams& a) {
    TreeShape t{};
    t.members = a.group * a.rows;
    t.workers = t.members <= kTileRows ? 1u : 0u;
    t.pairs = t.workers ? 1 : (t.members + 2 * kTileRows - 1) / (2 * kTileRows);
    t.row_cap = t.members < 2 * kTileRows ? t.members : 2 * kTileRows;
    const uint64_t blocks = (static_cast<uint64_t>(a.cache_rows) + kKvBlock - 1) / kKvBlock;
    // Short caches stay whole: cutting them saves less than the second kernel costs. One token of one
    // sequence (four sets): caches of two blocks 9.2 us whole and 10.7 cut, of four 11.8 and 10.8 (and
    // 2.5 us less for the host), of eight 17.1 and 11.5. 256 sets of one token: eight blocks 20.9 whole
    // and 21.6 cut; 64 sets of 256 rows: eight blocks 26.0 and 39.4.
    const uint64_t sets = static_cast<uint64_t>(a.batch) * a.hkv * t.pairs;
    t.cut = blocks > (sets >= 48 ? 8 : 4);
    t.ctas = grid_for(t.cut ? sets * blocks : sets, 1);
    t.ranges = t.workers ? 2 * t.ctas : t.ctas;
    t.slot_floats = (static_cast<uint64_t>(t.row_cap) * (a.width + 2) + 7) / 8 * 8;
    return t;
}

// Dynamic shared memory: the queries of two tiles (a second buffer where it fits and a tree call can
// use it) and the ring of key and value blocks.
uint32_t shared_bytes(const AttnParams& a, bool tree, TcParams* p) {
    const uint32_t block = a.width * kTileRows * 2;
    p->query_buffers = tree && 2 * block <= 32 * 1024 ? 2 : 1;
    const uint32_t room = (kDynamicBytes - 1024) / block - 2 * p->query_buffers;
    p->stages = (room < kMaxStages ? room : kMaxStages) / 2 * 2;
    return 1024 + (p->query_buffers * 2 + p->stages) * block;
}

}  // namespace

bool attention_tc_takes(const AttnParams& p) {
    return p.width % kTile == 0 && p.width <= kMaxWidth && p.k.planes <= 0x7FFFFFFFull && p.v.planes <= 0x7FFFFFFFull;
}

uint64_t attention_tc_workspace(const AttnParams& a) {
    const TreeShape t = tree_shape(a);
    if (!t.cut) return 0;
    return static_cast<uint64_t>(t.ranges) * 2 * t.slot_floats * sizeof(float);
}

template <class Leaf, Mode MODE>
static int launch_leaf(TcParams& p, uint32_t grid, uint32_t dynamic, const TreeShape* shape, cudaStream_t stream) {
    CUtensorMap k_map, v_map;
    if (!make_block_map(&k_map, p.a.k) || !make_block_map(&v_map, p.a.v)) {
        return fail(IOMB_ERR_DEVICE, "attention: the tensor map could not be encoded");
    }
    const int rc = allow_full_shared_memory(reinterpret_cast<const void*>(&attention_tc_kernel<Leaf, MODE>));
    if (rc != IOMB_OK) return rc;
    attention_tc_kernel<Leaf, MODE><<<grid, kThreads, dynamic, stream>>>(p, k_map, v_map);
    if constexpr (MODE != kPacked) {
        if (shape->cut) {
            const int status = check_launch("sdpa_tree launch");
            if (status != IOMB_OK) return status;
            // The join's CTAs may be set up while the last ranges finish; they wait before they read.
            cudaLaunchConfig_t config{};
            config.gridDim = dim3(p.a.batch * p.a.hkv * p.pairs, (p.row_cap + kJoinRows - 1) / kJoinRows);
            config.blockDim = dim3(kJoinWarps * 32);
            config.stream = stream;
            cudaLaunchAttribute early{};
            early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
            early.val.programmaticStreamSerializationAllowed = 1;
            config.attrs = &early;
            config.numAttrs = 1;
            if (cudaLaunchKernelEx(&config, attention_join_kernel<Leaf>, static_cast<const TcParams&>(p)) != cudaSuccess) {
                return check_launch("sdpa_tree join launch");
            }
        }
    }
    return check_launch(MODE != kPacked ? "sdpa_tree launch" : "sdpa_packed launch");
}

int launch_attention_tc(const AttnParams& a, bool tree, bool bf16, void* workspace, cudaStream_t stream) {
    TcParams p{};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    if (tree) {
        const TreeShape t = tree_shape(a);
        p.members = t.members;
        p.ranges = t.ranges;
        p.cut = t.cut ? 1u : 0u;
        // (decodes of 64 sequences: 31.6 us at none, 26.7 at one or two, 29.9 at five; eight trees of 64
        // nodes: 74.7 at none, 72.9 at two, 69.8 at five)
        p.set_cost = t.workers ? 2 : 5;
        p.lane_shift = t.members <= 32 ? 32 : t.members <= 64 ? 64 : 0;
        p.pairs = t.pairs;
        p.row_cap = t.row_cap;
        p.slot_floats = t.slot_floats;
        p.partial = static_cast<float*>(workspace);
        const uint32_t dynamic = shared_bytes(a, true, &p);
        if (t.workers) {
            return bf16 ? launch_leaf<LeafBf16, kWorkers>(p, t.ctas, dynamic, &t, stream)
                        : launch_leaf<LeafF16, kWorkers>(p, t.ctas, dynamic, &t, stream);
        }
        return bf16 ? launch_leaf<LeafBf16, kShared>(p, t.ctas, dynamic, &t, stream)
                    : launch_leaf<LeafF16, kShared>(p, t.ctas, dynamic, &t, stream);
    }
    // As many heads of a group per tile as divide it, up to eight (16 rows each): heads of one
    // group read the same tokens, and short sequences fill the tile.
    p.pack = 1;
    while (p.pack < 8 && a.group % (p.pack * 2) == 0) p.pack *= 2;
    p.tile_rows = kTileRows / p.pack;
    p.head_tiles = a.hq / p.pack;
    p.members = 0;
    p.pairs = 1;
    const uint64_t units = (static_cast<uint64_t>(a.rows) / (2 * p.tile_rows) + (a.batch < a.rows ? a.batch : a.rows))
            * p.head_tiles;
    if (units > 0x7FFFFFFFull) return fail(IOMB_ERR_UNSUPPORTED, "sdpa_packed: too many rows for one launch");
    const uint32_t dynamic = shared_bytes(a, false, &p);
    return bf16 ? launch_leaf<LeafBf16, kPacked>(p, static_cast<uint32_t>(units), dynamic, nullptr, stream)
                : launch_leaf<LeafF16, kPacked>(p, static_cast<uint32_t>(units), dynamic, nullptr, stream);
}

int prepare_attention_kernels() {
    for (const void* kernel : {reinterpret_cast<const void*>(&attention_tc_kernel<LeafBf16, kPacked>),
                               reinterpret_cast<const void*>(&attention_tc_kernel<LeafF16, kPacked>),
                               reinterpret_cast<const void*>(&attention_tc_kernel<LeafBf16, kShared>),
                               reinterpret_cast<const void*>(&attention_tc_kernel<LeafF16, kShared>),
                               reinterpret_cast<const void*>(&attention_tc_kernel<LeafBf16, kWorkers>),
                               reinterpret_cast<const void*>(&attention_tc_kernel<LeafF16, kWorkers>)}) {
        const int rc = allow_full_shared_memory(kernel);
        if (rc != IOMB_OK) return rc;
    }
    return IOMB_OK;
}

}  // namespace iomb

extern "C" int iomb_sdpa_wait_timeouts(unsigned int* count) {
    using namespace iomb;
    if (count == nullptr) return fail(IOMB_ERR_INVALID_ARGUMENT, "null result");
    if (cudaMemcpyFromSymbol(count, g_attention_timeouts, sizeof *count) != cudaSuccess) {
        return check_launch("attention timeout counter");
    }
    return IOMB_OK;
}
