// Attention over packed prompts (iomb_sdpa_packed) and of drafted token trees over a KV cache
// (iomb_sdpa_tree): admission, and the kernel that takes any head width.
//
// One warp computes one output row (attention.cuh). It reads every visible key twice and every
// visible value once per query head, with no tensor core: bound by issue slots, about 1 TFLOP/s.
// It serves head widths that are no multiple of 16 or exceed 128; the others run on the tensor
// cores (attention_tc.cu).
#include <math.h>
#include <stdio.h>

#include "attention.cuh"

namespace iomb {

constexpr int kRowWarpsPerCta = 8;

template <class Leaf>
__global__ void __launch_bounds__(kRowWarpsPerCta * 32)
packed_rows_kernel(const AttnParams p) {
    const bool ok = warp_borders_ok(p);
    const uint64_t warp = static_cast<uint64_t>(blockIdx.x) * kRowWarpsPerCta + (threadIdx.x >> 5);
    const uint64_t warps = static_cast<uint64_t>(gridDim.x) * kRowWarpsPerCta;
    if (warp == 0 && (threadIdx.x & 31u) == 0) *p.status = ok ? 0u : 1u;
    if (!ok) return;
    const uint64_t items = static_cast<uint64_t>(p.rows) * p.hq;
    for (uint64_t item = warp; item < items; item += warps) {
        const uint32_t h = static_cast<uint32_t>(item % p.hq);
        const uint32_t row = static_cast<uint32_t>(item / p.hq);
        // The last border at or before the row begins its sequence.
        if (row < p.offsets[0] || row >= p.offsets[p.batch]) continue;
        uint32_t low = 0, high = p.batch;
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2;
            if (p.offsets[mid] <= row) low = mid; else high = mid;
        }
        attend_row<Leaf>(p, 0, h, row, CausalRows{p.offsets[low], row});
    }
}

template <class Leaf>
__global__ void __launch_bounds__(kRowWarpsPerCta * 32)
tree_rows_kernel(const AttnParams p) {
    const uint64_t warp = static_cast<uint64_t>(blockIdx.x) * kRowWarpsPerCta + (threadIdx.x >> 5);
    const uint64_t warps = static_cast<uint64_t>(gridDim.x) * kRowWarpsPerCta;
    const uint64_t items = static_cast<uint64_t>(p.batch) * p.hq * p.rows;
    for (uint64_t item = warp; item < items; item += warps) {
        const uint32_t node = static_cast<uint32_t>(item % p.rows);
        const uint64_t rest = item / p.rows;
        const uint32_t h = static_cast<uint32_t>(rest % p.hq);
        const uint32_t b = static_cast<uint32_t>(rest / p.hq);
        const TreeExtent e = tree_extent(p, b);
        if (node >= e.nodes) continue;
        const int32_t* parents = p.parents != nullptr ? p.parents + static_cast<uint64_t>(b) * p.rows : nullptr;
        attend_row<Leaf>(p, b, h, node, TreeRow{e.length, node, parents});
    }
    if (warp == 0) {
        const bool bad = warp_tree_bad(p);
        if ((threadIdx.x & 31u) == 0) *p.status = bad ? 1u : 0u;
    }
}

// ---- admission ----------------------------------------------------------------------------------

static AttnOperand attn_operand(const iomb_view& view, const ViewFacts& f, int axis_b, int axis_h) {
    AttnOperand o{};
    o.base = static_cast<unsigned char*>(view.base);
    o.plane0 = view.plane_offset;
    o.stride_b = axis_b >= 0 ? view.plane_strides[axis_b] : 0;
    o.stride_h = axis_h >= 0 ? view.plane_strides[axis_h] : 0;
    o.planes = f.max_plane + 1;
    o.tile_rows = static_cast<uint32_t>(f.tile_rows);
    o.tile_cols = static_cast<uint32_t>(f.tile_cols);
    return o;
}

static bool aligned4(const void* address) { return reinterpret_cast<uintptr_t>(address) % 4 == 0; }

// What both operators ask of q, k, v and out; `lead` is the axis of the heads.
static int admit(const char* name, const iomb_view* q, const iomb_view* k, const iomb_view* v,
                 const iomb_view* out, uint32_t lead, float scale, const uint32_t* status, AttnParams* p) {
    char text[200];
    auto refuse = [&](int code, const char* why) {
        snprintf(text, sizeof text, "%s: %s", name, why);
        return fail(code, text);
    };
    ViewFacts fq{}, fk{}, fv{}, fo{};
    int rc = check_view(q, name, &fq);
    if (rc == IOMB_OK) rc = check_view(k, name, &fk);
    if (rc == IOMB_OK) rc = check_view(v, name, &fv);
    if (rc == IOMB_OK) rc = check_view(out, name, &fo);
    if (rc != IOMB_OK) return rc;
    if (q->rank != 3 + lead || k->rank != q->rank || v->rank != q->rank || out->rank != 2 + lead) {
        return refuse(IOMB_ERR_INVALID_ARGUMENT, lead ? "ranks must be q, k, v four and out three"
                                                      : "ranks must be q, k, v three and out two");
    }
    if (q->dtype != k->dtype || q->dtype != v->dtype || q->dtype != out->dtype) {
        return refuse(IOMB_ERR_INVALID_ARGUMENT, "encodings differ");
    }
    if (q->dtype != IOMB_BF16 && q->dtype != IOMB_F16) {
        return refuse(IOMB_ERR_UNSUPPORTED, "leaf must be BF16 or F16");
    }
    const uint64_t hq = q->dims[lead], hkv = k->dims[lead];
    if (lead == 1 && (k->dims[0] != q->dims[0] || out->dims[0] != q->dims[0])) {
        return refuse(IOMB_ERR_INVALID_ARGUMENT, "batch extents differ");
    }
    for (uint32_t i = 0; i < k->rank; ++i) {
        if (k->dims[i] != v->dims[i]) return refuse(IOMB_ERR_INVALID_ARGUMENT, "k and v shapes differ");
    }
    if (hq % hkv != 0) {
        return refuse(IOMB_ERR_INVALID_ARGUMENT, "query heads are not a multiple of the key/value heads");
    }
    if (fk.cols != fq.cols) return refuse(IOMB_ERR_INVALID_ARGUMENT, "head widths differ");
    if (fq.cols > kMaxHeadWidth) return refuse(IOMB_ERR_UNSUPPORTED, "head width exceeds 256");
    if (fo.rows != fq.rows || fo.cols != hq * fq.cols) {
        return refuse(IOMB_ERR_INVALID_ARGUMENT, "out must hold one row of Hq * D per row of q");
    }
    if (fq.rows > kMaxAttnRows || fk.rows > kMaxAttnRows || hq > kMaxAttnExtent || (lead == 1 && q->dims[0] > kMaxAttnExtent)) {
        return refuse(IOMB_ERR_UNSUPPORTED, "an extent exceeds the kernel limit");
    }
    if (!(scale > 0.0f) || !isfinite(scale)) {
        return refuse(IOMB_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
    }
    if (status == nullptr || !aligned4(status)) {
        return refuse(IOMB_ERR_INVALID_ARGUMENT, "status must be a device word");
    }
    if (storage_overlaps(*out, fo, *q, fq) || storage_overlaps(*out, fo, *k, fk) || storage_overlaps(*out, fo, *v, fv)) {
        return refuse(IOMB_ERR_INVALID_ARGUMENT, "the output overlaps an input");
    }
    const int ab = lead ? 0 : -1, ah = static_cast<int>(lead);
    p->q = attn_operand(*q, fq, ab, ah);
    p->k = attn_operand(*k, fk, ab, ah);
    p->v = attn_operand(*v, fv, ab, ah);
    p->out = attn_operand(*out, fo, ab, -1);
    p->hq = static_cast<uint32_t>(hq);
    p->hkv = static_cast<uint32_t>(hkv);
    p->group = static_cast<uint32_t>(hq / hkv);
    p->width = static_cast<uint32_t>(fq.cols);
    p->rows = static_cast<uint32_t>(fq.rows);
    p->cache_rows = static_cast<uint32_t>(fk.rows);
    p->scale = scale;
    p->status = const_cast<uint32_t*>(status);
    return IOMB_OK;
}

}  // namespace iomb

extern "C" int iomb_sdpa_packed(const iomb_view* q, const iomb_view* k, const iomb_view* v, const iomb_view* out,
                                const uint32_t* offsets, uint32_t sequences, float scale, uint32_t* status,
                                void* stream) {
    using namespace iomb;
    AttnParams p{};
    const int rc = admit("sdpa_packed", q, k, v, out, 0, scale, status, &p);
    if (rc != IOMB_OK) return rc;
    if (p.cache_rows != p.rows) return fail(IOMB_ERR_INVALID_ARGUMENT, "sdpa_packed: q and k hold different rows");
    if (offsets == nullptr || !aligned4(offsets)) {
        return fail(IOMB_ERR_INVALID_ARGUMENT, "sdpa_packed: offsets must be a device array of words");
    }
    if (sequences == 0 || sequences > (1u << 20)) {
        return fail(sequences == 0 ? IOMB_ERR_INVALID_ARGUMENT : IOMB_ERR_UNSUPPORTED,
                    "sdpa_packed: one to 2^20 sequences");
    }
    p.batch = sequences;
    p.offsets = offsets;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf16 = q->dtype == IOMB_BF16;
    if (attention_tc_takes(p)) return launch_attention_tc(p, false, bf16, nullptr, s);
    const uint64_t rows = static_cast<uint64_t>(p.rows) * p.hq;
    const unsigned grid = grid_for((rows + kRowWarpsPerCta - 1) / kRowWarpsPerCta, 8);
    if (bf16) packed_rows_kernel<LeafBf16><<<grid, kRowWarpsPerCta * 32, 0, s>>>(p);
    else packed_rows_kernel<LeafF16><<<grid, kRowWarpsPerCta * 32, 0, s>>>(p);
    return check_launch("sdpa_packed launch");
}

extern "C" int iomb_sdpa_tree_workspace_bytes(const iomb_view* q, const iomb_view* k, uint64_t* bytes) {
    using namespace iomb;
    if (bytes == nullptr) return fail(IOMB_ERR_INVALID_ARGUMENT, "sdpa_tree: null result");
    ViewFacts fq{}, fk{};
    int rc = check_view(q, "sdpa_tree q", &fq);
    if (rc == IOMB_OK) rc = check_view(k, "sdpa_tree k", &fk);
    if (rc != IOMB_OK) return rc;
    if (q->rank != 4 || k->rank != 4 || q->dims[0] != k->dims[0] || q->dims[1] % k->dims[1] != 0 || fq.cols != fk.cols) {
        return fail(IOMB_ERR_INVALID_ARGUMENT, "sdpa_tree: shapes must be q [B,Hq,N,D] and k [B,Hkv,C,D], Hq a multiple of Hkv");
    }
    if (q->dims[0] > kMaxAttnExtent || q->dims[1] > kMaxAttnExtent || fq.rows > kMaxTreeNodes || fk.rows > kMaxAttnRows
            || fq.cols > kMaxHeadWidth) {
        return fail(IOMB_ERR_UNSUPPORTED, "sdpa_tree: an extent exceeds the kernel limit");
    }
    AttnParams p{};
    p.k = p.v = attn_operand(*k, fk, 0, 1);
    p.hkv = static_cast<uint32_t>(k->dims[1]);
    p.group = static_cast<uint32_t>(q->dims[1] / k->dims[1]);
    p.width = static_cast<uint32_t>(fq.cols);
    p.rows = static_cast<uint32_t>(fq.rows);
    p.cache_rows = static_cast<uint32_t>(fk.rows);
    p.batch = static_cast<uint32_t>(q->dims[0]);
    *bytes = attention_tc_takes(p) ? attention_tc_workspace(p) : 0;
    return IOMB_OK;
}

extern "C" int iomb_sdpa_tree(const iomb_view* q, const iomb_view* k, const iomb_view* v, const iomb_view* out,
                              const uint32_t* lengths, const int32_t* parents, const uint32_t* counts, float scale,
                              void* workspace, uint64_t workspace_bytes, uint32_t* status, void* stream) {
    using namespace iomb;
    AttnParams p{};
    const int rc = admit("sdpa_tree", q, k, v, out, 1, scale, status, &p);
    if (rc != IOMB_OK) return rc;
    if (p.rows > kMaxTreeNodes) return fail(IOMB_ERR_UNSUPPORTED, "sdpa_tree: a tree holds at most 256 nodes");
    if (lengths == nullptr || !aligned4(lengths) || !aligned4(parents) || !aligned4(counts)) {
        return fail(IOMB_ERR_INVALID_ARGUMENT, "sdpa_tree: lengths, parents and counts are device arrays of words");
    }
    p.batch = static_cast<uint32_t>(q->dims[0]);
    p.lengths = lengths;
    p.parents = parents;
    p.counts = counts;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf16 = q->dtype == IOMB_BF16;
    if (attention_tc_takes(p)) {
        const uint64_t need = attention_tc_workspace(p);
        if (need != 0 && (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 32 != 0)) {
            return fail(IOMB_ERR_INVALID_ARGUMENT,
                        "sdpa_tree: the workspace is smaller than iomb_sdpa_tree_workspace_bytes or not 32-byte aligned");
        }
        return launch_attention_tc(p, true, bf16, workspace, s);
    }
    const uint64_t rows = static_cast<uint64_t>(p.batch) * p.hq * p.rows;
    const unsigned grid = grid_for((rows + kRowWarpsPerCta - 1) / kRowWarpsPerCta, 8);
    if (bf16) tree_rows_kernel<LeafBf16><<<grid, kRowWarpsPerCta * 32, 0, s>>>(p);
    else tree_rows_kernel<LeafF16><<<grid, kRowWarpsPerCta * 32, 0, s>>>(p);
    return check_launch("sdpa_tree launch");
}
