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
#include <cuda_fp16.h>

#include "host.hpp"

namespace iomb {

constexpr int kScoreThreads = 256;
constexpr uint32_t kMaxTop = 32;

struct ScoreParams {
    Operand logits, tokens, logprob, entropy, top_value, top_token;
    Leading leading;
    uint32_t rows, vocab, top;
    uint32_t has_entropy;
    uint32_t token_bits, token_signed;
    uint32_t* status;
};

struct ScoreBf16 {
    static constexpr uint32_t kBytes = 2;
    static __device__ __forceinline__ float load(const unsigned char* at) {
        return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at)) << 16);
    }
};
struct ScoreF16 {
    static constexpr uint32_t kBytes = 2;
    static __device__ __forceinline__ float load(const unsigned char* at) {
        return __half2float(*reinterpret_cast<const __half*>(at));
    }
};
struct ScoreF32 {
    static constexpr uint32_t kBytes = 4;
    static __device__ __forceinline__ float load(const unsigned char* at) {
        return *reinterpret_cast<const float*>(at);
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

template <class Leaf>
__global__ void __launch_bounds__(kScoreThreads)
score_rows_kernel(const ScoreParams p) {
    if (blockIdx.x == gridDim.x - 1) {
        report_tokens(p);
        return;
    }
    __shared__ float shared[kScoreThreads / 32];
    __shared__ float shared2[kScoreThreads / 32];
    __shared__ uint64_t best[kScoreThreads / 32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint64_t index = blockIdx.x / p.rows;
    const uint32_t row = static_cast<uint32_t>(blockIdx.x % p.rows);
    const uint64_t plane = operand_plane(p.logits, p.leading, index);
    auto at = [&](uint32_t c) {
        return Leaf::load(p.logits.base + score_slot(p.logits, plane, row, c) * Leaf::kBytes);
    };
    const float kInf = __int_as_float(0x7F800000);
    float m = -kInf;
    bool odd = false;
    for (uint32_t c = threadIdx.x; c < p.vocab; c += kScoreThreads) {
        const float x = at(c);
        odd = odd || x != x || x == kInf;
        m = fmaxf(m, x);
    }
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (lane == 0) shared[warp] = m;
    odd = __syncthreads_or(odd ? 1 : 0) != 0;
    for (uint32_t w = 0; w < kScoreThreads / 32; ++w) m = fmaxf(m, shared[w]);
    odd = odd || m == -kInf;
    __syncthreads();
    float z = 0.0f, t = 0.0f;
    for (uint32_t c = threadIdx.x; c < p.vocab; c += kScoreThreads) {
        const float y = at(c) - m;
        const float e = expf(y);
        z += e;
        if (e > 0.0f) t = __fmaf_rn(e, y, t);
    }
    for (int d = 16; d > 0; d >>= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, d);
        t += __shfl_xor_sync(0xffffffffu, t, d);
    }
    if (lane == 0) { shared[warp] = z; shared2[warp] = t; }
    __syncthreads();
    z = 0.0f;
    t = 0.0f;
    for (uint32_t w = 0; w < kScoreThreads / 32; ++w) { z += shared[w]; t += shared2[w]; }
    const float kNan = __int_as_float(0x7FC00000);
    const float log_z = logf(z);
    if (threadIdx.x == 0) {
        uint32_t token;
        if (score_token(p, operand_plane(p.tokens, p.leading, index), row, &token)) {
            const uint64_t slot = score_slot(p.logprob, operand_plane(p.logprob, p.leading, index), 0, row);
            reinterpret_cast<float*>(p.logprob.base)[slot] = odd ? kNan : (at(token) - m) - log_z;
        }
        if (p.has_entropy) {
            const uint64_t slot = score_slot(p.entropy, operand_plane(p.entropy, p.leading, index), 0, row);
            reinterpret_cast<float*>(p.entropy.base)[slot] = odd ? kNan : log_z - t / z;
        }
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < p.top; ++k) {
        uint64_t key = 0;
        for (uint32_t c = threadIdx.x; c < p.vocab; c += kScoreThreads) {
            const uint64_t one = score_key(at(c), c);
            if (one < last && one > key) key = one;
        }
        for (int d = 16; d > 0; d >>= 1) {
            const uint64_t other = __shfl_xor_sync(0xffffffffu, key, d);
            key = other > key ? other : key;
        }
        __syncthreads();
        if (lane == 0) best[warp] = key;
        __syncthreads();
        for (uint32_t w = 0; w < kScoreThreads / 32; ++w) key = best[w] > key ? best[w] : key;
        last = key;
        if (threadIdx.x == 0) {
            const uint32_t c = 0xFFFFFFFFu - static_cast<uint32_t>(key);
            reinterpret_cast<float*>(p.top_value.base)[score_slot(
                    p.top_value, operand_plane(p.top_value, p.leading, index), row, k)] = odd ? kNan : (at(c) - m) - log_z;
            reinterpret_cast<uint32_t*>(p.top_token.base)[score_slot(
                    p.top_token, operand_plane(p.top_token, p.leading, index), row, k)] = c;
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
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(facts[0].planes * rows) + 1;
    switch (logits->dtype) {
        case IOMB_BF16: score_rows_kernel<ScoreBf16><<<grid, kScoreThreads, 0, s>>>(p); break;
        case IOMB_F16: score_rows_kernel<ScoreF16><<<grid, kScoreThreads, 0, s>>>(p); break;
        default: score_rows_kernel<ScoreF32><<<grid, kScoreThreads, 0, s>>>(p); break;
    }
    return check_launch("token_logprobs launch");
}
