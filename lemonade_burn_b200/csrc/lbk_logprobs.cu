// Log probabilities of given tokens, entropy and the best alternatives of rows of logits.
//
//   c = scale * x;  lse = log sum_j exp(c_j);  logprob(token) = c_token - lse;  H = lse - sum_j p_j c_j
//   alternatives: the `top` largest logits, the lower id first among equal ones, with their log probabilities
//
// The reference has the greedy token only (crates/lb-model/src/sample.rs:17-25).
#include <cfloat>

#include "lbk_dense_dev.cuh"
#include "lbk_tree.cuh"

namespace lbk {

namespace {

using dense::get;

struct ScoreParams {
    const void *logits;
    size_t pitch;
    int vocab;
    const int *tokens;
    int given;
    float scale;
    int top;
    float *logprobs, *entropy;
    int *top_ids;
    float *top_logprobs;
};

// A place in the order of the alternatives: larger values first, then lower ids; every NaN in front of every number, as a sort has it; 0 is
// behind every place.
__device__ __forceinline__ unsigned long long order_key(float x, int id) {
    const unsigned bits = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
    const unsigned value = x != x ? 0xffffffffu : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return static_cast<unsigned long long>(value) << 32 | static_cast<unsigned>(~id);
}
__device__ __forceinline__ int key_id(unsigned long long key) { return static_cast<int>(~static_cast<unsigned>(key)); }

template <typename T>
__global__ void __launch_bounds__(256) logprobs_kernel(const ScoreParams p) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    __shared__ float s_red[32];
    __shared__ unsigned long long s_key[8];
    const int tid = threadIdx.x;
    const size_t row = blockIdx.x;
    const T *x = static_cast<const T *>(p.logits) + row * p.pitch;
    float m = -FLT_MAX;
    for (int i = tid; i < p.vocab; i += 256) m = fmaxf(m, get(x + i));
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) s_red[tid >> 5] = m;
    __syncthreads();
    for (int w = 0; w < 8; ++w) m = fmaxf(m, s_red[w]);
    float s = 0.0f, t = 0.0f;
    for (int i = tid; i < p.vocab; i += 256) {
        const float d = (get(x + i) - m) * p.scale, e = expf(d);
        s += e;
        t += e * fmaxf(d, -1000.0f);  // 0 * -inf is nothing here
    }
    __syncthreads();
    s = dense::block_sum<256>(s, s_red);
    t = dense::block_sum<256>(t, s_red);
    const float log_s = logf(s);
    auto logprob = [&](float v) { return (v - m) * p.scale - log_s; };
    if (tid == 0 && p.entropy) p.entropy[row] = log_s - t / s;
    for (int g = tid; g < p.given; g += 256) {
        const int token = p.tokens[row * p.given + g];
        p.logprobs[row * p.given + g] = token >= 0 && token < p.vocab ? logprob(get(x + token)) : __uint_as_float(0x7fc00000u);
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        unsigned long long best = 0;
        for (int i = tid; i < p.vocab; i += 256) {
            const unsigned long long key = order_key(get(x + i), i);
            if (key < last && key > best) best = key;
        }
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if ((tid & 31) == 0) s_key[tid >> 5] = best;
        __syncthreads();
        for (int w = 0; w < 8; ++w) best = max(best, s_key[w]);
        __syncthreads();
        last = best;
        if (tid == 0) {
            const int id = key_id(best);
            p.top_ids[row * p.top + k] = id;
            p.top_logprobs[row * p.top + k] = logprob(get(x + id));
        }
    }
}

}  // namespace
}  // namespace lbk

using namespace lbk;

extern "C" {

int lbk_token_logprobs(lbk_ctx *c, int dtype, const void *logits_dev, size_t pitch, size_t rows, size_t vocab, const int32_t *tokens_dev, size_t given, float scale,
                       size_t top, float *logprobs_dev, float *entropy_dev, int32_t *top_ids_dev, float *top_logprobs_dev, void *stream) {
    LBK_TREE_PRE("lbk_token_logprobs");
    if (rows == 0) return LBK_OK;
    if (!logits_dev || (given && (!tokens_dev || !logprobs_dev)) || (top && (!top_ids_dev || !top_logprobs_dev)))
        return fail(LBK_ERR_INVALID, "lbk_token_logprobs: null buffer");
    if (dtype != LBK_DTYPE_F32 && dtype != LBK_DTYPE_BF16) return fail(LBK_ERR_INVALID, "lbk_token_logprobs: unknown type %d", dtype);
    if (vocab == 0 || pitch < vocab || top > vocab) return fail(LBK_ERR_SHAPE, "lbk_token_logprobs: rows of %zu values, %zu apart, %zu alternatives", vocab, pitch, top);
    if (!(scale > 0.0f) || scale > FLT_MAX) return fail(LBK_ERR_INVALID, "lbk_token_logprobs: the scale is a positive number");
    if (top > LBK_LOGPROBS_TOP || vocab > (1u << 30) || given > (1u << 20) || rows > (1u << 26))
        return fail(LBK_ERR_UNSUPPORTED, "lbk_token_logprobs: at most %d alternatives, 2^30 values and 2^20 tokens a row, 2^26 rows", LBK_LOGPROBS_TOP);
    const ScoreParams p{logits_dev, pitch, static_cast<int>(vocab), tokens_dev, static_cast<int>(given), scale, static_cast<int>(top), logprobs_dev, entropy_dev, top_ids_dev,
                        top_logprobs_dev};
    LBK_CUDA(launch_chained(dtype == LBK_DTYPE_F32 ? logprobs_kernel<float> : logprobs_kernel<uint16_t>, dim3(static_cast<unsigned>(rows)), dim3(256), 0, st, p));
    ctx->launches++;
    return LBK_OK;
}

}  // extern "C"
