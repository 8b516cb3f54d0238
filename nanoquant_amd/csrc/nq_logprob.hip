// Log probabilities of given tokens, the entropy and the most probable alternatives.
#include <cmath>

#include <type_traits>

#include "nq_common.h"
#include "nq_paged.h"

namespace nq {
namespace {

struct ScoreArgs {
    const void* logits;
    int64_t batch_stride, row_stride;
    const int64_t* tokens;
    int64_t token_batch_stride, token_stride;
    float* logprobs;
    float* entropy;
    int64_t* top_tokens;
    float* top_logprobs;
    float scale;        // log2(e) / temperature
    double per_degree;  // 1 / temperature
    int rows, vocab, top;
};

template <typename T>
__device__ inline float logit(const void* row, int64_t at) {
    if constexpr (std::is_same_v<T, float>) return static_cast<const float*>(row)[at];
    else return T::to_float(static_cast<const uint16_t*>(row)[at]);
}

// Keys that order logits as torch.argmax does: a NaN before everything, equal ones by their index. 0 is no key.
__device__ inline uint64_t order_key(float x, int at) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 becomes 0
    const uint32_t k = x != x ? 0xFFFFFFFFu : u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
    return static_cast<uint64_t>(k) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(at));
}

// A block a row, the row read once for each thing that it makes.
template <typename T>
__global__ __launch_bounds__(256) void score_kernel(const ScoreArgs a) {
    __shared__ uint64_t s_key[256];
    __shared__ float s_sum[256], s_dev[256];
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x, b = row / a.rows, r = row - b * a.rows;
    const int64_t start = b * a.batch_stride + r * a.row_stride;
    const void* x = static_cast<const char*>(a.logits) + start * (std::is_same_v<T, float> ? 4 : 2);
    auto largest_below = [&](uint64_t bound) {  // among the keys below it
        uint64_t best = 0;
        for (int i = t; i < a.vocab; i += 256) {
            const uint64_t k = order_key(logit<T>(x, i), i);
            if (k < bound && k > best) best = k;
        }
        __syncthreads();
        s_key[t] = best;
        __syncthreads();
        for (int n = 128; n > 0; n >>= 1) {
            if (t < n && s_key[t + n] > s_key[t]) s_key[t] = s_key[t + n];
            __syncthreads();
        }
        return s_key[0];
    };
    const uint64_t first = largest_below(~uint64_t{0});
    const float m = logit<T>(x, 0xFFFFFFFFu - static_cast<uint32_t>(first));
    float sum = 0.0f, dev = 0.0f;
    for (int i = t; i < a.vocab; i += 256) {
        const float d = (logit<T>(x, i) - m) * a.scale, e = __builtin_amdgcn_exp2f(d);
        sum += e;
        dev += e * fmaxf(d, -1000.0f);  // of a token that is masked, 0
    }
    s_sum[t] = sum;
    s_dev[t] = dev;
    __syncthreads();
    for (int n = 128; n > 0; n >>= 1) {
        if (t < n) {
            s_sum[t] += s_sum[t + n];
            s_dev[t] += s_dev[t + n];
        }
        __syncthreads();
    }
    const float log_sum = log2f(s_sum[0]);
    constexpr float kLn2 = 0.69314718055994530942f;
    // in fp64: the difference of two fp32 logits may be more than fp32 holds
    auto logprob = [&](float v) { return static_cast<float>((static_cast<double>(v) - m) * a.per_degree - static_cast<double>(kLn2) * log_sum); };
    if (t == 0) {
        const int64_t token = a.tokens[b * a.token_batch_stride + r * a.token_stride];
        a.logprobs[row] = token >= 0 && token < a.vocab ? logprob(logit<T>(x, token)) : 0.0f;
        a.entropy[row] = kLn2 * (log_sum - s_dev[0] / s_sum[0]);
    }
    uint64_t key = first;
    for (int k = 0; k < a.top; ++k) {
        if (k > 0) key = largest_below(key);
        if (t == 0) {
            const uint32_t at = 0xFFFFFFFFu - static_cast<uint32_t>(key);
            a.top_tokens[row * a.top + k] = at;
            a.top_logprobs[row * a.top + k] = logprob(logit<T>(x, at));
        }
    }
}

constexpr int64_t kMaxVocab = int64_t{1} << 30, kMaxTop = 64;

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" {

size_t nq_token_logprobs_workspace_bytes(int64_t batch, int64_t rows, int64_t vocab, int64_t top) {
    return 16;
}

int nq_token_logprobs(int dtype, const void* logits, int64_t batch_stride, int64_t row_stride, const int64_t* tokens,
                      int64_t token_batch_stride, int64_t token_stride, double temperature, int64_t top, float* logprobs,
                      float* entropy, int64_t* top_tokens, float* top_logprobs, int64_t batch, int64_t rows, int64_t vocab,
                      void* workspace, size_t workspace_bytes, nq_stream_t stream) {
    const char* name = "nq_token_logprobs";
    if (dtype != NQ_F16 && dtype != NQ_BF16 && dtype != NQ_F32) return fail(NQ_ERR_DTYPE, "%s: unsupported dtype %d", name, dtype);
    if (batch < 0 || rows < 0 || vocab <= 0 || top < 0 || top > vocab || !(temperature > 0.0) || std::isinf(temperature))
        return fail(NQ_ERR_INVALID_ARGUMENT, "%s: bad sizes or temperature", name);
    if ((rows > 1 && row_stride < vocab) || (batch > 1 && batch_stride < vocab))
        return fail(NQ_ERR_SHAPE, "%s: rows of logits overlap", name);
    if (batch == 0 || rows == 0) return NQ_OK;
    if (vocab > kMaxVocab || top > kMaxTop || rows > kMaxThreads / 256 / batch || temperature < 0x1p-64 || temperature > 0x1p64)
        return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large, or a temperature outside 2^-64 to 2^64", name);
    if (!logits || !tokens || !logprobs || !entropy || (top && (!top_tokens || !top_logprobs)))
        return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(logits, dtype == NQ_F32 ? 4 : 2) || !aligned(tokens, 8) || !aligned(logprobs, 4) || !aligned(entropy, 4) ||
        !aligned(top_tokens, 8) || !aligned(top_logprobs, 4))
        return fail(NQ_ERR_ALIGNMENT, "%s: tensors must be aligned to their elements", name);
    ScoreArgs a{};
    a.logits = logits;
    a.batch_stride = batch_stride;
    a.row_stride = row_stride;
    a.tokens = tokens;
    a.token_batch_stride = token_batch_stride;
    a.token_stride = token_stride;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.top_tokens = top_tokens;
    a.top_logprobs = top_logprobs;
    a.scale = static_cast<float>(1.44269504088896340736 / temperature);
    a.per_degree = 1.0 / temperature;
    a.rows = static_cast<int>(rows);
    a.vocab = static_cast<int>(vocab);
    a.top = static_cast<int>(top);
    const dim3 grid(static_cast<unsigned>(batch * rows));
    hipStream_t st = as_stream(stream);
    if (dtype == NQ_F32) score_kernel<float><<<grid, 256, 0, st>>>(a);
    else if (dtype == NQ_F16) score_kernel<F16><<<grid, 256, 0, st>>>(a);
    else score_kernel<BF16><<<grid, 256, 0, st>>>(a);
    return check_launch(name);
}

}  // extern "C"
