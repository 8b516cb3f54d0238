// Log probabilities of given tokens, the entropy and the most probable alternatives.
//
// All rows' chunks (32 or 16 logits a thread of a block, in the 16-bit types and in fp32) are one line of units, cut into equal
// shares for the blocks. A block goes through its share once: sums of e = 2^d and e d, d = (x - ref) log2(e) / T, with each
// wave's ref moved up to its largest logit wherever that is 8 octaves above it; and the `top` largest logits so far, as keys
// that order them. A row that lies in one share is finished by its block, parts of others are joined by join_kernel.
#include <algorithm>
#include <cmath>

#include "nq_common.h"
#include "nq_logits.h"
#include "nq_paged.h"
#include "nq_wave.h"

namespace nq {
namespace {

constexpr int kCUs = 256;
constexpr int kMaxTop = 64, kGroups = 64;  // of threads
constexpr int kHeld = 2048;                // keys that a block holds
constexpr float kLn2 = 0.69314718055994530942f;

// Keys that order logits as torch.argmax does: a NaN before everything, equal ones by their index. 0 is no key.
__device__ inline uint64_t order_key(float x, int at) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 becomes 0
    const uint32_t k = x != x ? 0xFFFFFFFFu : u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
    return static_cast<uint64_t>(k) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(at));
}
__device__ inline int key_index(uint64_t key) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key)); }
__device__ inline float key_logit(uint64_t key) {  // -inf of no key
    const uint32_t k = static_cast<uint32_t>(key >> 32);
    return key == 0 ? -INFINITY : __builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}

struct Sums {
    float ref, s, d;  // sum of e and of e d
    // the same of two sets of logits; a set whose logits are all -inf has s = 0
    __device__ void join(const Sums& o, float scale) {
        const float top = fmaxf(ref, o.ref);
        move(top, scale);
        Sums other = o;
        other.move(top, scale);
        s += other.s;
        d += other.d;
    }
    __device__ void move(float to, float scale) {
        const float by = (ref - to) * scale, f = __builtin_amdgcn_exp2f(by);
        if (s != 0.0f) {  // also where it is NaN
            d = f == 0.0f ? 0.0f : f * fmaf(by, s, d);
            s *= f;
        }
        ref = to;
    }
};

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
    int chunks;      // of a row
    int64_t share;   // chunks of a block
    int64_t units;   // of all rows
    float4* sums;    // [blocks][2]: ref, s, d, 1 where the keys are not all there
    uint64_t* keys;  // [blocks][2][top]
    __device__ int64_t first(int64_t row) const {  // element
        const int64_t b = row / rows;
        return b * batch_stride + (row - b * rows) * row_stride;
    }
};

// A row's results but for its alternatives; log p of a logit.
template <typename T>
struct Scored {
    float ref, log_sum;
    double per_degree;
    __device__ Scored(const ScoreArgs& a, const Sums& sums) : ref(sums.ref), log_sum(log2f(sums.s)), per_degree(a.per_degree) {}
    // in fp64: the difference of two fp32 logits may be more than fp32 holds
    __device__ float logprob(float x) const {
        return static_cast<float>((static_cast<double>(x) - ref) * per_degree - static_cast<double>(kLn2) * log_sum);
    }
    __device__ void store(const ScoreArgs& a, int64_t row, const Sums& sums) const {  // one thread
        const int64_t b = row / a.rows, token = a.tokens[b * a.token_batch_stride + (row - b * a.rows) * a.token_stride];
        const bool there = token >= 0 && token < a.vocab;
        a.logprobs[row] = there ? logprob(Elem<T>::get(a.logits, a.first(row) + token)) : 0.0f;
        a.entropy[row] = kLn2 * (log_sum - sums.d / sums.s);
    }
    __device__ void store_top(const ScoreArgs& a, int64_t row, int k, uint64_t key) const {
        a.top_tokens[row * a.top + k] = key_index(key);
        a.top_logprobs[row * a.top + k] = logprob(key_logit(key));
    }
};

// The largest key below `bound` of those that `key(i)` gives for i < n. All threads of the block; `red`: one entry a wave.
template <int kThreads, typename Key>
__device__ inline uint64_t block_largest(uint64_t bound, int n, uint64_t* red, Key key) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t k = key(i);
        if (k < bound && k > best) best = k;
    }
    best = wave_largest(best);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) best = red[w] > best ? red[w] : best;
    return best;
}

// The alternatives of a row, one after the other: where there is a NaN, or more keys were met than a block holds.
template <typename T, int kThreads>
__device__ inline void slow_top(const ScoreArgs& a, int64_t row, const Scored<T>& scored, uint64_t* red) {
    uint64_t key = ~uint64_t{0};
    const int64_t first = a.first(row);
    for (int k = 0; k < a.top; ++k) {
        key = block_largest<kThreads>(key, a.vocab, red, [&](int i) { return order_key(Elem<T>::get(a.logits, first + i), i); });
        if (threadIdx.x == 0) scored.store_top(a, row, k, key);
    }
}

// The `top` largest keys among those held, sorted, and the last of them as a bound for what comes.
struct Held {
    uint64_t keys[kHeld], best[kMaxTop], group[kGroups];
    uint64_t bound;  // keys below it are none of the largest; 0 at first
    int count;
};
template <int kThreads>
__device__ inline void keep_largest(Held& held, int n, int top) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t key = held.keys[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += held.keys[j] > key ? 1 : 0;
        if (rank < top) held.best[rank] = key;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(n, top); i += kThreads) held.keys[i] = held.best[i];
    if (threadIdx.x == 0) {
        held.count = min(n, top);
        if (n >= top) held.bound = held.best[top - 1];
    }
    __syncthreads();
}

template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads, kThreads == 256 ? 5 : 4) void score_kernel(const ScoreArgs a) {
    constexpr int N = Elem<T>::N, kBatch = 4 * N, kWaves = kThreads / 64;
    using Row = LogitRow<T, kThreads, kBatch>;
    __shared__ Held held;
    __shared__ Sums wave_sums[kWaves];
    __shared__ uint64_t red[kWaves];
    const int t = threadIdx.x;
    int64_t u = blockIdx.x * a.share;
    const int64_t end = min(u + a.share, a.units);
    for (int segment = 0; u < end; ++segment) {
        const int64_t at_row = u / a.chunks;
        const int c0 = static_cast<int>(u - at_row * a.chunks), c1 = static_cast<int>(min<int64_t>(a.chunks, c0 + end - u));
        u += c1 - c0;
        const Row row(a.logits, a.first(at_row), a.vocab);
        Sums sums{-INFINITY, 0.0f, 0.0f};
        float limit = -INFINITY;
        bool spilled = false;
        if (a.top) {
            __syncthreads();  // the segment before has been read
            if (t == 0) {
                held.bound = 0;
                held.count = 0;
            }
            __syncthreads();
        }
        int had = 0;  // keys held before this chunk
        for (int c = c0; c < c1; ++c) {
            u32x4 v[Row::kPieces];
            row.load(c, v);
            float x[kBatch];
            row.unpack(c, v, x);
            float piece_most[Row::kPieces];
#pragma unroll
            for (int p = 0; p < Row::kPieces; ++p) {
                piece_most[p] = x[N * p];
#pragma unroll
                for (int i = 1; i < N; ++i) piece_most[p] = fmaxf(piece_most[p], x[N * p + i]);
            }
            static_assert(Row::kPieces == 4, "a chunk is four pieces a thread");
            const float most = fmaxf(fmaxf(piece_most[0], piece_most[1]), fmaxf(piece_most[2], piece_most[3]));
            if (__any(most > limit)) {
                sums.move(wave_max(fmaxf(most, sums.ref)), a.scale);
                limit = sums.ref + 8.0f / a.scale;
            }
            const float ref = sums.ref == -INFINITY ? 0.0f : sums.ref;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const float d = (x[i] - ref) * a.scale, e = __builtin_amdgcn_exp2f(d);
                sums.s += e;
                sums.d = fmaf(e, fmaxf(d, -1000.0f), sums.d);  // 0 of a logit of -inf
            }
            if (a.top == 0 || spilled) continue;
            // logit e of a piece, e known to nobody before: these parts run seldom, and unrolled their compares would take the
            // scalar registers of everything
            auto pick = [&](const u32x4& w, int e) {
                const int word = 4 * e / N;
                const uint32_t u = word & 2 ? (word & 1 ? w[3] : w[2]) : (word & 1 ? w[1] : w[0]);
                if constexpr (N == 4) return __builtin_bit_cast(float, u);
                else return T::to_float(static_cast<uint16_t>(u >> (16 * (e & 1))));
            };
            auto inside = [&](int at) { return static_cast<unsigned>(at) < static_cast<unsigned>(a.vocab); };
            // a bound from this chunk: the top-th largest of 64 groups of threads' largest
            auto sharpen = [&] {
                uint64_t key = 0;
                const int p = piece_most[0] == most ? 0 : piece_most[1] == most ? 1 : piece_most[2] == most ? 2 : 3;
                const u32x4 w = p & 2 ? (p & 1 ? v[3] : v[2]) : (p & 1 ? v[1] : v[0]);
#pragma unroll 1
                for (int e = 0; e < N; ++e) {
                    const int at = row.element(c, N * p + e);
                    if (pick(w, e) == most && inside(at) && key == 0) key = order_key(most, at);
                }
#pragma unroll
                for (int off = 1; off < kThreads / kGroups; off <<= 1) {
                    const uint64_t other = static_cast<uint64_t>(__shfl_xor(static_cast<long long>(key), off, 64));
                    key = other > key ? other : key;
                }
                if (t % (kThreads / kGroups) == 0) held.group[t / (kThreads / kGroups)] = key;
                __syncthreads();
                if (t < kGroups) {
                    key = held.group[t];
                    int rank = 0;
                    for (int j = 0; j < kGroups; ++j) rank += held.group[j] > key ? 1 : 0;
                    if (rank == a.top - 1 && key > held.bound) held.bound = key;  // keys are different but for 0
                }
                __syncthreads();
            };
            auto hold = [&] {  // returns how many are held with this chunk's
                const uint64_t bound = held.bound;
                const float least = key_logit(bound);
#pragma unroll
                for (int p = 0; p < Row::kPieces; ++p) {
                    if (!__any(piece_most[p] >= least)) continue;
#pragma unroll 1
                    for (int e = 0; e < N; ++e) {
                        const float y = pick(v[p], e);
                        const int at = row.element(c, N * p + e);
                        if (y >= least && inside(at) && order_key(y, at) >= bound) {
                            const int place = atomicAdd(&held.count, 1);
                            if (place < kHeld) held.keys[place] = order_key(y, at);
                        }
                    }
                }
                __syncthreads();
                return held.count;
            };
            if (c == c0) sharpen();
            int n = hold();
            if (n > kHeld && c > c0) {
                __syncthreads();
                if (t == 0) held.count = had;
                sharpen();
                n = hold();
            }
            spilled = n > kHeld;
            if (!spilled && (c == c0 || c + 1 == c1 || n > 2 * a.top + 32)) {
                keep_largest<kThreads>(held, n, a.top);
                n = min(n, a.top);
            }
            had = n;
            __syncthreads();
        }
        // the block's sums
        sums.s = wave_sum(sums.s);
        sums.d = wave_sum(sums.d);
        if ((t & 63) == 0) wave_sums[t >> 6] = sums;
        __syncthreads();
        Sums all = wave_sums[0];
        for (int w = 1; w < kWaves; ++w) all.join(wave_sums[w], a.scale);
        if (c0 == 0 && c1 == a.chunks) {
            const Scored<T> scored(a, all);
            if (t == 0) scored.store(a, at_row, all);
            if (a.top == 0) {
            } else if (spilled || all.s != all.s) {
                slow_top<T, kThreads>(a, at_row, scored, red);
            } else if (t < a.top) {
                scored.store_top(a, at_row, t, held.keys[t]);
            }
        } else {
            const int64_t part = static_cast<int64_t>(blockIdx.x) * 2 + (segment > 0);
            if (t == 0) a.sums[part] = float4{all.ref, all.s, all.d, spilled ? 1.0f : 0.0f};
            if (t < a.top) a.keys[part * a.top + t] = !spilled && t < had ? held.keys[t] : 0;
        }
        __syncthreads();  // wave_sums
    }
}

// A block a row: joins the parts that several blocks left of it.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const ScoreArgs a) {
    constexpr int kFew = 1024;
    __shared__ uint64_t keys[kFew];
    __shared__ uint64_t red[4];
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x, first = row * a.chunks;
    const int64_t b0 = first / a.share, b1 = (first + a.chunks - 1) / a.share;
    if (b0 == b1) return;
    const int n = static_cast<int>(b1 - b0) + 1;
    auto part = [&](int i) { return (b0 + i) * 2 + ((b0 + i) * a.share < first ? 1 : 0); };
    // every wave joins all the parts, a lane every 64th
    Sums all{-INFINITY, 0.0f, 0.0f};
    bool lost = false;
    for (int i = t & 63; i < n; i += 64) {
        const float4 p = a.sums[part(i)];
        all.join(Sums{p.x, p.y, p.z}, a.scale);
        lost |= p.w != 0.0f;
    }
    for (int off = 1; off < 64; off <<= 1) {
        // joined in the same order by both lanes
        const Sums other{__shfl_xor(all.ref, off, 64), __shfl_xor(all.s, off, 64), __shfl_xor(all.d, off, 64)};
        if (t & off) {
            Sums low = other;
            low.join(all, a.scale);
            all = low;
        } else {
            all.join(other, a.scale);
        }
    }
    const Scored<T> scored(a, all);
    if (t == 0) scored.store(a, row, all);
    if (a.top == 0) return;
    if (__any(lost) || all.s != all.s) {
        slow_top<T, 256>(a, row, scored, red);
        return;
    }
    const int count = n * a.top;
    auto key_of = [&](int i) { return a.keys[part(i / a.top) * a.top + i % a.top]; };
    if (count > kFew) {
        uint64_t key = ~uint64_t{0};
        for (int k = 0; k < a.top; ++k) {
            key = block_largest<256>(key, count, red, key_of);
            if (t == 0) scored.store_top(a, row, k, key);
        }
        return;
    }
    for (int i = t; i < count; i += 256) keys[i] = key_of(i);
    __syncthreads();
    for (int i = t; i < count; i += 256) {
        const uint64_t key = keys[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += keys[j] > key ? 1 : 0;
        if (key != 0 && rank < a.top) scored.store_top(a, row, rank, key);
    }
}

constexpr int64_t kMaxVocab = int64_t{1} << 30;

struct Plan {
    bool wide = false;  // blocks of 1024 threads, else of 256
    int64_t chunks = 0, share = 0, blocks = 0;
    size_t sums = 0, bytes = 0;
    bool joined() const { return share % chunks != 0; }
};

Plan make_plan(int64_t rows, int64_t vocab, int64_t top, int piece) {
    Plan p;
    p.wide = rows < 128 && vocab >= 16384;
    const int64_t chunk = (p.wide ? 1024 : 256) * 4 * piece;
    p.chunks = ceil_div(vocab + piece - 1, chunk);
    const int64_t units = rows * p.chunks;
    if (p.wide) p.share = p.chunks <= 2 ? p.chunks : ceil_div(units, 2 * kCUs);
    else if (rows >= kCUs && rows <= 8 * kCUs) p.share = p.chunks;
    else p.share = ceil_div(units, 8 * kCUs);
    p.blocks = ceil_div(units, p.share);
    p.sums = static_cast<size_t>(p.blocks) * 2 * sizeof(float4);
    p.bytes = p.joined() ? p.sums + static_cast<size_t>(p.blocks) * 2 * top * sizeof(uint64_t) : 16;
    return p;
}

// A call's plan; no bytes where there is none. The pieces of fp32 rows are shorter: whatever the type, it is given theirs.
Plan plan_of(int64_t batch, int64_t rows, int64_t vocab, int64_t top, int piece) {
    if (batch <= 0 || rows <= 0 || vocab <= 0 || top < 0 || top > vocab || vocab > kMaxVocab || top > kMaxTop ||
        rows > kMaxThreads / 256 / batch)
        return Plan{};
    return make_plan(batch * rows, vocab, top, piece);
}

template <typename T>
void launch_score(const ScoreArgs& a, const Plan& p, int64_t rows, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(p.blocks));
    if (p.wide) score_kernel<T, 1024><<<grid, 1024, 0, st>>>(a);
    else score_kernel<T, 256><<<grid, 256, 0, st>>>(a);
    if (p.joined()) join_kernel<T><<<dim3(static_cast<unsigned>(rows)), 256, 0, st>>>(a);
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" {

size_t nq_token_logprobs_workspace_bytes(int64_t batch, int64_t rows, int64_t vocab, int64_t top) {
    return std::max(plan_of(batch, rows, vocab, top, Elem<F32>::N).bytes, plan_of(batch, rows, vocab, top, Elem<F16>::N).bytes);
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
    const Plan plan = plan_of(batch, rows, vocab, top, dtype == NQ_F32 ? Elem<F32>::N : Elem<F16>::N);
    if (!aligned(workspace, 16)) return fail(NQ_ERR_ALIGNMENT, "%s: the workspace must be 16-byte aligned", name);
    if (!workspace || workspace_bytes < plan.bytes)
        return fail(NQ_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", name, workspace ? workspace_bytes : size_t{0}, plan.bytes);
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
    a.chunks = static_cast<int>(plan.chunks);
    a.share = plan.share;
    a.units = batch * rows * plan.chunks;
    a.sums = static_cast<float4*>(workspace);
    a.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + plan.sums);
    hipStream_t st = as_stream(stream);
    if (dtype == NQ_F32) launch_score<F32>(a, plan, batch * rows, st);
    else if (dtype == NQ_F16) launch_score<F16>(a, plan, batch * rows, st);
    else launch_score<BF16>(a, plan, batch * rows, st);
    return check_launch(name);
}

}  // extern "C"
