// Verification of drafted tokens: softmax statistics of every row of logits, the accept tests, and one token by inverse CDF
// from the row where the drafts end. Three launches:
//   1. row_stats_kernel, a block per (row, chunk of 4096 logits): the chunk's largest logit m_c (with its index) and
//      z_c = sum exp((x - m_c) / T);
//   2. chunk_sums_kernel, a block per (sequence, chunk): joins the rows' statistics, walks the accept tests
//      u q(x) < p(x) and adds up its chunk of w = max(p - q, 0) and of p for the row that the walk ends at;
//   3. pick_token_kernel, a block per sequence: the chunk in which the running sum of w passes u times its total, then the
//      index within it.
// Probabilities and their sums are fp64: the token is where a running sum over up to 10^5 terms passes a number, and its
// fp32 rounding would move a visible share of the borders between tokens.
#include <algorithm>

#include "nq_common.h"

namespace nq {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;                   // logits a thread
constexpr int kChunk = kThreads * kPer;    // logits a block

struct F32 {};

template <typename T>
struct Elem {
    typedef uint16_t type;
    __device__ static float get(const void* p, int64_t i) { return T::to_float(static_cast<const uint16_t*>(p)[i]); }
};
template <>
struct Elem<F32> {
    __device__ static float get(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
};

// (order of x, index) as one number whose maximum is torch.argmax's choice: the first largest, the first NaN if there is one.
__device__ inline uint64_t rank_of(float x, uint32_t index) {
    uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 counts as 0
    u = x != x ? 0xFFFFFFFFu : (u >> 31 ? ~u : u | 0x80000000u);
    return static_cast<uint64_t>(u) << 32 | static_cast<uint32_t>(~index);
}
__device__ inline uint32_t rank_index(uint64_t r) { return ~static_cast<uint32_t>(r); }
// the value; NaN where it was one
__device__ inline float rank_value(uint64_t r) {
    const uint32_t u = static_cast<uint32_t>(r >> 32);
    return __builtin_bit_cast(float, u >> 31 ? u & 0x7FFFFFFFu : ~u);
}
__device__ inline bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

__device__ inline uint64_t wave_max64(uint64_t v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = max(v, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(v), off, 64)));
    return v;
}
__device__ inline double wave_sum64(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

struct Stat {
    uint64_t rank;  // of the largest logit
    double z;       // sum exp((x - largest) / T); 0 where the largest is no finite number
};

struct VerifyArgs {
    const void* logits;
    int64_t row_stride;
    const int64_t* draft;
    const float* draft_probs;
    const float* uniforms;
    double inv_t;  // 0: greedy
    int64_t* accepted;
    int64_t* tokens;
    int64_t vocab;
    int drafts, chunks;
    Stat* stats;   // [batch * (drafts + 1)][chunks]
    double2* sums; // [batch][chunks]: of w and of p
};

template <typename T>
__global__ __launch_bounds__(kThreads) void row_stats_kernel(const VerifyArgs a) {
    __shared__ uint64_t ranks[kThreads / 64];
    __shared__ double zs[kThreads / 64];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t row = blockIdx.x / a.chunks;
    const int64_t base = static_cast<int64_t>(blockIdx.x - row * a.chunks) * kChunk;
    float x[kPer];
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int64_t j = base + t + i * kThreads;
        x[i] = j < a.vocab ? Elem<T>::get(a.logits, row * a.row_stride + j) : -INFINITY;
        if (j < a.vocab) best = max(best, rank_of(x[i], static_cast<uint32_t>(j)));
    }
    best = wave_max64(best);
    if (lane == 0) ranks[wave] = best;
    __syncthreads();
    best = max(max(ranks[0], ranks[1]), max(ranks[2], ranks[3]));
    const float m = rank_value(best);
    double z = 0.0;
    if (finite(m) && a.inv_t != 0.0) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) z += exp((static_cast<double>(x[i]) - m) * a.inv_t);
    }
    z = wave_sum64(z);
    if (lane == 0) zs[wave] = z;
    __syncthreads();
    if (t == 0) a.stats[blockIdx.x] = Stat{best, (zs[0] + zs[1]) + (zs[2] + zs[3])};
}

// A row's statistics from its chunks', in every lane of the wave that calls it.
__device__ inline Stat join_row(const VerifyArgs& a, int64_t row, int lane) {
    uint64_t best = 0;
    for (int c = lane; c < a.chunks; c += 64) best = max(best, a.stats[row * a.chunks + c].rank);
    best = wave_max64(best);
    const float m = rank_value(best);
    double z = 0.0;
    if (finite(m))
        for (int c = lane; c < a.chunks; c += 64) {
            const Stat s = a.stats[row * a.chunks + c];
            const float mc = rank_value(s.rank);
            if (finite(mc)) z += s.z * exp((static_cast<double>(mc) - m) * a.inv_t);  // a chunk of -inf adds nothing
        }
    return Stat{best, wave_sum64(z)};
}

// Where a sequence's drafts end.
struct Walk {
    int kept;       // accepted drafts: the row that the next token comes from
    bool less_q;    // that row's draft was turned down: w = max(p - q, 0)
    Stat stat;      // of that row
};

template <typename T>
__device__ Walk walk(const VerifyArgs& a, int64_t b) {
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    __shared__ int ends;  // 2 * row + (1: turned down)
    if (t == 0) ends = 2 * a.drafts;
    __syncthreads();
    for (int i = wave; i <= a.drafts; i += kThreads / 64) {
        const int64_t row = b * (a.drafts + 1) + i;
        if (i == a.drafts) break;
        const int64_t x = a.draft[b * a.drafts + i];
        if (x < 0 || x >= a.vocab) {
            if (lane == 0) atomicMin(&ends, 2 * i);
            break;
        }
        const Stat s = join_row(a, row, lane);
        const float m = rank_value(s.rank);
        double p = 0.0;
        if (a.inv_t == 0.0 || !finite(m)) p = finite(m) && rank_index(s.rank) == x ? 1.0 : 0.0;
        else p = exp((static_cast<double>(Elem<T>::get(a.logits, row * a.row_stride + x)) - m) * a.inv_t) / s.z;
        const double q = a.draft_probs && a.inv_t != 0.0 ? a.draft_probs[(b * a.drafts + i) * a.vocab + x] : 1.0;
        const double u = a.uniforms[b * (a.drafts + 1) + i];
        if (!(u * q < p)) {
            if (lane == 0) atomicMin(&ends, 2 * i + 1);
            break;
        }
    }
    __syncthreads();
    Walk w;
    w.kept = ends >> 1;
    w.less_q = ends & 1;
    w.stat = join_row(a, b * (a.drafts + 1) + w.kept, lane);
    return w;
}

// p and w of token j.
template <typename T>
__device__ inline double2 weights(const VerifyArgs& a, int64_t b, const Walk& w, int64_t j, int64_t x) {
    const int64_t row = b * (a.drafts + 1) + w.kept;
    const double p =
        exp((static_cast<double>(Elem<T>::get(a.logits, row * a.row_stride + j)) - rank_value(w.stat.rank)) * a.inv_t) / w.stat.z;
    if (!w.less_q) return double2{p, p};
    const double q = a.draft_probs ? a.draft_probs[(b * a.drafts + w.kept) * a.vocab + j] : (j == x ? 1.0 : 0.0);
    return double2{p > q ? p - q : 0.0, p};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void chunk_sums_kernel(const VerifyArgs a) {
    __shared__ double2 part[kThreads / 64];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t b = blockIdx.x / a.chunks;
    const int64_t base = static_cast<int64_t>(blockIdx.x - b * a.chunks) * kChunk;
    const Walk w = walk<T>(a, b);
    if (a.inv_t == 0.0 || !finite(rank_value(w.stat.rank))) return;  // the token is the argmax
    const int64_t x = w.less_q ? a.draft[b * a.drafts + w.kept] : -1;
    double2 s = {0.0, 0.0};
    for (int i = 0; i < kPer; ++i) {
        const int64_t j = base + t + i * kThreads;
        if (j >= a.vocab) break;
        const double2 e = weights<T>(a, b, w, j, x);
        s.x += e.x;
        s.y += e.y;
    }
    s.x = wave_sum64(s.x);
    s.y = wave_sum64(s.y);
    if (lane == 0) part[wave] = s;
    __syncthreads();
    if (t == 0)
        a.sums[blockIdx.x] = double2{(part[0].x + part[1].x) + (part[2].x + part[3].x), (part[0].y + part[1].y) + (part[2].y + part[3].y)};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pick_token_kernel(const VerifyArgs a) {
    __shared__ int s_chunk, s_last;
    __shared__ double s_left;
    __shared__ int64_t s_index[2];
    __shared__ double part[kThreads];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t b = blockIdx.x;
    const Walk w = walk<T>(a, b);
    int64_t token = rank_index(w.stat.rank);
    if (a.inv_t != 0.0 && finite(rank_value(w.stat.rank))) {
        const double2* sums = a.sums + b * a.chunks;
        if (wave == 0) {
            double total = 0.0, total_p = 0.0;
            for (int c = lane; c < a.chunks; c += 64) {
                total += sums[c].x;
                total_p += sums[c].y;
            }
            total = wave_sum64(total);
            total_p = wave_sum64(total_p);
            const bool plain = !(total > 0.0);
            const double target = a.uniforms[b * (a.drafts + 1) + a.drafts] * (plain ? total_p : total);
            // the first chunk whose running sum passes the target; the last one with a positive sum where rounding hides it
            double run = 0.0, left = 0.0;
            int chunk = -1, last = 0;
            for (int c0 = 0; c0 < a.chunks && chunk < 0; c0 += 64) {
                const int c = c0 + lane;
                const double v = c < a.chunks ? (plain ? sums[c].y : sums[c].x) : 0.0;
                double incl = v;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const double up = __shfl_up(incl, off, 64);
                    if (lane >= off) incl += up;
                }
                const uint64_t pass = __ballot(v > 0.0 && run + incl > target);
                const uint64_t some = __ballot(v > 0.0);
                if (some) last = c0 + 63 - __builtin_clzll(some);
                if (pass) {
                    const int at = __builtin_ctzll(pass);
                    chunk = c0 + at;
                    left = target - (run + __shfl(incl - v, at, 64));
                }
                run += __shfl(incl, 63, 64);
            }
            if (lane == 0) {
                s_chunk = chunk < 0 ? last : chunk;
                s_left = chunk < 0 ? INFINITY : left;
                s_last = plain;
            }
        }
        if (t == 0) {
            s_index[0] = INT64_MAX;  // the first index that passes
            s_index[1] = -1;         // the last one with a positive weight
        }
        __syncthreads();
        const bool plain = s_last;
        const int64_t x = w.less_q ? a.draft[b * a.drafts + w.kept] : -1;
        const int64_t base = static_cast<int64_t>(s_chunk) * kChunk + t * kPer;
        double v[kPer], sum = 0.0;
        for (int i = 0; i < kPer; ++i) {
            v[i] = 0.0;
            if (base + i < a.vocab) {
                const double2 e = weights<T>(a, b, w, base + i, x);
                v[i] = plain ? e.y : e.x;
            }
            sum += v[i];
        }
        part[t] = sum;
        __syncthreads();
        double run = 0.0;
        for (int i = 0; i < t; ++i) run += part[i];
        int64_t first = INT64_MAX, last = -1;
        for (int i = 0; i < kPer; ++i) {
            run += v[i];
            if (v[i] > 0.0) {
                last = base + i;
                if (run > s_left && first == INT64_MAX) first = base + i;
            }
        }
        atomicMin(reinterpret_cast<unsigned long long*>(&s_index[0]), static_cast<unsigned long long>(first));
        if (last >= 0) atomicMax(reinterpret_cast<long long*>(&s_index[1]), static_cast<long long>(last));
        __syncthreads();
        token = s_index[0] != INT64_MAX ? s_index[0] : s_index[1];
    }
    if (t == 0) a.accepted[b] = w.kept;
    for (int i = t; i <= a.drafts; i += kThreads)
        a.tokens[b * (a.drafts + 1) + i] = i < w.kept ? a.draft[b * a.drafts + i] : (i == w.kept ? token : -1);
}

template <typename T>
void launch_verify(const VerifyArgs& a, int64_t batch, hipStream_t st) {
    const int64_t rows = batch * (a.drafts + 1);
    row_stats_kernel<T><<<dim3(static_cast<unsigned>(rows * a.chunks)), kThreads, 0, st>>>(a);
    chunk_sums_kernel<T><<<dim3(static_cast<unsigned>(batch * a.chunks)), kThreads, 0, st>>>(a);
    pick_token_kernel<T><<<dim3(static_cast<unsigned>(batch)), kThreads, 0, st>>>(a);
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" {

size_t nq_verify_drafts_workspace_bytes(int64_t batch, int64_t drafts, int64_t vocab) {
    if (batch <= 0 || drafts < 0 || vocab <= 0 || vocab > INT32_MAX || batch > INT32_MAX || drafts > INT32_MAX / 2) return 0;
    const int64_t chunks = ceil_div(vocab, kChunk);
    if (batch * (drafts + 1) > (int64_t{1} << 23) / chunks) return 0;  // blocks of 256 threads
    return static_cast<size_t>(batch) * (drafts + 2) * chunks * 16;
}

int nq_verify_drafts(int dtype, const void* logits, int64_t row_stride, const int64_t* draft, const float* draft_probs,
                     const float* uniforms, float temperature, int64_t* accepted, int64_t* tokens, int64_t batch,
                     int64_t drafts, int64_t vocab, void* workspace, size_t workspace_bytes, nq_stream_t stream) {
    const char* name = "nq_verify_drafts";
    if (dtype != NQ_F16 && dtype != NQ_BF16 && dtype != NQ_F32) return fail(NQ_ERR_DTYPE, "%s: unsupported dtype %d", name, dtype);
    if (batch < 0 || drafts < 0 || vocab <= 0) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: bad sizes", name);
    if (row_stride < vocab) return fail(NQ_ERR_SHAPE, "%s: rows of logits overlap", name);
    if (!(temperature >= 0.0f) || temperature > 3.402823466e38f)
        return fail(NQ_ERR_INVALID_ARGUMENT, "%s: the temperature must be a finite number from 0", name);
    if (batch == 0) return NQ_OK;
    const size_t need = nq_verify_drafts_workspace_bytes(batch, drafts, vocab);
    if (need == 0) return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large", name);
    if (!logits || (!draft && drafts) || !uniforms || !accepted || !tokens || !workspace)
        return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(logits, dtype == NQ_F32 ? 4 : 2) || !aligned(draft, 8) || !aligned(draft_probs, 4) || !aligned(uniforms, 4) ||
        !aligned(accepted, 8) || !aligned(tokens, 8) || !aligned(workspace, 16))
        return fail(NQ_ERR_ALIGNMENT, "%s: misaligned pointer", name);
    if (workspace_bytes < need)
        return fail(NQ_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", name, workspace_bytes, need);
    VerifyArgs a{};
    a.logits = logits;
    a.row_stride = row_stride;
    a.draft = draft;
    a.draft_probs = draft_probs;
    a.uniforms = uniforms;
    a.inv_t = temperature > 0.0f ? 1.0 / static_cast<double>(temperature) : 0.0;
    a.accepted = accepted;
    a.tokens = tokens;
    a.vocab = vocab;
    a.drafts = static_cast<int>(drafts);
    a.chunks = static_cast<int>(ceil_div(vocab, kChunk));
    a.stats = static_cast<Stat*>(workspace);
    a.sums = reinterpret_cast<double2*>(a.stats + batch * (drafts + 1) * a.chunks);
    if (dtype == NQ_F16) launch_verify<F16>(a, batch, as_stream(stream));
    else if (dtype == NQ_BF16) launch_verify<BF16>(a, batch, as_stream(stream));
    else launch_verify<F32>(a, batch, as_stream(stream));
    return check_launch(name);
}

}  // extern "C"
