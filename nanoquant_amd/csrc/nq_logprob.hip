// Log probabilities of given tokens, the entropy and the most probable alternatives.
//
// All rows' chunks (32 or 16 logits a thread of a block, in the 16-bit types and in fp32) are one line of units, cut into equal
// shares for the blocks. A block goes through its share once: sums of e = 2^d and e d, d = x log2(e) / T - ref, with each
// wave's ref moved up to its largest logit wherever that is 8 octaves above it; and the `top` largest logits so far, each wave's
// in its lanes. A row that lies in one share is finished by its block, parts of others are joined by join_kernel.
//
// Bound by the read: 2111 rows of 100003 bf16 logits with the largest, 422 MB, 84 us (5.0 TB/s, a
// large copy's rate); 777 rows of 32000 in fp16, 50 MB, 14.5 us in one launch. Few rows by latency: one row of 32000 in
// fp32 with five alternatives 8.6 us, of which the launch and the first chunk's way, the sums and the lists' join are one chain;
// 64 rows of 100003 with twenty alternatives 11.8 and 5.8 the join's. The 2111 rows
// with several passes over each row 589 us; in one pass with the alternatives in LDS 143; with them in lanes and bounds from
// ballots 102; with five blocks a CU 93.
#include <algorithm>
#include <cmath>

#include "nq_common.h"
#include "nq_logits.h"
#include "nq_paged.h"
#include "nq_wave.h"

namespace nq {
namespace {

constexpr int kCUs = 256;
constexpr int kPerCU = 5;    // blocks of 256 threads: registers for more would go to scratch
constexpr int kMaxTop = 64;  // a wave's lanes
constexpr float kLn2 = 0.69314718055994530942f;

// Keys that order logits as torch.argmax does: a NaN before everything, equal ones by their index. Below 2^32 is no key.
__device__ inline uint32_t order_bits(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 becomes 0
    return x != x ? 0xFFFFFFFFu : u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ inline float from_order_bits(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ inline uint64_t order_key(float x, int at) {
    return static_cast<uint64_t>(order_bits(x)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(at));
}
__device__ inline bool is_key(uint64_t key) { return key >> 32 != 0; }
__device__ inline int key_index(uint64_t key) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key)); }
__device__ inline float key_logit(uint64_t key) {
    return is_key(key) ? from_order_bits(static_cast<uint32_t>(key >> 32)) : -INFINITY;
}

// Of e = 2^d and e d, d = x scale - ref: what ref has of a rounding, all d have in common, and log p = x scale - ref - log2 s.
struct Sums {
    float ref, s, d;
    // the same of two sets of logits; a set whose logits are all -inf has s = 0
    __device__ void join(const Sums& o) {
        const float top = fmaxf(ref, o.ref);
        move(top);
        Sums other = o;
        other.move(top);
        s += other.s;
        d += other.d;
    }
    __device__ void move(float to) {
        const float by = ref - to, f = __builtin_amdgcn_exp2f(by);
        if (s != 0.0f) {  // also where it is NaN
            d = f == 0.0f ? 0.0f : f * fmaf(by, s, d);
            s *= f;
        }
        ref = to;
    }
};

// Of all lanes' sums, the same in the whole wave.
__device__ inline Sums joined(Sums sums) {
    sums.move(wave_max(sums.ref));
    sums.s = wave_add(sums.s);
    sums.d = wave_add(sums.d);
    return sums;
}

struct ScoreArgs {
    const void* logits;
    int64_t batch_stride, row_stride;
    const int64_t* tokens;
    int64_t token_batch_stride, token_stride;
    float* logprobs;
    float* entropy;
    int64_t* top_tokens;
    float* top_logprobs;
    float scale;  // log2(e) / temperature
    int rows, vocab, top;
    int chunks;      // of a row, up to a whole number of shares where its parts are blocks'
    int full;        // those that it has
    int64_t share;   // chunks of a block
    int64_t units;   // of all rows
    float4* sums;    // [blocks][2]: ref, s, d
    uint64_t* keys;  // [blocks][2][top]
    __device__ int64_t first(int64_t row) const {  // element
        const int64_t b = row / rows;
        return b * batch_stride + (row - b * rows) * row_stride;
    }
};

// A row's given token and its logit, read before the row is.
template <typename T>
struct Given {
    bool there = false;
    float x = 0.0f;
    __device__ Given(const ScoreArgs& a, int64_t row, bool wanted) {
        if (!wanted) return;
        const int64_t b = row / a.rows, token = a.tokens[b * a.token_batch_stride + (row - b * a.rows) * a.token_stride];
        there = token >= 0 && token < a.vocab;
        if (there) x = Elem<T>::get(a.logits, a.first(row) + token);
    }
};

// A row's results from its sums, whose ref is given apart: twice as wide where it has to be.
struct Scored {
    double scale, ref;
    float log_sum;
    __device__ Scored(const ScoreArgs& a, const Sums& sums, double ref_) : scale(a.scale), ref(ref_), log_sum(log2f(sums.s)) {}
    // in fp64: x scale and ref may be large and nearly the same, and their difference more than fp32 holds
    __device__ float logprob(float x) const { return static_cast<float>((x * scale - ref - log_sum) * 0.69314718055994530942); }
    template <typename T>
    __device__ void store(const ScoreArgs& a, int64_t row, const Sums& sums, const Given<T>& given) const {  // one thread
        a.logprobs[row] = given.there ? logprob(given.x) : 0.0f;
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

// The alternatives of a row, one after the other: where there is a NaN.
template <typename T, int kThreads>
__device__ inline void slow_top(const ScoreArgs& a, int64_t row, const Scored& scored, uint64_t* red) {
    uint64_t key = ~uint64_t{0};
    const int64_t first = a.first(row);
    for (int k = 0; k < a.top; ++k) {
        key = block_largest<kThreads>(key, a.vocab, red, [&](int i) { return order_key(Elem<T>::get(a.logits, first + i), i); });
        if (threadIdx.x == 0) scored.store_top(a, row, k, key);
    }
}

// The `top` largest keys that a wave has met, the largest in lane 0, and a logit below which none is one of them.
struct TopList {
    uint64_t key = 0;
    float least = -INFINITY;
    __device__ void insert(uint64_t k, int top) {  // the same for the wave
        const int place = __popcll(__ballot(key > k)), lane = threadIdx.x & 63;
        if (place >= top) return;
        const uint64_t before = dpp<0x138, 0xF>(key);  // wave_shr:1
        key = lane < place ? key : lane == place ? k : before;
        least = fmaxf(least, key_logit(read_lane(key, top - 1)));
    }
    // Each lane has the largest of some logits: at least the upper half of the top-th largest's bits, a bit at a time
    __device__ void sharpen(float largest, int top) {
        const uint32_t mine = order_bits(largest);
        uint32_t bound = 0;
#pragma unroll
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t more = bound | 1u << bit;
            bound = __popcll(__ballot(mine >= more)) >= top ? more : bound;
        }
        if (bound >= 0x00800000u) least = fmaxf(least, from_order_bits(bound));  // else -inf, or no number
    }
};

// A row's sums where logits times the scale are too large for fp32, and ref, the scaled largest logit.
template <typename T, int kThreads>
__device__ inline Sums slow_sums(const ScoreArgs& a, int64_t row, uint64_t* red, Sums* wave_sums, double& ref) {
    const int64_t first = a.first(row);
    auto at = [&](int i) { return Elem<T>::get(a.logits, first + i); };
    const float most = key_logit(block_largest<kThreads>(~uint64_t{0}, a.vocab, red, [&](int i) { return order_key(at(i), i); }));
    Sums sums{0.0f, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
        const float d = (at(i) - most) * a.scale, e = __builtin_amdgcn_exp2f(d);
        sums.s += e;
        sums.d = fmaf(e, fmaxf(d, -1000.0f), sums.d);
    }
    sums.s = wave_add(sums.s);
    sums.d = wave_add(sums.d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) wave_sums[threadIdx.x >> 6] = sums;
    __syncthreads();
    sums = wave_sums[0];
    for (int w = 1; w < kThreads / 64; ++w) sums.join(wave_sums[w]);
    ref = static_cast<double>(most) * a.scale;
    return sums;
}
// Beyond this what ref is rounded by moves the exponentials by an octave and more. Infinities too.
__device__ inline bool leaves_fp32(const Sums& sums) { return fabsf(sums.ref) > 0x1p24f; }

template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads, kThreads == 256 ? kPerCU : 4) void score_kernel(const ScoreArgs a) {
    constexpr int N = Elem<T>::N, kBatch = 4 * N, kWaves = kThreads / 64;
    using Row = LogitRow<T, kThreads, kBatch>;
    static_assert(Row::kPieces == 4, "a chunk is four pieces a thread");
    __shared__ uint64_t keys[kWaves * kMaxTop];
    __shared__ float lane_most[2][kWaves][64];
    __shared__ uint32_t lane_words[kWaves][16];
    __shared__ int key_count[2];  // of this segment, of the next
    __shared__ Sums wave_sums[kWaves];
    __shared__ uint64_t red[kWaves];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int64_t u = blockIdx.x * a.share;
    const int64_t end = min(u + a.share, a.units);
    if (t == 0) key_count[0] = 0;
    for (int segment = 0; u < end; ++segment) {
        const int64_t at_row = u / a.chunks;
        const int c0 = static_cast<int>(u - at_row * a.chunks), c1 = static_cast<int>(min<int64_t>(a.chunks, c0 + end - u));
        u += c1 - c0;
        const bool whole = c0 == 0 && c1 == a.chunks;
        const int last = min(c1, a.full);
        const Row row(a.logits, a.first(at_row), a.vocab);
        u32x4 next[4];
        row.load_once(c0, next);
        const Given<T> given(a, at_row, whole && t == 0);
        Sums sums{-INFINITY, 0.0f, 0.0f};
        float limit = -INFINITY;
        TopList list;
        float most_yet = -INFINITY;
        int turn = 0;
        for (int c = c0; c < last; ++c) {
            u32x4 v[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) v[p] = next[p];
            if (c + 1 < last) row.load_once(c + 1, next);
            const bool edge = row.at_edge(c);
            if (edge) {
#pragma unroll
                for (int p = 0; p < 4; ++p) v[p] = row.cleared(c, p, v[p]);
            }
            // nothing unpacked is kept from here to there: what that would take in registers costs more than unpacking again
            auto forget = [&] {
#pragma unroll
                for (int p = 0; p < 4; ++p) asm volatile("" : "+v"(v[p]));
            };
            float piece_most[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                float x[N];
                Elem<T>::unpack(v[p], x);
                piece_most[p] = x[0];
#pragma unroll
                for (int i = 1; i < N; ++i) piece_most[p] = fmaxf(piece_most[p], x[i]);
            }
            const float most = fmaxf(fmaxf(piece_most[0], piece_most[1]), fmaxf(piece_most[2], piece_most[3]));
            if (__any(most > limit)) {
                sums.move(fmaxf(wave_max(most) * a.scale, sums.ref));
                limit = (sums.ref + 8.0f) / a.scale;
            }
            const float ref = sums.ref == -INFINITY ? 0.0f : sums.ref;
            float s = 0.0f, d = NAN;
            if (!edge) {
                d = 0.0f;
                forget();
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    float x[N];
                    Elem<T>::unpack(v[p], x);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float by = fmaf(x[i], a.scale, -ref), e = __builtin_amdgcn_exp2f(by);
                        s += e;
                        d = fmaf(e, by, d);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (__any(d != d)) {  // a logit of -inf adds nothing, but 0 times it does
                s = d = 0.0f;
                forget();
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    float x[N];
                    Elem<T>::unpack(v[p], x);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float by = fmaf(x[i], a.scale, -ref), e = __builtin_amdgcn_exp2f(by);
                        s += e;
                        d = fmaf(e, fmaxf(by, -1000.0f), d);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            sums.s += s;
            sums.d += d;
            if (a.top == 0) continue;
            most_yet = fmaxf(most_yet, most);
            // a bound from all waves, the block's lanes in 64 groups: chunks 0, 1, 2, 4, 8 ...
            if (((c - c0) & (c - c0 - 1)) == 0) {
                lane_most[turn][wave][lane] = most_yet;
                __syncthreads();
                float x = lane_most[turn][0][lane];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) x = fmaxf(x, lane_most[turn][w][lane]);
                list.sharpen(x, a.top);
                turn ^= 1;
            }
            uint64_t some = __ballot(most >= list.least);
            if (__popcll(some) > 16) {  // which takes as long as a few insertions
                list.sharpen(most, a.top);
                some = __ballot(most >= list.least);
            }
            if (some == 0) continue;
            forget();
            auto hold = [&](float y, int at, bool here) {  // of each lane a logit
                uint64_t todo = __ballot(here && y >= list.least);
                if (todo == 0) return;
                const uint64_t key = order_key(y, at);
                todo &= __ballot(static_cast<unsigned>(at) < static_cast<unsigned>(a.vocab) && key > read_lane(list.key, a.top - 1));
                while (todo != 0) {
                    list.insert(read_lane(key, __builtin_ctzll(todo)), a.top);
                    todo &= todo - 1;
                }
            };
            constexpr int kEach = N / 4;  // logits of a word
            auto logit_of = [](uint32_t word, int i) {
                if constexpr (kEach == 1) return __builtin_bit_cast(float, word);
                else return T::to_float(static_cast<uint16_t>(word >> (16 * i)));
            };
            if (__popcll(some) <= 8) {
                // a lane's logits go through LDS to as many lanes
                for (; some != 0; some &= some - 1) {
                    const int from = __builtin_ctzll(some);
                    wave_handover();
                    if (lane == from) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) lane_words[wave][i] = v[i / 4][i % 4];
                    }
                    wave_handover();
                    const int i = lane % kBatch;
                    hold(logit_of(lane_words[wave][i / kEach], i % kEach), row.element_of(c, 64 * wave + from, i), lane < kBatch);
                }
                continue;
            }
            // logit e of every lane's piece in turn; unrolled the compares would take the scalar registers of everything
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                if (__any(piece_most[p] >= list.least)) {
                    const uint32_t w0 = v[p][0], w1 = v[p][1], w2 = v[p][2], w3 = v[p][3];
                    const int first = row.element(c, N * p);
#pragma unroll 1
                    for (int e = 0; e < N; ++e) {
                        const int word = e / kEach;
                        hold(logit_of(word == 0 ? w0 : word == 1 ? w1 : word == 2 ? w2 : w3, e % kEach), first + e, true);
                    }
                }
            }
        }
        // the waves' sums and lists
        sums.s = wave_add(sums.s);
        sums.d = wave_add(sums.d);
        if (segment > 0 && a.top == 0) __syncthreads();  // the ones before have been read; with lists the first chunk saw to that
        if (lane == 0) wave_sums[wave] = sums;
        if (a.top) {
            const int n = __popcll(__ballot(is_key(list.key)));  // the first n lanes'
            int at = 0;
            if (lane == 0) at = atomicAdd(&key_count[segment & 1], n);
            at = __builtin_amdgcn_readfirstlane(at);
            if (lane < n) keys[at + lane] = list.key;
        }
        __syncthreads();
        if (t == 0) key_count[(segment + 1) & 1] = 0;
        Sums all = joined(lane < kWaves ? wave_sums[lane] : Sums{-INFINITY, 0.0f, 0.0f});
        const int64_t part = static_cast<int64_t>(blockIdx.x) * 2 + (segment > 0);
        double ref = all.ref;
        if (whole) {
            if (leaves_fp32(all)) all = slow_sums<T, kThreads>(a, at_row, red, wave_sums, ref);
        } else if (t == 0) {
            a.sums[part] = float4{all.ref, all.s, all.d, 0.0f};
        }
        const Scored scored(a, all, ref);
        if (whole && t == 0) scored.store(a, at_row, all, given);
        if (whole && a.top && all.s != all.s) {
            slow_top<T, kThreads>(a, at_row, scored, red);
            continue;
        }
        if (a.top == 0) continue;
        const int n = key_count[segment & 1];
        for (int i = t; i < n; i += kThreads) {
            const uint64_t key = keys[i];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) rank += keys[j] > key ? 1 : 0;
            if (rank >= a.top) continue;
            if (whole) scored.store_top(a, at_row, rank, key);
            else a.keys[part * a.top + rank] = key;
        }
        if (!whole && n + t < a.top) a.keys[part * a.top + n + t] = 0;
    }
}

// A block a row: joins the parts that several blocks left of it.
template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads) void join_kernel(const ScoreArgs a) {
    constexpr int kFew = kThreads * 4;
    __shared__ uint64_t keys[kFew];
    __shared__ uint64_t red[kThreads / 64];
    __shared__ Sums wave_sums[kThreads / 64];
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x, first = row * a.chunks;
    const int64_t b0 = first / a.share, b1 = (first + a.chunks - 1) / a.share;
    if (b0 == b1) return;
    const Given<T> given(a, row, t == 0);
    const int n = static_cast<int>(b1 - b0) + 1, count = n * a.top;
    auto part = [&](int i) { return (b0 + i) * 2 + ((b0 + i) * a.share < first ? 1 : 0); };
    auto key_of = [&](int i) { return a.keys[part(i / a.top) * a.top + i % a.top]; };
    if (count <= kFew)
        for (int i = t; i < count; i += kThreads) keys[i] = key_of(i);
    // every wave joins all the parts, a lane every 64th
    Sums all{-INFINITY, 0.0f, 0.0f};
    for (int i = t & 63; i < n; i += 64) {
        const float4 p = a.sums[part(i)];
        all.join(Sums{p.x, p.y, p.z});
    }
    all = joined(all);
    double ref = all.ref;
    if (leaves_fp32(all)) all = slow_sums<T, kThreads>(a, row, red, wave_sums, ref);
    const Scored scored(a, all, ref);
    if (t == 0) scored.store(a, row, all, given);
    if (a.top == 0) return;
    if (all.s != all.s) {
        slow_top<T, kThreads>(a, row, scored, red);
        return;
    }
    if (count > kFew) {
        uint64_t key = ~uint64_t{0};
        for (int k = 0; k < a.top; ++k) {
            key = block_largest<kThreads>(key, count, red, key_of);
            if (t == 0) scored.store_top(a, row, k, key);
        }
        return;
    }
    __syncthreads();
    for (int i = t; i < count; i += kThreads) {
        const uint64_t key = keys[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < count; ++j) rank += keys[j] > key ? 1 : 0;
        if (is_key(key) && rank < a.top) scored.store_top(a, row, rank, key);
    }
}

constexpr int64_t kMaxVocab = int64_t{1} << 30;

struct Plan {
    bool wide = false;  // blocks of 1024 threads, else of 256
    int64_t chunks = 0, full = 0, share = 0, blocks = 0;
    size_t sums = 0, bytes = 0;
    bool joined() const { return share % chunks != 0; }
};

Plan make_plan(int64_t rows, int64_t vocab, int64_t top, int piece) {
    Plan p;
    // Rows that leave CUs idle are for wide blocks, one a CU: 150 rows of 32000 9.1 us a block of 256 threads for 8192 logits, 7.0 a
    // block of 1024 a row; 300 rows 9.0 and 12.3. (fp16 without alternatives) Each row in as many alike parts as there are CUs for
    // it, so that no block has parts of two: 180 rows of 128000 in fp32 with the largest 20.9 us, 26.5 in equal shares of all.
    p.wide = rows <= kCUs && vocab >= 8192;
    const int64_t chunk = (p.wide ? 1024 : 256) * 4 * piece;
    p.full = ceil_div(vocab + piece - 1, chunk);
    // Whole rows need no second launch to join their parts, 5 us: 100 rows of 16000 11.2 us, 15.0 cut. In bf16, 777 of 32000 15.4 and
    // 19.6, 400 of 16000 7.1 and 10.0. Few long rows leave a CU one block or two, which takes what the join would: of 128000, 257 rows
    // 20.2 and 20.2, with five alternatives 28.8 and 26.0, 513 34.5 and 34.8, 777 50.4 and 47.5, 1280 68.2 and 68.7; in fp32 28.1 and
    // 27.0, 36.1 and 35.5, 54.9 and 54.4, 81.4 and 79.0, 122.8 and 123.1.
    if (p.wide) p.share = p.full <= 2 ? p.full : ceil_div(p.full, kCUs / rows);
    else if (rows <= kPerCU * kCUs) p.share = p.full;
    else p.share = ceil_div(rows * p.full, kPerCU * kCUs);
    p.chunks = p.wide ? ceil_div(p.full, p.share) * p.share : p.full;
    p.blocks = ceil_div(rows * p.chunks, p.share);
    p.sums = static_cast<size_t>(p.blocks) * 2 * sizeof(float4);
    p.bytes = p.joined() ? p.sums + static_cast<size_t>(p.blocks) * 2 * top * sizeof(uint64_t) : 0;
    return p;
}

// A call's plan; no blocks where there is none.
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
    if (!p.joined()) return;
    // of few parts a wave a row
    const dim3 all(static_cast<unsigned>(rows));
    if ((ceil_div(p.chunks, p.share) + 1) * a.top <= 128) join_kernel<T, 64><<<all, 64, 0, st>>>(a);
    else join_kernel<T, 256><<<all, 256, 0, st>>>(a);
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
    if (plan.bytes && (!workspace || workspace_bytes < plan.bytes))
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
    a.rows = static_cast<int>(rows);
    a.vocab = static_cast<int>(vocab);
    a.top = static_cast<int>(top);
    a.chunks = static_cast<int>(plan.chunks);
    a.full = static_cast<int>(plan.full);
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
