// Verification of drafted tokens: softmax statistics of every row of logits, the accept tests, and one token by inverse CDF
// from the row where the drafts end:
//   1. row_stats_kernel, a block per (row, chunk of one or more parts of 4096 logits): the chunk's largest logit m_c (with its
//      index) and z_c = sum exp((x - m_c) / T);
//   2. the accept tests u q(x) < p(x) with the rows' joined statistics, and part_sums_kernel, a block per (sequence, 4096
//      logits): the sums of w = max(p - q, 0) and of p over its part of the row that the tests ended at. Up to three blocks a
//      CU every block makes its sequence's tests itself, beyond that a launch of their own does, a block a sequence: seven
//      drafts against 100000 bf16 logits 26.4 us against 28.2 for 16 sequences, 37.2 against 38.2 for 32, 61.2 against 59.4
//      for 64 (42.3 against 41.4 and 70.0 against 65.5 for 32 and 64 in fp32);
//   3. pick_token_kernel, a block per sequence: the part in which the running sum of w passes u times its total, then the
//      index within it.
// Probabilities and their sums are fp64: the token is where a running sum over up to 10^5 terms passes a number, and fp32
// rounding would move a visible share of the borders between tokens.
#include <algorithm>
#include <cfloat>

#include "nq_common.h"
#include "nq_wave.h"

namespace nq {
namespace {

constexpr int kThreads = 256, kCUs = 256;
struct F32 {};

// Logits come in aligned pieces of 16 bytes, whatever the row's alignment: piece k of a row holds its elements
// k * N - lead .. + N - 1, of which those outside the row (of its first and last piece) are not used.
template <typename T>
struct Elem {
    static constexpr int N = 8;
    __device__ static float get(const void* p, int64_t i) { return T::to_float(static_cast<const uint16_t*>(p)[i]); }
    __device__ static void unpack(const u32x4& v, float* x) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = T::to_float(static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1))));
    }
};
template <>
struct Elem<F32> {
    static constexpr int N = 4;
    __device__ static float get(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
    __device__ static void unpack(const u32x4& v, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = v[i];  // of the vector's element itself, bit_cast takes the first
            x[i] = __builtin_bit_cast(float, w);
        }
    }
};

constexpr int kPart = 4096;             // logits a block takes at a time
constexpr int kBatch = kPart / kThreads;  // and a thread of row_stats_kernel's

template <typename T>
struct Row {
    static constexpr int N = Elem<T>::N, kPieces = kBatch / N;
    const u32x4* pieces;
    int lead, vocab, last;  // piece
    __device__ Row(const void* logits, int64_t first, int64_t vocab_) {
        constexpr int size = 16 / N;
        const char* at = static_cast<const char*>(logits) + first * size;
        const int off = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
        pieces = reinterpret_cast<const u32x4*>(at - off);
        lead = off / size;
        vocab = static_cast<int>(vocab_);
        last = (vocab + lead - 1) / N;
    }
    // Part k of a row is its elements k kPart - lead on; element i of this thread's is element(k, i).
    __device__ int element(int k, int i) const {
        return (k * (kPieces * kThreads) + (i / N) * kThreads + static_cast<int>(threadIdx.x)) * N - lead + i % N;
    }
    __device__ void load(int k, u32x4* v) const {  // past the last piece, which is not used, the last
#pragma unroll
        for (int i = 0; i < kPieces; ++i) v[i] = pieces[min((k * kPieces + i) * kThreads + static_cast<int>(threadIdx.x), last)];
    }
    // -inf for what lies outside the row
    __device__ void unpack(int k, const u32x4* v, float* x) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) Elem<T>::unpack(v[i], x + N * i);
        if (k == 0 || (k + 1) * (kBatch * kThreads) - lead > vocab) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) x[i] = static_cast<unsigned>(element(k, i)) < static_cast<unsigned>(vocab) ? x[i] : -INFINITY;
        }
    }
};

// exp(d) for d <= 0 as p t: n = round(128 d / ln2), t = 2^(n / 128) from a table, with n / 128's whole part added to its
// exponent, and a polynomial p of |r| <= ln2 / 256 (table-driven exp, Tang 1989), whose first term left out is below 2^-49. n
// comes as the low bits of a sum with 1.5 * 2^52. The copy in LDS has i << 13 taken from the upper word of entry i, so that
// all of n << 13 is added to it (an exponent's one is 2^20). A table of 32 entries, a copy in every pair of LDS banks, and one
// term more cost 10%: the arithmetic bounds this, not the table's reads.
constexpr int kTable = 128;
__device__ const double kPowers[kTable] = {  // 2^(i / 128)
    0x1.0000000000000p+0, 0x1.0163da9fb3335p+0, 0x1.02c9a3e778061p+0, 0x1.04315e86e7f85p+0, 0x1.059b0d3158574p+0,
    0x1.0706b29ddf6dep+0, 0x1.0874518759bc8p+0, 0x1.09e3ecac6f383p+0, 0x1.0b5586cf9890fp+0, 0x1.0cc922b7247f7p+0,
    0x1.0e3ec32d3d1a2p+0, 0x1.0fb66affed31bp+0, 0x1.11301d0125b51p+0, 0x1.12abdc06c31ccp+0, 0x1.1429aaea92de0p+0,
    0x1.15a98c8a58e51p+0, 0x1.172b83c7d517bp+0, 0x1.18af9388c8deap+0, 0x1.1a35beb6fcb75p+0, 0x1.1bbe084045cd4p+0,
    0x1.1d4873168b9aap+0, 0x1.1ed5022fcd91dp+0, 0x1.2063b88628cd6p+0, 0x1.21f49917ddc96p+0, 0x1.2387a6e756238p+0,
    0x1.251ce4fb2a63fp+0, 0x1.26b4565e27cddp+0, 0x1.284dfe1f56381p+0, 0x1.29e9df51fdee1p+0, 0x1.2b87fd0dad990p+0,
    0x1.2d285a6e4030bp+0, 0x1.2ecafa93e2f56p+0, 0x1.306fe0a31b715p+0, 0x1.32170fc4cd831p+0, 0x1.33c08b26416ffp+0,
    0x1.356c55f929ff1p+0, 0x1.371a7373aa9cbp+0, 0x1.38cae6d05d866p+0, 0x1.3a7db34e59ff7p+0, 0x1.3c32dc313a8e5p+0,
    0x1.3dea64c123422p+0, 0x1.3fa4504ac801cp+0, 0x1.4160a21f72e2ap+0, 0x1.431f5d950a897p+0, 0x1.44e086061892dp+0,
    0x1.46a41ed1d0057p+0, 0x1.486a2b5c13cd0p+0, 0x1.4a32af0d7d3dep+0, 0x1.4bfdad5362a27p+0, 0x1.4dcb299fddd0dp+0,
    0x1.4f9b2769d2ca7p+0, 0x1.516daa2cf6642p+0, 0x1.5342b569d4f82p+0, 0x1.551a4ca5d920fp+0, 0x1.56f4736b527dap+0,
    0x1.58d12d497c7fdp+0, 0x1.5ab07dd485429p+0, 0x1.5c9268a5946b7p+0, 0x1.5e76f15ad2148p+0, 0x1.605e1b976dc09p+0,
    0x1.6247eb03a5585p+0, 0x1.6434634ccc320p+0, 0x1.6623882552225p+0, 0x1.68155d44ca973p+0, 0x1.6a09e667f3bcdp+0,
    0x1.6c012750bdabfp+0, 0x1.6dfb23c651a2fp+0, 0x1.6ff7df9519484p+0, 0x1.71f75e8ec5f74p+0, 0x1.73f9a48a58174p+0,
    0x1.75feb564267c9p+0, 0x1.780694fde5d3fp+0, 0x1.7a11473eb0187p+0, 0x1.7c1ed0130c132p+0, 0x1.7e2f336cf4e62p+0,
    0x1.80427543e1a12p+0, 0x1.82589994cce13p+0, 0x1.8471a4623c7adp+0, 0x1.868d99b4492edp+0, 0x1.88ac7d98a6699p+0,
    0x1.8ace5422aa0dbp+0, 0x1.8cf3216b5448cp+0, 0x1.8f1ae99157736p+0, 0x1.9145b0b91ffc6p+0, 0x1.93737b0cdc5e5p+0,
    0x1.95a44cbc8520fp+0, 0x1.97d829fde4e50p+0, 0x1.9a0f170ca07bap+0, 0x1.9c49182a3f090p+0, 0x1.9e86319e32323p+0,
    0x1.a0c667b5de565p+0, 0x1.a309bec4a2d33p+0, 0x1.a5503b23e255dp+0, 0x1.a799e1330b358p+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ac36bbfd3f37ap+0, 0x1.ae89f995ad3adp+0, 0x1.b0e07298db666p+0, 0x1.b33a2b84f15fbp+0, 0x1.b59728de5593ap+0,
    0x1.b7f76f2fb5e47p+0, 0x1.ba5b030a1064ap+0, 0x1.bcc1e904bc1d2p+0, 0x1.bf2c25bd71e09p+0, 0x1.c199bdd85529cp+0,
    0x1.c40ab5fffd07ap+0, 0x1.c67f12e57d14bp+0, 0x1.c8f6d9406e7b5p+0, 0x1.cb720dcef9069p+0, 0x1.cdf0b555dc3fap+0,
    0x1.d072d4a07897cp+0, 0x1.d2f87080d89f2p+0, 0x1.d5818dcfba487p+0, 0x1.d80e316c98398p+0, 0x1.da9e603db3285p+0,
    0x1.dd321f301b460p+0, 0x1.dfc97337b9b5fp+0, 0x1.e264614f5a129p+0, 0x1.e502ee78b3ff6p+0, 0x1.e7a51fbc74c83p+0,
    0x1.ea4afa2a490dap+0, 0x1.ecf482d8e67f1p+0, 0x1.efa1bee615a27p+0, 0x1.f252b376bba97p+0, 0x1.f50765b6e4540p+0,
    0x1.f7bfdad9cbe14p+0, 0x1.fa7c1819e90d8p+0, 0x1.fd3c22b8f71f1p+0,
};
__device__ inline void fill_table(double* table) {
    if (threadIdx.x < kTable)
        table[threadIdx.x] = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, kPowers[threadIdx.x]) - (static_cast<uint64_t>(threadIdx.x) << 45));
}
__device__ inline uint32_t exp_reduce(double d, double& p) {  // n, p
    constexpr double kMagic = 6755399441055744.0;
    const double sum = fma(d, kTable * 1.4426950408889634, kMagic);
    const double r = fma(sum - kMagic, -0.6931471805599453 / kTable, d);
    p = fma(r, 1.0 / 24, 1.0 / 6);
    p = fma(r, p, 0.5);
    p = fma(r, p, 1.0);
    p = fma(r, p, 1.0);
    return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, sum));
}
__device__ inline double exp_power(uint32_t n, uint32_t add, const double* table) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    u32x2 bits = __builtin_bit_cast(u32x2, table[n & (kTable - 1)]);
    bits.y += add << 13;
    return __builtin_bit_cast(double, bits);
}
// For sums in which there is a 1 as well: below -700 exp(d) counts as exp(-700), which is nothing beside it.
__device__ inline void exp_parts(double d, const double* table, double& p, double& t) {
    const uint32_t n = exp_reduce(fmax(d, -700.0), p);
    t = exp_power(n, n, table);
}
__device__ inline double exp_of(double d, const double* table) {
    double p, t;
    exp_parts(d, table, p, t);
    return p * t;
}
// For what is compared with 0: subnormal where exp(d) is, and 0 below that (about -745). The whole part of n / 128 goes in last.
__device__ inline double exp_or_zero(double d, const double* table) {
    double p;
    const uint32_t n = exp_reduce(fmax(d, -1100.0), p);
    return __builtin_ldexp(p * exp_power(n, n & (kTable - 1), table), static_cast<int>(n) >> 7);
}

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

struct Stat {
    uint64_t rank;  // of the largest logit
    double z;       // sum exp((x - largest) / T); 0 where the largest is no finite number
};

// Where a sequence's drafts end.
struct Walk {
    int kept;    // accepted drafts: the row that the next token comes from
    int draft;   // that row's draft where it was turned down (w = max(p - q, 0)), else -1
    Stat stat;   // of that row
    double inv_z;
};
static_assert(sizeof(Stat) == 16 && sizeof(Walk) == 32, "as the workspace's size counts them");

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
    int drafts, chunks, parts, row_parts;  // chunks a row, parts a chunk and a row
    Stat* stats;    // [batch * (drafts + 1)][chunks]
    double2* sums;  // [batch][row_parts]: of w and of p
    Walk* walks;    // [batch]
};

// A chunk is a.parts parts. A thread goes through its own with its own running maximum, so that the block meets once, at
// the end. Bound by arithmetic: about 18 instructions an element, 11 of them fp64; 512 rows of 100003 bf16 logits, 102 MB, take
// 44 us, where 29 are the instructions' issue and 20 a copy's rate.
template <typename T>
__global__ __launch_bounds__(kThreads) void row_stats_kernel(const VerifyArgs a) {
    __shared__ double table[kTable];
    __shared__ uint64_t ranks[kThreads / 64];
    __shared__ double zs[kThreads / 64];
    __shared__ uint32_t index;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t row = blockIdx.x / a.chunks;
    const int k0 = static_cast<int>(blockIdx.x - row * a.chunks) * a.parts;
    const Row<T> src(a.logits, row * a.row_stride, a.vocab);
    const int n = min(a.parts, a.row_parts - k0);
    u32x4 v[Row<T>::kPieces];
    src.load(k0, v);
    fill_table(table);
    if (t == 0) index = 0xFFFFFFFFu;
    __syncthreads();
    float m = -INFINITY;
    bool odd = false;  // some element is a NaN
    int found = k0;                   // the part that m is of
    double z = 0.0;
    for (int k = 0; k < n; ++k) {
        float x[kBatch];
        src.unpack(k0 + k, v, x);
        if (k + 1 < n) src.load(k0 + k + 1, v);
        float top = x[0];
#pragma unroll
        for (int i = 0; i < kBatch; i += 2) {
            top = fmaxf(top, fmaxf(x[i], x[i + 1]));
            odd |= __builtin_isunordered(x[i], x[i + 1]);
        }
        if (top > m) {
            z *= exp_of((static_cast<double>(m) - top) * a.inv_t, table);
            m = top;
            found = k0 + k;
        }
        const double base = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            double p, power;
            // the difference first: x / T and m / T, rounded, would be off by more than 1 apart where T is small
            exp_parts((static_cast<double>(x[i]) - base) * a.inv_t, table, p, power);
            z = fma(p, power, z);
        }
    }
    // the largest of the block, and its first index: only threads that hold it look for it again, those with a NaN in all of
    // their parts
    float nan = m;
    int nan_at = found;
    if (odd) {
        for (int k = n - 1; k >= 0; --k) {
            float x[kBatch];
            src.load(k0 + k, v);
            src.unpack(k0 + k, v, x);
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (x[i] != x[i]) {
                    nan = x[i];
                    nan_at = k0 + k;
                }
        }
    }
    const uint64_t own = rank_of(nan, 0xFFFFFFFFu);
    uint64_t best = wave_largest(own);
    if (lane == 0) ranks[wave] = best;
    __syncthreads();
    best = max(max(ranks[0], ranks[1]), max(ranks[2], ranks[3]));
    if (own == best) {
        float x[kBatch];
        src.load(nan_at, v);
        src.unpack(nan_at, v, x);
        uint32_t at = 0xFFFFFFFFu;
#pragma unroll
        for (int i = kBatch - 1; i >= 0; --i) {
            const int j = src.element(nan_at, i);
            if (j >= 0 && j < src.vocab && rank_of(x[i], 0xFFFFFFFFu) == best) at = static_cast<uint32_t>(j);
        }
        if (at != 0xFFFFFFFFu) atomicMin(&index, at);
    }
    const float top = rank_value(best);
    z = finite(top) && m != -INFINITY ? z * exp_of((static_cast<double>(m) - top) * a.inv_t, table) : 0.0;
    z = wave_total(z);
    if (lane == 0) zs[wave] = z;
    __syncthreads();
    if (t == 0) a.stats[blockIdx.x] = Stat{(best & ~uint64_t{0xFFFFFFFFu}) | static_cast<uint32_t>(~index), (zs[0] + zs[1]) + (zs[2] + zs[3])};
}

// A row's statistics from its chunks', in the 16 lanes that call it together.
__device__ inline Stat join_row(const VerifyArgs& a, int64_t row, const double* table) {
    const int l = threadIdx.x & 15;
    const Stat* stats = a.stats + row * a.chunks;
    uint64_t best = 0;
    for (int c = l; c < a.chunks; c += 16) best = max(best, stats[c].rank);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) best = max(best, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(best), off, 64)));
    const float m = rank_value(best);
    double z = 0.0;
    if (finite(m))
        for (int c = l; c < a.chunks; c += 16) {
            const Stat s = stats[c];
            const float mc = rank_value(s.rank);
            if (finite(mc)) z += s.z * exp_of((static_cast<double>(mc) - m) * a.inv_t, table);  // -inf adds nothing
        }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) z += __shfl_xor(z, off, 64);
    return Stat{best, z};
}

// Where the drafts of sequence b end, by the whole block: 16 lanes a row, blockDim / 16 rows at a time, whose tests do not wait
// for each other.
template <typename T, int kThreads>
__device__ inline Walk walk_of(const VerifyArgs& a, int64_t b, const double* table) {
    __shared__ int end;  // 2 * row + (1: turned down) of the first row that ends the drafts
    __shared__ Stat stats[kThreads / 16];
    const int t = threadIdx.x, group = t >> 4;
    if (t == 0) end = INT32_MAX;
    __syncthreads();
    for (int i0 = 0;; i0 += kThreads / 16) {
        const int i = i0 + group;
        if (i <= a.drafts) {
            const int64_t row = b * (a.drafts + 1) + i;
            const int64_t x = i < a.drafts ? a.draft[b * a.drafts + i] : -1;
            const bool real = x >= 0 && x < a.vocab;
            const double u = a.uniforms[row];
            const float logit = real ? Elem<T>::get(a.logits, row * a.row_stride + x) : 0.0f;
            const float qx = real && a.draft_probs ? a.draft_probs[(b * a.drafts + i) * a.vocab + x] : 1.0f;
            const Stat st = join_row(a, row, table);
            const float m = rank_value(st.rank);
            double p = 0.0;
            if (a.inv_t == 0.0 || !finite(m)) p = finite(m) && rank_index(st.rank) == x ? 1.0 : 0.0;
            else if (logit != -INFINITY) p = exp_or_zero((static_cast<double>(logit) - m) * a.inv_t, table) / st.z;
            const double q = a.inv_t != 0.0 ? qx : 1.0;
            if ((t & 15) == 0) {
                stats[group] = st;
                if (!real) atomicMin(&end, 2 * i);
                else if (!(u * q < p)) atomicMin(&end, 2 * i + 1);
            }
        }
        __syncthreads();
        if (end != INT32_MAX) break;  // the last row ends them at the latest
        __syncthreads();
    }
    const int at = end;
    const Stat st = stats[(at >> 1) % (kThreads / 16)];
    const int64_t draft = at & 1 ? a.draft[b * a.drafts + (at >> 1)] : -1;
    return Walk{at >> 1, static_cast<int>(draft), st, 1.0 / st.z};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void walk_kernel(const VerifyArgs a) {
    __shared__ double table[kTable];
    fill_table(table);
    const Walk walk = walk_of<T, kThreads>(a, blockIdx.x, table);
    if (threadIdx.x == 0) a.walks[blockIdx.x] = walk;
}

// A part of a row, a piece a thread of 4096 / N: its p and w.
template <typename T>
struct Part {
    static constexpr int N = Elem<T>::N, kThreads = kPart / N;
    int first;  // the piece's first element
    double p[N], w[N];
    __device__ Part(const VerifyArgs& a, int64_t b, int part, const Walk& walk, const double* table) {
        const Row<T> src(a.logits, (b * (a.drafts + 1) + walk.kept) * a.row_stride, a.vocab);
        const int piece = part * kThreads + static_cast<int>(threadIdx.x);
        first = piece * N - src.lead;
        const u32x4 v = src.pieces[min(piece, src.last)];
        float x[N], q[N];
        const bool inside = first >= 0 && first + N <= src.vocab;
        if (walk.draft >= 0 && a.draft_probs) {
            const float* row = a.draft_probs + (b * a.drafts + walk.kept) * a.vocab;
            typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));  // any row begins at a multiple of 4 bytes
            if (inside) {
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    const f32x4a four = *reinterpret_cast<const f32x4a*>(row + first + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[i + e] = four[e];
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) q[i] = row[min(max(first + i, 0), src.vocab - 1)];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) q[i] = first + i == walk.draft ? 1.0f : 0.0f;
        }
        Elem<T>::unpack(v, x);
        const double top = rank_value(walk.stat.rank);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool none = x[i] == -INFINITY || !(inside || static_cast<unsigned>(first + i) < static_cast<unsigned>(src.vocab));
            p[i] = none ? 0.0 : exp_or_zero((static_cast<double>(x[i]) - top) * a.inv_t, table) * walk.inv_z;
            w[i] = walk.draft >= 0 ? (p[i] > q[i] ? p[i] - q[i] : 0.0) : p[i];
        }
    }
};

// Bound by latency too, of the statistics, of the tests, then of the part: 12 us for 64 sequences of 25 parts.
template <typename T, bool kTests>
__global__ __launch_bounds__(Part<T>::kThreads) void part_sums_kernel(const VerifyArgs a) {
    constexpr int kWaves = Part<T>::kThreads / 64;
    __shared__ double table[kTable];
    __shared__ double2 sums[kWaves];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t b = blockIdx.x / a.row_parts;
    fill_table(table);
    Walk walk;
    if constexpr (kTests) {
        walk = walk_of<T, Part<T>::kThreads>(a, b, table);
    } else {
        walk = a.walks[b];
        __syncthreads();
    }
    const int at = static_cast<int>(blockIdx.x - b * a.row_parts);
    if (kTests && at == 0 && t == 0) a.walks[b] = walk;
    if (a.inv_t == 0.0 || !finite(rank_value(walk.stat.rank))) return;  // the token is the argmax
    const Part<T> part(a, b, at, walk, table);
    double2 s = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < Part<T>::N; ++i) {
        s.x += part.w[i];
        s.y += part.p[i];
    }
    s.x = wave_total(s.x);
    s.y = wave_total(s.y);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    if (t == 0) {
        for (int i = 1; i < kWaves; ++i) {
            s.x += sums[i].x;
            s.y += sums[i].y;
        }
        a.sums[blockIdx.x] = s;
    }
}

// Bound by latency: what does not depend on the walk is loaded with it. 4 to 5 us.
template <typename T>
__global__ __launch_bounds__(Part<T>::kThreads) void pick_token_kernel(const VerifyArgs a) {
    constexpr int N = Elem<T>::N, kThreads = Part<T>::kThreads, kWaves = kThreads / 64;
    __shared__ double table[kTable];
    __shared__ int s_part, s_plain;
    __shared__ double s_target, s_before;
    __shared__ int s_first, s_last;
    __shared__ double sums_of[kWaves];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t b = blockIdx.x;
    const double2* sums = a.sums + b * a.row_parts;
    const double2 own = wave == 0 && lane < a.row_parts ? sums[lane] : double2{0.0, 0.0};
    const double u = a.uniforms[b * (a.drafts + 1) + a.drafts];
    const int64_t draft = t < a.drafts ? a.draft[b * a.drafts + t] : -1;
    const Walk walk = a.walks[b];
    fill_table(table);
    int64_t token = rank_index(walk.stat.rank);
    if (a.inv_t != 0.0 && finite(rank_value(walk.stat.rank))) {
        if (wave == 0) {
            double total = own.x, total_p = own.y;
            for (int c = lane + 64; c < a.row_parts; c += 64) {
                total += sums[c].x;
                total_p += sums[c].y;
            }
            total = wave_total(total);
            total_p = wave_total(total_p);
            const bool plain = !(total > 0.0);  // nothing left: the row itself
            const double target = u * (plain ? total_p : total);
            // the first part whose running sum passes the target; the last one with a positive sum where rounding hides it
            double run = 0.0, before = 0.0;
            int found = -1, last = 0;
            for (int c0 = 0; c0 < a.row_parts && found < 0; c0 += 64) {
                const double2 both = c0 == 0 ? own : c0 + lane < a.row_parts ? sums[c0 + lane] : double2{0.0, 0.0};
                const double v = plain ? both.y : both.x;
                const double incl = wave_scan(v);
                const uint64_t pass = __ballot(v > 0.0 && run + incl > target);
                const uint64_t some = __ballot(v > 0.0);
                if (some) last = c0 + 63 - __builtin_clzll(some);
                if (pass) {
                    const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(pass));
                    found = c0 + at;
                    before = run + read_lane(incl - v, at);
                }
                run += read_lane(incl, 63);
            }
            if (lane == 0) {
                s_part = found < 0 ? last : found;
                s_target = found < 0 ? INFINITY : target;
                s_before = before;
                s_plain = plain;
                s_first = INT32_MAX;  // the first index that passes
                s_last = -1;          // the last one with a positive weight
            }
        }
        __syncthreads();
        const bool plain = s_plain;
        const double target = s_target;
        const Part<T> part(a, b, s_part, walk, table);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) sum += plain ? part.p[i] : part.w[i];
        const double incl = wave_scan(sum);
        if (lane == 63) sums_of[wave] = incl;
        __syncthreads();
        double run = s_before + wave_total(lane < wave ? sums_of[lane % kWaves] : 0.0) + (incl - sum);
        int first = INT32_MAX, last = -1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const double weight = plain ? part.p[i] : part.w[i];
            run += weight;
            if (weight > 0.0) {
                last = part.first + i;
                if (run > target) first = min(first, last);
            }
        }
        // of a wave its first lane that passes and its last one with a weight
        const uint64_t passes = __ballot(first != INT32_MAX), some = __ballot(last >= 0);
        if (passes && lane == __builtin_ctzll(passes)) atomicMin(&s_first, first);
        if (some && lane == 63 - __builtin_clzll(some)) atomicMax(&s_last, last);
        __syncthreads();
        token = s_first != INT32_MAX ? s_first : s_last;
    }
    if (t == 0) a.accepted[b] = walk.kept;
    for (int i = t; i <= a.drafts; i += kThreads) {
        const int64_t kept = i == t ? draft : a.draft[b * a.drafts + min(i, a.drafts - 1)];
        a.tokens[b * (a.drafts + 1) + i] = i < walk.kept ? kept : (i == walk.kept ? token : -1);
    }
}

// Parts of a row, which may begin up to 7 elements into its first piece; chunks of a row, each of as many parts as make all
// rows' chunks come into the card at once (8 blocks a CU), for a block's fixed part (its table, reductions of 64-bit numbers)
// costs as much as half a part, and a second round of blocks as much as the first: 512 rows of 25 parts in 4 chunks each 62.3
// us a call, in 7 of four parts 63.3.
int64_t row_parts_of(int64_t vocab) { return ceil_div(vocab + 7, kBatch * kThreads); }
int64_t parts_of(int64_t rows, int64_t vocab) {
    const int64_t most = std::max<int64_t>(1, 2048 / rows);
    return ceil_div(row_parts_of(vocab), most);
}
int64_t chunks_of(int64_t rows, int64_t vocab) { return ceil_div(row_parts_of(vocab), parts_of(rows, vocab)); }

template <typename T>
void launch_verify(const VerifyArgs& a, int64_t batch, hipStream_t st) {
    const int64_t rows = batch * (a.drafts + 1);
    row_stats_kernel<T><<<dim3(static_cast<unsigned>(rows * a.chunks)), kThreads, 0, st>>>(a);
    const dim3 grid(static_cast<unsigned>(batch * a.row_parts));
    if (batch * a.row_parts <= 3 * kCUs) {
        part_sums_kernel<T, true><<<grid, Part<T>::kThreads, 0, st>>>(a);
    } else {
        walk_kernel<T><<<dim3(static_cast<unsigned>(batch)), kThreads, 0, st>>>(a);
        part_sums_kernel<T, false><<<grid, Part<T>::kThreads, 0, st>>>(a);
    }
    pick_token_kernel<T><<<dim3(static_cast<unsigned>(batch)), Part<T>::kThreads, 0, st>>>(a);
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" {

size_t nq_verify_drafts_workspace_bytes(int64_t batch, int64_t drafts, int64_t vocab) {
    if (batch <= 0 || drafts < 0 || vocab <= 0 || vocab > (1 << 30) || batch > INT32_MAX || drafts > INT32_MAX / 2) return 0;
    if (batch > (int64_t{1} << 23) / (drafts + 1)) return 0;
    const int64_t chunks = chunks_of(batch * (drafts + 1), vocab);
    if (batch * (drafts + 1) > (int64_t{1} << 23) / chunks || batch > (int64_t{1} << 23) / row_parts_of(vocab)) return 0;
    return static_cast<size_t>(batch) * (((drafts + 1) * chunks + row_parts_of(vocab)) * 16 + 32);
}

int nq_verify_drafts(int dtype, const void* logits, int64_t row_stride, const int64_t* draft, const float* draft_probs,
                     const float* uniforms, double temperature, int64_t* accepted, int64_t* tokens, int64_t batch,
                     int64_t drafts, int64_t vocab, void* workspace, size_t workspace_bytes, nq_stream_t stream) {
    const char* name = "nq_verify_drafts";
    if (dtype != NQ_F16 && dtype != NQ_BF16 && dtype != NQ_F32) return fail(NQ_ERR_DTYPE, "%s: unsupported dtype %d", name, dtype);
    if (batch < 0 || drafts < 0 || vocab <= 0) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: bad sizes", name);
    if (row_stride < vocab) return fail(NQ_ERR_SHAPE, "%s: rows of logits overlap", name);
    if (!(temperature >= 0.0 && temperature <= DBL_MAX))
        return fail(NQ_ERR_INVALID_ARGUMENT, "%s: the temperature must be a finite number from 0", name);
    if (batch == 0) return NQ_OK;
    const size_t need = nq_verify_drafts_workspace_bytes(batch, drafts, vocab);
    const int64_t part_threads = dtype == NQ_F32 ? Part<F32>::kThreads : Part<F16>::kThreads;
    if (need == 0 || batch * row_parts_of(vocab) > UINT32_MAX / part_threads)  // a launch's threads are counted in 32 bits
        return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large", name);
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
    // finite, so that 0 stays 0: two logits that differ are 2^-149 apart at least, far enough for any such temperature
    a.inv_t = temperature > 0.0 ? std::min(1.0 / temperature, DBL_MAX) : 0.0;
    a.accepted = accepted;
    a.tokens = tokens;
    a.vocab = vocab;
    a.drafts = static_cast<int>(drafts);
    a.chunks = static_cast<int>(chunks_of(batch * (drafts + 1), vocab));
    a.parts = static_cast<int>(parts_of(batch * (drafts + 1), vocab));
    a.row_parts = static_cast<int>(row_parts_of(vocab));
    a.stats = static_cast<Stat*>(workspace);
    a.sums = reinterpret_cast<double2*>(a.stats + batch * (drafts + 1) * a.chunks);
    a.walks = reinterpret_cast<Walk*>(a.sums + batch * a.row_parts);
    if (dtype == NQ_F16) launch_verify<F16>(a, batch, as_stream(stream));
    else if (dtype == NQ_BF16) launch_verify<BF16>(a, batch, as_stream(stream));
    else launch_verify<F32>(a, batch, as_stream(stream));
    return check_launch(name);
}

}  // extern "C"
