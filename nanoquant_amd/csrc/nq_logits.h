// Rows of logits in the types that the kernels take, read in aligned pieces.
#pragma once

#include "nq_common.h"

namespace nq {

struct F32 {};

// Logits come in aligned pieces of 16 bytes, whatever the row's alignment: piece k of a row holds its elements
// k * N - lead .. + N - 1, of which those outside the row (of its first and last piece) are not used.
template <typename T>
struct Elem {
    static constexpr int N = 8;
    static constexpr uint32_t kNone = T::ONE_PAIR == 0x3C003C00u ? 0xFC00FC00u : 0xFF80FF80u;  // -inf
    __device__ static float get(const void* p, int64_t i) { return T::to_float(static_cast<const uint16_t*>(p)[i]); }
    __device__ static void unpack(const u32x4& v, float* x) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = T::to_float(static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1))));
    }
};
template <>
struct Elem<F32> {
    static constexpr int N = 4;
    static constexpr uint32_t kNone = 0xFF800000u;
    __device__ static float get(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
    __device__ static void unpack(const u32x4& v, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = v[i];  // of the vector's element itself, bit_cast takes the first
            x[i] = __builtin_bit_cast(float, w);
        }
    }
};

// A row as blocks of kThreads threads take it, kBatch logits a thread at a time.
template <typename T, int kThreads, int kBatch>
struct LogitRow {
    static constexpr int N = Elem<T>::N, kPieces = kBatch / N;
    const u32x4* pieces;
    int lead, vocab, last;  // piece
    __device__ LogitRow(const void* logits, int64_t first, int64_t vocab_) {
        constexpr int size = 16 / N;
        const char* at = static_cast<const char*>(logits) + first * size;
        const int off = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
        pieces = reinterpret_cast<const u32x4*>(at - off);
        lead = off / size;
        vocab = static_cast<int>(vocab_);
        last = (vocab + lead - 1) / N;
    }
    // Part k of a row is its elements k kBatch kThreads - lead on; element i of this thread's is element(k, i).
    __device__ int element(int k, int i) const { return element_of(k, static_cast<int>(threadIdx.x), i); }
    __device__ int element_of(int k, int thread, int i) const {
        return (k * (kPieces * kThreads) + (i / N) * kThreads + thread) * N - lead + i % N;
    }
    __device__ void load(int k, u32x4* v) const {  // past the last piece, which is not used, the last
#pragma unroll
        for (int i = 0; i < kPieces; ++i) v[i] = pieces[min((k * kPieces + i) * kThreads + static_cast<int>(threadIdx.x), last)];
    }
    __device__ void load_once(int k, u32x4* v) const {  // the same of what is not read again
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            v[i] = __builtin_nontemporal_load(pieces + min((k * kPieces + i) * kThreads + static_cast<int>(threadIdx.x), last));
    }
    __device__ bool at_edge(int k) const { return (k == 0 && lead > 0) || (k + 1) * (kBatch * kThreads) - lead > vocab; }
    // Piece p of this thread's in part k with -inf for what lies outside the row
    __device__ u32x4 cleared(int k, int p, u32x4 v) const {
        constexpr int each = N / 4;  // logits of a word
        const int first = element(k, N * p);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t keep = 0;
#pragma unroll
            for (int i = 0; i < each; ++i)
                if (static_cast<unsigned>(first + each * w + i) < static_cast<unsigned>(vocab))
                    keep |= (each == 1 ? 0xFFFFFFFFu : 0xFFFFu) << (16 * i);
            v[w] = bit_select(keep, v[w], Elem<T>::kNone);
        }
        return v;
    }
    // -inf for what lies outside the row
    __device__ void unpack(int k, const u32x4* v, float* x) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) Elem<T>::unpack(v[i], x + N * i);
        if (at_edge(k)) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                x[i] = static_cast<unsigned>(element(k, i)) < static_cast<unsigned>(vocab) ? x[i] : -INFINITY;
        }
    }
};

}  // namespace nq
