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

}  // namespace nq
