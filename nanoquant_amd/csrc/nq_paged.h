// What the kernels of the paged cache share: its pages, and the checks of a call's arguments.
#pragma once

#include "nq_common.h"

namespace nq {

// A pointer that is the same for the whole wave, in scalar registers.
__device__ inline const uint16_t* uniform(const uint16_t* p) {
    const uint64_t u = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u)), hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u >> 32));
    return reinterpret_cast<const uint16_t*>(static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ inline const u32x4* vec(const uint16_t* p) { return reinterpret_cast<const u32x4*>(p); }

// The page of position p of a sequence, -1 where there is none.
struct Pages {
    const int32_t* table;
    int64_t table_stride;
    int table_pages, pages, page_size;
    uint32_t inverse;  // 2^shift / page_size, rounded up: with 2^31 below that, exact for what is below 2^31
    int shift;
    Pages() = default;
    Pages(const int32_t* table_, int64_t stride, int64_t table_pages_, int64_t pages_, int64_t page_size_)
        : table(table_), table_stride(stride), table_pages(static_cast<int>(table_pages_)), pages(static_cast<int>(pages_)),
          page_size(static_cast<int>(page_size_)), shift(31) {
        while ((int64_t{1} << (shift - 31)) < page_size_) ++shift;
        inverse = static_cast<uint32_t>((uint64_t{1} << shift) / static_cast<uint64_t>(page_size_) + 1);
    }
    __device__ int slot_of(int key) const {  // key / page_size, in three instructions instead of thirty
        return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(key)) * inverse >> shift);
    }
    __device__ int64_t capacity() const { return static_cast<int64_t>(table_pages) * page_size; }
    __device__ int page(int b, int slot) const {
        const int at = table[static_cast<int64_t>(b) * table_stride + slot];
        return at >= 0 && at < pages ? at : -1;
    }
};

constexpr int64_t kMaxThreads = int64_t{1} << 31;  // of a launch, which counts them in 32 bits
constexpr int64_t kMaxKeys = int64_t{1} << 30;

inline int check_pages(const char* name, const void* k_pages, const void* v_pages, int64_t pages, int64_t page_size,
                const int32_t* table, int64_t table_stride, int64_t table_pages, const int64_t* positions) {
    if (!k_pages || !v_pages || !table || !positions) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(k_pages, 16) || !aligned(v_pages, 16))
        return fail(NQ_ERR_ALIGNMENT, "%s: pages must be 16-byte aligned", name);
    if (!aligned(table, 4) || !aligned(positions, 8))
        return fail(NQ_ERR_ALIGNMENT, "%s: table must be 4-byte and positions 8-byte aligned", name);
    return NQ_OK;
}

inline int check_sizes(const char* name, int dtype, int64_t pages, int64_t page_size, int64_t table_stride, int64_t table_pages,
                int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim) {
    if (dtype != NQ_F16 && dtype != NQ_BF16) return fail(NQ_ERR_DTYPE, "%s: unsupported dtype %d", name, dtype);
    if (batch < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || pages <= 0 || page_size <= 0 ||
        table_pages <= 0)
        return fail(NQ_ERR_INVALID_ARGUMENT, "%s: bad sizes", name);
    if (table_stride < table_pages) return fail(NQ_ERR_SHAPE, "%s: table rows overlap", name);
    if (heads % kv_heads) return fail(NQ_ERR_SHAPE, "%s: heads must be a multiple of kv_heads", name);
    if (pages > INT32_MAX || page_size > kMaxKeys || table_pages > kMaxKeys || page_size * table_pages > kMaxKeys ||
        batch > INT32_MAX || tokens > INT32_MAX || heads > 65536 || head_dim > 65536)
        return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large", name);
    return NQ_OK;
}

}  // namespace nq
