// Pages of a KV cache copied within its pools.
#include <algorithm>

#include "nq_common.h"
#include "nq_paged.h"

namespace nq {
namespace {

constexpr int kPools = 256;  // of a launch: their addresses go with its arguments, 2 KB of the 4 that there are
constexpr int kLoads = 4;    // of a thread
constexpr int kChunk = 256 * kLoads;

struct CopyArgs {
    const int32_t* source;
    const int32_t* target;
    int64_t units;  // of a page
    int chunks;     // of kChunk units a page
    int pages;
    void* pools[kPools];
};

// A block copies kChunk units of one page in one pool, each thread's loads before its stores. One launch copies the pages of up
// to 128 layers. Bound by the read and the write: 61 pages of 64 pools, 512 MB both ways, 102 us (5.0 TB/s; a copy of 2 GiB
// runs at 4.9 to 5.1), 5 pages of 64 pools, 63 MB, 12.8 us (4.9 TB/s); 17 MB 4.9 us, most of it a launch's beginning and end.
template <typename Unit>
__global__ __launch_bounds__(256) void copy_pages_kernel(const CopyArgs a) {
    const int move = static_cast<int>(blockIdx.x) / a.chunks, chunk = static_cast<int>(blockIdx.x) - move * a.chunks;
    const int from = a.source[move], to = a.target[move];
    if (from < 0 || from >= a.pages || to < 0 || to >= a.pages || from == to) return;
    Unit* pool = static_cast<Unit*>(a.pools[blockIdx.y]);
    const Unit* src = pool + from * a.units;
    Unit* dst = pool + to * a.units;
    const int64_t at = static_cast<int64_t>(chunk) * kChunk + threadIdx.x;
    Unit x[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
        if (at + 256 * i < a.units) x[i] = src[at + 256 * i];
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
        if (at + 256 * i < a.units) dst[at + 256 * i] = x[i];
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" int nq_copy_pages(void* const* pools, int64_t count, int64_t pages, int64_t page_bytes, const int32_t* source,
                             const int32_t* target, int64_t moves, nq_stream_t stream) {
    const char* name = "nq_copy_pages";
    if (count < 0 || pages <= 0 || page_bytes <= 0 || moves < 0) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: bad sizes", name);
    if (count == 0 || moves == 0) return NQ_OK;
    if (!pools || !source || !target) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(source, 4) || !aligned(target, 4)) return fail(NQ_ERR_ALIGNMENT, "%s: page numbers must be 4-byte aligned", name);
    bool wide = page_bytes % 16 == 0;
    for (int64_t i = 0; i < count; ++i) {
        if (!pools[i]) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pool", name);
        wide = wide && aligned(pools[i], 16);
    }
    CopyArgs a{};
    a.units = wide ? page_bytes / 16 : page_bytes;
    const int64_t chunks = ceil_div(a.units, kChunk), blocks = kMaxThreads / 256;
    if (pages > INT32_MAX || chunks > blocks) return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large", name);
    a.chunks = static_cast<int>(chunks);
    a.pages = static_cast<int>(pages);
    const int64_t per_move = std::min(moves, blocks / chunks);
    const int64_t per_pool = std::min<int64_t>({count, kPools, blocks / (per_move * chunks)});
    hipStream_t st = as_stream(stream);
    for (int64_t p = 0; p < count; p += per_pool)
        for (int64_t m = 0; m < moves; m += per_move) {
            const int64_t np = std::min(per_pool, count - p), nm = std::min(per_move, moves - m);
            std::copy(pools + p, pools + p + np, a.pools);
            a.source = source + m;
            a.target = target + m;
            const dim3 grid(static_cast<unsigned>(nm * chunks), static_cast<unsigned>(np));
            if (wide) copy_pages_kernel<u32x4><<<grid, 256, 0, st>>>(a);
            else copy_pages_kernel<uint8_t><<<grid, 256, 0, st>>>(a);
        }
    return check_launch(name);
}
