// A KV cache in pages: the rotary write of new tokens and the attention that reads it.
#include <algorithm>

#include "nq_common.h"

namespace nq {
namespace {

__device__ inline const u32x4* vec(const uint16_t* p) { return reinterpret_cast<const u32x4*>(p); }

// The page of position p of a sequence, -1 where there is none.
struct Pages {
    const int32_t* table;
    int64_t table_stride;
    int table_pages, pages, page_size;
    __device__ int64_t capacity() const { return static_cast<int64_t>(table_pages) * page_size; }
    __device__ int page(int b, int slot) const {
        const int at = table[static_cast<int64_t>(b) * table_stride + slot];
        return at >= 0 && at < pages ? at : -1;
    }
};

struct WriteArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    int64_t q_stride, k_stride, v_stride;  // elements between tokens
    const void* cos;
    const void* sin;  // [batch * tokens][head_dim]
    const int64_t* positions;
    Pages pages;
    uint16_t* k_pages;
    uint16_t* v_pages;
    uint16_t* q_out;
    int64_t rows;  // batch * tokens
    int tokens, heads, kv_heads, head_dim;
};

// Eight entries of a table row in fp32.
template <typename T, typename R>
__device__ inline void table8(const void* base, int64_t at, float* f) {
    if constexpr (sizeof(R) == 4) {
        const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + at);
        const f32x4 a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = a[i];
            f[4 + i] = b[i];
        }
    } else {
        const u32x4 a = *vec(static_cast<const uint16_t*>(base) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = T::to_float(static_cast<uint16_t>(a[i >> 1] >> (16 * (i & 1))));
    }
}

// One thread per (token, head of q, k or v, eight dimensions d of the first half): it holds d and d + D / 2, the rotary pair,
// so x0 cos0 - x1 sin0 and x1 cos1 + x0 sin1 take two 16-byte loads and two stores.
template <typename T, typename R>
__global__ __launch_bounds__(256) void paged_write_kernel(const WriteArgs a) {
    const int half = a.head_dim / 2;
    const int parts = half / 8;
    const int slots = (a.heads + 2 * a.kv_heads) * parts;  // threads a token
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = id / slots;
    if (row >= a.rows) return;
    const int slot = static_cast<int>(id - row * slots);
    const int head = slot / parts;
    const int d = 8 * (slot - head * parts);
    const int64_t p = a.positions[row];
    const bool real = p >= 0 && p < a.pages.capacity();
    if (head < a.heads && !real) {
        uint16_t* dst = a.q_out + (row * a.heads + head) * a.head_dim + d;
        *reinterpret_cast<u32x4*>(dst) = u32x4{0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4*>(dst + half) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    if (!real) return;
    const uint16_t* src;
    uint16_t* dst;
    if (head < a.heads) {
        src = a.q + row * a.q_stride + static_cast<int64_t>(head) * a.head_dim + d;
        dst = a.q_out + (row * a.heads + head) * a.head_dim + d;
    } else {
        const int slot_page = static_cast<int>(p) / a.pages.page_size;
        const int page = a.pages.page(static_cast<int>(row / a.tokens), slot_page);
        if (page < 0) return;
        const bool key = head < a.heads + a.kv_heads;
        const int h = head - a.heads - (key ? 0 : a.kv_heads);
        src = (key ? a.k + row * a.k_stride : a.v + row * a.v_stride) + static_cast<int64_t>(h) * a.head_dim + d;
        const int64_t at = (static_cast<int64_t>(page) * a.kv_heads + h) * a.pages.page_size + (static_cast<int>(p) - slot_page * a.pages.page_size);
        dst = (key ? a.k_pages : a.v_pages) + at * a.head_dim + d;
    }
    u32x4 lo = *vec(src), hi = *vec(src + half);
    if (head < a.heads + a.kv_heads) {
        float c0[8], s0[8], c1[8], s1[8];
        const int64_t at = row * a.head_dim + d;
        table8<T, R>(a.cos, at, c0);
        table8<T, R>(a.sin, at, s0);
        table8<T, R>(a.cos, at + half, c1);
        table8<T, R>(a.sin, at + half, s1);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t r0 = 0, r1 = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 2 * w + h;
                const float x0 = T::to_float(static_cast<uint16_t>(lo[w] >> (16 * h)));
                const float x1 = T::to_float(static_cast<uint16_t>(hi[w] >> (16 * h)));
                r0 |= static_cast<uint32_t>(T::from_float(x0 * c0[i] - x1 * s0[i])) << (16 * h);
                r1 |= static_cast<uint32_t>(T::from_float(x1 * c1[i] + x0 * s1[i])) << (16 * h);
            }
            lo[w] = r0;
            hi[w] = r1;
        }
    }
    *reinterpret_cast<u32x4*>(dst) = lo;
    *reinterpret_cast<u32x4*>(dst + half) = hi;
}

struct PagedArgs {
    const uint16_t* q;
    int64_t q_stride;
    const uint16_t* k_pages;
    const uint16_t* v_pages;
    Pages pages;
    const int64_t* positions;
    uint16_t* out;
    int batch, tokens, heads, kv_heads;
    int window, sinks;  // window 0: none
    float scaling;
};

// One wave per (sequence, token, head), one key at a time: lane l holds dimensions l and, of 128, l + 64.
template <typename T, int D>
__global__ __launch_bounds__(64) void paged_simple_kernel(const PagedArgs a) {
    constexpr int N = D / 64;
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x / a.heads;  // b * tokens + t
    const int h = static_cast<int>(blockIdx.x - row * a.heads);
    const int b = static_cast<int>(row / a.tokens);
    const int kvh = h / (a.heads / a.kv_heads);
    const int64_t p64 = a.positions[row];
    const bool real = p64 >= 0 && p64 < a.pages.capacity();
    const int p = real ? static_cast<int>(p64) : -1;
    const int start = a.window > 0 ? max(0, p - a.window + 1) : 0;
    float q[N], o[N], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < N; ++i) {
        q[i] = T::to_float(a.q[row * a.q_stride + h * D + lane + 64 * i]) * a.scaling;
        o[i] = 0.0f;
    }
    for (int j = 0; j <= p; ++j) {
        if (j < start && j >= a.sinks) j = start;
        const int page = a.pages.page(b, j / a.pages.page_size);
        if (page < 0) continue;
        const int64_t at =
            ((static_cast<int64_t>(page) * a.kv_heads + kvh) * a.pages.page_size + j % a.pages.page_size) * D + lane;
        float s = 0.0f;
        for (int i = 0; i < N; ++i) s += q[i] * T::to_float(a.k_pages[at + 64 * i]);
        s = wave_sum(s);
        const float mn = fmaxf(m, s);
        const float keep = mn == -INFINITY ? 1.0f : expf(m - mn), e = mn == -INFINITY ? 0.0f : expf(s - mn);
        m = mn;
        l = l * keep + e;
        for (int i = 0; i < N; ++i) o[i] = o[i] * keep + e * T::to_float(a.v_pages[at + 64 * i]);
    }
    for (int i = 0; i < N; ++i) a.out[(row * a.heads + h) * D + lane + 64 * i] = T::from_float(l == 0.0f ? 0.0f : o[i] / l);
}

constexpr int64_t kMaxKeys = int64_t{1} << 30;

int check_pages(const char* name, const void* k_pages, const void* v_pages, int64_t pages, int64_t page_size,
                const int32_t* table, int64_t table_stride, int64_t table_pages, const int64_t* positions) {
    if (!k_pages || !v_pages || !table || !positions) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(k_pages, 16) || !aligned(v_pages, 16))
        return fail(NQ_ERR_ALIGNMENT, "%s: pages must be 16-byte aligned", name);
    if (!aligned(table, 4) || !aligned(positions, 8))
        return fail(NQ_ERR_ALIGNMENT, "%s: table must be 4-byte and positions 8-byte aligned", name);
    return NQ_OK;
}

int check_sizes(const char* name, int dtype, int64_t pages, int64_t page_size, int64_t table_stride, int64_t table_pages,
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

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" {

int nq_paged_rope_write(int dtype, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                        int64_t v_stride, const void* rope_cos, const void* rope_sin, int rope_float32,
                        const int64_t* positions, const int32_t* table, int64_t table_stride, int64_t table_pages,
                        void* k_pages, void* v_pages, int64_t pages, int64_t page_size, void* q_out, int64_t batch,
                        int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, nq_stream_t stream) {
    const char* name = "nq_paged_rope_write";
    if (int st = check_sizes(name, dtype, pages, page_size, table_stride, table_pages, batch, tokens, heads, kv_heads, head_dim))
        return st;
    if (head_dim % 16) return fail(NQ_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 16", name);
    if (q_stride < heads * head_dim || k_stride < kv_heads * head_dim || v_stride < kv_heads * head_dim || q_stride % 8 ||
        k_stride % 8 || v_stride % 8)
        return fail(NQ_ERR_SHAPE, "%s: token strides must hold the heads and be multiples of 8", name);
    if (batch == 0 || tokens == 0) return NQ_OK;
    const int64_t slots = (heads + 2 * kv_heads) * (head_dim / 16);
    if (batch * tokens > (int64_t{INT32_MAX} * 256) / slots) return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large", name);
    if (int st = check_pages(name, k_pages, v_pages, pages, page_size, table, table_stride, table_pages, positions)) return st;
    for (const void* p : {q, k, v, rope_cos, rope_sin, static_cast<const void*>(q_out)}) {
        if (!p) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
        if (!aligned(p, 16)) return fail(NQ_ERR_ALIGNMENT, "%s: tensors must be 16-byte aligned", name);
    }
    WriteArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.cos = rope_cos;
    a.sin = rope_sin;
    a.positions = positions;
    a.pages = Pages{table, table_stride, static_cast<int>(table_pages), static_cast<int>(pages), static_cast<int>(page_size)};
    a.k_pages = static_cast<uint16_t*>(k_pages);
    a.v_pages = static_cast<uint16_t*>(v_pages);
    a.q_out = static_cast<uint16_t*>(q_out);
    a.rows = batch * tokens;
    a.tokens = static_cast<int>(tokens);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.head_dim = static_cast<int>(head_dim);
    const dim3 grid(static_cast<unsigned>(ceil_div(a.rows * slots, 256)));
    hipStream_t st = as_stream(stream);
    if (dtype == NQ_F16) {
        if (rope_float32) paged_write_kernel<F16, float><<<grid, 256, 0, st>>>(a);
        else paged_write_kernel<F16, uint16_t><<<grid, 256, 0, st>>>(a);
    } else {
        if (rope_float32) paged_write_kernel<BF16, float><<<grid, 256, 0, st>>>(a);
        else paged_write_kernel<BF16, uint16_t><<<grid, 256, 0, st>>>(a);
    }
    return check_launch(name);
}

size_t nq_paged_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                          int64_t table_pages, int64_t page_size) {
    return 0;
}

int nq_paged_attention(int dtype, const void* q, int64_t q_stride, const void* k_pages, const void* v_pages, int64_t pages,
                       int64_t page_size, const int32_t* table, int64_t table_stride, int64_t table_pages,
                       const int64_t* positions, void* out, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                       int64_t head_dim, int64_t window, int64_t sinks, float scaling, void* workspace,
                       size_t workspace_bytes, nq_stream_t stream) {
    const char* name = "nq_paged_attention";
    if (int st = check_sizes(name, dtype, pages, page_size, table_stride, table_pages, batch, tokens, heads, kv_heads, head_dim))
        return st;
    if (head_dim != 64 && head_dim != 128) return fail(NQ_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", name);
    if (page_size % 16) return fail(NQ_ERR_UNSUPPORTED, "%s: page_size must be a multiple of 16", name);
    if (window < 0 || sinks < 0) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: negative window or sinks", name);
    if (q_stride < heads * head_dim || q_stride % 8)
        return fail(NQ_ERR_SHAPE, "%s: the token stride must hold the heads and be a multiple of 8", name);
    if (batch == 0 || tokens == 0) return NQ_OK;
    if (batch * tokens > INT32_MAX / heads) return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large", name);
    if (int st = check_pages(name, k_pages, v_pages, pages, page_size, table, table_stride, table_pages, positions)) return st;
    if (!q || !out) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(q, 16) || !aligned(out, 16)) return fail(NQ_ERR_ALIGNMENT, "%s: tensors must be 16-byte aligned", name);
    PagedArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.q_stride = q_stride;
    a.k_pages = static_cast<const uint16_t*>(k_pages);
    a.v_pages = static_cast<const uint16_t*>(v_pages);
    a.pages = Pages{table, table_stride, static_cast<int>(table_pages), static_cast<int>(pages), static_cast<int>(page_size)};
    a.positions = positions;
    a.out = static_cast<uint16_t*>(out);
    a.batch = static_cast<int>(batch);
    a.tokens = static_cast<int>(tokens);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.window = static_cast<int>(std::min(window, kMaxKeys));
    a.sinks = static_cast<int>(std::min(sinks, kMaxKeys));
    a.scaling = scaling;
    const dim3 grid(static_cast<unsigned>(batch * tokens * heads));
    hipStream_t st = as_stream(stream);
    if (dtype == NQ_F16) {
        if (head_dim == 64) paged_simple_kernel<F16, 64><<<grid, 64, 0, st>>>(a);
        else paged_simple_kernel<F16, 128><<<grid, 64, 0, st>>>(a);
    } else {
        if (head_dim == 64) paged_simple_kernel<BF16, 64><<<grid, 64, 0, st>>>(a);
        else paged_simple_kernel<BF16, 128><<<grid, 64, 0, st>>>(a);
    }
    return check_launch(name);
}

}  // extern "C"
