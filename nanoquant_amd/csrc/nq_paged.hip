// A KV cache in pages: the rotary write of new tokens and the attention that reads it.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nq_common.h"
#include "nq_paged_few.h"
#include "nq_paged_rows.h"
#include "nq_wave.h"

namespace nq {
namespace {

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
// so x0 cos0 - x1 sin0 and x1 cos1 + x0 sin1 take two 16-byte loads and two stores. Bound by memory: 2158 tokens of 64 heads of
// 8 kv heads, 105 MB in 22.6 us, launch and all (4.6 TB/s; a large copy runs at 5.1); one token by the launch, 8.4 us.
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
        const int slot_page = a.pages.slot_of(static_cast<int>(p));
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

// Where the partial results of an (entry, kv head) lie: n blocks from `first` on took part, the first with its slot, the others
// with their slot 0.
struct Parts {
    int place0, first, n;
    __device__ int64_t row(const PagedArgs& a, int i, int row) const {
        return static_cast<int64_t>(i == 0 ? place0 : (first + i) * 2) * a.rows_kept + row;
    }
};
__device__ inline Parts parts_of(const PagedArgs& a, int seg) {
    const int2 d = a.desc[seg];
    return Parts{d.x, d.x >> 1, d.y - (d.x >> 1) + 1};
}

// Adds what the blocks left of one row of an (entry, kv head), for few rows of which many blocks may hold a part: the threads
// in groups of D / 4, a group every Groups-th part. Bound by latency: where the parts lie, then the parts, then their sums;
// 3.3 to 3.9 us for one token of 32 kv heads in eight parts each, 5.0 for 40 rows of 72 (sequence, kv head) pairs.
template <typename T, int D>
__global__ __launch_bounds__(256) void few_join_kernel(const PagedArgs a, int group) {
    constexpr int L4 = D / 4, Groups = 256 / L4, kAhead = 4;
    __shared__ float red[Groups][D];
    __shared__ float2 stat[Groups];
    const int t = threadIdx.x;
    const int seg = static_cast<int>(blockIdx.x) / a.rows_kept;
    const int row = static_cast<int>(blockIdx.x) - seg * a.rows_kept;
    const Parts parts = parts_of(a, seg);
    if (parts.n == 1) return;
    const int entry = seg / a.kv_heads, kvh = seg - entry * a.kv_heads;
    const int b = entry / a.row_groups;
    const int r = (entry - b * a.row_groups) * group + row;
    if (r >= a.tokens * a.groups) return;
    const int grp = t / L4, at = 4 * (t % L4);
    float M = -INFINITY, L = 0.0f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = grp; i0 < parts.n; i0 += kAhead * Groups) {
        float2 ml[kAhead];
        f32x4 x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {  // those past the last read it again
            const int64_t p = parts.row(a, min(i0 + i * Groups, parts.n - 1), row);
            ml[i] = a.part_ml[p];
            x[i] = *reinterpret_cast<const f32x4*>(a.part_o + p * D + at);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) top = fmaxf(top, ml[i].x);
        const float mu = top == -INFINITY ? 0.0f : top;
        const float keep = __builtin_amdgcn_exp2f(M - mu);
        M = top;
        L *= keep;
        o *= keep;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const float f = __builtin_amdgcn_exp2f(ml[i].x - mu);
            const bool in = i0 + i * Groups < parts.n;
            L = in ? fmaf(f, ml[i].y, L) : L;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = in ? fmaf(f, x[i][e], o[e]) : o[e];
        }
    }
    *reinterpret_cast<f32x4*>(&red[grp][at]) = o;
    if (at == 0) stat[grp] = float2{M, L};
    __syncthreads();
    if (t < D / 2) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < Groups; ++i) top = fmaxf(top, stat[i].x);
        const float mu = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
        for (int i = 0; i < Groups; ++i) {
            const float f = __builtin_amdgcn_exp2f(stat[i].x - mu);
            sum = fmaf(f, stat[i].y, sum);
            x = fmaf(f, red[i][2 * t], x);
            y = fmaf(f, red[i][2 * t + 1], y);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        *reinterpret_cast<uint32_t*>(a.out + out_row(a, b, kvh, r) * D + 2 * t) = pack2<T>(x * inv, y * inv);
    }
}

// The same for many rows, of which a few blocks hold a part: D / 8 threads a row, eight dimensions each, the parts one after
// the other. 7 us for 5600 rows of 8 kv heads.
template <typename T, int D>
__global__ __launch_bounds__(256) void rows_join_kernel(const PagedArgs a, int group) {
    constexpr int C = D / 8, Rows = 256 / C;
    const int t = threadIdx.x;
    const int blocks = (a.rows_kept + Rows - 1) / Rows;
    const int seg = static_cast<int>(blockIdx.x) / blocks;
    const Parts parts = parts_of(a, seg);
    if (parts.n == 1) return;
    const int row = (static_cast<int>(blockIdx.x) - seg * blocks) * Rows + t / C;
    const int entry = seg / a.kv_heads, kvh = seg - entry * a.kv_heads;
    const int b = entry / a.row_groups;
    const int r = (entry - b * a.row_groups) * group + row;
    if (row >= a.rows_kept || r >= a.tokens * a.groups) return;
    const int at = 8 * (t % C);
    float M = -INFINITY, L = 0.0f;
    f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
    for (int i0 = 0; i0 < parts.n; i0 += 4) {
        float2 ml[4];
        f32x4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // those past the last read it again, with a weight of zero
            const int64_t p = parts.row(a, min(i0 + i, parts.n - 1), row);
            ml[i] = a.part_ml[p];
            x[i] = *reinterpret_cast<const f32x4*>(a.part_o + p * D + at);
            y[i] = *reinterpret_cast<const f32x4*>(a.part_o + p * D + at + 4);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i].x);
        const float mu = top == -INFINITY ? 0.0f : top;
        const float keep = __builtin_amdgcn_exp2f(M - mu);
        M = top;
        L *= keep;
        lo *= keep;
        hi *= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i0 + i >= parts.n) continue;
            const float f = __builtin_amdgcn_exp2f(ml[i].x - mu);
            L += f * ml[i].y;
            lo += f * x[i];
            hi += f * y[i];
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    *reinterpret_cast<u32x4*>(a.out + out_row(a, b, kvh, r) * D + at) =
        u32x4{pack2<T>(lo[0] * inv, lo[1] * inv), pack2<T>(lo[2] * inv, lo[3] * inv), pack2<T>(hi[0] * inv, hi[1] * inv),
              pack2<T>(hi[2] * inv, hi[3] * inv)};
}

// Which kernel a call runs, how many sequences a launch takes, and what it needs of the workspace.
struct Plan {
    bool few;            // few_kernel, else rows_kernel
    bool shared;
    int tiles;           // row tiles: of 16 rows a wave (few), of 32
    int64_t group;       // rows of a row group
    int64_t row_groups, rows_kept, batch, blocks;
    size_t part_o, part_ml, desc, spans, bytes;
};

// `max_keys` that a row group may see, `mean_keys` one among the others
Plan make_plan(int64_t batch, int64_t tokens, int64_t groups, int64_t kv_heads, int64_t head_dim, int64_t max_keys, int64_t mean_keys) {
    Plan p{};
    const int64_t rows = tokens * groups;
    // Times in tiles of 64 keys, as rows_kernel takes them with 128 rows a block (1 us), from measurements of 11 and 29 shapes;
    // `fill` is how often its row groups fill the card, `longest` and `mean` are what a row group may see.
    const double fill = static_cast<double>(ceil_div(rows, 128) * batch * kv_heads) / kCUs;
    const double longest = max_keys / 64.0, mean = mean_keys / 64.0;
    // few_kernel reads at the card's rate whatever the grid, 1.9 for a card full, and joins for 7 more than rows_kernel takes.
    // 64 rows a sequence and 8 kv heads: 9 sequences in 2900 keys 45 us against 56, 32 sequences 91 against 78; a sequence of
    // 64 tokens and 32 kv heads in 8000 keys 48 us against 131, in 64 keys 18 against 11. Past 3200 keys its shares are worth
    // more than that whatever the grid: one long sequence among short ones would have a row group's block run on alone.
    p.few = rows <= 16 || (rows <= 64 && (longest > 50.0 || longest * (1.0 - 1.9 * fill) > 7.0));
    if (p.few) {
        p.tiles = static_cast<int>(ceil_div(rows, 16));
        p.group = 16 * p.tiles;
        // One row tile also without shares, a block an (entry, kv head): no plan of shares and no join, 4 us, but a block is as
        // long as its sequence. 32 kv heads of one sequence of 480 keys 8.8 us against 10.6, of 1000 13.2 against 11.7, of
        // eight sequences of 2000 43.8 against 46.5, of 1 to 4000 57 against 51; 8 kv heads of 64 sequences of 1 to 4000 keys
        // 108.7 against 109.9. Not past 4096 keys, where one long sequence would run on alone.
        p.shared = rows > 16 || max_keys > std::max<int64_t>(640, std::min<int64_t>(4096, 8 * batch * kv_heads));
        p.blocks = p.tiles < 3 || head_dim == 64 ? 2 * kCUs : kCUs;  // FewShape's
    } else {
        // Two row tiles a wave where the rows fill them, and a grid of them the card nearly twice: 64 heads of 8 kv heads, a
        // prompt of 2000 tokens 93 us against 106, but 1500 tokens in 8000 keys 461 against 406, and 64 sequences of 64 rows in
        // 1000 keys 93 against 60. With the work shared the card is always full: 700 tokens in 8000 keys 222 us against 233,
        // but 800 tokens of 32 kv heads, which leave an eighth of the row tiles empty, 174 against 158.
        const int64_t large = ceil_div(rows, 256);
        const bool full = 2 * large * 15 <= ceil_div(rows, 128) * 16;
        p.tiles = full && large * batch * kv_heads >= 7 * kCUs / 4 ? 2 : 1;
        // Shares make up for a grid that leaves CUs without work, or runs a round more for a few blocks, and cost 25: 700 tokens
        // of 64 heads of 8 kv heads in 2000 keys 81 us against 70, in 4000 128 against 132, in 8000 222 against 262; 200 tokens
        // of 32 kv heads in 2000 keys 45 against 41, in 4000 53 against 74.
        p.shared = p.tiles == 1 && std::max(longest, std::ceil(fill) * mean) > fill * mean + 25.0;
        if (p.shared && full) p.tiles = 2;
        p.group = 128 * p.tiles;
        p.blocks = kCUs;
    }
    p.row_groups = ceil_div(rows, p.group);
    p.rows_kept = std::min(rows, p.group);
    p.batch = batch;
    if (p.shared) {
        const int64_t entries = p.few ? kFewEntries : kEntries;
        if (p.row_groups > entries) p.shared = false;  // a prompt this long fills the card
        p.batch = std::min({batch, std::max<int64_t>(1, entries / p.row_groups),
                            std::max<int64_t>(1, kMaxThreads / 256 / (p.row_groups * kv_heads * p.rows_kept))});
    }
    if (!p.shared) {
        const int threads = p.few || p.tiles == 2 ? 256 : 512;
        p.batch = std::min(batch, std::max<int64_t>(1, kMaxThreads / threads / (p.row_groups * kv_heads)));
        return p;
    }
    p.part_o = static_cast<size_t>(p.blocks) * 2 * p.rows_kept * head_dim * sizeof(float);
    p.part_ml = static_cast<size_t>(p.blocks) * 2 * p.rows_kept * sizeof(float2);
    p.spans = static_cast<size_t>(p.batch) * p.row_groups * sizeof(int4);
    p.desc = static_cast<size_t>(p.batch) * p.row_groups * kv_heads * sizeof(int2);
    p.part_ml = static_cast<size_t>(ceil_div(p.part_ml, 16) * 16);
    p.bytes = p.part_o + p.part_ml + p.spans + p.desc;
    return p;
}

// The plan of a call. A window makes row groups shorter than the table; the workspace's size does not know it, so its plan has to
// make do with that.
Plan plan_of(int64_t batch, int64_t tokens, int64_t groups, int64_t kv_heads, int64_t head_dim, int64_t max_keys, int64_t window,
             int64_t sinks) {
    const Plan p = make_plan(batch, tokens, groups, kv_heads, head_dim, max_keys, std::max(max_keys - tokens / 2, max_keys / 2));
    if (window == 0) return p;
    const int64_t visible = std::min(max_keys, window + sinks + std::min(tokens, ceil_div(256, groups)) + 64);
    const Plan q = make_plan(batch, tokens, groups, kv_heads, head_dim, visible, visible);
    return q.bytes <= p.bytes ? q : p;
}

template <typename T, int D>
void launch_slice(const PagedArgs& a, const Plan& plan, hipStream_t st) {
    const unsigned segs = static_cast<unsigned>(static_cast<int64_t>(a.batch) * a.row_groups * a.kv_heads);
    const dim3 grid(static_cast<unsigned>(plan.blocks));
    if (plan.few) {
        if (!plan.shared) few_kernel<T, D, 1, false><<<dim3(segs), 64 * kWaves, 0, st>>>(a);
        else if (plan.tiles == 1) few_kernel<T, D, 1, true><<<grid, 64 * kWaves, 0, st>>>(a);
        else if (plan.tiles == 2) few_kernel<T, D, 2, true><<<grid, 64 * kWaves, 0, st>>>(a);
        else if (plan.tiles == 3) few_kernel<T, D, 3, true><<<grid, 64 * kWaves, 0, st>>>(a);
        else few_kernel<T, D, 4, true><<<grid, 64 * kWaves, 0, st>>>(a);
    } else if (plan.shared) {
        const int entries = a.batch * a.row_groups;
        spans_kernel<<<dim3(static_cast<unsigned>(ceil_div(entries, 4))), 256, 0, st>>>(a, static_cast<int>(plan.group), entries);
        if (plan.tiles == 1) rows_kernel<T, D, 1, true><<<grid, 512, 0, st>>>(a);
        else rows_kernel<T, D, 2, true><<<grid, 256, 0, st>>>(a);
    } else {
        if (plan.tiles == 1) rows_kernel<T, D, 1, false><<<dim3(segs), 512, 0, st>>>(a);
        else rows_kernel<T, D, 2, false><<<dim3(segs), 256, 0, st>>>(a);
    }
    const int group = static_cast<int>(plan.group);
    if (!plan.shared) return;
    if (plan.few) few_join_kernel<T, D><<<dim3(segs * static_cast<unsigned>(a.rows_kept)), 256, 0, st>>>(a, group);
    else rows_join_kernel<T, D><<<dim3(segs * static_cast<unsigned>(ceil_div(a.rows_kept, 256 / (D / 8)))), 256, 0, st>>>(a, group);
}

template <typename T, int D>
void launch_paged(PagedArgs a, const Plan& plan, char* ws, hipStream_t st) {
    a.row_groups = static_cast<int>(plan.row_groups);
    a.rows_kept = static_cast<int>(plan.rows_kept);
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + plan.part_o);
    a.spans = reinterpret_cast<int4*>(ws + plan.part_o + plan.part_ml);
    a.desc = reinterpret_cast<int2*>(ws + plan.part_o + plan.part_ml + plan.spans);
    const int64_t batch = a.batch;
    for (int64_t b = 0; b < batch; b += plan.batch) {
        PagedArgs s = a;
        s.batch = static_cast<int>(std::min(plan.batch, batch - b));
        s.q += b * a.tokens * a.q_stride;
        s.positions += b * a.tokens;
        s.pages.table += b * a.pages.table_stride;
        s.out += b * a.tokens * a.heads * D;
        launch_slice<T, D>(s, plan, st);
    }
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
    if (batch * tokens > kMaxThreads / slots) return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large", name);
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
    a.pages = Pages(table, table_stride, table_pages, pages, page_size);
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
    if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 65536 || batch > INT32_MAX ||
        tokens > INT32_MAX || batch * tokens > INT32_MAX / heads || table_pages <= 0 || page_size <= 0 ||
        table_pages > kMaxKeys || page_size > kMaxKeys)
        return 0;
    return plan_of(batch, tokens, heads / kv_heads, kv_heads, head_dim, table_pages * page_size, 0, 0).bytes;
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
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16))
        return fail(NQ_ERR_ALIGNMENT, "%s: q, out and the workspace must be 16-byte aligned", name);
    window = std::min(window, kMaxKeys);
    sinks = std::min(sinks, kMaxKeys);
    const Plan plan = plan_of(batch, tokens, heads / kv_heads, kv_heads, head_dim, table_pages * page_size, window, sinks);
    const size_t need = plan.bytes;
    if (need && (!workspace || workspace_bytes < need))
        return fail(NQ_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", name, workspace ? workspace_bytes : size_t{0}, need);
    PagedArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.q_stride = q_stride;
    a.k_pages = static_cast<const uint16_t*>(k_pages);
    a.v_pages = static_cast<const uint16_t*>(v_pages);
    a.pages = Pages(table, table_stride, table_pages, pages, page_size);
    a.positions = positions;
    a.out = static_cast<uint16_t*>(out);
    a.batch = static_cast<int>(batch);
    a.tokens = static_cast<int>(tokens);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.groups = static_cast<int>(heads / kv_heads);
    a.window = static_cast<int>(window);
    a.sinks = static_cast<int>(sinks);
    a.scale = scaling * 1.44269504088896340736f;  // exp(x) = exp2(x log2(e))
    char* ws = static_cast<char*>(workspace);
    hipStream_t st = as_stream(stream);
    if (dtype == NQ_F16) {
        if (head_dim == 64) launch_paged<F16, 64>(a, plan, ws, st);
        else launch_paged<F16, 128>(a, plan, ws, st);
    } else {
        if (head_dim == 64) launch_paged<BF16, 64>(a, plan, ws, st);
        else launch_paged<BF16, 128>(a, plan, ws, st);
    }
    return check_launch(name);
}

}  // extern "C"
