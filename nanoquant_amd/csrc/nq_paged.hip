// A KV cache in pages: the rotary write of new tokens and the attention that reads it.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nq_common.h"
#include "nq_paged_few.h"
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

// ---------------------------------------------------------------- many rows

constexpr int kKeys = 64;   // keys of a tile

// An entry's tiles, for the blocks that share the work of all: a wave per entry, its tokens over the lanes. 4.7 us; in every
// block of rows_kernel, whose entries have hundreds of tokens, it would cost more.
__global__ __launch_bounds__(256) void spans_kernel(const PagedArgs a, int group, int entries) {
    const int entry = static_cast<int>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (entry >= entries) return;
    const int b = entry / a.row_groups;
    const int first = (entry - b * a.row_groups) * group;
    const int t0 = first / a.groups, t1 = min(a.tokens - 1, (first + group - 1) / a.groups);
    int lo = INT32_MAX, hi = -1;
    for (int t = t0 + (threadIdx.x & 63); t <= t1; t += 64) {
        const int p = real_position(a, static_cast<int64_t>(b) * a.tokens + t);
        if (p >= 0) lo = min(lo, p);
        hi = max(hi, p);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        lo = min(lo, __shfl_xor(lo, off, 64));
        hi = max(hi, __shfl_xor(hi, off, 64));
    }
    if ((threadIdx.x & 63) == 0) {
        const Tiles r = tiles_between<kKeys>(a, lo, hi);
        a.spans[entry] = int4{r.sink_tiles, r.window_tile, r.count, 0};
    }
}

// Attention of many rows per sequence over its pages, tiles of 64 keys that a block's waves share, K and V row-major in rings of
// four tiles by DMA:
//   S^T = K Q^T      v_mfma_f32_32x32x16, A = 32 keys x 16 dimensions, B = 32 rows of queries
//   O^T += V^T P^T   A = 32 dimensions x 16 keys, read transposed, B = P^T: S^T's accumulator layout already, with keys
//                    4 kg .. +3 and 8 + 4 kg .. +3 of each 16 in lane group kg
// A tile that every row sees whole runs in a loop that orders products and exponentials by hand: scores of its first 32 keys;
// scores of the others among the first ones' exponentials; values of the first among the others' exponentials; values of the
// others. Left to the scheduler, half of the exponentials stood in front of the products (349 us against 338 for the chunk
// below, page lookups for 64 tiles at a time included).
// RW 2: 4 waves of 64 rows, which read every operand for two row tiles. One wave a SIMD: what it waits for, nobody fills.
// RW 1: 8 waves, 32 rows each, of which waves w and w + 4 have the same rows and take the tiles in turn, so two waves a SIMD
// fill each other's waits; they read each operand twice as often as RW 2's for the same rows. Their sums are joined through
// LDS. (A half of each tile's keys to either, in step at every barrier: a prompt of 1000 tokens 28.5 us against 25.3.)
// Bound by products and exponentials of a wave in turn: 4001 tokens of 64 heads of 8 kv heads under a window of 2047, RW 2,
// 329 us (822 TFLOP/s, where a large matrix product runs at 1345): of a tile's 5500 cycles 2050 are products, 2000 vector
// instructions, of which about half overlap, 1100 waits for LDS and barriers, 480 scalar instructions. A prompt of 1000 tokens,
// 32 heads, RW 1: 25.3 us, of which the longest row group's 16 tiles take 16.
// kShared: the work of all row groups in equal shares over the grid, as few_kernel's; otherwise a block takes a row group,
// the last ones (the longest of a prompt) first.
template <typename T, int D, int RW, bool kShared>
__global__ __launch_bounds__(RW == 1 ? 512 : 256, RW == 1 ? 2 : 1) void rows_kernel(const PagedArgs a) {
    constexpr int NW = RW == 1 ? 8 : 4;  // waves
    constexpr int C = D / 8;             // 16-byte chunks of a row
    constexpr int RowsPer = 64 / C;      // rows of one DMA instruction
    constexpr int Instr = 16 / RowsPer;  // instructions for 16 rows
    constexpr int Group = 128 * RW;
    constexpr int KT = D / 16, DT = D / 32, KG = KT / 2;
    constexpr int TileElems = kKeys * D, kStep = RW == 1 ? 2 : 1;  // tiles from one of a wave's to its next
    __shared__ __attribute__((aligned(16))) uint16_t kring[4][TileElems], vring[4][TileElems];
    __shared__ int spans[2][4];
    __shared__ int64_t pre[kShared ? kEntries + 1 : 1];
    __shared__ int64_t wave_total[NW];
    __shared__ int s_entry;
    __shared__ int s_tainted[2];  // as few_kernel's
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int rwave = wave & 3, grp = wave >> 2;  // its rows, and of the two halves of RW 1
    const int c = lane & 31, kg = lane >> 5;
    const int entries = a.batch * a.row_groups;

    if (t < 2) s_tainted[t] = 0;
    Shares shares{};
    int entry, slot = 0, turn = 0;
    int64_t u = 0;
    if constexpr (kShared) {
        shares = make_shares<64 * NW, kCUs>(a, entries, kLeastTiles, pre, wave_total, &s_entry, [&](int e) { return a.spans[e].z + kStart; });
        if (shares.entry < 0) return;
        entry = shares.entry;
        u = shares.first;
    } else {
        const int order = static_cast<int>(blockIdx.x) / (a.batch * a.kv_heads);
        const int rest = static_cast<int>(blockIdx.x) - order * a.batch * a.kv_heads;
        entry = rest / a.kv_heads * a.row_groups + a.row_groups - 1 - order;
    }

    uint32_t koff[Instr], voff[Instr];
#pragma unroll
    for (int j = 0; j < Instr; ++j) {
        const int row = j * RowsPer + lane / C, pos = lane % C;
        const int kswz = D == 128 ? row : row >> 1;
        const int vswz = D == 128 ? ((row & 3) << 2) | (row >> 2) : (((row >> 1) & 1) << 2) | (row >> 2);
        koff[j] = static_cast<uint32_t>(row * D * 2 + 16 * (pos ^ (kswz & (C - 1))));
        voff[j] = static_cast<uint32_t>(row * D * 2 + 16 * (pos ^ vswz));
    }
    const uint32_t klds = __builtin_amdgcn_readfirstlane(lds_addr(&kring[0][0])) + static_cast<uint32_t>(rwave) * (16 * D * 2);
    const uint32_t vlds = __builtin_amdgcn_readfirstlane(lds_addr(&vring[0][0])) + static_cast<uint32_t>(rwave) * (16 * D * 2);
    // positive, so that the largest product is the largest score: the queries take a negative factor's sign, and are zero for
    // a factor of zero
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
    // the row of 16 keys that this lane names in a transposed read, and the place of its four dimensions
    const int vr = 4 * kg + ((lane & 15) >> 2);
    const int dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    auto read_k = [&](const uint16_t* half, int kt) {
        const int kswz = D == 128 ? c : c >> 1;
        return *vec(half + c * D + 8 * ((2 * kt + kg) ^ (kswz & (C - 1))));
    };
    auto read_v = [&](const uint16_t* half, int k2, int dt) {
        uint2 part[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = vr + 8 * e;
            const int vswz = D == 128 ? ((row & 3) << 2) | (row >> 2) : (((row >> 1) & 1) << 2) | (row >> 2);
            const int d = 32 * dt + dim;
            part[e] = read_transposed(half + (16 * k2 + row) * D + 8 * ((d >> 3) ^ vswz) + (d & 7));
        }
        return u32x4{part[0].x, part[0].y, part[1].x, part[1].y};
    };

    while (true) {
        const int b = entry / a.row_groups;
        const int row0 = (entry - b * a.row_groups) * Group + rwave * (32 * RW);
        const int rows = a.tokens * a.groups;
        int kvh, first = 0, n, count;
        int64_t seg = 0;
        Tiles tiles;
        if constexpr (kShared) {
            const int64_t seg0 = pre[entry] * a.kv_heads;
            const int units = __builtin_amdgcn_readfirstlane(static_cast<int>(pre[entry + 1] - pre[entry]));
            count = units - kStart;
            kvh = __builtin_amdgcn_readfirstlane(quotient(u - seg0, units));
            seg = seg0 + static_cast<int64_t>(kvh) * units;
            first = max(0, __builtin_amdgcn_readfirstlane(static_cast<int>(u - seg)) - kStart);
            u = min(shares.end, seg + units);
            n = __builtin_amdgcn_readfirstlane(static_cast<int>(u - seg)) - kStart - first;
            if (n <= 0) return;  // the share ended before its first tile
            const int4 sp = a.spans[entry];
            tiles = Tiles{__builtin_amdgcn_readfirstlane(sp.x), __builtin_amdgcn_readfirstlane(sp.y), sp.z};
        } else {
            kvh = static_cast<int>(blockIdx.x) % a.kv_heads;
        }

        // a wave brings a quarter of a tile: 16 keys, which lie in one page. Where they are, for 64 tiles at a time, a lane each:
        // a scalar load and a division for every tile stood in its way
        int my_page = 0, my_rest = 0, my_there = 0;
        uint32_t there = 0u;  // bit 4 (it % 4) + i: the page of keys 16 i .. +15 of tile `it` is there
        auto look_up = [&](int it) {
            const int key = tiles.at(first + min(it + lane, n - 1)) * kKeys;
            my_there = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = (key + 16 * i) / a.pages.page_size;
                const int page = at < a.pages.table_pages ? a.pages.page(b, at) : -1;
                my_there |= page >= 0 ? 1 << i : 0;
                if (i == rwave) {
                    my_page = max(page, 0);
                    my_rest = key + 16 * i - at * a.pages.page_size;
                }
            }
        };
        auto place = [&](int it) {
            if ((it & 63) < kStep) look_up(it & ~63);
            const int at = it & 63, by = 4 * (it & 3);
            there = (there & ~(15u << by)) | static_cast<uint32_t>(__builtin_amdgcn_readlane(my_there, at)) << by;
            const int page = __builtin_amdgcn_readlane(my_page, at), rest = __builtin_amdgcn_readlane(my_rest, at);
            return ((static_cast<int64_t>(page) * a.kv_heads + kvh) * a.pages.page_size + rest) * D;
        };
        auto issue_k = [&](int it, int64_t from) {
            const uint16_t* p = uniform(a.k_pages + from);
#pragma unroll
            for (int j = 0; j < Instr; ++j) dma16_lds(p, koff[j], klds + static_cast<uint32_t>(it & 3) * (TileElems * 2) + 1024u * j);
        };
        auto issue_v = [&](int it, int64_t from) {
            const uint16_t* p = uniform(a.v_pages + from);
#pragma unroll
            for (int j = 0; j < Instr; ++j) dma16_lds(p, voff[j], vlds + static_cast<uint32_t>(it & 3) * (TileElems * 2) + 1024u * j);
        };
        // The waves of a group send for their tiles: all of them three ahead, every other one the next ahead.
        constexpr int kOut = 2 * Instr;  // instructions of a wave, a tile
        auto issue = [&](int it) {
            const int64_t from = place(it);
            issue_k(it, from);
            issue_v(it, from);
        };
        auto begin = [&] {
            for (int it = grp; it < (RW == 1 ? 4 : 3) && it < n; it += kStep) issue(it);
        };
        if constexpr (kShared) begin();  // while the queries come

        u32x4 qf[RW][KT];
        int last[RW], start[RW];
        int lo = INT32_MAX, hi = -1, all_start = 0;
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u, keep_q = a.scale == 0.0f ? 0u : 0xFFFFFFFFu;
#pragma unroll
        for (int rw = 0; rw < RW; ++rw) {
            const int r = min(row0 + 32 * rw + c, rows - 1);
            const int tok = r / a.groups;
            const int64_t q_row = static_cast<int64_t>(b) * a.tokens + tok;
            last[rw] = row0 + 32 * rw + c < rows ? real_position(a, q_row) : -1;
            start[rw] = a.window > 0 ? max(0, last[rw] - a.window + 1) : 0;
            if (last[rw] >= 0) {
                lo = min(lo, last[rw]);
                all_start = max(all_start, start[rw]);
            }
            hi = max(hi, last[rw]);
            const uint16_t* src = a.q + q_row * a.q_stride + static_cast<int64_t>(kvh * a.groups + r - tok * a.groups) * D + 8 * kg;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) qf[rw][kt] = *vec(src + 16 * kt);
        }
#pragma unroll
        for (int rw = 0; rw < RW; ++rw)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
                for (int w = 0; w < 4; ++w) qf[rw][kt][w] = (qf[rw][kt][w] ^ flip) & keep_q;
                // in accumulation registers, from which the products take them as they are: the vector registers hold the rest
                if constexpr (RW == 2) asm volatile("" : "+a"(qf[rw][kt]));
            }
        lo = least_of<32>(lo);
        hi = largest_of<32>(hi);
        all_start = largest_of<32>(all_start);
        const int any_start = a.window > 0 ? max(0, lo == INT32_MAX ? 0 : lo - a.window + 1) : 0;  // the first key of some row
        if constexpr (!kShared) {
            if (lane == 0) {
                spans[0][rwave] = lo;
                spans[1][rwave] = hi;
            }
            __syncthreads();
            int blo = INT32_MAX, bhi = -1;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                blo = min(blo, spans[0][w]);
                bhi = max(bhi, spans[1][w]);
            }
            tiles = tiles_between<kKeys>(a, blo, bhi);
            tiles.sink_tiles = __builtin_amdgcn_readfirstlane(tiles.sink_tiles);
            tiles.window_tile = __builtin_amdgcn_readfirstlane(tiles.window_tile);
            count = n = __builtin_amdgcn_readfirstlane(tiles.count);
            begin();
        }

        f32x16 o[RW][DT];
        float m[RW], l[RW];
#pragma unroll
        for (int rw = 0; rw < RW; ++rw) {
            m[rw] = -INFINITY;
            l[rw] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[rw][dt][i] = 0.0f;
        }
        auto live = [&](int key0) {  // some row of the wave sees some key of 32
            return key0 <= hi && (key0 + 32 > any_start || key0 < a.sinks);
        };
        // scores that a row does not see become -inf; returns whether every row sees every key, and what some row sees: the
        // lane's key 8 (i / 4) + 4 kg + i % 4 in bit 8 (i / 4) + i % 4
        auto mask = [&](f32x16 (&s)[RW], int half0, uint32_t pages, uint32_t& some) {  // pages: 2 bits
            const bool whole = pages == 3u && half0 + 31 <= lo && (half0 >= all_start || half0 + 32 <= a.sinks);
            some = 0xFFFFFFFFu;
            if (!whole) {
                some = 0u;
                const uint32_t pages_there = (pages & 1u ? 0xFFFFu : 0u) | (pages & 2u ? 0xFFFF0000u : 0u);
#pragma unroll
                for (int rw = 0; rw < RW; ++rw) {
                    const uint32_t seen = (seen_bits(half0, last[rw], start[rw], a.sinks) & pages_there) >> (4 * kg);
                    some |= seen;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[rw][i] = or_minus_inf(s[rw][i], seen, 8 * (i >> 2) + (i & 3));
                }
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) some |= __shfl_xor(some, off, 64);
            }
            return whole;
        };
        // The reference point of the exponentials follows the running maximum only once that is 8 above it: exponentials up to
        // 2^8 round the same, and most steps rescale nothing. What the sums so far have to be multiplied by, if so.
        auto follow = [&](const f32x16 (&s)[RW], float (&keep)[RW]) {
            float top[RW];
            bool grows = false;
#pragma unroll
            for (int rw = 0; rw < RW; ++rw) {
                top[rw] = s[rw][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top[rw] = fmaxf(top[rw], s[rw][i]);
                top[rw] = max_xor32(top[rw]) * scale;
                grows |= top[rw] > m[rw] + kSlack;
            }
            const bool any = __any(grows);
            if (any) {
#pragma unroll
                for (int rw = 0; rw < RW; ++rw) {
                    const float mn = fmaxf(m[rw], top[rw]);
                    keep[rw] = __builtin_amdgcn_exp2f(m[rw] - (mn == -INFINITY ? 0.0f : mn));
                    m[rw] = mn;
                    l[rw] *= keep[rw];
                }
            }
            return any;
        };
        auto rescale = [&](const float (&keep)[RW]) {
#pragma unroll
            for (int rw = 0; rw < RW; ++rw)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[rw][dt][i] *= keep[rw];
        };
        // two probabilities of a row tile; rounded, and into its sum as rounded
        auto exp2x2 = [&](const f32x16 (&s)[RW], int rw, int w) {
            const float mu = m[rw] == -INFINITY ? 0.0f : m[rw];
            return float2{__builtin_amdgcn_exp2f(fmaf(s[rw][2 * w], scale, -mu)),
                          __builtin_amdgcn_exp2f(fmaf(s[rw][2 * w + 1], scale, -mu))};
        };
        auto keep2 = [&](float2 e, u32x4 (&p)[RW][2], int rw, int w) {
            p[rw][w >> 2][w & 3] = pack2<T>(e.x, e.y);
            l[rw] = T::dot2(p[rw][w >> 2][w & 3], T::ONE_PAIR, l[rw]);
        };
        // `kProducts` products, and half q of the probabilities spread among them in this order: the exponentials of one step are
        // rounded in the next
        auto among = [&](const f32x16 (&s)[RW], u32x4 (&p)[RW][2], int q, auto products, auto&& product) {
            constexpr int kProducts = decltype(products)::value, kEach = 4 * RW / kProducts;
            float2 e[kEach];
#pragma unroll
            for (int x = 0; x <= kProducts; ++x) {
                if (x < kProducts) product(x);
                float2 next[kEach];
#pragma unroll
                for (int y = 0; y < kEach; ++y) {
                    const int at = 4 * RW * q + kEach * x + y;
                    if (x < kProducts) next[y] = exp2x2(s, at / 8, at % 8);
                    if (x > 0) keep2(e[y], p, (at - kEach) / 8, (at - kEach) % 8);
                    e[y] = next[y];
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // O^T += V^T P^T of 32 keys; values that no row sees are cleared
        auto values = [&](const uint16_t* half, const u32x4 (&p)[RW][2], bool whole, uint32_t some) {
            float zero = 0.0f;
            u32x4 vf[2][DT];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) vf[0][dt] = read_v(half, 0, dt);
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                if (k2 == 0) {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) vf[1][dt] = read_v(half, 1, dt);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (!whole) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t keep = pair_mask(some, 16 * k2 + 8 * (w >> 1) + 2 * (w & 1));
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            vf[k2][dt][w] &= keep;
                            zero = T::dot2(vf[k2][dt][w], 0u, zero);  // NaN where one is not finite
                        }
                    }
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int rw = 0; rw < RW; ++rw) o[rw][dt] = mfma32x32x16<T>(vf[k2][dt], p[rw][k2], o[rw][dt]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (zero != zero) s_tainted[turn] = 1;
        };
        u32x4 kf[2][KG];
        // S^T = K Q^T of 32 keys, operands read ahead of the products that run, the first half of them by `come` if `begun`
        auto scores = [&](const uint16_t* half, f32x16 (&s)[RW], bool begun) {
            if (!begun) {
#pragma unroll
                for (int e = 0; e < KG; ++e) kf[0][e] = read_k(half, e);
            }
#pragma unroll
            for (int rw = 0; rw < RW; ++rw)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[rw][i] = 0.0f;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (q == 0) {
#pragma unroll
                    for (int e = 0; e < KG; ++e) kf[1][e] = read_k(half, KG + e);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < KG; ++e)
#pragma unroll
                    for (int rw = 0; rw < RW; ++rw) s[rw] = mfma32x32x16<T>(kf[q][e], qf[rw][KG * q + e], s[rw]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };

        int key0;
        auto come = [&](int it) {  // waits for a tile, and sends for one where the group's tile before it was
            if constexpr (RW == 2) {
                const int behind = min(n - 1 - it, 2);  // tiles out behind this one
                if (behind == 2) wait_vmcnt<2 * kOut>();
                else if (behind == 1) wait_vmcnt<kOut>();
                else wait_vmcnt<0>();
            } else {
                if (it < 2 && it + 2 < n) wait_vmcnt<kOut>();
                else wait_vmcnt<0>();
            }
            barrier_keep_dma();
#pragma unroll
            for (int e = 0; e < KG; ++e) kf[0][e] = read_k(kring[it & 3], e);
            if ((RW == 2 || it >= 2) && it + 4 - kStep < n) issue(it + 4 - kStep);
            key0 = tiles.at(first + it) * kKeys;
        };
        auto all_whole = [&](int it) {  // every row sees all of the tile
            return it < n && (there >> (4 * (it & 3)) & 15u) == 15u && key0 + kKeys - 1 <= lo && (key0 >= all_start || key0 + kKeys <= a.sinks);
        };
        // the groups take the same number of steps, the last of which may be none of the second's
        const int end = RW == 1 ? ((n + 1) & ~1) + grp : n;
        int it = grp;
        come(it);
        while (it < end) {
            {
                // tiles that every row sees whole, in a loop of their own (with the others in one, its registers did not
                // suffice): the exponentials of a half among the products of the other
                while (all_whole(it)) {
                    const uint16_t* kt0 = kring[it & 3];
                    const uint16_t* vt0 = vring[it & 3];
                    f32x16 s[2][RW];
                    u32x4 p[2][RW][2], vf[2][DT];
                    float keep[RW];
                    scores(kt0, s[0], true);
#pragma unroll
                    for (int e = 0; e < KG; ++e) kf[0][e] = read_k(kt0 + 32 * D, e);
                    if (follow(s[0], keep)) rescale(keep);
#pragma unroll
                    for (int rw = 0; rw < RW; ++rw)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[1][rw][i] = 0.0f;
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
#pragma unroll
                        for (int e = 0; e < KG; ++e) {
                            if (q == 0) kf[1][e] = read_k(kt0 + 32 * D, KG + e);
                            else if (e < DT) vf[0][e] = read_v(vt0, 0, e);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                        among(s[0], p[0], q, std::integral_constant<int, KG * RW>{}, [&](int x) {
                            const int e = x / RW, rw = x % RW;
                            s[1][rw] = mfma32x32x16<T>(kf[q][e], qf[rw][KG * q + e], s[1][rw]);
                        });
                    }
                    const bool grew = follow(s[1], keep);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) vf[1 - q][dt] = q == 0 ? read_v(vt0, 1, dt) : read_v(vt0 + 32 * D, 0, dt);
                        __builtin_amdgcn_sched_barrier(0);
                        among(s[1], p[1], q, std::integral_constant<int, DT * RW>{}, [&](int x) {
                            const int dt = x / RW, rw = x % RW;
                            o[rw][dt] = mfma32x32x16<T>(vf[q][dt], p[0][rw][q], o[rw][dt]);
                        });
                    }
                    // or they are made behind the branch, where they are used
#pragma unroll
                    for (int rw = 0; rw < RW; ++rw) asm volatile("" : "+v"(p[1][rw][0]), "+v"(p[1][rw][1]));
                    if (grew) rescale(keep);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        if (q == 0) {
#pragma unroll
                            for (int dt = 0; dt < DT; ++dt) vf[1][dt] = read_v(vt0 + 32 * D, 1, dt);
                        }
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int rw = 0; rw < RW; ++rw) o[rw][dt] = mfma32x32x16<T>(vf[q][dt], p[1][rw][q], o[rw][dt]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    it += kStep;
                    if (it >= end) break;
                    come(it);
                }
                if (it >= end) break;
            }
            const uint16_t* kt0 = kring[it & 3];
            const uint16_t* vt0 = vring[it & 3];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (it >= n || !live(key0 + 32 * h)) continue;
                f32x16 s[RW];
                scores(kt0 + 32 * h * D, s, false);
                uint32_t some;
                const bool whole = mask(s, key0 + 32 * h, there >> (4 * (it & 3) + 2 * h) & 3u, some);
                float keep[RW];
                if (follow(s, keep)) rescale(keep);
                u32x4 p[RW][2];
#pragma unroll
                for (int rw = 0; rw < RW; ++rw)
#pragma unroll
                    for (int w = 0; w < 8; ++w) keep2(exp2x2(s, rw, w), p, rw, w);
                values(vt0 + 32 * h * D, p, whole, some);
            }
            it += kStep;
            if (it < end) come(it);
        }

        const bool done = first == 0 && n == count;
        __syncthreads();
        const bool tainted = s_tainted[turn] != 0;
        if (tainted) {
            const int group0 = (entry - b * a.row_groups) * Group;
            slow_rows<T, D>(a, Rows<PagedArgs>{b, group0, min(Group, rows - group0)}, kvh, tiles, kKeys, first, n, done,
                            (static_cast<int64_t>(blockIdx.x) * 2 + slot) * a.rows_kept);
        }
        // the halves' sums: the second group's through the key ring, its statistics through the value ring's first 2 KB
        if (RW == 1 && !tainted) {
            float* red = reinterpret_cast<float*>(&kring[0][0]);
            float* stat = reinterpret_cast<float*>(&vring[0][0]);
            static_assert(RW == 2 || sizeof(kring) >= DT * 16 * 256 * sizeof(float), "the key ring holds a group's sums");
            if (grp == 1) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) red[(16 * dt + i) * 256 + (t & 255)] = o[0][dt][i];
                stat[t & 255] = m[0];
                stat[256 + (t & 255)] = l[0];
            }
            __syncthreads();
            if (grp == 0) {
                const float m1 = stat[t], mn = fmaxf(m[0], m1);
                const float mu = mn == -INFINITY ? 0.0f : mn;
                const float f0 = __builtin_amdgcn_exp2f(m[0] - mu), f1 = __builtin_amdgcn_exp2f(m1 - mu);
                m[0] = mn;
                l[0] = l[0] * f0 + stat[256 + t] * f1;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[0][dt][i] = o[0][dt][i] * f0 + red[(16 * dt + i) * 256 + t] * f1;
            }
        }
        // a wave's rows through LDS, a row tile at a time, then whole rows to memory
        uint16_t* ob = (RW == 1 ? &vring[0][0] + 1024 : &kring[0][0]) + rwave * (32 * D);
        if (grp == 0 && !tainted) {
#pragma unroll
            for (int rw = 0; rw < RW; ++rw) {
                float L = l[rw] + __shfl_xor(l[rw], 32, 64);
                float M = m[rw];
                if (last[rw] < 0) {  // padding took part where the tile was whole
                    L = 0.0f;
                    M = -INFINITY;
                }
                const float inv = 1.0f / L;
                if (kShared && !done) {
                    const int at = rwave * (32 * RW) + 32 * rw + c;
                    if (row0 + 32 * rw + c < rows) {
                        const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + slot) * a.rows_kept + at;
                        if (kg == 0) a.part_ml[part] = float2{M, L};
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int g4 = 0; g4 < 4; ++g4) {
                                f32x4 x;
#pragma unroll
                                for (int e = 0; e < 4; ++e) x[e] = L == 0.0f ? 0.0f : o[rw][dt][4 * g4 + e];
                                *reinterpret_cast<f32x4*>(a.part_o + part * D + 32 * dt + 8 * g4 + 4 * kg) = x;
                            }
                    }
                    continue;
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) {
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = L == 0.0f ? 0.0f : o[rw][dt][4 * g4 + e] * inv;
                        *reinterpret_cast<uint2*>(ob + c * D + 8 * ((4 * dt + g4) ^ (c & (C - 1))) + 4 * kg) =
                            uint2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
                    }
#pragma unroll
                for (int j = 0; j < 32 / RowsPer; ++j) {
                    const int r = RowsPer * j + lane / C, ch = lane % C;
                    const u32x4 v = *vec(ob + r * D + 8 * (ch ^ (r & (C - 1))));
                    const int at_row = row0 + 32 * rw + r;
                    if (at_row < rows) *reinterpret_cast<u32x4*>(a.out + out_row(a, b, kvh, at_row) * D + 8 * ch) = v;
                }
            }
        }
        if constexpr (!kShared) return;
        if (first == 0 && t == 0)
            a.desc[entry * a.kv_heads + kvh] =
                int2{static_cast<int>(blockIdx.x) * 2 + slot, static_cast<int>((seg + count + kStart - 1) / shares.share)};
        if (u >= shares.end) return;
        slot = 1;
        if (kvh + 1 == a.kv_heads) ++entry;
        if (t == 0) s_tainted[turn ^ 1] = 0;
        turn ^= 1;
        __syncthreads();
    }
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
    a.pages = Pages{table, table_stride, static_cast<int>(table_pages), static_cast<int>(pages), static_cast<int>(page_size)};
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
