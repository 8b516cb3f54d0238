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

constexpr int kTile = 32;          // keys a wave takes at a time
constexpr int kWaves = 4;          // of a block
constexpr int kBlocks = 256;       // one a CU: its rings take most of the LDS
constexpr int kEntries = 2048;     // (sequence, row group) pairs of a launch, whose key counts every block adds up
constexpr int kLeastShare = 4;     // tiles a block takes at least: one a wave
constexpr float kSlack = 8.0f;
constexpr int64_t kMaxGrid = 1 << 23;  // blocks of 256 threads: their count stays in 32 bits

struct PagedArgs {
    const uint16_t* q;
    int64_t q_stride;
    const uint16_t* k_pages;
    const uint16_t* v_pages;
    Pages pages;
    const int64_t* positions;
    uint16_t* out;
    int batch, tokens, heads, kv_heads, groups;
    int window, sinks;  // window 0: none
    float scale;        // times log2(e)
    int row_groups, rows_kept;  // row groups a (sequence, kv head), rows of one that there are
    int2* desc;         // [batch * row_groups * kv_heads]: {first block * 2 + its slot, last block}
    float* part_o;      // [kBlocks][2][rows_kept][D]
    float2* part_ml;    // the same rows' {maximum, sum}
};

// A position that the table holds, -1 for any other.
__device__ inline int real_position(const PagedArgs& a, int64_t row) {
    const int64_t p = a.positions[row];
    return p >= 0 && p < a.pages.capacity() ? static_cast<int>(p) : -1;
}

// The key tiles that the rows of an entry see: `sink_tiles` from the front, then those from window_tile on.
struct Tiles {
    int sink_tiles, window_tile, count;
    __device__ int at(int i) const { return i < sink_tiles ? i : window_tile + i - sink_tiles; }
};

template <int RT>
__device__ inline Tiles tiles_of(const PagedArgs& a, int entry) {
    const int b = entry / a.row_groups;
    const int first = (entry - b * a.row_groups) * (16 * RT);  // row of the sequence
    const int t0 = first / a.groups, t1 = min(a.tokens - 1, (first + 16 * RT - 1) / a.groups);
    int lo = INT32_MAX, hi = -1;
    for (int t = t0; t <= t1; ++t) {
        const int p = real_position(a, static_cast<int64_t>(b) * a.tokens + t);
        if (p >= 0) lo = min(lo, p);
        hi = max(hi, p);
    }
    Tiles r{0, 0, 1};  // nothing to see: one masked tile
    if (hi >= 0) {
        const int start = a.window > 0 ? max(0, lo - a.window + 1) : 0;
        r.window_tile = start / kTile;
        r.sink_tiles = min(r.window_tile, (min(a.sinks, start) + kTile - 1) / kTile);
        r.count = r.sink_tiles + hi / kTile - r.window_tile + 1;
    }
    return r;
}

template <typename T>
__device__ inline uint32_t pack2(float a, float b) {
    return static_cast<uint32_t>(T::from_float(a)) | (static_cast<uint32_t>(T::from_float(b)) << 16);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// Lane i of 16 gives the address of 4 values: a [4][16] tile whose row r is what lanes 4 r .. +3 name; it gets column i.
__device__ inline uint2 read_transposed(const uint16_t* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

__device__ inline float wave_cols_max(float v) {  // over the four lane groups that hold a column
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

// Attention of a few rows (query head of a kv head's group, token) per sequence over its pages. All work is one line of
// units (entry = (sequence, row group), kv head, tile of 32 keys), cut into equal shares for the blocks, so the lengths need
// not be known on the host nor be alike; a (entry, kv head) that lies in one block is finished there, of the others the blocks
// leave sums in the workspace that few_join_kernel adds. A wave takes every fourth tile of a share and keeps two in flight
// (DMA into its own ring: no barriers), and computes
//   S^T = K Q^T      v_mfma_f32_16x16x32, A = 16 keys x 32 dimensions, B = 16 rows of queries
//   O^T += V^T P^T   A = 16 dimensions x 32 keys, read transposed from the row-major tile, B = P^T: S^T's accumulator layout
//                    already, with keys 4 g .. +3 and 16 + 4 g .. +3 in lane group g
// and the probabilities' sums as one more product with ones, from the rounded values that the value product takes.
template <typename T, int D, int RT>
__global__ __launch_bounds__(64 * kWaves, 1) void few_kernel(const PagedArgs a) {
    constexpr int C = D / 8;                  // 16-byte chunks of a row
    constexpr int RowsPer = 64 / C;           // rows of one DMA instruction
    constexpr int Instr = 16 / RowsPer;       // instructions for 16 rows
    constexpr int PerTile = 4 * Instr;        // K and V, two 16-row halves
    constexpr int TileElems = kTile * D;
    __shared__ __attribute__((aligned(16))) uint16_t ring[kWaves][2][2][TileElems];
    __shared__ int64_t pre[kEntries + 1];
    __shared__ int64_t wave_total[kWaves];
    __shared__ float stat_m[kWaves][16 * RT], stat_l[kWaves][16 * RT];
    __shared__ int s_entry;
    static_assert(sizeof(ring) >= sizeof(float) * kWaves * 16 * D, "the rings hold the waves' sums of 16 rows");
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int entries = a.batch * a.row_groups;

    // the shares
    {
        const int per = (entries + 64 * kWaves - 1) / (64 * kWaves);
        int64_t sum = 0;
        for (int i = 0; i < per; ++i) {
            const int e = t * per + i;
            if (e < entries) {
                pre[e] = sum;
                sum += tiles_of<RT>(a, e).count;
            }
        }
        int64_t incl = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int64_t up = __shfl_up(incl, off, 64);
            if (lane >= off) incl += up;
        }
        if (lane == 63) wave_total[wave] = incl;
        if (t == 0) s_entry = 0;
        __syncthreads();
        int64_t before = incl - sum;
        for (int w = 0; w < wave; ++w) before += wave_total[w];
        for (int i = 0; i < per; ++i) {
            const int e = t * per + i;
            if (e < entries) pre[e] += before;
        }
        if (t == 0) pre[entries] = wave_total[0] + wave_total[1] + wave_total[2] + wave_total[3];
        __syncthreads();
    }
    const int64_t total = pre[entries] * a.kv_heads;
    int64_t share = (total + kBlocks - 1) / kBlocks;
    share = share < kLeastShare ? kLeastShare : share;
    int64_t u = blockIdx.x * share;
    const int64_t end = min(u + share, total);
    if (u >= end) return;
    for (int e = t; e < entries; e += 64 * kWaves)
        if (pre[e] * a.kv_heads <= u && u < pre[e + 1] * a.kv_heads) s_entry = e;
    __syncthreads();
    int entry = __builtin_amdgcn_readfirstlane(s_entry);

    uint32_t voff[Instr];
#pragma unroll
    for (int j = 0; j < Instr; ++j) {
        const int row = j * RowsPer + lane / C;
        const int swz = D == 128 ? row : row >> 1;
        voff[j] = static_cast<uint32_t>(row * D * 2 + 16 * ((lane % C) ^ (swz & (C - 1))));
    }
    const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_addr(&ring[wave][0][0][0]));
    int slot = 0;
    while (true) {
        const int64_t seg0 = pre[entry] * a.kv_heads;
        const int count = static_cast<int>(pre[entry + 1] - pre[entry]);
        const int kvh = __builtin_amdgcn_readfirstlane(static_cast<int>((u - seg0) / count));
        const int64_t seg = seg0 + static_cast<int64_t>(kvh) * count;
        const int first = __builtin_amdgcn_readfirstlane(static_cast<int>(u - seg));
        const int n = __builtin_amdgcn_readfirstlane(static_cast<int>(min<int64_t>(end - u, count - first)));
        const int b = entry / a.row_groups;
        const int row0 = (entry - b * a.row_groups) * (16 * RT);
        const int rows = min(16 * RT, a.tokens * a.groups - row0);
        Tiles tiles = tiles_of<RT>(a, entry);
        tiles.sink_tiles = __builtin_amdgcn_readfirstlane(tiles.sink_tiles);
        tiles.window_tile = __builtin_amdgcn_readfirstlane(tiles.window_tile);

        u32x4 qf[RT][D / 32];
        int last[RT], start[RT];
        int all_last = INT32_MAX, all_start = 0;  // what every row sees
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = min(16 * rt + c, rows - 1) + row0;
            const int tok = r / a.groups;
            const int64_t q_row = static_cast<int64_t>(b) * a.tokens + tok;
            last[rt] = 16 * rt + c < rows ? real_position(a, q_row) : -1;
            start[rt] = a.window > 0 ? max(0, last[rt] - a.window + 1) : 0;
            if (last[rt] >= 0) {
                all_last = min(all_last, last[rt]);
                all_start = max(all_start, start[rt]);
            }
            const uint16_t* src = a.q + q_row * a.q_stride + static_cast<int64_t>(kvh * a.groups + r - tok * a.groups) * D + 8 * g;
#pragma unroll
            for (int kt = 0; kt < D / 32; ++kt) qf[rt][kt] = *vec(src + 32 * kt);
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) {
            all_last = min(all_last, __shfl_xor(all_last, off, 64));
            all_start = max(all_start, __shfl_xor(all_start, off, 64));
        }
        all_last = __builtin_amdgcn_readfirstlane(all_last);
        all_start = __builtin_amdgcn_readfirstlane(all_start);

        f32x4 o[RT][D / 16], lsum[RT];
        float m[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY;
            lsum[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

        const __attribute__((address_space(4))) int32_t* table =
            (const __attribute__((address_space(4))) int32_t*)(a.pages.table + static_cast<int64_t>(b) * a.pages.table_stride);
        // the pages of a tile's halves, -1 where there is none (past the table's end too)
        auto page_of = [&](int key) {
            const int at = key / a.pages.page_size;
            if (at >= a.pages.table_pages) return -1;
            const int page = table[at];
            return page >= 0 && page < a.pages.pages ? page : -1;
        };
        auto issue = [&](int i, int buf) {
            const int key0 = tiles.at(first + wave + kWaves * i) * kTile;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = key0 + 16 * h;
                const int page = __builtin_amdgcn_readfirstlane(max(0, page_of(key)));
                const int64_t at = ((static_cast<int64_t>(page) * a.kv_heads + kvh) * a.pages.page_size + key % a.pages.page_size) * D;
                const uint32_t lds = ring_lds + static_cast<uint32_t>(buf * 2 * TileElems + h * 16 * D) * 2u;
#pragma unroll
                for (int j = 0; j < Instr; ++j) dma16_lds(a.k_pages + at, voff[j], lds + 1024u * j);
#pragma unroll
                for (int j = 0; j < Instr; ++j) dma16_lds(a.v_pages + at, voff[j], lds + 2u * TileElems + 1024u * j);
            }
        };
        const int mine = n > wave ? (n - wave + kWaves - 1) / kWaves : 0;
        if (mine > 0) issue(0, 0);
        if (mine > 1) issue(1, 1);
        for (int i = 0; i < mine; ++i) {
            const int buf = i & 1;
            if (i + 1 < mine) wait_vmcnt<PerTile>();
            else wait_vmcnt<0>();
            asm volatile("" ::: "memory");
            const uint16_t* kb = ring[wave][buf][0];
            const uint16_t* vb = ring[wave][buf][1];
            const int key0 = tiles.at(first + wave + kWaves * i) * kTile;
            u32x4 kf[2][D / 32];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int kt = 0; kt < D / 32; ++kt) {
                    const int swz = D == 128 ? c : c >> 1;
                    kf[h][kt] = *vec(kb + (16 * h + c) * D + 8 * ((4 * kt + g) ^ (swz & (C - 1))));
                }
            // which of the lane's keys (16 h + 4 g + i in bit 4 h + i) are there
            const bool there0 = page_of(key0) >= 0, there1 = page_of(key0 + 16) >= 0;
            const bool whole = there0 && there1 && key0 + kTile - 1 <= all_last &&
                               (key0 >= all_start || key0 + kTile <= a.sinks);
            uint32_t some = 0;  // seen by some row of the wave's
            u32x4 pf[RT];
            uint32_t seen[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int kt = 0; kt < D / 32; ++kt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) s[h] = mfma16x16x32<T>(kf[h][kt], qf[rt][kt], s[h]);
                seen[rt] = 0xFF;
                if (!whole) {
                    seen[rt] = 0;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + 16 * h + 4 * g + e;
                            const bool see = (h ? there1 : there0) && key <= last[rt] && (key >= start[rt] || key < a.sinks);
                            seen[rt] |= see ? 1u << (4 * h + e) : 0u;
                        }
                    some |= seen[rt];
                }
                float top = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[h][e] = (seen[rt] >> (4 * h + e)) & 1 ? s[h][e] * a.scale : -INFINITY;
                        top = fmaxf(top, s[h][e]);
                    }
                top = wave_cols_max(top);
                if (__any(top > m[rt] + kSlack)) {
                    const float mn = fmaxf(m[rt], top);
                    const float keep = __builtin_amdgcn_exp2f(m[rt] - (mn == -INFINITY ? 0.0f : mn));
                    m[rt] = mn;
                    lsum[rt] *= keep;
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] *= keep;
                }
                const float mu = m[rt] == -INFINITY ? 0.0f : m[rt];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[h][e] = __builtin_amdgcn_exp2f(s[h][e] - mu);
                    pf[rt][2 * h] = pack2<T>(s[h][0], s[h][1]);
                    pf[rt][2 * h + 1] = pack2<T>(s[h][2], s[h][3]);
                }
                lsum[rt] = mfma16x16x32<T>(u32x4{T::ONE_PAIR, T::ONE_PAIR, T::ONE_PAIR, T::ONE_PAIR}, pf[rt], lsum[rt]);
            }
            u32x4 vf[D / 16];
            const int vr = 4 * g + (c >> 2);  // of 16: the row whose address the lane gives
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) {
                const int swz = D == 128 ? vr : vr >> 1;
                const int at = 8 * ((2 * dt + ((c >> 1) & 1)) ^ (swz & (C - 1))) + 4 * (c & 1);
                const uint2 lo = read_transposed(vb + vr * D + at), hi = read_transposed(vb + (16 + vr) * D + at);
                vf[dt] = u32x4{lo.x, lo.y, hi.x, hi.y};
            }
            bool tainted = false;
            if (!whole) {
                // values that no row sees are cleared (0 * NaN would reach every row); where a value that some rows see is
                // not finite, the rows' sums are made one by one
#pragma unroll
                for (int off = 1; off < 16; off <<= 1) some |= __shfl_xor(some, off, 64);
                float zero = 0.0f;
                u32x4 keep;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    keep[w] = ((some >> (2 * w)) & 1 ? 0xFFFFu : 0u) | ((some >> (2 * w + 1)) & 1 ? 0xFFFF0000u : 0u);
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) {
                    vf[dt] &= keep;
#pragma unroll
                    for (int w = 0; w < 4; ++w) zero = T::dot2(vf[dt][w], 0u, zero);
                }
                tainted = __any(zero != zero);
            }
            if (!tainted) {
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma16x16x32<T>(vf[dt], pf[rt], o[rt][dt]);
            } else {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    for (int k = 0; k < kTile; ++k) {
                        const int from = 16 * ((k & 15) >> 2) + c;  // the lane that has the key's probability
                        const int at = 4 * (k >> 4) + (k & 3);
                        const uint32_t mine2 = at & 4 ? (at & 2 ? pf[rt][3] : pf[rt][2]) : (at & 2 ? pf[rt][1] : pf[rt][0]);
                        const uint32_t pair = __shfl(mine2, from, 64);
                        const bool see = (__shfl(seen[rt], from, 64) >> at) & 1;
                        const float p = T::to_float(static_cast<uint16_t>(pair >> (16 * (at & 1))));
                        const int swz = D == 128 ? k : k >> 1;
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int d = 16 * dt + 4 * g + e;
                                const float v = T::to_float(vb[k * D + 8 * ((d >> 3) ^ (swz & (C - 1))) + (d & 7)]);
                                o[rt][dt][e] = see ? fmaf(p, v, o[rt][dt][e]) : o[rt][dt][e];
                            }
                    }
            }
            if (i + 2 < mine) {
                __builtin_amdgcn_s_waitcnt(0xF | (0x3 << 14) | (0x7 << 4));  // the buffer's reads have ended (lgkmcnt 0)
                issue(i + 2, buf);
            }
        }

        // the waves' sums, joined through the rings a row group at a time
        const bool done = first == 0 && n == count;
        const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + slot) * a.rows_kept;
        float* red = reinterpret_cast<float*>(&ring[0][0][0][0]);
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (rt > 0) __syncthreads();
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt)
                *reinterpret_cast<f32x4*>(red + (wave * 16 + c) * D + 4 * ((4 * dt + g) ^ c)) = o[rt][dt];
            if (g == 0) {  // a row of padding took part where the tile was whole: -inf says that its sums are none
                stat_m[wave][c] = last[rt] < 0 ? -INFINITY : m[rt];
                stat_l[wave][c] = lsum[rt][0];
            }
            __syncthreads();
            for (int id = t; id < 16 * C; id += 64 * kWaves) {
                const int row = id / C, ch = id % C;
                if (16 * rt + row >= rows) continue;
                float M = stat_m[0][row];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) M = fmaxf(M, stat_m[w][row]);
                const float mu = M == -INFINITY ? 0.0f : M;
                float L = 0.0f;
                f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    if (stat_m[w][row] == -INFINITY) continue;
                    const float f = __builtin_amdgcn_exp2f(stat_m[w][row] - mu);
                    L += f * stat_l[w][row];
                    lo += f * *reinterpret_cast<const f32x4*>(red + (w * 16 + row) * D + 4 * ((2 * ch) ^ row));
                    hi += f * *reinterpret_cast<const f32x4*>(red + (w * 16 + row) * D + 4 * ((2 * ch + 1) ^ row));
                }
                const int r = row0 + 16 * rt + row;
                if (done) {
                    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                    const int tok = r / a.groups;
                    const int64_t at = ((static_cast<int64_t>(b) * a.tokens + tok) * a.heads + kvh * a.groups + r - tok * a.groups) * D;
                    *reinterpret_cast<u32x4*>(a.out + at + 8 * ch) =
                        u32x4{pack2<T>(lo[0] * inv, lo[1] * inv), pack2<T>(lo[2] * inv, lo[3] * inv),
                              pack2<T>(hi[0] * inv, hi[1] * inv), pack2<T>(hi[2] * inv, hi[3] * inv)};
                } else {
                    float* dst = a.part_o + (part + 16 * rt + row) * D + 8 * ch;
                    *reinterpret_cast<f32x4*>(dst) = lo;
                    *reinterpret_cast<f32x4*>(dst + 4) = hi;
                    if (ch == 0) a.part_ml[part + 16 * rt + row] = float2{M, L};
                }
            }
        }
        if (first == 0 && t == 0)
            a.desc[entry * a.kv_heads + kvh] =
                int2{static_cast<int>(blockIdx.x) * 2 + slot, static_cast<int>((seg + count - 1) / share)};
        u += n;
        if (u >= end) return;
        slot = 1;  // a share's first and last (entry, kv head) are the ones that it may not finish
        if (kvh + 1 == a.kv_heads) ++entry;
        __syncthreads();
    }
}

// Adds what the blocks left of one row of an (entry, kv head): the threads in groups of D / 4, a group a partial result.
template <typename T, int D, int RT>
__global__ __launch_bounds__(256) void few_join_kernel(const PagedArgs a) {
    constexpr int L4 = D / 4, Groups = 256 / L4;
    __shared__ float red[Groups][D];
    __shared__ float tops[4], sums[4];
    const int t = threadIdx.x;
    const int seg = static_cast<int>(blockIdx.x) / a.rows_kept;
    const int row = static_cast<int>(blockIdx.x) - seg * a.rows_kept;
    const int2 d = a.desc[seg];
    const int first = d.x >> 1, n = d.y - first + 1;
    if (n == 1) return;
    const int entry = seg / a.kv_heads, kvh = seg - entry * a.kv_heads;
    const int b = entry / a.row_groups;
    const int r = (entry - b * a.row_groups) * (16 * RT) + row;
    if (r >= a.tokens * a.groups) return;
    // partial i: the first block's slot, then slot 0 of those behind it
    auto place = [&](int i) { return static_cast<int64_t>(i == 0 ? d.x : (first + i) * 2) * a.rows_kept + row; };
    static_assert(kBlocks == 256, "a thread a block's statistics");
    const float2 ml = t < n ? a.part_ml[place(t)] : float2{-INFINITY, 0.0f};
    float top = ml.x;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    if ((t & 63) == 0) tops[t >> 6] = top;
    __syncthreads();
    const float M = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float mu = M == -INFINITY ? 0.0f : M;
    const float l = wave_sum(ml.y * __builtin_amdgcn_exp2f(ml.x - mu));
    if ((t & 63) == 0) sums[t >> 6] = l;
    const int grp = t / L4, at = 4 * (t % L4);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i = grp; i < n; i += Groups) {
        const int64_t p = place(i);
        const float f = __builtin_amdgcn_exp2f(a.part_ml[p].x - mu);
        o += f * *reinterpret_cast<const f32x4*>(a.part_o + p * D + at);
    }
    *reinterpret_cast<f32x4*>(&red[grp][at]) = o;
    __syncthreads();
    if (t < D / 2) {
        const float L = sums[0] + sums[1] + sums[2] + sums[3];
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        float x = 0.0f, y = 0.0f;
        for (int i = 0; i < Groups; ++i) {
            x += red[i][2 * t];
            y += red[i][2 * t + 1];
        }
        const int tok = r / a.groups;
        const int64_t to = ((static_cast<int64_t>(b) * a.tokens + tok) * a.heads + kvh * a.groups + r - tok * a.groups) * D;
        *reinterpret_cast<uint32_t*>(a.out + to + 2 * t) = pack2<T>(x * inv, y * inv);
    }
}

int row_tiles(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

// Sequences of a launch, and what it needs of the workspace.
struct FewPlan {
    int64_t rt, row_groups, rows_kept, batch;
    size_t part_o, part_ml, desc, bytes;
};

FewPlan few_plan(int64_t batch, int64_t tokens, int64_t groups, int64_t kv_heads, int64_t head_dim) {
    FewPlan p{};
    p.rt = row_tiles(tokens * groups);
    p.row_groups = ceil_div(tokens * groups, 16 * p.rt);
    p.rows_kept = std::min(tokens * groups, 16 * p.rt);
    p.batch = std::min({batch, std::max<int64_t>(1, kEntries / p.row_groups),
                        std::max<int64_t>(1, kMaxGrid / (p.row_groups * kv_heads * p.rows_kept))});
    p.part_o = static_cast<size_t>(kBlocks) * 2 * p.rows_kept * head_dim * sizeof(float);
    p.part_ml = static_cast<size_t>(kBlocks) * 2 * p.rows_kept * sizeof(float2);
    p.desc = static_cast<size_t>(p.batch) * p.row_groups * kv_heads * sizeof(int2);
    p.bytes = p.part_o + p.part_ml + p.desc;
    return p;
}

template <typename T, int D, int RT>
void launch_few(const PagedArgs& a, hipStream_t st) {
    few_kernel<T, D, RT><<<dim3(kBlocks), 64 * kWaves, 0, st>>>(a);
    few_join_kernel<T, D, RT><<<dim3(static_cast<unsigned>(a.batch * a.row_groups * a.kv_heads * a.rows_kept)), 256, 0, st>>>(a);
}

template <typename T, int D>
void launch_paged(PagedArgs a, const FewPlan& plan, char* ws, hipStream_t st) {
    a.row_groups = static_cast<int>(plan.row_groups);
    a.rows_kept = static_cast<int>(plan.rows_kept);
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + plan.part_o);
    a.desc = reinterpret_cast<int2*>(ws + plan.part_o + plan.part_ml);
    const int batch = a.batch;
    for (int b = 0; b < batch; b += static_cast<int>(plan.batch)) {
        PagedArgs s = a;
        s.batch = std::min(static_cast<int>(plan.batch), batch - b);
        s.q += static_cast<int64_t>(b) * a.tokens * a.q_stride;
        s.positions += static_cast<int64_t>(b) * a.tokens;
        s.pages.table += b * a.pages.table_stride;
        s.out += static_cast<int64_t>(b) * a.tokens * a.heads * D;
        if (plan.rt == 1) launch_few<T, D, 1>(s, st);
        else if (plan.rt == 2) launch_few<T, D, 2>(s, st);
        else launch_few<T, D, 4>(s, st);
    }
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
    if (batch * tokens > kMaxGrid * 256 / slots) return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large", name);
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
        tokens > INT32_MAX || batch * tokens > INT32_MAX / heads)
        return 0;
    return few_plan(batch, tokens, heads / kv_heads, kv_heads, head_dim).bytes;
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
    const size_t need = nq_paged_attention_workspace_bytes(batch, tokens, heads, kv_heads, head_dim, table_pages, page_size);
    if (!workspace || workspace_bytes < need)
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
    a.window = static_cast<int>(std::min(window, kMaxKeys));
    a.sinks = static_cast<int>(std::min(sinks, kMaxKeys));
    a.scale = scaling * 1.44269504088896340736f;  // exp(x) = exp2(x log2(e))
    const FewPlan plan = few_plan(batch, tokens, heads / kv_heads, kv_heads, head_dim);
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
