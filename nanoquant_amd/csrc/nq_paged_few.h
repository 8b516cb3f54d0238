// Attention of a few rows per sequence over the pages of a cache: what few_kernel, its launches and the kernels beside it share.
#pragma once

#include <type_traits>

#include "nq_common.h"
#include "nq_paged.h"
#include "nq_wave.h"

namespace nq {
namespace {

constexpr int kTileShift = 5, kTile = 1 << kTileShift;  // keys a wave of few_kernel takes at a time
constexpr int kWaves = 4;          // of a block
constexpr int kCUs = 256;
// (sequence, row group) pairs of a launch, whose key counts every block adds up in LDS: 8 KB, with which two blocks still fit a
// CU where its rings let them (FewShape; rows_kernel of 64 dimensions)
constexpr int kFewEntries = 512, kEntries = 1024;
constexpr int kLeastShare = 4;     // tiles a block of few_kernel takes at least: one a wave
constexpr int kLeastTiles = 8;     // the same of rows_kernel's
// what an (entry, kv head) costs on top of its tiles, in tiles: its queries, its first tiles' way from memory, its sums' join.
// Uncounted, blocks that have many short ones end last: five tokens of nine sequences of 300 to 6000 keys 53 us against 46, 17
// sequences' next tokens 66 against 63.5; two chunks of 700 tokens, heads of 64, 147 against 145.
constexpr int kFewStart = 8, kStart = 4;
constexpr float kSlack = 8.0f;

struct PagedArgs {
    static constexpr bool kGroups = false;
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
    int4* spans;        // [batch * row_groups]: Tiles, for rows_kernel's shares
    int2* desc;         // [batch * row_groups * kv_heads]: {first block * 2 + its slot, last block}
    float* part_o;      // [blocks][2][rows_kept][D]
    float2* part_ml;    // the same rows' {maximum, sum}
};

// x / n of 0 <= x < 2^21 by `per`, 1 / n rounded: (x + 1/2) / n is 1 / 2n from an integer at least, and the product off by 2^-23 of
// itself at most. Thirty instructions fewer than a division, in what a block does before its first load.
__device__ inline int small_quotient(int x, float per) { return static_cast<int>((static_cast<float>(x) + 0.5f) * per); }

// The same where groups of sequences have their leading pages in common: an entry is a group's row group (row t of member i:
// i * tokens * groups + t) over the shared keys, or a sequence's over its own. Entries of groups come first.
struct GroupArgs : PagedArgs {
    static constexpr bool kGroups = true;
    const int32_t* members;  // [sharing][most]
    const int32_t* shared;   // [sharing]: pages in common
    int sharing, most;       // groups, and places of one
    // Of a group's entries and of the sequences': row groups (a sequence's are row_groups), rows of one, and those that there
    // are. Each entry's first part has a place of its own among the workspace's parts, the later ones their block's.
    int group_rows, group_tile, group_kept, own_tile;  // rows_kept: a sequence's
    int64_t own_first, group_later, own_later;         // rows
    int group_shift, own_shift;                        // of the tiles: powers of two
    // inverses: a launch lists 2^17 members' rows at most
    float per_most, per_each, per_groups, per_tokens, per_group_rows, per_row_groups;
    __device__ int row_group_of(int entry, bool of_group) const {  // of an entry's number among its kind
        return entry - small_quotient(entry, of_group ? per_group_rows : per_row_groups) * (of_group ? group_rows : row_groups);
    }
    int* place;              // [batch]: where a sequence stands in `members`; -1: nowhere
    __device__ int entries_of_groups() const { return sharing * group_rows; }
    __device__ int64_t first_part(int entry, int kvh) const {
        const int own = entry - entries_of_groups();
        if (own < 0) return (static_cast<int64_t>(entry) * kv_heads + kvh) * group_kept;
        return own_first + (static_cast<int64_t>(own) * kv_heads + kvh) * rows_kept;
    }
    __device__ int64_t later_part(int entry, int block) const {
        const bool of_group = entry < entries_of_groups();
        return (of_group ? group_later : own_later) + static_cast<int64_t>(block) * (of_group ? group_tile : own_tile);
    }
};

// A position that the table holds, -1 for any other.
__device__ inline int real_position(const PagedArgs& a, int64_t row) {
    const int64_t p = a.positions[row];
    return p >= 0 && p < a.pages.capacity() ? static_cast<int>(p) : -1;
}

__device__ inline int64_t out_row(const PagedArgs& a, int b, int kvh, int r) {  // row r of a sequence and kv head
    const int tok = r / a.groups;
    return (static_cast<int64_t>(b) * a.tokens + tok) * a.heads + kvh * a.groups + r - tok * a.groups;
}

// The key tiles that a group of rows sees: `sink_tiles` from the front, then those from window_tile on.
struct Tiles {
    int sink_tiles, window_tile, count;
    int front = 0;
    __device__ int at(int i) const { return i < sink_tiles ? front + i : window_tile + i - sink_tiles; }
};

// of rows whose real positions go from lo to hi (hi -1: none, which is one masked tile)
template <int kKeys>
__device__ inline Tiles tiles_between(const PagedArgs& a, int lo, int hi) {
    Tiles r{0, 0, 1};
    if (hi >= 0) {
        const int start = a.window > 0 ? max(0, lo - a.window + 1) : 0;
        r.window_tile = start / kKeys;
        r.sink_tiles = min(r.window_tile, (min(a.sinks, start) + kKeys - 1) / kKeys);
        r.count = r.sink_tiles + hi / kKeys - r.window_tile + 1;
    }
    return r;
}

// The same among the keys from `from` to before `to` (a group's shared ones, a member's others), tiles of 2^shift.
__device__ inline Tiles tiles_within(const PagedArgs& a, int shift, int lo, int hi, int from, int to) {
    Tiles r{0, from >> shift, 1, from >> shift};
    const int last = min(hi, to - 1);
    if (last < from) return r;
    const int start = a.window > 0 ? max(from, lo - a.window + 1) : from;
    const int sinks = min(a.sinks, min(start, to)), sink_tiles = sinks > from ? ((sinks - 1) >> shift) + 1 - r.front : 0;
    if (start > last) {  // the window begins behind them
        r.sink_tiles = sink_tiles;
        r.count = max(1, sink_tiles);
        return r;
    }
    r.window_tile = start >> shift;
    r.sink_tiles = min(r.window_tile - r.front, sink_tiles);
    r.count = r.sink_tiles + (last >> shift) - r.window_tile + 1;
    return r;
}

// Row groups of `group` rows (token t, query head g of a kv head's G: row t G + g); entry = (sequence, row group).
__device__ inline int2 span_of_tokens(const PagedArgs& a, int b, int t0, int t1) {  // the least and the largest position
    int lo = INT32_MAX, hi = -1;
    for (int t = t0; t <= t1; t += 8) {
        int p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = real_position(a, static_cast<int64_t>(b) * a.tokens + min(t + i, t1));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo = p[i] >= 0 ? min(lo, p[i]) : lo;
            hi = max(hi, p[i]);
        }
    }
    return int2{lo, hi};
}
__device__ inline Tiles tiles_of_few(const PagedArgs& a, int entry, int group) {
    const int b = entry / a.row_groups;
    const int first = (entry - b * a.row_groups) * group;
    const int2 span = span_of_tokens(a, b, first / a.groups, min(a.tokens - 1, (first + group - 1) / a.groups));
    return tiles_between<kTile>(a, span.x, span.y);
}

constexpr int kNobody = INT32_MAX, kIdle = 1 << 30;  // a sequence without tokens leads only where no other does
constexpr int kSequenceBits = 10;  // of a batch's: each has an entry

// What the blocks of a launch with groups work out before they take their shares, in LDS.
template <int kEntries>
struct GroupPlan {
    int place[kEntries];  // of a sequence: the last place that names it, -1
    // of an entry: the sequence by whose row of the table its pages are found, with its place in the group above it until
    // tiles_of_plan; kNobody. The first place that has a token: rows of later ones may lack pages that their windows are past
    int lead[kEntries];
    int ends[kEntries];   // of a group: the shared keys
    int2 spans[kEntries];
    uint8_t slow[kEntries];  // of a group's entry: the tiles in which some member's window begins
    __device__ int from(int b, float per_most) const {  // of a sequence's own keys
        return place[b] < 0 ? 0 : ends[small_quotient(place[b], per_most)];
    }
};
// All threads of the block.
template <int kThreads, int kEntries>
__device__ inline void plan_groups(const GroupArgs& a, GroupPlan<kEntries>& plan) {
    static_assert(kEntries <= 1 << kSequenceBits, "a sequence's number fits below its place, of 2^17, and kIdle");
    const int t = threadIdx.x, first = a.entries_of_groups(), each = a.tokens * a.groups, own = a.batch * a.row_groups;
    auto span_of = [&](int e) {
        const int b = small_quotient(e, a.per_row_groups), row = (e - b * a.row_groups) << a.own_shift;
        if (a.tokens == 1) {
            const int p = real_position(a, b);
            return int2{p >= 0 ? p : INT32_MAX, p};
        }
        const int t0 = small_quotient(row, a.per_groups), t1 = small_quotient(min(row + a.own_tile, each) - 1, a.per_groups);
        return span_of_tokens(a, b, t0, t1);
    };
    // what all threads load first, together
    int2 span = {0, 0};
    if (t < own) span = span_of(t);
    const int member = t < a.sharing * a.most ? a.members[t] : -1;
    for (int g = t; g < a.sharing; g += kThreads) plan.ends[g] = min(max(a.shared[g], 0), a.pages.table_pages) * a.pages.page_size;
    for (int b = t; b < a.batch; b += kThreads) plan.place[b] = -1;
    for (int e = t; e < first; e += kThreads) {
        plan.spans[e] = int2{INT32_MAX, -1};
        plan.lead[e] = kNobody;
    }
    __syncthreads();
    for (int at = t; at < a.sharing * a.most; at += kThreads) {
        const int b = at == t ? member : a.members[at];
        if (b >= 0 && b < a.batch && plan.ends[small_quotient(at, a.per_most)] > 0) atomicMax(&plan.place[b], at);
    }
    __syncthreads();
    for (int e = t; e < own; e += kThreads) {
        const int b = small_quotient(e, a.per_row_groups), at = plan.place[b], row = (e - b * a.row_groups) << a.own_shift;
        const int rows = min(a.own_tile, each - row);
        if (e != t) span = span_of(e);
        plan.spans[first + e] = span;
        plan.lead[first + e] = b;
        if (at < 0) continue;
        const int g = small_quotient(at, a.per_most), in_group = at - g * a.most, row0 = in_group * each + row;
        const int lead = in_group << kSequenceBits | b;
        for (int i = row0 >> a.group_shift; i <= (row0 + rows - 1) >> a.group_shift; ++i) {
            atomicMin(&plan.spans[g * a.group_rows + i].x, span.x);
            atomicMax(&plan.spans[g * a.group_rows + i].y, span.y);
            atomicMin(&plan.lead[g * a.group_rows + i], span.y < 0 ? lead | kIdle : lead);
        }
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int b = t; b < a.batch; b += kThreads) a.place[b] = plan.place[b];
}
// The tiles of 2^shift keys of an entry, whose span turns into their places. 0: nobody's
template <int kEntries>
__device__ inline int tiles_of_plan(const GroupArgs& a, GroupPlan<kEntries>& plan, int e, int shift) {
    if (plan.lead[e] == kNobody) return 0;
    plan.lead[e] &= (1 << kSequenceBits) - 1;
    const int of_groups = a.entries_of_groups();
    const int from = e < of_groups ? 0 : plan.from(plan.lead[e], a.per_most);
    const int to = e < of_groups ? plan.ends[small_quotient(e, a.per_group_rows)] : INT32_MAX;
    const Tiles r = tiles_within(a, shift, plan.spans[e].x, plan.spans[e].y, from, to);
    int slow = 0;
    if (e < of_groups && a.window > 0 && r.count > r.sink_tiles)
        slow = (min(max(0, plan.spans[e].y - a.window + 1), to - 1) >> shift) - r.window_tile + 1;
    plan.slow[e] = static_cast<uint8_t>(min(max(slow, 0), 255));
    plan.spans[e] = int2{r.sink_tiles, r.window_tile};
    return r.count;
}

// Which keys of a tile a row sees, a bit a key: arithmetic on words, since compares of every key with every row would each
// hold a pair of scalar registers.
__device__ inline uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : 0xFFFFFFFFu >> (32 - n); }
__device__ inline uint32_t seen_bits(int key0, int last, int start, int sinks) {  // of keys key0 .. key0 + 31
    return low_bits(last - key0 + 1) & (~low_bits(start - key0) | low_bits(sinks - key0));
}
__device__ inline uint32_t bit_mask(uint32_t bits, int i) {
    return static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(bits), i, 1));
}
__device__ inline float or_minus_inf(float x, uint32_t bits, int i) {  // x where bit i is set
    return __builtin_bit_cast(float, bit_select(bit_mask(bits, i), __builtin_bit_cast(uint32_t, x), 0xFF800000u));
}
// both halves of a pair under bits i and i + 1
__device__ inline uint32_t pair_mask(uint32_t bits, int i) { return bit_select(0xFFFFu, bit_mask(bits, i), bit_mask(bits, i + 1)); }

template <typename T>
__device__ inline uint32_t pack2(float a, float b);
template <>
__device__ inline uint32_t pack2<F16>(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
}
template <>
__device__ inline uint32_t pack2<BF16>(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// All work of a launch is one line of units (entry, kv head, tile of keys), cut into equal shares for the blocks, so lengths
// need neither be known on the host nor be alike. `count(e)`: the tiles of an entry and its charge; pre[e]: those of the entries
// before it.
struct Shares {
    int64_t share, first, end;  // units a block, and this block's
    int64_t base;               // the first unit of all
    int block;                  // this one, of those that have shares
    int entry;                  // of the first unit; -1: nothing to do
    __device__ int block_of(int64_t unit) const;
};
// a / b for 0 <= a < 2^53 and b > 0, the same for the wave: the quotient in fp64 is off by less than its distance from the next
// integer. Of small a as small_quotient, with a reciprocal that is off by 2^-23.
__device__ inline int64_t quotient(int64_t a, int64_t b) {
    if (a < 1 << 20) return small_quotient(static_cast<int>(a), __builtin_amdgcn_rcpf(static_cast<float>(b)));
    return static_cast<int64_t>(static_cast<double>(a) / static_cast<double>(b));
}
__device__ inline int Shares::block_of(int64_t unit) const { return static_cast<int>(quotient(unit - base, share)); }

// Sum: in what a wave's are added up, where they are exact
template <int kThreads, typename Sum, typename Count>
__device__ inline void prefix_sums(int entries, int64_t* pre, int64_t* wave_total, Count count) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int per = (entries + kThreads - 1) / kThreads;
    int64_t sum = 0;
    for (int i = 0; i < per; ++i) {
        const int e = t * per + i;
        if (e < entries) {
            pre[e] = sum;
            sum += count(e);
        }
    }
    const int64_t incl = static_cast<int64_t>(wave_scan(static_cast<Sum>(sum)));
    if (lane == 63) wave_total[wave] = incl;
    __syncthreads();
    int64_t before = incl - sum;
    for (int w = 0; w < wave; ++w) before += wave_total[w];
    for (int i = 0; i < per; ++i) {
        const int e = t * per + i;
        if (e < entries) pre[e] += before;
    }
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) all += wave_total[w];
    if (t == 0) pre[entries] = all;
    __syncthreads();
}
// The share of one of `blocks` blocks in the units of entries e0 to e1 - 1, but for its first entry; `end` <= `first`: nothing.
__device__ inline Shares share_of(const PagedArgs& a, int e0, int e1, int block, int blocks, int least, const int64_t* pre) {
    Shares r;
    r.base = pre[e0] * a.kv_heads;
    r.block = block;
    const int64_t total = pre[e1] * a.kv_heads - r.base;
    r.share = max<int64_t>(quotient(total + blocks - 1, blocks), least);
    r.first = r.base + block * r.share;
    r.end = min(r.first + r.share, r.base + total);
    r.entry = -1;
    return r;
}
__device__ inline bool holds_unit(const PagedArgs& a, const int64_t* pre, int e, int64_t unit) {
    return pre[e] * a.kv_heads <= unit && unit < pre[e + 1] * a.kv_heads;
}
template <int kThreads>
__device__ inline Shares take_share(const PagedArgs& a, int e0, int e1, int block, int blocks, int least, const int64_t* pre,
                                    int* s_entry) {
    Shares r = share_of(a, e0, e1, block, blocks, least, pre);
    if (r.first >= r.end) return r;
    for (int e = e0 + static_cast<int>(threadIdx.x); e < e1; e += kThreads)
        if (holds_unit(a, pre, e, r.first)) *s_entry = e;
    __syncthreads();
    r.entry = __builtin_amdgcn_readfirstlane(*s_entry);
    return r;
}
template <int kThreads, int kBlocks, typename Sum, typename Count>
__device__ inline Shares make_shares(const PagedArgs& a, int entries, int least, int64_t* pre, int64_t* wave_total,
                                     int* s_entry, Count count) {
    prefix_sums<kThreads, Sum>(entries, pre, wave_total, count);
    return take_share<kThreads>(a, 0, entries, static_cast<int>(blockIdx.x), kBlocks, least, pre, s_entry);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// Rows row0 on of an entry's row group, of which `rows` there are: where a row's query lies, and which keys it sees.
struct RowAt {
    int64_t q_row;  // (sequence, token)
    int head;       // of the kv head's group
    int position;   // -1: padding
    int last;       // its position, or the last of the entry's keys where that is before it
};
template <typename Args>
struct Rows {
    int b, row0, rows;
    int from = 0, to = INT32_MAX;  // the entry's keys
    int group = -1;                // of sequences; -1: sequence b's own
    const int* place = nullptr;    // GroupPlan's
    __device__ RowAt at(const Args& a, int row) const {
        const int r = row0 + row;
        if constexpr (Args::kGroups) {
            if (group >= 0) {
                const int i = small_quotient(r, a.per_each), left = r - i * a.tokens * a.groups, tok = small_quotient(left, a.per_groups);
                const int m = a.members[group * a.most + i];
                if (m < 0 || m >= a.batch || place[m] != group * a.most + i) return RowAt{0, 0, -1, -1};
                const int64_t q_row = static_cast<int64_t>(m) * a.tokens + tok;
                const int p = real_position(a, q_row);
                return RowAt{q_row, left - tok * a.groups, p, min(p, to - 1)};
            }
        }
        int tok;
        if constexpr (Args::kGroups) tok = small_quotient(r, a.per_groups);
        else tok = r / a.groups;
        const int64_t q_row = static_cast<int64_t>(b) * a.tokens + tok;
        const int p = real_position(a, q_row);
        return RowAt{q_row, r - tok * a.groups, p, p};
    }
    __device__ bool holds(int key) const { return !Args::kGroups || (key >= from && key < to); }
    __device__ uint32_t held_bits(int key0) const {  // of keys key0 .. key0 + 31
        return Args::kGroups ? ~low_bits(from - key0) & low_bits(to - key0) : 0xFFFFFFFFu;
    }
    __device__ bool holds_tile(int key0) const { return !Args::kGroups || (key0 >= from && key0 <= to - kTile); }
};

// Lane i of 16 gives the address of 4 values: a [4][16] tile whose row r is what lanes 4 r .. +3 name; it gets column i.
__device__ inline uint2 read_transposed(const uint16_t* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

// A value that some rows of a product see and others do not reaches the others too where it is not finite (0 * inf, 0 * NaN).
// A block that finds one in a tile that its rows see in part makes its result here instead: a wave a row, a key at a time,
// with lane l at dimensions l and, of 128, l + 64. For data of which no speed is asked.
template <typename T, int D, typename Args>
__device__ inline void slow_rows(const Args& a, const Rows<Args>& rows, int kvh, const Tiles& tiles, int keys, int first, int n,
                                 bool done, int64_t part, int wave, int waves) {
    constexpr int N = D / 64;
    const int lane = threadIdx.x & 63;
    for (int row = wave; row < rows.rows; row += waves) {
        const RowAt at_row = rows.at(a, row);
        const int last = at_row.last, start = a.window > 0 ? max(0, at_row.position - a.window + 1) : 0;
        const uint16_t* q = a.q + at_row.q_row * a.q_stride + static_cast<int64_t>(kvh * a.groups + at_row.head) * D + lane;
        float o[N], m = -INFINITY, l = 0.0f;
        for (int i = 0; i < N; ++i) o[i] = 0.0f;
        for (int tile = first; tile < first + n; ++tile)
            for (int key = tiles.at(tile) * keys; key < (tiles.at(tile) + 1) * keys; ++key) {
                const int slot = a.pages.slot_of(key);
                const int page = slot < a.pages.table_pages ? a.pages.page(rows.b, slot) : -1;
                if (key > last || !rows.holds(key) || !(key >= start || key < a.sinks) || page < 0) continue;
                const int64_t at = ((static_cast<int64_t>(page) * a.kv_heads + kvh) * a.pages.page_size + key - slot * a.pages.page_size) * D + lane;
                float s = 0.0f;
                for (int i = 0; i < N; ++i) s = fmaf(T::to_float(q[64 * i]), T::to_float(a.k_pages[at + 64 * i]), s);
                s = wave_sum(s) * a.scale;
                const float top = fmaxf(m, s);
                const float keep = __builtin_amdgcn_exp2f(m - top), e = __builtin_amdgcn_exp2f(s - top);
                const bool none = top == -INFINITY && s == s;  // scores of -inf so far
                m = top;
                l = none ? 0.0f : fmaf(l, keep, e);
                for (int i = 0; i < N; ++i) o[i] = none ? 0.0f : fmaf(e, T::to_float(a.v_pages[at + 64 * i]), o[i] * keep);
            }
        for (int i = 0; i < N; ++i) {
            if (done) a.out[out_row(a, rows.b, kvh, rows.row0 + row) * D + lane + 64 * i] = T::from_float(l == 0.0f ? 0.0f : o[i] / l);
            else a.part_o[(part + row) * D + lane + 64 * i] = o[i];
        }
        if (!done && lane == 0) a.part_ml[part + row] = float2{m, l};
    }
}

// Attention of a few rows (query head of a kv head's group, token) per sequence over its pages: p_j = 2^(s_j - m), out =
// sum p_j v_j / sum p_j of s = q k scale log2(e), with m moved up to the running maximum wherever that is more than 8 above it.
// kShared: an (entry, kv head) that lies in one block's share is finished there, of the others the blocks leave sums in the
// workspace that few_join_kernel adds; otherwise a block has an (entry, kv head) for itself. A wave takes every fourth tile of
// its block's, and its own ring (DMA, no barriers) takes the next tile's keys as soon as these have been read, its values
// likewise, and computes
//   S^T = K Q^T      v_mfma_f32_16x16x32, A = 16 keys x 32 dimensions, B = 16 rows of queries
//   O^T += V^T P^T   A = 16 dimensions x 32 keys, read transposed from the row-major tile, B = P^T: S^T's accumulator layout
//                    already, with keys 4 g .. +3 and 16 + 4 g .. +3 in lane group g
// and the probabilities' sums as one more product with ones, from the rounded values that the value product takes (rounded to
// the type as that product's operand, so what is divided by is the sum of what was taken).
// Bound by the read of keys and values: 64 sequences of 4000 to 16000 keys, 8 kv heads, 2.67 GB in 460 us, join and all (5.8
// TB/s), 17 of 20 to 8000 63.5 us (4.7 TB/s). Small calls by latency: 1000 keys of 32 kv heads 8.9 us and 3.3 the join. Two
// blocks on a CU hold as much in flight as one with rings twice as large and hide each other's waits (with keys and values sent
// for on their own, 81 -> 66 us for the 17 sequences); three and four row tiles of 128 dimensions need the registers of both.
// With GroupArgs nothing is finished by a block: an entry's first part has a place of its own in the workspace, later ones their
// block's, and group_join_kernel adds up each row's shared keys and its own.
template <int D, int RT>
struct FewShape {
    static constexpr bool kWide = RT >= 3 && D == 128;  // too many registers for two blocks on a CU
    static constexpr int kPerCU = kWide ? 1 : 2, kBlocks = kPerCU * kCUs;
    static constexpr int kStages = kWide || D == 64 ? 2 : 1;  // tiles in a wave's ring: 16 KB, 32 where a block has the CU
};

template <int W>
struct FewMarks {
    float stat_m[W][16], stat_l[W][16];
    int tainted[2];  // a value that is not finite in a tile that the rows see in part: this (entry, kv head)'s, the next's
};

// Barriers of the waves that work together: of a whole block, or of kWaves of its waves among others. All of a block's waves
// are on their CU until the last has ended, so those that wait do not keep the others out.
struct BlockSync {
    __device__ void operator()() const { __syncthreads(); }
};
template <int kWaves_>
struct WavesSync {
    int* arrived;  // in LDS, 0 at first
    int due = 0;
    __device__ void operator()() {
        due += kWaves_;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");  // of all lanes' writes
        __builtin_amdgcn_wave_barrier();
        if ((threadIdx.x & 63) == 0) __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        while (__hip_atomic_load(arrived, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) < due) __builtin_amdgcn_s_sleep(1);
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    }
};

// What W waves do with their share, thread t of them; without shares, with `entry`.
template <typename T, int D, int RT, bool kShared, int W, int kCharge, typename Args, int kPlanned, typename Sync>
__device__ __forceinline__ void few_segments(const Args& a, const Shares& shares, int entry,
                                             uint16_t (&ring)[W][FewShape<D, RT>::kStages][2][kTile * D], const int64_t* pre,
                                             const int2* spans, const GroupPlan<kPlanned>& plan, FewMarks<W>& marks, int t, Sync sync) {
    using Shape = FewShape<D, RT>;
    constexpr bool kGroups = Args::kGroups;
    constexpr int C = D / 8;                  // 16-byte chunks of a row
    constexpr int RowsPer = 64 / C;           // rows of one DMA instruction
    constexpr int Instr = 16 / RowsPer;       // instructions for 16 rows
    constexpr int Half = 2 * Instr;           // for a tile's keys, or its values
    constexpr int S = Shape::kStages, TileElems = kTile * D;
    static_assert(sizeof(ring) >= sizeof(float) * W * 16 * D, "the rings hold the waves' sums of 16 rows");
    const int lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int c = lane & 15, g = lane >> 4;
    int64_t u = kShared ? shares.first : 0;
    int of_groups = 0;  // entries, which come first
    if constexpr (kGroups) of_groups = a.entries_of_groups();
    uint32_t voff[Instr];
#pragma unroll
    for (int j = 0; j < Instr; ++j) {
        const int row = j * RowsPer + lane / C;
        const int swz = D == 128 ? row : row >> 1;
        voff[j] = static_cast<uint32_t>(row * D * 2 + 16 * ((lane % C) ^ (swz & (C - 1))));
    }
    const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_addr(&ring[wave][0][0][0]));
    int slot = 0, turn = 0;
    while (true) {
        int kvh, first = 0, n, units = 0;
        Rows<Args> rows{};
        int64_t seg = 0;
        Tiles tiles;
        if constexpr (kShared) {
            const int64_t seg0 = pre[entry] * a.kv_heads;
            units = __builtin_amdgcn_readfirstlane(static_cast<int>(pre[entry + 1] - pre[entry]));
            kvh = __builtin_amdgcn_readfirstlane(static_cast<int>(quotient(u - seg0, units)));
            seg = seg0 + static_cast<int64_t>(kvh) * units;
            first = max(0, __builtin_amdgcn_readfirstlane(static_cast<int>(u - seg)) - kCharge);
            u = min(shares.end, seg + units);
            n = __builtin_amdgcn_readfirstlane(static_cast<int>(u - seg)) - kCharge - first;
            if (n <= 0) return;  // the share ended before its first tile
            tiles = Tiles{__builtin_amdgcn_readfirstlane(spans[entry].x), __builtin_amdgcn_readfirstlane(spans[entry].y), units - kCharge};
            if constexpr (kGroups) {
                rows.place = plan.place;
                rows.b = __builtin_amdgcn_readfirstlane(plan.lead[entry]);
                if (entry < of_groups) {
                    rows.group = __builtin_amdgcn_readfirstlane(small_quotient(entry, a.per_group_rows));
                    rows.to = __builtin_amdgcn_readfirstlane(plan.ends[rows.group]);
                } else {
                    rows.from = __builtin_amdgcn_readfirstlane(plan.from(rows.b, a.per_most));
                }
                tiles.front = rows.from / kTile;
            }
        } else {
            kvh = static_cast<int>(blockIdx.x) - entry * a.kv_heads;
            const Tiles r = tiles_of_few(a, entry, 16 * RT);
            n = __builtin_amdgcn_readfirstlane(r.count);
            tiles = Tiles{__builtin_amdgcn_readfirstlane(r.sink_tiles), __builtin_amdgcn_readfirstlane(r.window_tile), n};
        }
        const int count = tiles.count;
        if constexpr (kGroups) {
            const bool of_group = rows.group >= 0;
            rows.row0 = __builtin_amdgcn_readfirstlane(a.row_group_of(of_group ? entry : entry - of_groups, of_group)) * (16 * RT);
            rows.rows = min(16 * RT, (of_group ? a.most : 1) * a.tokens * a.groups - rows.row0);
        } else {
            rows.b = entry / a.row_groups;
            rows.row0 = (entry - rows.b * a.row_groups) * (16 * RT);
            rows.rows = min(16 * RT, a.tokens * a.groups - rows.row0);
        }

        const __attribute__((address_space(4))) int32_t* table =
            (const __attribute__((address_space(4))) int32_t*)(a.pages.table + static_cast<int64_t>(rows.b) * a.pages.table_stride);
        // the page of a table's slot, -1 where there is none (past the table's end too)
        auto page_of = [&](int slot) {
            if (slot >= a.pages.table_pages) return -1;
            const int page = table[slot];
            return page >= 0 && page < a.pages.pages ? page : -1;
        };
        // a tile's keys and values go out on their own, the next ones as soon as these have been read
        struct Places {
            int64_t at[2];  // of the halves, in elements
            int there;      // bit h: half h's page is there
        };
        auto places_of = [&](int i) {
            const int key0 = tiles.at(first + wave + W * i) * kTile;
            Places p;
            p.there = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = key0 + 16 * h, slot = __builtin_amdgcn_readfirstlane(a.pages.slot_of(key));
                const int page = __builtin_amdgcn_readfirstlane(page_of(slot));
                p.there |= page >= 0 ? 1 << h : 0;
                p.at[h] = ((static_cast<int64_t>(max(page, 0)) * a.kv_heads + kvh) * a.pages.page_size + key - slot * a.pages.page_size) * D;
            }
            return p;
        };
        auto issue = [&](const uint16_t* pool, const Places& p, int stage, int which) {
            const uint32_t lds = ring_lds + static_cast<uint32_t>((stage * 2 + which) * TileElems) * 2u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint16_t* from = uniform(pool + p.at[h]);
#pragma unroll
                for (int j = 0; j < Instr; ++j) dma16_lds(from, voff[j], lds + static_cast<uint32_t>(h * 16 * D) * 2u + 1024u * j);
            }
        };
        u32x4 qf[RT][D / 32];
        int last[RT], start[RT];
        int all_last = INT32_MAX, all_start = 0;  // what every row sees
        auto fetch_queries = [&] {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const RowAt row = rows.at(a, min(16 * rt + c, rows.rows - 1));
                last[rt] = 16 * rt + c < rows.rows ? row.last : -1;
                start[rt] = a.window > 0 ? max(0, row.position - a.window + 1) : 0;
                if (last[rt] >= 0) {
                    all_last = min(all_last, last[rt]);
                    all_start = max(all_start, start[rt]);
                }
                const uint16_t* src = a.q + row.q_row * a.q_stride + static_cast<int64_t>(kvh * a.groups + row.head) * D + 8 * g;
#pragma unroll
                for (int kt = 0; kt < D / 32; ++kt) qf[rt][kt] = *vec(src + 32 * kt);
            }
        };
        // loads come back in the order in which they went out: of a group, where the rows lie is loaded before the queries are,
        // and the tiles would have to come first
        if constexpr (kGroups) fetch_queries();
        const int mine = n > wave ? (n - wave + W - 1) / W : 0;
        int there[S] = {};  // of the tiles that are out, the oldest first
#pragma unroll
        for (int st = 0; st < S; ++st)
            if (st < mine) {
                const Places p = places_of(st);
                there[st] = p.there;
                issue(a.k_pages, p, st, 0);
                issue(a.v_pages, p, st, 1);
            }

        if constexpr (!kGroups) fetch_queries();
        all_last = least_of<16>(all_last);
        all_start = largest_of<16>(all_start);

        f32x4 o[RT][D / 16], lsum[RT];
        float m[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY;
            lsum[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

        // waits until the oldest outstanding part (a tile's keys, or values) has come, `behind` parts having gone out since
        auto wait_part = [&](int behind) {
            if (behind >= 3) wait_vmcnt<(S == 2 ? 3 : 1) * Half>();
            else if (behind == 2) wait_vmcnt<(S == 2 ? 2 : 1) * Half>();
            else if (behind == 1) wait_vmcnt<Half>();
            else wait_vmcnt<0>();
            asm volatile("" ::: "memory");
        };
        auto reads_ended = [] { __builtin_amdgcn_s_waitcnt(0xF | (0x3 << 14) | (0x7 << 4)); };  // lgkmcnt 0
        for (int i = 0; i < mine; ++i) {
            const int stage = S == 1 ? 0 : i & 1, ahead = min(mine - 1 - i, S - 1);  // tiles out behind this one
            const uint16_t* kb = ring[wave][stage][0];
            const uint16_t* vb = ring[wave][stage][1];
            const int key0 = tiles.at(first + wave + W * i) * kTile;
            const bool more = i + S < mine;
            Places next{};
            if (more) next = places_of(i + S);
            wait_part(1 + 2 * ahead);
            u32x4 kf[2][D / 32];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int kt = 0; kt < D / 32; ++kt) {
                    const int swz = D == 128 ? c : c >> 1;
                    kf[h][kt] = *vec(kb + (16 * h + c) * D + 8 * ((4 * kt + g) ^ (swz & (C - 1))));
                }
            if (more) {
                reads_ended();
                issue(a.k_pages, next, stage, 0);
            }
            const bool whole = there[0] == 3 && key0 + kTile - 1 <= all_last &&
                               (key0 >= all_start || key0 + kTile <= a.sinks) && rows.holds_tile(key0);
            const uint32_t pages_there = ((there[0] & 1 ? 0xFFFFu : 0u) | (there[0] & 2 ? 0xFFFF0000u : 0u)) & rows.held_bits(key0);
            uint32_t some = 0;  // seen by some row of the wave's
            u32x4 pf[RT];
            f32x4 s[RT][2];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int h = 0; h < 2; ++h) s[rt][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kt = 0; kt < D / 32; ++kt)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) s[rt][h] = mfma16x16x32<T>(kf[h][kt], qf[rt][kt], s[rt][h]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int h = 0; h < 2; ++h) s[rt][h] *= a.scale;
            if (!whole) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    // the lane's key 16 h + 4 g + e in bit 16 h + e
                    const uint32_t seen = (seen_bits(key0, last[rt], start[rt], a.sinks) & pages_there) >> (4 * g);
                    some |= seen;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[rt][h][e] = or_minus_inf(s[rt][h][e], seen, 16 * h + e);
                }
            }
            // the reference point of the exponentials follows the running maximum only once that is 8 above it: exponentials
            // up to 2^8 round the same, and most tiles rescale nothing
            float top[RT];
            bool grows = false;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                top[rt] = fmaxf(fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), fmaxf(s[rt][0][2], s[rt][0][3])),
                                fmaxf(fmaxf(s[rt][1][0], s[rt][1][1]), fmaxf(s[rt][1][2], s[rt][1][3])));
                top[rt] = max_xor32(max_xor16(top[rt]));  // the lane groups that hold a column
                grows |= top[rt] > m[rt] + kSlack;
            }
            if (__any(grows)) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const float mn = fmaxf(m[rt], top[rt]);
                    const float keep = __builtin_amdgcn_exp2f(m[rt] - (mn == -INFINITY ? 0.0f : mn));
                    m[rt] = mn;
                    lsum[rt] *= keep;
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] *= keep;
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float mu = m[rt] == -INFINITY ? 0.0f : m[rt];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[rt][h][e] = __builtin_amdgcn_exp2f(s[rt][h][e] - mu);
                    pf[rt][2 * h] = pack2<T>(s[rt][h][0], s[rt][h][1]);
                    pf[rt][2 * h + 1] = pack2<T>(s[rt][h][2], s[rt][h][3]);
                }
                lsum[rt] = mfma16x16x32<T>(u32x4{T::ONE_PAIR, T::ONE_PAIR, T::ONE_PAIR, T::ONE_PAIR}, pf[rt], lsum[rt]);
            }
            const int vr = 4 * g + (c >> 2);  // of 16: the row whose address the lane gives
            auto read_v = [&](int dt) {
                const int swz = D == 128 ? vr : vr >> 1;
                const int at = 8 * ((2 * dt + ((c >> 1) & 1)) ^ (swz & (C - 1))) + 4 * (c & 1);
                const uint2 lo = read_transposed(vb + vr * D + at), hi = read_transposed(vb + (16 + vr) * D + at);
                return u32x4{lo.x, lo.y, hi.x, hi.y};
            };
            u32x4 keep;
            if (!whole) {
                some = or_row16(some);
#pragma unroll
                for (int w = 0; w < 4; ++w) keep[w] = pair_mask(some, 16 * (w >> 1) + 2 * (w & 1));
            }
            float zero = 0.0f;
            constexpr int kAhead = 4;  // dimension tiles read together
            wait_part(2 * ahead + more);
#pragma unroll
            for (int d0 = 0; d0 < D / 16; d0 += kAhead) {
                u32x4 vf[kAhead];
#pragma unroll
                for (int e = 0; e < kAhead; ++e) vf[e] = read_v(d0 + e);
                if (!whole) {  // values that no row sees are cleared: rows behind a sequence's last, pages that are not there
#pragma unroll
                    for (int e = 0; e < kAhead; ++e)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            vf[e][w] &= keep[w];
                            zero = T::dot2(vf[e][w], 0u, zero);  // NaN where one is not finite
                        }
                }
#pragma unroll
                for (int e = 0; e < kAhead; ++e)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) o[rt][d0 + e] = mfma16x16x32<T>(vf[e], pf[rt], o[rt][d0 + e]);
            }
            if (zero != zero) marks.tainted[turn] = 1;
            if (more) {
                reads_ended();
                issue(a.v_pages, next, stage, 1);
            }
#pragma unroll
            for (int st = 0; st + 1 < S; ++st) there[st] = there[st + 1];
            there[S - 1] = next.there;
        }

        // the waves' sums, joined through the rings a row group at a time
        const bool done = !kGroups && first == 0 && n == count;
        int64_t part;
        if constexpr (kGroups) part = first == 0 ? a.first_part(entry, kvh) : a.later_part(entry, shares.block);
        else part = (static_cast<int64_t>(shares.block) * 2 + slot) * a.rows_kept;
        float* red = reinterpret_cast<float*>(&ring[0][0][0][0]);
        sync();
        const bool tainted = marks.tainted[turn] != 0;
        if (tainted) slow_rows<T, D>(a, rows, kvh, tiles, kTile, first, n, done, part, wave, W);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (tainted) break;
            if (rt > 0) sync();
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt)
                *reinterpret_cast<f32x4*>(red + (wave * 16 + c) * D + 4 * ((4 * dt + g) ^ c)) = o[rt][dt];
            if (g == 0) {  // a row of padding took part where the tile was whole: its sums are none
                marks.stat_m[wave][c] = last[rt] < 0 ? -INFINITY : m[rt];
                marks.stat_l[wave][c] = last[rt] < 0 ? 0.0f : lsum[rt][0];
            }
            sync();
            for (int id = t; id < 16 * C; id += 64 * W) {
                const int row = id / C, ch = id % C;
                if (16 * rt + row >= rows.rows) continue;
                float M = marks.stat_m[0][row];
#pragma unroll
                for (int w = 1; w < W; ++w) M = fmaxf(M, marks.stat_m[w][row]);
                const float mu = M == -INFINITY ? 0.0f : M;
                float L = 0.0f;
                f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    if (marks.stat_l[w][row] == 0.0f) continue;
                    const float f = __builtin_amdgcn_exp2f(marks.stat_m[w][row] - mu);
                    L += f * marks.stat_l[w][row];
                    lo += f * *reinterpret_cast<const f32x4*>(red + (w * 16 + row) * D + 4 * ((2 * ch) ^ row));
                    hi += f * *reinterpret_cast<const f32x4*>(red + (w * 16 + row) * D + 4 * ((2 * ch + 1) ^ row));
                }
                const int r = rows.row0 + 16 * rt + row;
                if (done) {
                    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                    *reinterpret_cast<u32x4*>(a.out + out_row(a, rows.b, kvh, r) * D + 8 * ch) =
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
        if constexpr (!kShared) return;
        if (first == 0 && t == 0)
            a.desc[entry * a.kv_heads + kvh] = int2{shares.block * 2 + slot, shares.block_of(seg + units - 1)};
        if (u >= shares.end) return;
        slot = 1;  // a share's first and last (entry, kv head) are the ones that it may not finish
        if (kvh + 1 == a.kv_heads) {
            ++entry;
            if constexpr (kGroups)
                while (pre[entry + 1] == pre[entry]) ++entry;  // nobody's; another one holds the unit u
        }
        if (t == 0) marks.tainted[turn ^ 1] = 0;
        turn ^= 1;
        sync();
    }
}

template <typename T, int D, int RT, bool kShared, typename Args = PagedArgs>
__global__ __launch_bounds__(64 * kWaves, (FewShape<D, RT>::kPerCU)) void few_kernel(const Args a) {
    using Shape = FewShape<D, RT>;
    constexpr bool kGroups = Args::kGroups;
    constexpr int kEntries = kShared ? kFewEntries : 0;
    static_assert(kShared || !kGroups, "entries with groups are shared out");
    __shared__ __attribute__((aligned(16))) uint16_t ring[kWaves][Shape::kStages][2][kTile * D];
    __shared__ int64_t pre[kEntries + 1];
    __shared__ int2 own_spans[kShared && !kGroups ? kEntries : 1];  // {sink_tiles, window_tile}
    __shared__ GroupPlan<kGroups ? kEntries : 1> plan;
    __shared__ int64_t wave_total[kWaves];
    __shared__ FewMarks<kWaves> marks;
    __shared__ int s_entry;
    if (threadIdx.x < 2) marks.tainted[threadIdx.x] = 0;
    Shares shares{};
    int entry;
    if constexpr (kShared) {
        int entries = a.batch * a.row_groups;
        if constexpr (kGroups) {
            plan_groups<64 * kWaves>(a, plan);
            entries += a.entries_of_groups();
        }
        using Sum = std::conditional_t<kGroups, int, double>;
        shares = make_shares<64 * kWaves, Shape::kBlocks, Sum>(a, entries, kLeastShare, pre, wave_total, &s_entry, [&](int e) {
            if constexpr (kGroups) {
                const int n = tiles_of_plan(a, plan, e, kTileShift);
                return n == 0 ? 0 : n + kFewStart;
            } else {
                const Tiles r = tiles_of_few(a, e, 16 * RT);
                own_spans[e] = int2{r.sink_tiles, r.window_tile};
                return r.count + kFewStart;
            }
        });
        if (shares.entry < 0) return;
        entry = shares.entry;
    } else {
        entry = static_cast<int>(blockIdx.x) / a.kv_heads;
        __syncthreads();  // the marks are cleared before any wave sets one (make_shares has barriers of its own)
    }
    const int2* spans = own_spans;
    if constexpr (kGroups) spans = plan.spans;
    few_segments<T, D, RT, kShared, kWaves, kFewStart>(a, shares, entry, ring, pre, spans, plan, marks,
                                                       static_cast<int>(threadIdx.x), BlockSync{});
}

}  // namespace
}  // namespace nq
