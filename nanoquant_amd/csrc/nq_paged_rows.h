// Attention of many rows per sequence over the pages of a cache: rows_kernel and what it needs.
#pragma once

#include <type_traits>

#include "nq_paged_few.h"

namespace nq {
namespace {

constexpr int kKeysShift = 6, kKeys = 1 << kKeysShift;  // keys of a tile

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
// 319 us (848 TFLOP/s, where a large matrix product runs at 1345): of a tile's 5500 cycles 2050 are products, 2000 vector
// instructions, of which about half overlap, 1100 waits for LDS and barriers, 480 scalar instructions. A prompt of 1000 tokens,
// 32 heads, RW 1: 25.3 us, of which the longest row group's 16 tiles take 16.
// kShared: the work of all row groups in equal shares over the grid, as few_kernel's; otherwise a block takes a row group,
// the last ones (the longest of a prompt) first.
// With GroupArgs: the entries of groups only, each over the keys that its members share; every part goes to the workspace.
template <int D>
struct RowsRings {
    uint16_t k[4][kKeys * D], v[4][kKeys * D];
};
struct RowsMarks {
    int spans[2][4];
    int tainted[2];  // as few_kernel's
};

// What a block does with its share; without shares, with `entry`.
template <typename T, int D, int RW, bool kShared, int kCharge, typename Args, int kPlanned>
__device__ __forceinline__ void rows_segments(const Args& a, const Shares& shares, int entry, RowsRings<D>& rings, const int64_t* pre,
                                              const GroupPlan<kPlanned>& plan, RowsMarks& marks) {
    constexpr bool kGroups = Args::kGroups;
    constexpr int C = D / 8;             // 16-byte chunks of a row
    constexpr int RowsPer = 64 / C;      // rows of one DMA instruction
    constexpr int Instr = 16 / RowsPer;  // instructions for 16 rows
    constexpr int Group = 128 * RW;
    constexpr int KT = D / 16, DT = D / 32, KG = KT / 2;
    constexpr int TileElems = kKeys * D, kStep = RW == 1 ? 2 : 1;  // tiles from one of a wave's to its next
    auto& kring = rings.k;
    auto& vring = rings.v;
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int rwave = wave & 3, grp = wave >> 2;  // its rows, and of the two halves of RW 1
    const int c = lane & 31, kg = lane >> 5;
    int slot = 0, turn = 0;
    int64_t u = kShared ? shares.first : 0;

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
        // row 0 is the first of all row groups here
        Rows<Args> rows{};
        int row0;
        if constexpr (kGroups) {
            rows.b = __builtin_amdgcn_readfirstlane(plan.lead[entry]);
            rows.group = __builtin_amdgcn_readfirstlane(small_quotient(entry, a.per_group_rows));
            rows.place = plan.place;
            rows.to = __builtin_amdgcn_readfirstlane(plan.ends[rows.group]);
            rows.rows = a.most * a.tokens * a.groups;
            row0 = (entry - rows.group * a.group_rows) * Group;
        } else {
            rows.b = entry / a.row_groups;
            rows.rows = a.tokens * a.groups;
            row0 = (entry - rows.b * a.row_groups) * Group;
        }
        const int group0 = row0;
        row0 += rwave * (32 * RW);
        int kvh, first = 0, n, count, units = 0;
        int64_t seg = 0;
        Tiles tiles;
        if constexpr (kShared) {
            const int64_t seg0 = pre[entry] * a.kv_heads;
            units = __builtin_amdgcn_readfirstlane(static_cast<int>(pre[entry + 1] - pre[entry]));
            int charge = kCharge;
            if constexpr (kGroups) charge += __builtin_amdgcn_readfirstlane(static_cast<int>(plan.slow[entry]));
            count = units - charge;
            kvh = __builtin_amdgcn_readfirstlane(static_cast<int>(quotient(u - seg0, units)));
            seg = seg0 + static_cast<int64_t>(kvh) * units;
            first = max(0, __builtin_amdgcn_readfirstlane(static_cast<int>(u - seg)) - charge);
            u = min(shares.end, seg + units);
            n = __builtin_amdgcn_readfirstlane(static_cast<int>(u - seg)) - charge - first;
            if (n <= 0) return;  // the share ended before its first tile
            if constexpr (kGroups) {
                tiles = Tiles{__builtin_amdgcn_readfirstlane(plan.spans[entry].x), __builtin_amdgcn_readfirstlane(plan.spans[entry].y), count};
            } else {
                const int4 sp = a.spans[entry];
                tiles = Tiles{__builtin_amdgcn_readfirstlane(sp.x), __builtin_amdgcn_readfirstlane(sp.y), sp.z};
            }
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
                const int at = a.pages.slot_of(key + 16 * i);
                const int page = at < a.pages.table_pages ? a.pages.page(rows.b, at) : -1;
                my_there |= page >= 0 ? 1 << i : 0;
                if (i == rwave) {
                    my_page = max(page, 0);
                    my_rest = key + 16 * i - at * a.pages.page_size;
                }
            }
        };
        auto place = [&](int it) {
            if ((it & 63) < kStep && !(kGroups && it < kStep)) look_up(it & ~63);
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
        // loads come back in the order in which they went out: of a group, where the rows lie is loaded before the queries are,
        // and the tiles would have to come first; and the pages are looked up before
        if constexpr (kGroups) look_up(0);
        else if constexpr (kShared) begin();  // while the queries come

        u32x4 qf[RW][KT];
        int last[RW], start[RW];
        int lo = INT32_MAX, hi = -1, all_start = 0, any_of = INT32_MAX;
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u, keep_q = a.scale == 0.0f ? 0u : 0xFFFFFFFFu;
#pragma unroll
        for (int rw = 0; rw < RW; ++rw) {
            const RowAt row = rows.at(a, min(row0 + 32 * rw + c, rows.rows - 1));
            last[rw] = row0 + 32 * rw + c < rows.rows ? row.last : -1;
            start[rw] = a.window > 0 ? max(0, row.position - a.window + 1) : 0;
            if (last[rw] >= 0) {
                lo = min(lo, last[rw]);
                all_start = max(all_start, start[rw]);
                any_of = min(any_of, start[rw]);
            }
            hi = max(hi, last[rw]);
            const uint16_t* src = a.q + row.q_row * a.q_stride + static_cast<int64_t>(kvh * a.groups + row.head) * D + 8 * kg;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) qf[rw][kt] = *vec(src + 16 * kt);
        }
        if constexpr (kGroups) begin();
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
        int any_start = a.window > 0 ? max(0, lo == INT32_MAX ? 0 : lo - a.window + 1) : 0;  // the first key of some row
        if constexpr (kGroups) any_start = least_of<32>(any_of);  // lo is no position where the shared keys end before
        if constexpr (!kShared) {
            if (lane == 0) {
                marks.spans[0][rwave] = lo;
                marks.spans[1][rwave] = hi;
            }
            __syncthreads();
            int blo = INT32_MAX, bhi = -1;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                blo = min(blo, marks.spans[0][w]);
                bhi = max(bhi, marks.spans[1][w]);
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
                some = or_half32(some);
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
            if (zero != zero) marks.tainted[turn] = 1;
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

        const bool done = !kGroups && first == 0 && n == count;
        __syncthreads();
        const bool tainted = marks.tainted[turn] != 0;
        int64_t parts;
        if constexpr (kGroups) parts = first == 0 ? a.first_part(entry, kvh) : a.later_part(entry, shares.block);
        else parts = (static_cast<int64_t>(shares.block) * 2 + slot) * a.rows_kept;
        if (tainted) {
            Rows<Args> these = rows;
            these.row0 = group0;
            these.rows = min(Group, rows.rows - group0);
            slow_rows<T, D>(a, these, kvh, tiles, kKeys, first, n, done, parts, wave, static_cast<int>(blockDim.x) >> 6);
        }
        // the halves' sums: either wave of two with the same rows joins half of the dimensions, and has those of the other's from
        // the key ring, the statistics from the value ring's first 4 KB
        constexpr int DH = RW == 1 ? DT / 2 : DT, Cols = 32 * DH;  // of a wave
        const int col0 = RW == 1 ? grp * Cols : 0;
        f32x16 sums[RW][DH];
        int at_lane = lane;  // whose places are worked out here: kept through the loop, they would take its registers
        asm volatile("" : "+v"(at_lane));
        const int ec = at_lane & 31, ekg = at_lane >> 5;
        float* stage = reinterpret_cast<float*>(&kring[0][0]) + wave * (32 * Cols);  // of 32 rows
        static_assert(sizeof(kring) >= (RW == 1 ? 8 : 4) * 32 * Cols * sizeof(float), "the key ring holds all waves' sums of 32 rows");
        if constexpr (RW == 1) {
            if (!tainted) {
                float* theirs = reinterpret_cast<float*>(&kring[0][0]) + (wave ^ 4) * (32 * Cols) + at_lane;
                float* stat = reinterpret_cast<float*>(&vring[0][0]) + 64 * rwave + at_lane;
#pragma unroll
                for (int dt = 0; dt < DH; ++dt) {
                    if (grp == 0) {
                        sums[0][dt] = o[0][dt];
#pragma unroll
                        for (int i = 0; i < 16; ++i) theirs[(16 * dt + i) * 64] = o[0][DH + dt][i];
                    } else {
                        sums[0][dt] = o[0][DH + dt];
#pragma unroll
                        for (int i = 0; i < 16; ++i) theirs[(16 * dt + i) * 64] = o[0][dt][i];
                    }
                }
                stat[512 * grp] = m[0];
                stat[512 * grp + 256] = l[0];
                __syncthreads();
                const float m0 = stat[0], m1 = stat[512], mn = fmaxf(m0, m1);
                const float mu = mn == -INFINITY ? 0.0f : mn;
                const float f0 = __builtin_amdgcn_exp2f(m0 - mu), f1 = __builtin_amdgcn_exp2f(m1 - mu);
                m[0] = mn;
                l[0] = stat[256] * f0 + stat[768] * f1;
#pragma unroll
                for (int dt = 0; dt < DH; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float mine = sums[0][dt][i], other = stage[(16 * dt + i) * 64 + at_lane];
                        sums[0][dt][i] = (grp == 0 ? mine : other) * f0 + (grp == 0 ? other : mine) * f1;
                    }
            }
        } else {
#pragma unroll
            for (int rw = 0; rw < RW; ++rw)
#pragma unroll
                for (int dt = 0; dt < DH; ++dt) sums[rw][dt] = o[rw][dt];
        }
        // a wave's rows through LDS, a row tile at a time, then whole rows to memory
        constexpr int OC = Cols / 8, FC = Cols / 4;  // 16-byte chunks of a row, in the type and in fp32
        uint16_t* ob = (RW == 1 ? &vring[0][0] + 2048 : &kring[0][0]) + wave * (32 * Cols);
        if (!tainted) {
#pragma unroll
            for (int rw = 0; rw < RW; ++rw) {
                float L = l[rw] + __shfl_xor(l[rw], 32, 64);
                float M = m[rw];
                if (last[rw] < 0) {  // padding took part where the tile was whole
                    L = 0.0f;
                    M = -INFINITY;
                }
                const float inv = 1.0f / L;
                wave_handover();
                if (kShared && !done) {
                    const int64_t part = parts + rwave * (32 * RW) + 32 * rw;
                    if (ekg == 0 && col0 == 0 && row0 + 32 * rw + ec < rows.rows) a.part_ml[part + ec] = float2{M, L};
#pragma unroll
                    for (int dt = 0; dt < DH; ++dt)
#pragma unroll
                        for (int g4 = 0; g4 < 4; ++g4) {
                            f32x4 x;
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] = L == 0.0f ? 0.0f : sums[rw][dt][4 * g4 + e];
                            *reinterpret_cast<f32x4*>(stage + ec * Cols + 4 * ((8 * dt + 2 * g4 + ekg) ^ (ec & (FC - 1)))) = x;
                        }
                    wave_handover();
#pragma unroll
                    for (int j = 0; j < FC / 2; ++j) {
                        const int r = (64 * j + at_lane) / FC, ch = at_lane % FC;
                        const f32x4 x = *reinterpret_cast<const f32x4*>(stage + r * Cols + 4 * (ch ^ (r & (FC - 1))));
                        if (row0 + 32 * rw + r < rows.rows) *reinterpret_cast<f32x4*>(a.part_o + (part + r) * D + col0 + 4 * ch) = x;
                    }
                    continue;
                }
#pragma unroll
                for (int dt = 0; dt < DH; ++dt)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) {
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = L == 0.0f ? 0.0f : sums[rw][dt][4 * g4 + e] * inv;
                        *reinterpret_cast<uint2*>(ob + ec * Cols + 8 * ((4 * dt + g4) ^ (ec & (OC - 1))) + 4 * ekg) =
                            uint2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
                    }
                wave_handover();
#pragma unroll
                for (int j = 0; j < OC / 2; ++j) {
                    const int r = (64 * j + at_lane) / OC, ch = at_lane % OC;
                    const u32x4 v = *vec(ob + r * Cols + 8 * (ch ^ (r & (OC - 1))));
                    const int at_row = row0 + 32 * rw + r;
                    if (at_row < rows.rows)
                        *reinterpret_cast<u32x4*>(a.out + out_row(a, rows.b, kvh, at_row) * D + col0 + 8 * ch) = v;
                }
            }
        }
        if constexpr (!kShared) return;
        if (first == 0 && t == 0)
            a.desc[entry * a.kv_heads + kvh] =
                int2{shares.block * 2 + slot, shares.block_of(seg + units - 1)};
        if (u >= shares.end) return;
        slot = 1;
        if (kvh + 1 == a.kv_heads) {
            ++entry;
            if constexpr (kGroups)
                while (pre[entry + 1] == pre[entry]) ++entry;  // nobody's; another one holds the unit u
        }
        if (t == 0) marks.tainted[turn ^ 1] = 0;
        turn ^= 1;
        __syncthreads();
    }
}

template <typename T, int D, int RW, bool kShared>
__global__ __launch_bounds__(RW == 1 ? 512 : 256, RW == 1 ? 2 : 1) void rows_kernel(const PagedArgs a) {
    constexpr int NW = RW == 1 ? 8 : 4;  // waves
    __shared__ __attribute__((aligned(16))) RowsRings<D> rings;
    __shared__ RowsMarks marks;
    __shared__ int64_t pre[kShared ? kEntries + 1 : 1];
    __shared__ int64_t wave_total[NW];
    __shared__ int s_entry;
    __shared__ GroupPlan<1> plan;
    if (threadIdx.x < 2) marks.tainted[threadIdx.x] = 0;
    Shares shares{};
    int entry;
    if constexpr (kShared) {
        shares = make_shares<64 * NW, kCUs, double>(a, a.batch * a.row_groups, kLeastTiles, pre, wave_total, &s_entry,
                                            [&](int e) { return a.spans[e].z + kStart; });
        if (shares.entry < 0) return;
        entry = shares.entry;
    } else {
        const int order = static_cast<int>(blockIdx.x) / (a.batch * a.kv_heads);
        const int rest = static_cast<int>(blockIdx.x) - order * a.batch * a.kv_heads;
        entry = rest / a.kv_heads * a.row_groups + a.row_groups - 1 - order;
    }
    rows_segments<T, D, RW, kShared, kStart>(a, shares, entry, rings, pre, plan, marks);
}

}  // namespace
}  // namespace nq
