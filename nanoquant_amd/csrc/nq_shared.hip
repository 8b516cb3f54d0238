// Attention over the pages of a cache of which groups of sequences have the leading ones in common.
#include <algorithm>
#include <cmath>

#include "nq_common.h"
#include "nq_paged_few.h"
#include "nq_paged_rows.h"

namespace nq {
namespace {

// Adds up what few_kernel or shared_kernel left of a row: the parts of its group's shared keys and of its sequence's own. A wave
// a row, D / 4 lanes a part. Bound by its chain of loads (the sequence's place, its entries' blocks, their parts): 3.9 us for 128
// rows, 7.0 for 8192 of 128 dimensions, with several parts a row on their way at once (with half or twice as many 3 us more).
template <typename T, int D>
__global__ __launch_bounds__(256) void group_join_kernel(const GroupArgs a, uint32_t count) {
    constexpr int L4 = D / 4, Groups = 64 / L4, kAhead = 4;
    const int lane = threadIdx.x & 63;
    const uint32_t row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));  // (sequence, token, head)
    if (row >= count) return;
    const int token = static_cast<int>(row / static_cast<uint32_t>(a.heads));
    const int head = static_cast<int>(row) - token * a.heads;
    const int kvh = __builtin_amdgcn_readfirstlane(small_quotient(head, a.per_groups));
    const int b = __builtin_amdgcn_readfirstlane(small_quotient(token, a.per_tokens));
    const int r = (token - b * a.tokens) * a.groups + head - kvh * a.groups;
    const int at = a.place[b];
    struct Parts {
        int64_t first, later;  // rows of the first part and, were it one of the later ones, of the first block's
        int n, step;
    };
    auto parts_of = [&](int entry, int in_entry) {
        const int2 d = a.desc[entry * a.kv_heads + kvh];
        return Parts{a.first_part(entry, kvh) + in_entry, a.later_part(entry, d.x >> 1) + in_entry, d.y - (d.x >> 1) + 1,
                     entry < a.entries_of_groups() ? a.group_tile : a.own_tile};
    };
    Parts common{0, 0, 0, 0};
    if (at >= 0) {
        const int g = small_quotient(at, a.per_most), in_group = (at - g * a.most) * a.tokens * a.groups + r;
        common = parts_of(g * a.group_rows + (in_group >> a.group_shift), in_group & (a.group_tile - 1));
    }
    const Parts own = parts_of(a.entries_of_groups() + b * a.row_groups + (r >> a.own_shift), r & (a.own_tile - 1));
    const int n = common.n + own.n, grp = lane / L4, d0 = 4 * (lane % L4);
    float M = -INFINITY, L = 0.0f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = grp; i0 < n; i0 += kAhead * Groups) {
        float2 ml[kAhead];
        f32x4 x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {  // those past the last read it again
            const int part = min(i0 + i * Groups, n - 1);
            const bool of_common = part < common.n;
            const int k = of_common ? part : part - common.n;
            const int64_t later = (of_common ? common.later : own.later) + static_cast<int64_t>(k) * (of_common ? common.step : own.step);
            const int64_t from = k == 0 ? (of_common ? common.first : own.first) : later;
            ml[i] = a.part_ml[from];
            x[i] = *reinterpret_cast<const f32x4*>(a.part_o + from * D + d0);
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
            const bool in = i0 + i * Groups < n;
            L = in ? fmaf(f, ml[i].y, L) : L;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = in ? fmaf(f, x[i][e], o[e]) : o[e];
        }
    }
#pragma unroll
    for (int off = L4; off < 64; off <<= 1) {
        const float other = __shfl_xor(M, off, 64), top = fmaxf(M, other);
        const float mu = top == -INFINITY ? 0.0f : top;
        const float f0 = __builtin_amdgcn_exp2f(M - mu), f1 = __builtin_amdgcn_exp2f(other - mu);
        L = f0 * L + f1 * __shfl_xor(L, off, 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = f0 * o[e] + f1 * __shfl_xor(o[e], off, 64);
        M = top;
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (grp == 0)
        *reinterpret_cast<uint2*>(a.out + static_cast<int64_t>(row) * D + d0) =
            uint2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
}

// Groups of more than 32 rows: some of the blocks take their entries as rows_kernel does, the others the sequences' as
// few_kernel does, a team of two waves each, in equal shares; all of them work out the same list. One launch, since the
// sequences' part is bound by the read of keys and values and the groups' by products: in two launches, each on all CUs, 16
// sequences with 8000 shared keys 47 us against 36, 60 conversations 179 against 152, 128 samples under a window 221 against
// 161. Now, of 64 heads of 8 kv heads: 16 sequences with 8000 shared keys and 20 to 700 of their own 23 us, bound by latency
// (the list, the first tiles' way, the waves' join); 60 in five groups with 100 to 4000 of their own 146, bound by the read
// (5.0 TB/s, a large copy's rate); 128 under a window of 12011 keys 137 to 145, bound by rows_segments' products and exponentials, of
// which the tiles in which windows begin take twice. 11 sequences of 5 tokens, heads of 64, 5000 shared keys: 21 us. How many
// blocks either gets goes by what a unit takes of a CU, in ns: a tile of 64 keys and 128 rows, or one of 32 keys; and by how
// much longer the groups' blocks take for their beginning and their end.
constexpr float kGroupTime = 1200.0f, kGroupTime64 = 700.0f, kOwnTime = 400.0f, kOwnTime64 = 350.0f, kGroupMore = 4000.0f;
constexpr int kGroupStart = 8, kOwnStart = 4;  // what a segment costs on top of its tiles, in tiles
constexpr int kGroupTile = 128;
constexpr int kTeams = 4;  // of a block's waves, for sequences' own keys: 40 samples of a prompt, 32 kv heads, 48.0 us, two teams 49.8
constexpr int kLeastGroupTiles = 6;  // of a block's share, starts among them

// Blocks of kCUs for groups' work such that both parts end together, of the numbers 4 lane + 2.
template <int D>
__device__ inline int blocks_for_groups(int64_t group_units, int64_t own_units) {
    if (group_units == 0) return 0;
    const int n = 4 * (static_cast<int>(threadIdx.x) & 63) + 2;
    const float group_time = D == 128 ? kGroupTime : kGroupTime64, own_time = D == 128 ? kOwnTime : kOwnTime64;
    const float g = static_cast<float>(group_units) * group_time * __builtin_amdgcn_rcpf(static_cast<float>(n));
    const float s = static_cast<float>(own_units) * own_time * __builtin_amdgcn_rcpf(static_cast<float>(kCUs - n));
    const int late = __popcll(__ballot(g + kGroupMore > s));  // the lanes at which the groups' part ends last: the first ones
    return min(4 * late + 2, kCUs - 2);
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(512, 2) void shared_kernel(const GroupArgs a) {
    constexpr int kThreads = 512, W = kThreads / 64 / kTeams;  // waves of a team
    __shared__ __attribute__((aligned(16))) union {
        uint16_t few[kTeams][W][FewShape<D, RT>::kStages][2][kTile * D];
        RowsRings<D> rows;
    } rings;
    __shared__ int64_t pre[kEntries + 1];
    __shared__ GroupPlan<kEntries> plan;
    __shared__ int64_t wave_total[kThreads / 64];
    __shared__ union {
        FewMarks<W> few[kTeams];
        RowsMarks rows;
    } marks;
    __shared__ int first_entry[kTeams], arrived[kTeams];
    const int of_groups = a.entries_of_groups(), entries = of_groups + a.batch * a.row_groups;
    plan_groups<kThreads>(a, plan);
    prefix_sums<kThreads, int>(entries, pre, wave_total, [&](int e) {
        const int n = tiles_of_plan(a, plan, e, e < of_groups ? kKeysShift : kTileShift);
        // a tile that is masked takes twice as long
        return n == 0 ? 0 : e < of_groups ? n + kGroupStart + plan.slow[e] : n + kOwnStart;
    });
    const int block = static_cast<int>(blockIdx.x);
    const int for_groups = blocks_for_groups<D>(pre[of_groups] * a.kv_heads, (pre[entries] - pre[of_groups]) * a.kv_heads);
    if (block < for_groups) {
        if (threadIdx.x < 2) marks.rows.tainted[threadIdx.x] = 0;
        const Shares shares = take_share<kThreads>(a, 0, of_groups, block, for_groups, kLeastGroupTiles, pre, first_entry);
        if (shares.entry >= 0) rows_segments<T, D, 1, true, kGroupStart>(a, shares, shares.entry, rings.rows, pre, plan, marks.rows);
    } else {
        // the teams of the block go their own ways, so that one's first tiles come and its waves' sums are joined among the
        // others' products
        const int team = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / (64 * W)), at = kTeams * (block - for_groups);
        if (threadIdx.x < 2 * kTeams) marks.few[threadIdx.x >> 1].tainted[threadIdx.x & 1] = 0;
        if (threadIdx.x < kTeams) arrived[threadIdx.x] = 0;
        Shares shares = share_of(a, of_groups, entries, at + team, kTeams * (kCUs - for_groups), W, pre);
        const int64_t first = shares.first - team * shares.share;  // the block's first unit
        for (int e = of_groups + static_cast<int>(threadIdx.x); e < entries; e += kThreads)
#pragma unroll
            for (int i = 0; i < kTeams; ++i)
                if (holds_unit(a, pre, e, first + i * shares.share)) first_entry[i] = e;
        __syncthreads();
        if (shares.first >= shares.end) return;
        shares.entry = __builtin_amdgcn_readfirstlane(first_entry[team]);
        few_segments<T, D, RT, true, W, kOwnStart>(a, shares, shares.entry, rings.few[team], pre, plan.spans, plan, marks.few[team],
                                                   static_cast<int>(threadIdx.x) % (64 * W), WavesSync<W>{&arrived[team]});
    }
}

// What a call's launch lists, and what it needs of the workspace; tiles 0: a call for the plain attention.
struct Plan {
    int tiles = 0;      // of 16 rows a wave
    bool apart;         // shared_kernel, else few_kernel takes the groups' entries too
    int64_t group_rows, row_groups, group_tile, own_tile, group_kept, rows_kept;
    int64_t own_first, group_later, own_later;  // rows of parts
    size_t part_o, part_ml, desc, place, bytes;
};

Plan make_plan(int64_t batch, int64_t tokens, int64_t groups, int64_t kv_heads, int64_t head_dim, int64_t keys, int64_t sharing,
               int64_t most) {
    Plan p{};
    const int64_t each = tokens * groups, together = most * each;
    p.apart = together > 32;
    // Many rows a sequence are bound by products, of which sharing saves none: eight sequences of 16 tokens, 64 heads of 8 kv heads,
    // in 4000 shared keys 64.0 us against 55.8 of the plain attention, of 8 tokens 40.8 against 43.2.
    if (each > 64) return p;
    // Tables whose keys and values are read in the time that the shared kernel needs to begin and to join: two sequences in 4000
    // shared keys, 8 kv heads, 19.2 us against 16.2 of the plain attention (33 MB), 40 in 250 22.9 against 12.1 (57), eight of heads
    // of 64 in 4000 17.1 against 19.9 (67), four of 32 kv heads in 1000 16.4 against 20.5 (70), eight of 8 in 4000 24.8 against 29.2
    // (134). Wider tables say nothing of the keys in them: who calls this knows what it saves.
    const int64_t bytes = batch * keys * kv_heads * head_dim * 4;
    if (bytes < (p.apart ? int64_t{1} << 27 : int64_t{1} << 26)) return p;
    const int tiles = (p.apart ? each : together) > 16 ? 2 : 1;
    p.own_tile = 16 * tiles;
    p.group_tile = p.apart ? kGroupTile : p.own_tile;
    p.group_rows = ceil_div(together, p.group_tile);
    p.row_groups = ceil_div(each, p.own_tile);
    p.group_kept = std::min(together, p.group_tile);
    p.rows_kept = std::min(each, p.own_tile);
    const int64_t of_groups = sharing * p.group_rows, own = batch * p.row_groups;
    // Past the list of either kernel the plain attention reads every sequence's pages, of small groups also where the other's list
    // would hold them.
    if (of_groups + own > (p.apart ? kEntries : kFewEntries)) return p;
    if (batch * each * kv_heads > kMaxThreads / 64) return p;  // rows of group_join_kernel, a wave each
    if ((of_groups + own) * (keys / kTile + 512) > INT32_MAX) return p;  // units, which are added up in 32 bits
    constexpr int64_t kParts = (kTeams > 2 ? kTeams : 2) * kCUs;  // teams, or blocks, two on a CU
    p.own_first = kv_heads * of_groups * p.group_kept;
    p.own_later = p.own_first + kv_heads * own * p.rows_kept;
    p.group_later = p.apart ? p.own_later + kParts * p.own_tile : p.own_later;
    const int64_t parts = p.group_later + (p.apart ? kCUs : kParts) * p.group_tile;
    p.tiles = tiles;
    p.part_o = static_cast<size_t>(parts * head_dim) * sizeof(float);
    p.part_ml = static_cast<size_t>(ceil_div(parts, 2) * 2) * sizeof(float2);
    p.desc = static_cast<size_t>(ceil_div((of_groups + own) * kv_heads, 2) * 2) * sizeof(int2);
    p.place = static_cast<size_t>(batch) * sizeof(int);
    p.bytes = p.part_o + p.part_ml + p.desc + p.place;
    return p;
}

template <typename T, int D>
void launch_shared(GroupArgs a, const Plan& p, char* ws, hipStream_t st) {
    a.row_groups = static_cast<int>(p.row_groups);
    a.rows_kept = static_cast<int>(p.rows_kept);
    a.group_rows = static_cast<int>(p.group_rows);
    a.group_tile = static_cast<int>(p.group_tile);
    a.group_kept = static_cast<int>(p.group_kept);
    a.own_tile = static_cast<int>(p.own_tile);
    a.group_shift = __builtin_ctz(a.group_tile);
    a.own_shift = __builtin_ctz(a.own_tile);
    a.per_most = 1.0f / static_cast<float>(a.most);
    a.per_each = 1.0f / static_cast<float>(a.tokens * a.groups);
    a.per_groups = 1.0f / static_cast<float>(a.groups);
    a.per_tokens = 1.0f / static_cast<float>(a.tokens);
    a.per_group_rows = 1.0f / static_cast<float>(a.group_rows);
    a.per_row_groups = 1.0f / static_cast<float>(a.row_groups);
    a.own_first = p.own_first;
    a.group_later = p.group_later;
    a.own_later = p.own_later;
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + p.part_o);
    a.desc = reinterpret_cast<int2*>(ws + p.part_o + p.part_ml);
    a.place = reinterpret_cast<int*>(ws + p.part_o + p.part_ml + p.desc);
    if (p.apart) {
        if (p.tiles == 1) shared_kernel<T, D, 1><<<dim3(kCUs), 512, 0, st>>>(a);
        else shared_kernel<T, D, 2><<<dim3(kCUs), 512, 0, st>>>(a);
    } else {
        if (p.tiles == 1) few_kernel<T, D, 1, true, GroupArgs><<<dim3(FewShape<D, 1>::kBlocks), 64 * kWaves, 0, st>>>(a);
        else few_kernel<T, D, 2, true, GroupArgs><<<dim3(FewShape<D, 2>::kBlocks), 64 * kWaves, 0, st>>>(a);
    }
    const int64_t rows = static_cast<int64_t>(a.batch) * a.tokens * a.heads;
    group_join_kernel<T, D><<<dim3(static_cast<unsigned>(ceil_div(rows, 4))), 256, 0, st>>>(a, static_cast<uint32_t>(rows));
}

// A call's plan; tiles 0 where there is none.
Plan plan_of(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t table_pages,
             int64_t page_size, int64_t sharing, int64_t most) {
    if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 65536 || batch > INT32_MAX ||
        tokens > INT32_MAX || batch * tokens > INT32_MAX / heads || sharing <= 0 || most <= 0 || sharing > INT32_MAX ||
        most > INT32_MAX / sharing || most > INT32_MAX / (tokens * heads) || (head_dim != 64 && head_dim != 128) ||
        table_pages <= 0 || page_size <= 0 || table_pages > kMaxKeys / page_size)
        return Plan{};
    return make_plan(batch, tokens, heads / kv_heads, kv_heads, head_dim, table_pages * page_size, sharing, most);
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" {

size_t nq_paged_shared_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                 int64_t head_dim, int64_t table_pages, int64_t page_size, int64_t groups,
                                                 int64_t most) {
    return plan_of(batch, tokens, heads, kv_heads, head_dim, table_pages, page_size, groups, most).bytes;
}

int nq_paged_shared_attention(int dtype, const void* q, int64_t q_stride, const void* k_pages, const void* v_pages,
                              int64_t pages, int64_t page_size, const int32_t* table, int64_t table_stride, int64_t table_pages,
                              const int64_t* positions, const int32_t* members, const int32_t* shared, int64_t groups,
                              int64_t most, void* out, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                              int64_t head_dim, int64_t window, int64_t sinks, float scaling, void* workspace,
                              size_t workspace_bytes, nq_stream_t stream) {
    const char* name = "nq_paged_shared_attention";
    if (int st = check_sizes(name, dtype, pages, page_size, table_stride, table_pages, batch, tokens, heads, kv_heads, head_dim))
        return st;
    if (head_dim != 64 && head_dim != 128) return fail(NQ_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", name);
    if (page_size % 16) return fail(NQ_ERR_UNSUPPORTED, "%s: page_size must be a multiple of 16", name);
    if (window < 0 || sinks < 0 || groups < 0 || most < 0)
        return fail(NQ_ERR_INVALID_ARGUMENT, "%s: negative window, sinks, groups or members", name);
    if (q_stride < heads * head_dim || q_stride % 8)
        return fail(NQ_ERR_SHAPE, "%s: the token stride must hold the heads and be a multiple of 8", name);
    if (batch == 0 || tokens == 0) return NQ_OK;
    if (batch * tokens > INT32_MAX / heads) return fail(NQ_ERR_UNSUPPORTED, "%s: sizes too large", name);
    if (int st = check_pages(name, k_pages, v_pages, pages, page_size, table, table_stride, table_pages, positions)) return st;
    if (!q || !out || !members || !shared) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16) || !aligned(members, 4) || !aligned(shared, 4))
        return fail(NQ_ERR_ALIGNMENT, "%s: q, out and the workspace must be 16-byte aligned, the groups 4-byte", name);
    const Plan plan = plan_of(batch, tokens, heads, kv_heads, head_dim, table_pages, page_size, groups, most);
    if (plan.tiles == 0) return fail(NQ_ERR_UNSUPPORTED, "%s: no groups, or a call for nq_paged_attention", name);
    if (!workspace || workspace_bytes < plan.bytes)
        return fail(NQ_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", name, workspace ? workspace_bytes : size_t{0}, plan.bytes);
    GroupArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.q_stride = q_stride;
    a.k_pages = static_cast<const uint16_t*>(k_pages);
    a.v_pages = static_cast<const uint16_t*>(v_pages);
    a.pages = Pages(table, table_stride, table_pages, pages, page_size);
    a.positions = positions;
    a.members = members;
    a.shared = shared;
    a.sharing = static_cast<int>(groups);
    a.most = static_cast<int>(most);
    a.out = static_cast<uint16_t*>(out);
    a.batch = static_cast<int>(batch);
    a.tokens = static_cast<int>(tokens);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.groups = static_cast<int>(heads / kv_heads);
    a.window = static_cast<int>(std::min(window, kMaxKeys));
    a.sinks = static_cast<int>(std::min(sinks, kMaxKeys));
    a.scale = scaling * 1.44269504088896340736f;  // exp(x) = exp2(x log2(e))
    char* ws = static_cast<char*>(workspace);
    hipStream_t st = as_stream(stream);
    if (dtype == NQ_F16) {
        if (head_dim == 64) launch_shared<F16, 64>(a, plan, ws, st);
        else launch_shared<F16, 128>(a, plan, ws, st);
    } else {
        if (head_dim == 64) launch_shared<BF16, 64>(a, plan, ws, st);
        else launch_shared<BF16, 128>(a, plan, ws, st);
    }
    return check_launch(name);
}

}  // extern "C"
