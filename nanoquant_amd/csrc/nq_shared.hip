// Attention over the pages of a cache of which groups of sequences have the leading ones in common.
#include <algorithm>
#include <cmath>

#include "nq_common.h"
#include "nq_paged.h"

namespace nq {
namespace {

constexpr int kEntries = 1024;  // pieces of work that a launch lists

struct SharedArgs {
    const uint16_t* q;
    int64_t q_stride;
    const uint16_t* k_pages;
    const uint16_t* v_pages;
    Pages pages;
    const int64_t* positions;
    const int32_t* members;  // [groups][most]
    const int32_t* shared;   // [groups]: pages
    int groups, most;
    uint16_t* out;
    int batch, tokens, heads, kv_heads;
    int window, sinks;
    float scale;  // times log2(e)
};

// A wave a row, a key at a time, lane l at dimensions l and, of 128, l + 64.
template <typename T, int D>
__global__ __launch_bounds__(256) void shared_kernel(const SharedArgs a) {
    constexpr int N = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);  // (sequence, token, head)
    if (row >= static_cast<int64_t>(a.batch) * a.tokens * a.heads) return;
    const int64_t token = row / a.heads;
    const int head = static_cast<int>(row - token * a.heads), kvh = head / (a.heads / a.kv_heads);
    const int b = static_cast<int>(token / a.tokens);
    const int64_t p = a.positions[token];
    const int last = p >= 0 && p < a.pages.capacity() ? static_cast<int>(p) : -1;
    const int start = a.window > 0 ? max(0, last - a.window + 1) : 0;
    const uint16_t* q = a.q + token * a.q_stride + static_cast<int64_t>(head) * D + lane;
    float o[N], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < N; ++i) o[i] = 0.0f;
    for (int key = 0; key <= last; ++key) {
        const int page = a.pages.page(b, key / a.pages.page_size);
        if (!(key >= start || key < a.sinks) || page < 0) continue;
        const int64_t at = ((static_cast<int64_t>(page) * a.kv_heads + kvh) * a.pages.page_size + key % a.pages.page_size) * D + lane;
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
    for (int i = 0; i < N; ++i) a.out[row * D + lane + 64 * i] = T::from_float(l == 0.0f ? 0.0f : o[i] / l);
}

template <typename T>
void launch_shared(const SharedArgs& a, int64_t head_dim, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.batch) * a.tokens * a.heads, 4)));
    if (head_dim == 64) shared_kernel<T, 64><<<grid, 256, 0, st>>>(a);
    else shared_kernel<T, 128><<<grid, 256, 0, st>>>(a);
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" {

size_t nq_paged_shared_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                 int64_t head_dim, int64_t groups, int64_t most) {
    if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 65536 || batch > INT32_MAX ||
        tokens > INT32_MAX || batch * tokens > INT32_MAX / heads || groups <= 0 || most <= 0 || groups > kEntries || most > INT32_MAX / (tokens * heads))
        return 0;
    const int64_t rows = tokens * (heads / kv_heads);
    return groups * ceil_div(most * rows, 64) + batch * ceil_div(rows, 64) <= kEntries ? 16 : 0;
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
    if (!q || !out || (groups * most && (!members || !shared))) return fail(NQ_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16) || !aligned(members, 4) || !aligned(shared, 4))
        return fail(NQ_ERR_ALIGNMENT, "%s: q, out and the workspace must be 16-byte aligned, the groups 4-byte", name);
    SharedArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.q_stride = q_stride;
    a.k_pages = static_cast<const uint16_t*>(k_pages);
    a.v_pages = static_cast<const uint16_t*>(v_pages);
    a.pages = Pages{table, table_stride, static_cast<int>(table_pages), static_cast<int>(pages), static_cast<int>(page_size)};
    a.positions = positions;
    a.members = members;
    a.shared = shared;
    a.groups = static_cast<int>(groups);
    a.most = static_cast<int>(most);
    a.out = static_cast<uint16_t*>(out);
    a.batch = static_cast<int>(batch);
    a.tokens = static_cast<int>(tokens);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.window = static_cast<int>(std::min(window, kMaxKeys));
    a.sinks = static_cast<int>(std::min(sinks, kMaxKeys));
    a.scale = scaling * 1.44269504088896340736f;  // exp(x) = exp2(x log2(e))
    if (dtype == NQ_F16) launch_shared<F16>(a, head_dim, as_stream(stream));
    else launch_shared<BF16>(a, head_dim, as_stream(stream));
    return check_launch(name);
}

}  // extern "C"
