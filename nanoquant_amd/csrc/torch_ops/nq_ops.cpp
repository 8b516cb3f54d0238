// The torch.ops.binary_kernels operators' device implementations in C++: argument checks, output and
// scratch from torch's caching allocator, one call of the C ABI on torch's current stream.
//
// At decode sizes a launch takes a few microseconds and an operator implemented in Python spent 24 us on the
// host per call (dispatch into Python, its checks, ctypes), so eager calls were bound by it: 4096 x 4096,
// r = 1120, one row 23.5 -> 11.7 us a call, a module call of 21 rows on 4096 x 11008 34.7 -> 21.5. These
// implementations take the well-formed calls; a call that fails any check, or a library that has not been
// loaded yet, goes to the general operator of the same schema (namespace nanoquant_amd, implemented in Python),
// which loads the library, handles the empty sizes and raises the documented errors.
//
// The C ABI's functions come in as addresses (nq_ops_bind), so that this file needs no link to the HIP library.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <atomic>
#include <cmath>

#include "../../../include/nq_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// In the order of nq_ops_bind's array.
struct Library {
    decltype(&nq_gemv_workspace_bytes) gemv_bytes;
    decltype(&nq_gemv) gemv;
    decltype(&nq_gemm_onebit_workspace_bytes) onebit_bytes;
    decltype(&nq_gemm_onebit) onebit;
    decltype(&nq_gemm_nanoquant_workspace_bytes) nanoquant_bytes;
    decltype(&nq_gemm_nanoquant) nanoquant;
    decltype(&nq_paged_rope_write) paged_write;
    decltype(&nq_paged_attention_workspace_bytes) paged_attention_bytes;
    decltype(&nq_paged_attention) paged_attention;
    decltype(&nq_verify_drafts_workspace_bytes) verify_bytes;
    decltype(&nq_verify_drafts) verify;
};
constexpr int kFunctions = 11;
std::atomic<const Library*> g_library{nullptr};

int dtype_code(at::ScalarType t) { return t == at::kHalf ? NQ_F16 : NQ_BF16; }

// A tensor the kernels read where it lies: on `x`'s device, contiguous, of the given type.
bool plain(const Tensor& t, const Tensor& x, at::ScalarType type) {
    return t.device() == x.device() && t.scalar_type() == type && t.is_contiguous();
}

// A 1-D scale of `size` elements, or none.
bool scale_ok(const OptTensor& s, const Tensor& x, int64_t size) {
    return !s.has_value() || (s->dim() == 1 && s->size(0) == size && plain(*s, x, x.scalar_type()));
}

const void* data_of(const OptTensor& t) { return t.has_value() ? t->const_data_ptr() : nullptr; }

Tensor scratch(size_t bytes, const Tensor& x) {
    return at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
}

nq_stream_t stream_of(const Tensor& x) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.get_device()).stream();
}

template <typename F>
c10::TypedOperatorHandle<F> general(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

bool one_of(int64_t v, std::initializer_list<int64_t> choices) {
    for (int64_t c : choices)
        if (v == c) return true;
    return false;
}

Tensor gemv(const Tensor& x, const Tensor& s_in, const Tensor& v_words, const OptTensor& s_mid, const Tensor& u_words,
            const Tensor& s_out, int64_t th1, int64_t th2, int64_t rpw1, int64_t rpw2, int64_t acc1, int64_t acc2,
            int64_t pipe1, int64_t pipe2) {
    const Library* lib = g_library.load(std::memory_order_acquire);
    const auto type = x.scalar_type();
    if (lib && (type == at::kHalf || type == at::kBFloat16) && x.is_cuda() && x.is_contiguous() && x.dim() >= 1 &&
        x.numel() > 0 && v_words.dim() == 2 && u_words.dim() == 2 && s_out.dim() == 1) {
        const int64_t n = x.size(-1), r = v_words.size(0), m = s_out.size(0), batch = x.numel() / n;
        if (m > 0 && plain(s_in, x, type) && s_in.numel() == n && plain(s_out, x, type) && plain(v_words, x, at::kInt) &&
            v_words.size(1) == (n + 31) / 32 && plain(u_words, x, at::kInt) && u_words.size(0) == m &&
            u_words.size(1) == (r + 31) / 32 && scale_ok(s_mid, x, r) && one_of(th1, {64, 128, 256}) &&
            one_of(th2, {64, 128, 256}) && one_of(rpw1, {1, 2, 4, 8}) && one_of(rpw2, {1, 2, 4, 8}) &&
            one_of(acc1, {1, 2}) && one_of(acc2, {1, 2}) && one_of(pipe1, {1, 2, 4, 8, 16}) &&
            one_of(pipe2, {1, 2, 4, 8, 16})) {
            const c10::DeviceGuard guard(x.device());
            std::vector<int64_t> shape = x.sizes().vec();
            shape.back() = m;
            Tensor y = at::empty(shape, x.options());
            const size_t bytes = lib->gemv_bytes(batch, n, r, m);
            const Tensor ws = scratch(bytes, x);
            if (lib->gemv(dtype_code(type), x.const_data_ptr(), s_in.const_data_ptr(),
                          static_cast<const uint32_t*>(v_words.const_data_ptr()), data_of(s_mid),
                          static_cast<const uint32_t*>(u_words.const_data_ptr()), s_out.const_data_ptr(),
                          y.mutable_data_ptr(), batch, n, r, m, ws.mutable_data_ptr(), bytes, stream_of(x)) == NQ_OK)
                return y;
        }
    }
    static const auto op = general<decltype(gemv)>("nanoquant_amd::nanoquant_dyn_forward");
    return op.call(x, s_in, v_words, s_mid, u_words, s_out, th1, th2, rpw1, rpw2, acc1, acc2, pipe1, pipe2);
}

// What both GEMM operators ask of one stage: x [M, K] against Marlin words of K inputs and `out` outputs, with the
// reference's workspace size.
bool stage_ok(const Tensor& x, int64_t K, const Tensor& words, const OptTensor& scale_in, const OptTensor& scale_out,
              const Tensor& workspace) {
    if (words.dim() != 2 || !plain(words, x, at::kInt) || words.size(0) * 16 != K || words.size(1) % 32 != 0) return false;
    const int64_t out = words.size(1) * 2;
    return out > 0 && scale_ok(scale_in, x, K) && scale_ok(scale_out, x, out) && workspace.numel() >= out / 128 * 32;
}

bool x_ok(const Library* lib, const Tensor& x) {
    return lib && (x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16) && x.is_cuda() && x.is_contiguous() &&
           x.dim() == 2 && x.size(0) > 0 && x.size(1) > 0;
}

Tensor onebit(const Tensor& x, const Tensor& weight, const OptTensor& s_in, const OptTensor& s_out, const Tensor& workspace) {
    const Library* lib = g_library.load(std::memory_order_acquire);
    if (x_ok(lib, x) && stage_ok(x, x.size(1), weight, s_in, s_out, workspace)) {
        const c10::DeviceGuard guard(x.device());
        const int64_t M = x.size(0), K = x.size(1), N = weight.size(1) * 2;
        Tensor y = at::empty({M, N}, x.options());
        const size_t bytes = lib->onebit_bytes(M, K, N);
        const Tensor part = bytes ? scratch(bytes, x) : Tensor();
        if (lib->onebit(dtype_code(x.scalar_type()), x.const_data_ptr(), static_cast<const uint32_t*>(weight.const_data_ptr()),
                        data_of(s_in), data_of(s_out), y.mutable_data_ptr(), M, K, N,
                        bytes ? part.mutable_data_ptr() : nullptr, bytes, stream_of(x)) == NQ_OK)
            return y;
    }
    static const auto op = general<decltype(onebit)>("nanoquant_amd::marlin_onebit_forward");
    return op.call(x, weight, s_in, s_out, workspace);
}

Tensor nanoquant(const Tensor& x, const Tensor& v_words, const Tensor& u_words, const OptTensor& s_g, const OptTensor& s_l,
                 const OptTensor& s_h, const Tensor& workspace) {
    const Library* lib = g_library.load(std::memory_order_acquire);
    if (x_ok(lib, x) && stage_ok(x, x.size(1), v_words, s_g, s_l, workspace) &&
        stage_ok(x, v_words.size(1) * 2, u_words, std::nullopt, s_h, workspace)) {
        const c10::DeviceGuard guard(x.device());
        const int64_t M = x.size(0), n = x.size(1), r_pad = v_words.size(1) * 2, m = u_words.size(1) * 2;
        const Tensor imm = at::empty({M, r_pad}, x.options());
        Tensor y = at::empty({M, m}, x.options());
        const size_t bytes = lib->nanoquant_bytes(M, n, r_pad, m);
        const Tensor part = bytes ? scratch(bytes, x) : Tensor();
        if (lib->nanoquant(dtype_code(x.scalar_type()), x.const_data_ptr(),
                           static_cast<const uint32_t*>(v_words.const_data_ptr()),
                           static_cast<const uint32_t*>(u_words.const_data_ptr()), data_of(s_g), data_of(s_l), data_of(s_h),
                           imm.mutable_data_ptr(), y.mutable_data_ptr(), M, n, r_pad, m,
                           bytes ? part.mutable_data_ptr() : nullptr, bytes, stream_of(x)) == NQ_OK)
            return y;
    }
    static const auto op = general<decltype(nanoquant)>("nanoquant_amd::marlin_nanoquant_forward");
    return op.call(x, v_words, u_words, s_g, s_l, s_h, workspace);
}

// The paged cache's operators (nanoquant_amd/serve.py): the well-formed calls on memory that the kernels read where it lies.
// For any other call they give nothing, and the function in Python goes on to check it, to lay tensors out or to run torch ops.

bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

// Elements between the rows of x [batch, tokens, width], 0 where a kernel cannot read them.
int64_t row_stride(const Tensor& x, int64_t batch, int64_t tokens) {
    const int64_t width = x.size(2), stride = tokens > 1 ? x.stride(1) : batch > 1 ? x.stride(0) : width;
    const bool fits = x.stride(2) == 1 && stride % 8 == 0 && stride >= width && aligned16(x) &&
                      (tokens == 1 || batch == 1 || x.stride(0) == tokens * stride);
    return fits ? stride : 0;
}

// The pool [pages, kv_heads, page_size, head_dim], the table and the positions of a call whose tokens are like q.
bool pages_ok(const Library* lib, const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
              const Tensor& positions) {
    if (!lib || !q.is_cuda() || (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16) || q.dim() != 3 ||
        q.numel() == 0 || k_pages.dim() != 4 || k_pages.numel() == 0 || table.dim() != 2 || positions.dim() != 2)
        return false;
    const int64_t width = k_pages.size(1) * k_pages.size(3);
    return plain(k_pages, q, q.scalar_type()) && plain(v_pages, q, q.scalar_type()) && k_pages.sizes() == v_pages.sizes() &&
           aligned16(k_pages) && aligned16(v_pages) && plain(positions, q, at::kLong) && positions.size(0) == q.size(0) &&
           positions.size(1) == q.size(1) && q.size(2) % width == 0 && table.device() == q.device() &&
           table.scalar_type() == at::kInt && table.size(0) == q.size(0) && table.size(1) > 0 && table.stride(1) == 1 &&
           table.stride(0) >= table.size(1) && table.size(1) <= (int64_t{1} << 30) / k_pages.size(2);
}

OptTensor paged_write(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos, const Tensor& sin,
                      const Tensor& positions, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table) {
    const Library* lib = g_library.load(std::memory_order_acquire);
    if (!pages_ok(lib, q, k_pages, v_pages, table, positions)) return std::nullopt;
    const int64_t B = q.size(0), T = q.size(1), KV = k_pages.size(1), S = k_pages.size(2), D = k_pages.size(3);
    const auto type = q.scalar_type(), rope = cos.scalar_type();
    auto tokens_ok = [&](const Tensor& t) {
        return t.device() == q.device() && t.scalar_type() == type && t.dim() == 3 && t.size(0) == B && t.size(1) == T &&
               t.size(2) == KV * D;
    };
    auto table_ok = [&](const Tensor& t) {
        return plain(t, q, rope) && t.numel() == B * T * D && t.size(-1) == D && aligned16(t);
    };
    if (D % 16 || !tokens_ok(k) || !tokens_ok(v) || (rope != type && rope != at::kFloat) || cos.dim() == 0 ||
        cos.sizes() != sin.sizes() || !table_ok(cos) || !table_ok(sin))
        return std::nullopt;
    const int64_t qs = row_stride(q, B, T), ks = row_stride(k, B, T), vs = row_stride(v, B, T);
    if (qs == 0 || ks == 0 || vs == 0) return std::nullopt;
    const c10::DeviceGuard guard(q.device());
    Tensor out = at::empty(q.sizes(), q.options());
    if (lib->paged_write(dtype_code(type), q.const_data_ptr(), qs, k.const_data_ptr(), ks, v.const_data_ptr(), vs,
                         cos.const_data_ptr(), sin.const_data_ptr(), rope == at::kFloat,
                         static_cast<const int64_t*>(positions.const_data_ptr()), static_cast<const int32_t*>(table.const_data_ptr()),
                         table.stride(0), table.size(1), k_pages.mutable_data_ptr(), v_pages.mutable_data_ptr(), k_pages.size(0), S,
                         out.mutable_data_ptr(), B, T, q.size(2) / D, KV, D, stream_of(q)) != NQ_OK)
        return std::nullopt;
    return out;
}

OptTensor paged_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                          const Tensor& positions, int64_t window, int64_t sinks, std::optional<double> scale) {
    const Library* lib = g_library.load(std::memory_order_acquire);
    if (!pages_ok(lib, q, k_pages, v_pages, table, positions)) return std::nullopt;
    const int64_t B = q.size(0), T = q.size(1), KV = k_pages.size(1), S = k_pages.size(2), D = k_pages.size(3), H = q.size(2) / D;
    const int64_t qs = row_stride(q, B, T);
    if ((D != 64 && D != 128) || S % 16 || qs == 0 || window < 0 || sinks < 0) return std::nullopt;
    const c10::DeviceGuard guard(q.device());
    Tensor out = at::empty(q.sizes(), q.options());
    const size_t bytes = lib->paged_attention_bytes(B, T, H, KV, D, table.size(1), S);
    const Tensor ws = bytes ? scratch(bytes, q) : Tensor();
    const float factor = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(D)));
    if (lib->paged_attention(dtype_code(q.scalar_type()), q.const_data_ptr(), qs, k_pages.const_data_ptr(),
                             v_pages.const_data_ptr(), k_pages.size(0), S, static_cast<const int32_t*>(table.const_data_ptr()),
                             table.stride(0), table.size(1), static_cast<const int64_t*>(positions.const_data_ptr()),
                             out.mutable_data_ptr(), B, T, H, KV, D, window, sinks, factor,
                             bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(q)) != NQ_OK)
        return std::nullopt;
    return out;
}

// {accepted, tokens}, or an empty list.
std::vector<Tensor> verify(const Tensor& logits, const Tensor& drafts, const Tensor& uniforms, const OptTensor& draft_probs,
                           double temperature) {
    const Library* lib = g_library.load(std::memory_order_acquire);
    const auto type = logits.scalar_type();
    if (!lib || !logits.is_cuda() || logits.dim() != 3 || drafts.dim() != 2 || uniforms.dim() != 2 || logits.numel() == 0 ||
        (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat))
        return {};
    const int64_t B = logits.size(0), n = logits.size(1) - 1, V = logits.size(2);
    const int64_t stride = n > 0 ? logits.stride(1) : B > 1 ? logits.stride(0) : V;  // between rows
    if (logits.stride(2) != 1 || stride < V || (n > 0 && B > 1 && logits.stride(0) != (n + 1) * stride) ||
        !plain(drafts, logits, at::kLong) || drafts.size(0) != B || drafts.size(1) != n || !plain(uniforms, logits, at::kFloat) ||
        uniforms.size(0) != B || uniforms.size(1) != n + 1 || !(temperature >= 0.0) || std::isinf(temperature))
        return {};
    if (draft_probs.has_value() && (!plain(*draft_probs, logits, at::kFloat) || draft_probs->dim() != 3 ||
                                    draft_probs->size(0) != B || draft_probs->size(1) != n || draft_probs->size(2) != V))
        return {};
    const size_t bytes = lib->verify_bytes(B, n, V);
    if (bytes == 0) return {};
    const c10::DeviceGuard guard(logits.device());
    Tensor accepted = at::empty({B}, drafts.options()), tokens = at::empty({B, n + 1}, drafts.options());
    const Tensor ws = scratch(bytes, logits);
    if (lib->verify(type == at::kFloat ? NQ_F32 : dtype_code(type), logits.const_data_ptr(), stride,
                    static_cast<const int64_t*>(drafts.const_data_ptr()), static_cast<const float*>(data_of(draft_probs)),
                    static_cast<const float*>(uniforms.const_data_ptr()), temperature,
                    static_cast<int64_t*>(accepted.mutable_data_ptr()), static_cast<int64_t*>(tokens.mutable_data_ptr()), B, n, V,
                    ws.mutable_data_ptr(), bytes, stream_of(logits)) != NQ_OK)
        return {};
    return {accepted, tokens};
}

}  // namespace

// The addresses of the C ABI's functions, in Library's order, once the HIP library is loaded (the table lives as long
// as the process). Returns 0, or 1 where the count is not this build's.
extern "C" int nq_ops_bind(void* const* functions, int count) {
    if (count != kFunctions) return 1;
    static Library library;
    library.gemv_bytes = reinterpret_cast<decltype(library.gemv_bytes)>(functions[0]);
    library.gemv = reinterpret_cast<decltype(library.gemv)>(functions[1]);
    library.onebit_bytes = reinterpret_cast<decltype(library.onebit_bytes)>(functions[2]);
    library.onebit = reinterpret_cast<decltype(library.onebit)>(functions[3]);
    library.nanoquant_bytes = reinterpret_cast<decltype(library.nanoquant_bytes)>(functions[4]);
    library.nanoquant = reinterpret_cast<decltype(library.nanoquant)>(functions[5]);
    library.paged_write = reinterpret_cast<decltype(library.paged_write)>(functions[6]);
    library.paged_attention_bytes = reinterpret_cast<decltype(library.paged_attention_bytes)>(functions[7]);
    library.paged_attention = reinterpret_cast<decltype(library.paged_attention)>(functions[8]);
    library.verify_bytes = reinterpret_cast<decltype(library.verify_bytes)>(functions[9]);
    library.verify = reinterpret_cast<decltype(library.verify)>(functions[10]);
    g_library.store(&library, std::memory_order_release);
    return 0;
}

// Digest of the header that this library was built from, to be compared with nq_header_digest before binding.
extern "C" const char* nq_ops_header_digest(void) { return NQ_HEADER_DIGEST; }

TORCH_LIBRARY_IMPL(binary_kernels, CUDA, m) {
    m.impl("nanoquant_dyn_forward", &gemv);
    m.impl("marlin_onebit_forward", &onebit);
    m.impl("marlin_nanoquant_forward", &nanoquant);
}

TORCH_LIBRARY_IMPL(nanoquant_amd, CUDA, m) {
    m.impl("paged_rope_write", &paged_write);
    m.impl("paged_attention", &paged_attention);
    m.impl("verify_drafts", &verify);
}
