"""What serving many sequences at once needs beyond one static cache: a KV cache in pages, each sequence at a length of its
own, and the check of drafted tokens.

* :class:`PagedKVCache` holds the pools and the page table; ``NanoQuantLlama.forward`` takes it in place of a
  ``StaticKVCache``, with positions [B, T].
* :func:`paged_rope_write` rotates the new tokens' queries and keys and writes keys and values into the pages.
* :func:`paged_attention` is causal attention over the pages, for one new token a sequence, drafted tokens, prompts and
  chunks of prompts, optionally under a sliding window with a few first tokens that stay visible.
* :func:`verify_drafts` keeps or turns down drafted tokens by the model's logits and given random numbers.

Calls of well-laid-out tensors on the GPU go through the C++ of ``libnq_ops.so`` (``csrc/torch_ops/nq_ops.cpp``): a small call
is bound by its host path. What that does not take is checked, copied into place or refused here.

float16 and bfloat16 tensors on the GPU run the HIP library (``nq_paged_rope_write``, ``nq_paged_attention``,
``nq_verify_drafts``); CPU tensors, float32 models, calls that are differentiated, head sizes other than 64 and 128 and page
sizes that are no multiple of 16 run torch ops with the same results but for rounding, in float32, or in float64 where the
tensors are. The reference has no counterpart: its harness decodes one batch on Hugging Face's static cache and samples one
token a step (``src/nanoquant/kernel/test_decode.py:350-422``).
"""
from __future__ import annotations

import math
import sys

import torch

from . import _lib
from ._dispatch import launch as _launch, only_eager as _only_eager

_HALF = (torch.float16, torch.bfloat16)

_OPS = torch.library.Library("nanoquant_amd", "FRAGMENT")
for _schema in (
        "paged_rope_write(Tensor q, Tensor k, Tensor v, Tensor cos, Tensor sin, Tensor positions, Tensor(a!) k_pages, "
        "Tensor(b!) v_pages, Tensor table) -> Tensor?",
        "paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor positions, int window, int sinks, "
        "float? scale) -> Tensor?",
        "verify_drafts(Tensor logits, Tensor drafts, Tensor uniforms, Tensor? draft_probs, float temperature) -> Tensor[]"):
    _OPS.define(_schema)


def _native(name):
    """The operator in C++, or None where ``libnq_ops.so`` is missing or older."""
    if _lib.ops is None or not torch._C._dispatch_has_kernel_for_dispatch_key(f"nanoquant_amd::{name}", "CUDA"):
        return None
    return getattr(torch.ops.nanoquant_amd, name).default


_native_write, _native_attention, _native_verify = (_native(n) for n in ("paged_rope_write", "paged_attention", "verify_drafts"))


class PagedKVCache:
    """Per-layer K and V pools of ``pages`` pages of ``page_size`` positions, shared by ``batch`` sequences of up to
    ``max_len`` positions each, and the table that says where a sequence's positions lie.

    ``k[layer]`` and ``v[layer]`` are [pages, kv_heads, page_size, head_dim]; ``table`` is int32
    [batch, ceil(max_len / page_size)] on the device: position p of sequence b lies in page ``table[b, p // page_size]`` at row
    ``p % page_size``, and -1 is a page that is not there. The table's memory stays the same, so a captured graph follows its
    changes. ``window`` and ``sinks`` (0: none) are how the model's layers read the cache: a token sees the last ``window``
    positions and the first ``sinks``.

    ``reserve`` gives a sequence the pages that its next tokens need, ``trim`` takes back those that no later token will see,
    ``release`` all of them. A program may also fill the table itself, and then uses none of these: they write a sequence's row
    as they know it. Serve under ``torch.no_grad``, or what a model with gradients writes makes the pools part of its graph.
    """

    def __init__(self, shape, batch: int, pages: int, page_size: int, max_len: int, device, dtype, window: int = 0,
                 sinks: int = 0):
        if min(batch, pages, page_size, max_len) <= 0 or min(window, sinks) < 0:
            raise ValueError(f"bad sizes of a paged cache: batch {batch}, pages {pages}, page_size {page_size}, max_len "
                             f"{max_len}, window {window}, sinks {sinks}")
        self.batch, self.pages, self.page_size = batch, pages, page_size
        self.max_pages = -(-max_len // page_size)
        self.max_len = max_len
        self.window, self.sinks = window, sinks
        pool = (pages, shape.kv_heads, page_size, shape.head_dim)
        self.k = [torch.zeros(pool, device=device, dtype=dtype) for _ in range(shape.layers)]
        self.v = [torch.zeros(pool, device=device, dtype=dtype) for _ in range(shape.layers)]
        self.table = torch.full((batch, self.max_pages), -1, device=device, dtype=torch.int32)
        self._host = [[-1] * self.max_pages for _ in range(batch)]  # the table as the methods below left it
        self._free = list(range(pages - 1, -1, -1))

    def _row(self, sequence: int):
        if not 0 <= sequence < self.batch:
            raise IndexError(f"sequence {sequence} of {self.batch}")
        return self._host[sequence]

    def _store(self, sequence: int):
        self.table[sequence].copy_(torch.tensor(self._host[sequence], dtype=torch.int32))

    def reserve(self, sequence: int, length: int, start: int = 0) -> None:
        """Pages for the sequence's positions ``start`` to ``length - 1`` (those it has stay). RuntimeError, and no change,
        where the pool has too few left."""
        row = self._row(sequence)
        if not 0 <= start <= length <= self.max_len:
            raise ValueError(f"positions {start} to {length} do not fit max_len {self.max_len}")
        need = [i for i in range(start // self.page_size, -(-length // self.page_size)) if row[i] < 0]
        if len(need) > len(self._free):
            raise RuntimeError(f"the paged cache has {len(self._free)} pages left, sequence {sequence} needs {len(need)}")
        for i in need:
            row[i] = self._free.pop()
        if need:
            self._store(sequence)

    def _take_back(self, sequence: int, slots) -> int:
        row = self._row(sequence)
        gone = [i for i in slots if row[i] >= 0]
        for i in gone:
            self._free.append(row[i])
            row[i] = -1
        if gone:
            self._store(sequence)
        return len(gone)

    def trim(self, sequence: int, position: int) -> int:
        """Take back the pages that no token from ``position`` on sees under the window; returns their number. Calls in
        flight on other streams must have ended."""
        if self.window == 0:
            return 0
        first = min(max(0, position - self.window + 1) // self.page_size, self.max_pages)
        return self._take_back(sequence, range(-(-self.sinks // self.page_size), first))

    def release(self, sequence: int) -> int:
        """Take back all pages of a sequence; returns their number. Calls in flight on other streams must have ended."""
        return self._take_back(sequence, range(self.max_pages))


# ------------------------------------------------------------------------------------- arguments

def _check_pages(what, k_pages, v_pages, table, positions, dtype, device):
    """Shapes of a paged call; returns (batch, tokens, pages, kv_heads, page_size, head_dim)."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError(f"{what}: the pages of keys and values must be [pages, kv_heads, page_size, head_dim] alike, got "
                         f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if positions.dim() != 2 or table.dim() != 2 or table.shape[0] != positions.shape[0] or table.shape[1] == 0:
        raise ValueError(f"{what}: positions must be [batch, tokens] and the table [batch, pages of a sequence], got "
                         f"{tuple(positions.shape)} and {tuple(table.shape)}")
    if positions.dtype != torch.int64 or table.dtype != torch.int32:
        raise TypeError(f"{what}: positions must be int64 and the table int32, got {positions.dtype} and {table.dtype}")
    if k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise TypeError(f"{what}: the pages are {k_pages.dtype} and {v_pages.dtype}, the tokens {dtype}")
    for t in (k_pages, v_pages, table, positions):
        if t.device != device:
            raise ValueError(f"{what}: tensors on {t.device} and {device}")
    if 0 in k_pages.shape:
        raise ValueError(f"{what}: empty pages {tuple(k_pages.shape)}")
    return (*positions.shape, *k_pages.shape)


def _rows(x, batch, tokens):
    """x [batch, tokens, width] as rows a kernel can read, and the elements between two: itself, or a copy where its strides
    or alignment do not fit."""
    stride = x.stride(1) if tokens > 1 else x.stride(0) if batch > 1 else x.shape[2]
    if (x.stride(2) != 1 or stride % 8 or stride < x.shape[2] or x.data_ptr() % 16
            or (tokens > 1 and batch > 1 and x.stride(0) != tokens * stride)):
        x = torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
        stride = x.shape[2]
    return x, stride


def _table_rows(table):
    """The table with rows a kernel can read: itself, or a copy (``contiguous`` keeps the stride of a dimension of one element)."""
    if table.stride(0) >= table.shape[1] and (table.stride(1) == 1 or table.shape[1] == 1):
        return table
    return torch.empty(table.shape, dtype=table.dtype, device=table.device).copy_(table)


def _pool_fits(k_pages, v_pages):
    return (k_pages.is_contiguous() and v_pages.is_contiguous() and k_pages.data_ptr() % 16 == 0
            and v_pages.data_ptr() % 16 == 0)


# ------------------------------------------------------------------------------------- the pages

def paged_rope_write(q, k, v, cos, sin, positions, k_pages, v_pages, table):
    """Rotate the new tokens' queries and keys and write keys and values into the pages; returns the rotated queries
    [B, T, H * D].

    q [B, T, H * D], k and v [B, T, KV * D] (strided views are fine), cos and sin [B, T, D] (or [B * T, D]) in float32 or the
    tokens' type, positions int64 [B, T], pages [pages, KV, page_size, D], table int32 [B, pages of a sequence]. A position
    outside the table (-1 for padding) writes nothing and gives zero queries; a page that is not there is not written. Two
    tokens of a call must not name the same row of a page."""
    what = "paged_rope_write"
    if _native_write is not None and q.is_cuda and _only_eager(q, k, v, cos, sin, positions, k_pages, v_pages, table):
        out = _native_write(q, k, v, cos, sin, positions, k_pages, v_pages, table)
        if out is not None:
            return out
    B, T, N, KV, S, D = _check_pages(what, k_pages, v_pages, table, positions, q.dtype, q.device)
    if (q.dim() != 3 or q.shape[:2] != positions.shape or q.shape[2] % (KV * D) or q.shape[2] == 0
            or tuple(k.shape) != (B, T, KV * D) or v.shape != k.shape):
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit {B} x {T} tokens "
                         f"and pages of {KV} heads of {D}")
    if D % 2 or cos.numel() != B * T * D or sin.shape != cos.shape or cos.shape[-1] != D:
        raise ValueError(f"{what}: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be [{B}, {T}, {D}], {D} even")
    if k.dtype != q.dtype or v.dtype != q.dtype or cos.dtype != sin.dtype or cos.dtype not in (torch.float32, q.dtype):
        raise TypeError(f"{what}: q, k and v of one type, cos and sin of that or float32, got {q.dtype}, {k.dtype}, {v.dtype}, "
                        f"{cos.dtype}, {sin.dtype}")
    for t in (k, v, cos, sin):
        if t.device != q.device:
            raise ValueError(f"{what}: tensors on {t.device} and {q.device}")
    if (q.is_cuda and q.dtype in _HALF and D % 16 == 0 and _only_eager(q, k, v, cos, sin, positions, k_pages, v_pages, table)
            and _pool_fits(k_pages, v_pages) and table.shape[1] * S <= 1 << 30):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if out.numel() == 0:
            return out
        (q, qs), (k, ks), (v, vs) = _rows(q, B, T), _rows(k, B, T), _rows(v, B, T)
        cos, sin = _dense(cos), _dense(sin)
        table, positions = _table_rows(table), positions.contiguous()
        _launch(what, _lib.load().nq_paged_rope_write, q, _lib.dtype_code(q.dtype), q.data_ptr(), qs, k.data_ptr(), ks,
                v.data_ptr(), vs, cos.data_ptr(), sin.data_ptr(), cos.dtype == torch.float32, positions.data_ptr(),
                table.data_ptr(), table.stride(0), table.shape[1], k_pages.data_ptr(), v_pages.data_ptr(), N, S, out.data_ptr(),
                B, T, q.shape[2] // D, KV, D)
        return out
    wide = torch.promote_types(q.dtype, torch.float32)
    cos, sin = cos.reshape(B, T, 1, D).to(wide), sin.reshape(B, T, 1, D).to(wide)

    def rotate(x):
        x = x.reshape(B, T, -1, D).to(wide)
        return (x * cos + torch.cat((-x[..., D // 2:], x[..., :D // 2]), dim=-1) * sin).to(q.dtype)

    real = (positions >= 0) & (positions < table.shape[1] * S)
    at = torch.where(real, positions, 0)
    page = table.gather(1, at // S)
    here = (real & (page >= 0) & (page < N)).nonzero(as_tuple=True)
    rows, offsets = page[here].long(), (at % S)[here]
    k_pages[rows, :, offsets] = rotate(k)[here]
    v_pages[rows, :, offsets] = v.reshape(B, T, KV, D)[here]
    return torch.where(real.unsqueeze(-1), rotate(q).reshape(q.shape), 0)


def _dense(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def paged_attention(q, k_pages, v_pages, table, positions, window: int = 0, sinks: int = 0, scale: float | None = None):
    """Causal attention of rotated queries q [B, T, H * D] at ``positions`` int64 [B, T] over the sequences' pages, which hold
    the tokens' own keys and values already (:func:`paged_rope_write`); returns [B, T, H * D].

    A token at position p sees the keys j <= p whose page is there, with ``window`` > 0 only those with j > p - window or
    j < sinks. A token that sees none, or whose position is outside the table (-1 for padding), gets zeros. ``scale`` is
    D ** -0.5 unless given."""
    what = "paged_attention"
    if _native_attention is not None and q.is_cuda and _only_eager(q, k_pages, v_pages, table, positions):
        out = _native_attention(q, k_pages, v_pages, table, positions, window, sinks, scale)
        if out is not None:
            return out
    B, T, N, KV, S, D = _check_pages(what, k_pages, v_pages, table, positions, q.dtype, q.device)
    if q.dim() != 3 or q.shape[:2] != positions.shape or q.shape[2] % (KV * D) or q.shape[2] == 0:
        raise ValueError(f"{what}: q {tuple(q.shape)} does not fit {B} x {T} tokens and pages of {KV} heads of {D}")
    if window < 0 or sinks < 0:
        raise ValueError(f"{what}: negative window ({window}) or sinks ({sinks})")
    H = q.shape[2] // D
    scale = D ** -0.5 if scale is None else scale
    if (q.is_cuda and q.dtype in _HALF and (D == 128 or D == 64) and S % 16 == 0
            and _only_eager(q, positions, k_pages, v_pages, table) and _pool_fits(k_pages, v_pages)
            and table.shape[1] * S <= 1 << 30):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if out.numel() == 0:
            return out
        q, qs = _rows(q, B, T)
        table, positions = _table_rows(table), positions.contiguous()
        lib = _lib.load()
        nbytes = lib.nq_paged_attention_workspace_bytes(B, T, H, KV, D, table.shape[1], S)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        _launch(what, lib.nq_paged_attention, q, _lib.dtype_code(q.dtype), q.data_ptr(), qs, k_pages.data_ptr(),
                v_pages.data_ptr(), N, S, table.data_ptr(), table.stride(0), table.shape[1], positions.data_ptr(),
                out.data_ptr(), B, T, H, KV, D, window, sinks, scale, _lib.ptr(ws), nbytes)
        return out
    if q.device.type in ("cpu", "cuda") and torch.is_autocast_enabled(q.device.type):  # which would round the products' operands
        with torch.autocast(q.device.type, enabled=False):
            return paged_attention(q, k_pages, v_pages, table, positions, window, sinks, scale)
    wide = torch.promote_types(q.dtype, torch.float32)
    P = table.shape[1]
    page = table.long()
    there = (page >= 0) & (page < N)
    page = torch.where(there, page, 0)
    key = torch.arange(P * S, device=q.device)
    p = positions.view(B, T, 1)
    seen = (key <= p) & (p < P * S) & there.repeat_interleave(S, dim=1).unsqueeze(1)  # [B, T, L]
    if window:
        seen = seen & ((key > p - window) | (key < sinks))
    seen = seen.view(B, 1, 1, T, P * S)
    k = k_pages[page].transpose(1, 2).reshape(B, KV, 1, P * S, D).to(wide)
    v = v_pages[page].transpose(1, 2).reshape(B, KV, 1, P * S, D).to(wide)
    qg = q.reshape(B, T, KV, H // KV, D).permute(0, 2, 3, 1, 4).to(wide)  # [B, KV, G, T, D]
    if _only_eager(q, k_pages, v_pages, table, positions):
        scores = torch.matmul(qg, k.transpose(-1, -2).contiguous()) * scale
    else:
        # 0 * NaN again, in the gradients: queries of tokens that see nothing are none, and the products that are
        # differentiated take the finite keys; scores of the others are constants, for the tokens that see them
        qg = torch.where(seen.any(dim=-1, keepdim=True), qg, 0.0)
        finite = torch.isfinite(k)
        scores = torch.matmul(qg, torch.where(finite, k, 0.0).transpose(-1, -2).contiguous()) * scale
        other = torch.matmul(qg.detach(), k.detach().transpose(-1, -2).contiguous()) * scale
        scores = torch.where(finite.all(dim=-1).unsqueeze(-2), scores, other)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    # 0 * inf would reach tokens that do not see it: products with the finite values, then what the others make of the sums
    # of the tokens that do
    o = torch.matmul(e, torch.where(torch.isfinite(v), v, 0.0))
    up, down, nan = (torch.matmul(seen.float(), kind.float()) > 0 for kind in (v == math.inf, v == -math.inf, torch.isnan(v)))
    o = torch.where(up, math.inf, torch.where(down, -math.inf, o))
    o = torch.where(nan | (up & down), math.nan, o)
    total = e.sum(dim=-1, keepdim=True)
    o = torch.where(total == 0.0, 0.0, o / torch.where(total == 0.0, 1.0, total))  # 0 / 0 would have NaN for a gradient
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H * D).to(q.dtype)


def paged_rotary_attention(shape, layer: int, q, k, v, cos, sin, positions, cache: PagedKVCache):
    """A layer's attention between the q, k and v projections and o_proj: rotary embedding, write into the pages and
    attention over them under the cache's window and sinks. Arguments as :func:`paged_rope_write`; returns [B, T, H * D]."""
    k_pages, v_pages = cache.k[layer], cache.v[layer]
    dtype = k_pages.dtype
    q = paged_rope_write(q.to(dtype), k.to(dtype), v.to(dtype), cos, sin, positions, k_pages, v_pages, cache.table)
    return paged_attention(q, k_pages, v_pages, cache.table, positions, cache.window, cache.sinks, shape.head_dim ** -0.5)


# ------------------------------------------------------------------------------------- drafted tokens

def _logit_rows(x):
    """x [batch, rows, vocab] as evenly spaced rows, and the elements between two: itself, or a copy. The stride of a dimension
    of one element says nothing, and ``contiguous`` leaves it as it is."""
    batch, rows, vocab = x.shape
    stride = x.stride(1) if rows > 1 else x.stride(0) if batch > 1 else vocab
    if x.stride(2) != 1 or stride < vocab or (rows > 1 and batch > 1 and x.stride(0) != rows * stride):
        x = torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
        stride = vocab
    return x, stride


def verify_drafts(logits, drafts, uniforms, draft_probs=None, temperature: float = 1.0):
    """Keep or turn down drafted tokens so that what comes out is distributed as the model's own tokens.

    logits [B, n + 1, vocab] (float32, float16 or bfloat16; strided rows are fine): the model's after 0 .. n drafts;
    drafts int64 [B, n], the first entry outside the vocabulary (-1) ends a sequence's; uniforms float32 [B, n + 1] in [0, 1);
    draft_probs float32 [B, n, vocab]: the distributions that the drafts were drawn from, None where they were chosen
    without chance (a greedy drafter, a lookup). Returns ``(accepted [B], tokens [B, n + 1])``, both int64: the number of
    drafts kept, and those drafts, one token more, and -1 behind.

    With p = softmax(logits / temperature) (temperature 0: 1 at the first largest logit), draft i is kept while
    uniforms[i] * q_i(draft) < p_i(draft). The token more is the first index at which the running sum of w passes
    uniforms[n] times its total: w = max(p - q, 0) where a draft was turned down (p where that is zero), else p. A row with a
    NaN or an infinite largest logit turns its draft down and gives its argmax. Probabilities and sums are float64."""
    what = "verify_drafts"
    given = (logits, drafts, uniforms) if draft_probs is None else (logits, drafts, uniforms, draft_probs)
    if _native_verify is not None and logits.is_cuda and _only_eager(*given):
        out = _native_verify(logits, drafts, uniforms, draft_probs, temperature)
        if out:
            return tuple(out)
    if logits.dim() != 3 or drafts.dim() != 2 or logits.shape[0] != drafts.shape[0] or logits.shape[1] != drafts.shape[1] + 1:
        raise ValueError(f"{what}: logits must be [batch, drafts + 1, vocab] and drafts [batch, drafts], got "
                         f"{tuple(logits.shape)} and {tuple(drafts.shape)}")
    B, n = drafts.shape
    V = logits.shape[2]
    if V == 0 or tuple(uniforms.shape) != (B, n + 1) or (draft_probs is not None and tuple(draft_probs.shape) != (B, n, V)):
        raise ValueError(f"{what}: uniforms {tuple(uniforms.shape)} must be [{B}, {n + 1}] and draft_probs "
                         f"{None if draft_probs is None else tuple(draft_probs.shape)} [{B}, {n}, vocab {V}]")
    if (logits.dtype not in (torch.float32, *_HALF) or drafts.dtype != torch.int64 or uniforms.dtype != torch.float32
            or (draft_probs is not None and draft_probs.dtype != torch.float32)):
        raise TypeError(f"{what}: logits float32, float16 or bfloat16, drafts int64, uniforms and draft_probs float32")
    if not 0.0 <= temperature < math.inf:
        raise ValueError(f"{what}: the temperature must be a finite number from 0, got {temperature}")
    for t in given:
        if t.device != logits.device:
            raise ValueError(f"{what}: tensors on {t.device} and {logits.device}")
    if logits.is_cuda and V <= 1 << 30 and _only_eager(*given):
        accepted = torch.empty(B, dtype=torch.int64, device=logits.device)
        tokens = torch.empty(B, n + 1, dtype=torch.int64, device=logits.device)
        if B == 0:
            return accepted, tokens
        logits, stride = _logit_rows(logits)
        drafts, uniforms = drafts.contiguous(), uniforms.contiguous()
        if draft_probs is not None:
            draft_probs = draft_probs.contiguous()
        lib = _lib.load()
        nbytes = lib.nq_verify_drafts_workspace_bytes(B, n, V)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=logits.device)
        code = _lib.NQ_F32 if logits.dtype == torch.float32 else _lib.dtype_code(logits.dtype)
        _launch(what, lib.nq_verify_drafts, logits, code, logits.data_ptr(), stride, drafts.data_ptr(),
                _lib.ptr(draft_probs), uniforms.data_ptr(), temperature, accepted.data_ptr(), tokens.data_ptr(), B, n, V,
                ws.data_ptr(), nbytes)
        return accepted, tokens
    x, u = logits.double(), uniforms.double()
    top = x.amax(dim=-1, keepdim=True)  # NaN where the row has one
    best = x.argmax(dim=-1, keepdim=True)
    plain = torch.isfinite(top) if temperature else torch.zeros_like(top, dtype=torch.bool)
    # finite, so that 0 stays 0: two logits that differ are 2^-149 apart at least, far enough for any such temperature
    factor = min(1.0 / temperature, sys.float_info.max) if temperature else 1.0
    e = torch.exp((x - torch.where(plain, top, 0.0)) * factor)
    p = torch.where(plain, e / e.sum(dim=-1, keepdim=True), torch.zeros_like(e).scatter_(2, best, 1.0))
    real = (drafts >= 0) & (drafts < V)
    at = torch.where(real, drafts, 0).unsqueeze(-1)
    if draft_probs is None or not temperature:
        q = torch.zeros_like(p[:, :n]).scatter_(2, at, 1.0)
    else:
        q = draft_probs.double()
    sound = torch.isfinite(top[:, :n, 0])
    keep = real & sound & (u[:, :n] * q.gather(2, at)[..., 0] < p[:, :n].gather(2, at)[..., 0])
    accepted = keep.long().cumprod(dim=1).sum(dim=1)
    row = accepted.view(B, 1, 1)
    chosen = p.gather(1, row.expand(B, 1, V))[:, 0]
    q = torch.where(real.unsqueeze(-1), q, 0.0)  # where the drafts ended without one turned down: p itself
    q = torch.cat((q, torch.zeros_like(p[:, :1])), dim=1).gather(1, row.expand(B, 1, V))[:, 0]
    left = (chosen - q).clamp(min=0.0)
    left = torch.where(plain.gather(1, row)[:, 0] & (left.sum(dim=-1, keepdim=True) > 0.0), left, chosen)
    sums = left.cumsum(dim=-1)
    passed = (sums > u[:, n:] * sums[:, -1:]) & (left > 0.0)
    last = V - 1 - (left.flip(-1) > 0.0).int().argmax(dim=-1)  # where rounding hides the total
    token = torch.where(passed.any(dim=-1), passed.int().argmax(dim=-1), last).unsqueeze(-1)
    index = torch.arange(n + 1, device=logits.device)
    tokens = torch.cat((drafts, torch.full_like(token, -1)), dim=1)
    return accepted, torch.where(index < row[:, 0], tokens, torch.where(index == row[:, 0], token, -1))
