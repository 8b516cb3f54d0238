"""What serving many sequences at once needs beyond one static cache: a KV cache in pages, each sequence at a length of its
own, several answers to one prompt, the check of drafted tokens and the scores of given ones.

* :class:`PagedKVCache` holds the pools and the page table; ``NanoQuantLlama.forward`` takes it in place of a
  ``StaticKVCache``, with positions [B, T].
* :func:`paged_rope_write` rotates the new tokens' queries and keys and writes keys and values into the pages.
* :func:`paged_attention` is causal attention over the pages, for one new token a sequence, drafted tokens, prompts and
  chunks of prompts, optionally under a sliding window with a few first tokens that stay visible.
* :func:`paged_shared_attention` is the same for sequences of which groups have their leading pages in common, which
  :meth:`PagedKVCache.fork` makes; those keys and values are read once a group.
* :func:`copy_pages` copies pages within the pools of every layer.
* :func:`verify_drafts` keeps or turns down drafted tokens by the model's logits and given random numbers.
* :func:`token_logprobs` gives the log probabilities of given tokens, the entropy and the most probable alternatives.

Calls of well-laid-out tensors on the GPU go through the C++ of ``libnq_ops.so`` (``csrc/torch_ops/nq_ops.cpp``): a small call
is bound by its host path. What that does not take is checked, copied into place or refused here.

float16 and bfloat16 tensors on the GPU run the HIP library (``nq_paged_rope_write``, ``nq_paged_attention``,
``nq_verify_drafts``, ``nq_paged_shared_attention``, ``nq_copy_pages``, ``nq_token_logprobs``); CPU tensors, float32 models,
calls that are differentiated, head sizes other than 64 and 128 and page sizes that are no multiple of 16 run torch ops with the
same results but for rounding, in float32, or in float64 where the tensors are. Pages of any type are copied by the library,
and logits in float32 scored and verified by it. The reference has no counterpart: its harness decodes one batch on Hugging
Face's static cache and samples one token a step (``src/nanoquant/kernel/test_decode.py:350-422``).
"""
from __future__ import annotations

import ctypes
import math
import sys

import torch

from . import _lib
from ._dispatch import launch as _launch, only_eager as _only_eager, only_eager_many as _only_eager_many

_HALF = (torch.float16, torch.bfloat16)

_OPS = torch.library.Library("nanoquant_amd", "FRAGMENT")
for _schema in (
        "paged_rope_write(Tensor q, Tensor k, Tensor v, Tensor cos, Tensor sin, Tensor positions, Tensor(a!) k_pages, "
        "Tensor(b!) v_pages, Tensor table) -> Tensor?",
        "paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor positions, int window, int sinks, "
        "float? scale) -> Tensor?",
        "verify_drafts(Tensor logits, Tensor drafts, Tensor uniforms, Tensor? draft_probs, float temperature) -> Tensor[]",
        "paged_shared_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor positions, Tensor members, "
        "Tensor shared, int window, int sinks, float? scale) -> Tensor?",
        "copy_pages(Tensor(a!)[] pools, Tensor source, Tensor target) -> bool",
        "token_logprobs(Tensor logits, Tensor tokens, int top, float temperature) -> Tensor[]"):
    _OPS.define(_schema)


def _native(name):
    """The operator in C++, or None where ``libnq_ops.so`` is missing or older."""
    if _lib.ops is None or not torch._C._dispatch_has_kernel_for_dispatch_key(f"nanoquant_amd::{name}", "CUDA"):
        return None
    return getattr(torch.ops.nanoquant_amd, name).default


_native_write, _native_attention, _native_verify = (_native(n) for n in ("paged_rope_write", "paged_attention", "verify_drafts"))
_native_shared, _native_copy, _native_score = (_native(n) for n in ("paged_shared_attention", "copy_pages", "token_logprobs"))


# Bytes a layer, 0.2 us of reading, that sequences in two groups have to save beyond one: more groups than ever before take new
# tensors, and graphs captured earlier lose theirs. The attention's time goes by the keys, not by their groups: 48 sequences of 300
# keys behind 8192 shared ones in all, 32 heads, 85 us as one group, 83 as sixteen.
_WORTH_A_GROUP = 1 << 20


class PagedKVCache:
    """Per-layer K and V pools of ``pages`` pages of ``page_size`` positions, shared by ``batch`` sequences of up to
    ``max_len`` positions each, and the table that says where a sequence's positions lie.

    ``k[layer]`` and ``v[layer]`` are [pages, kv_heads, page_size, head_dim]; ``table`` is int32
    [batch, ceil(max_len / page_size)] on the device: position p of sequence b lies in page ``table[b, p // page_size]`` at row
    ``p % page_size``, and -1 is a page that is not there. The table's memory stays the same, so a captured graph follows its
    changes. ``window`` and ``sinks`` (0: none) are how the model's layers read the cache: a token sees the last ``window``
    positions and the first ``sinks``.

    ``reserve`` gives a sequence the pages that its next tokens need, ``trim`` takes back those that no later token will see,
    ``release`` all of them. ``fork`` lets sequences go on where another stands: they share its whole pages, which are counted
    and go back to the pool with the last that has them, and ``own`` gives a sequence copies of shared pages before something is
    written there. ``compact`` moves the pages that are in use to the front of the pools. A program may also fill the table
    itself, and then uses none of these: they write a sequence's row as they know it. Serve under ``torch.no_grad``, or what a
    model with gradients writes makes the pools part of its graph.

    ``members`` and ``shared`` (None before the first fork) say which sequences have their leading pages in common, as
    :func:`paged_shared_attention` takes it, and ``groups`` how many such groups there are; ``saved`` is what reading each
    group's pages once saves in a layer, in bytes. Their memory stays as long as no more groups and no larger ones come up than
    ever before, so a graph captured with the largest follows their changes; one captured before reads groups of nobody from
    then on, which is right, but reads each sequence's pages for itself. The model's layers use them from 100 MB saved on.
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
        self._owners = [0] * pages  # sequences that have a page
        self.members = self.shared = None
        self._outgrown = []  # those that graphs captured earlier read
        self.groups = self.saved = 0
        self._lists = []  # each group's sequences, and how many leading entries their rows have in common
        self._common = [0] * batch  # the same number, of a sequence's group
        self._missing = [0] * batch  # of those entries, the ones that the sequence has trimmed
        # Where a sequence's slots come from, trimmed ones too: (stretch, its end) one after the other. Slots of the same stretch
        # are the same page in every sequence that has one there. Stretches that sequences share end before ``_forked``
        self._stretches = batch
        self._lines = [[(b, self.max_pages)] for b in range(batch)]
        self._forked = [0] * batch

    def _row(self, sequence: int):
        if not 0 <= sequence < self.batch:
            raise IndexError(f"sequence {sequence} of {self.batch}")
        return self._host[sequence]

    def _store(self, sequence: int):
        self.table[sequence].copy_(torch.tensor(self._host[sequence], dtype=torch.int32))

    def _take(self) -> int:
        page = self._free.pop()
        self._owners[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._owners[page] -= 1
        if self._owners[page] == 0:
            self._free.append(page)

    def _copy(self, moves) -> None:
        source, target = torch.tensor(moves, dtype=torch.int32).t().contiguous().to(self.table.device).unbind(0)
        copy_pages([*self.k, *self.v], source, target)

    def _branch(self, sequence: int, line, slot: int) -> None:
        """The sequence's slots are those of ``line`` before ``slot`` and its own from there on."""
        kept, at = [], 0
        for stretch, end in line:
            if at < slot:
                at = min(end, slot)
                kept.append((stretch, at))
        self._lines[sequence] = [*kept, (self._stretches, self.max_pages)]
        self._stretches += 1
        self._forked[sequence] = slot

    def _reach(self, sequence: int, slots: int) -> int:
        """The sequence's last slot before ``slots`` that has a page, and one more."""
        row = self._host[sequence]
        while slots and row[slots - 1] < 0:
            slots -= 1
        return slots

    def _saves(self, common: int, missing) -> int:
        """Bytes a layer that reading the leading ``common`` slots once saves, of sequences that lack so many of them: what they
        still have, but for the one that has the most."""
        position = 2 * self.k[0][0, :, 0].numel() * self.k[0].element_size() if self.k else 0
        most = self.window + self.sinks if self.window else self.max_len
        seen = [min((common - n) * self.page_size, most) for n in missing]
        return position * (sum(seen) - max(seen))

    def _together(self, sequences, slots: int):
        """(bytes saved, groups, sequences in none) of sequences whose rows are alike before ``slots``: one group over what all
        of them still have some of, or two where some have no more than the first pages left and that costs the others much."""
        reach = {b: self._reach(b, slots) for b in sequences}
        best = (0, [], sequences)
        for least in sorted(set(reach.values()) - {0}):
            lists = [[b for b in sequences if reach[b] >= least], [b for b in sequences if 0 < reach[b] < least]]
            groups = [(x, min(reach[b] for b in x)) for x in lists if len(x) > 1]
            saved = sum(self._saves(n, [self._host[b][:n].count(-1) for b in x]) for x, n in groups)
            if groups and (not best[1] or saved >= best[0] + _WORTH_A_GROUP):
                best = (saved, groups, [b for b in sequences if not any(b in x for x, _ in groups)])
        return best

    def _regroup(self) -> None:
        """``members`` and ``shared`` of the sequences whose rows begin alike: all that do in one group, over the slots that all
        have in common, or in several where parts of them have so much more in common that it saves more. A slot that a sequence
        has trimmed is behind its window and so counts as alike."""
        self._lists = []
        part = None  # of the sequences in the lines' order: (sequences, bytes saved, groups, sequences in none)
        above = []   # (slots that some sequences have in common, their parts so far), from the fewest slots on
        before = []
        for line, b in sorted((self._lines[b], b) for b in range(self.batch) if self._forked[b]) + [([], -1)]:
            common = _alike(before, line)
            while above and above[-1][0] > common:
                slots, parts = above.pop()
                parts.append(part)
                everyone, groups, alone = (sum((p[i] for p in parts), []) for i in (0, 2, 3))
                best = self._together(everyone, slots)
                if groups:  # of the parts, and of those that are in none of them
                    saved, more, alone = self._together(alone, slots)
                    saved += sum(p[1] for p in parts)
                    if not best[1] or saved >= best[0] + _WORTH_A_GROUP:
                        best = (saved, groups + more, alone)
                part = (everyone, *best)
            if common == 0:
                self._lists += part[2] if part else []
            elif above and above[-1][0] == common:
                above[-1][1].append(part)
            else:
                above.append((common, [part]))
            part, before = ([b], 0, [], [b]), line
        self._common = [0] * self.batch
        for i, (sequences, common) in enumerate(self._lists):
            for b in sequences:
                self._common[b] = common
                self._missing[b] = self._host[b][:common].count(-1)
            self._lists[i] = (sorted(sequences, key=self._lead), common)
        self._add_up()
        self._lists.sort(key=lambda x: min(x[0]))
        lists, shared = [sequences for sequences, _ in self._lists], [common for _, common in self._lists]
        self.groups = len(lists)
        most = max(map(len, lists), default=0)
        if self.members is None or self.members.shape[0] < len(lists) or self.members.shape[1] < most:
            old = (0, 0) if self.members is None else self.members.shape
            shape = (max(old[0], len(lists)), max(old[1], most))
            if self.members is not None:
                self._outgrown.append((self.members.fill_(-1), self.shared.zero_()))
            with torch.inference_mode(False):  # as the table's, whose changes may come outside it
                self.members = torch.empty(shape, dtype=torch.int32, device=self.table.device)
                self.shared = torch.empty(shape[0], dtype=torch.int32, device=self.table.device)
        groups, most = self.members.shape
        lists += [[]] * (groups - len(lists))
        self.members.copy_(torch.tensor([x + [-1] * (most - len(x)) for x in lists], dtype=torch.int32).view(groups, most))
        self.shared.copy_(torch.tensor(shared + [0] * (groups - len(shared)), dtype=torch.int32))

    def _add_up(self) -> None:
        self.saved = sum(self._saves(common, [self._missing[b] for b in sequences]) for sequences, common in self._lists)

    def _lead(self, sequence: int):
        """The order of a group: what a sequence has, those behind it have no more of, so its row serves for theirs. (Trimmed slots
        begin where the sinks end in every row.)"""
        return self._missing[sequence], sequence

    def _reorder(self, sequence: int) -> None:
        """The groups after the sequence has trimmed some of the slots in common. While it has the last of them, only its place
        changes: 128 answers that trim one after the other would spend most of a step in ``_regroup``."""
        common = self._common[sequence]
        if self._host[sequence][common - 1] < 0:
            self._regroup()
            return
        at = next(i for i, (sequences, _) in enumerate(self._lists) if sequence in sequences)
        sequences = self._lists[at][0]
        self._missing[sequence] = self._host[sequence][:common].count(-1)
        self._add_up()
        order = sorted(sequences, key=self._lead)
        if order != sequences:
            sequences[:] = order
            self.members[at, :len(order)].copy_(torch.tensor(order, dtype=torch.int32))

    def reserve(self, sequence: int, length: int, start: int = 0) -> None:
        """Pages for the sequence's positions ``start`` to ``length - 1`` (those it has stay, shared ones too: a sequence that
        was set back needs ``own`` before it writes there). RuntimeError, and no change, where the pool has too few left."""
        row = self._row(sequence)
        if not 0 <= start <= length <= self.max_len:
            raise ValueError(f"positions {start} to {length} do not fit max_len {self.max_len}")
        need = [i for i in range(start // self.page_size, -(-length // self.page_size)) if row[i] < 0]
        if len(need) > len(self._free):
            raise RuntimeError(f"the paged cache has {len(self._free)} pages left, sequence {sequence} needs {len(need)}")
        for i in need:
            row[i] = self._take()
        if need:
            self._store(sequence)
            if need[0] < self._forked[sequence]:
                self._branch(sequence, self._lines[sequence], need[0])
                self._regroup()

    def _take_back(self, sequence: int, slots) -> int:
        row = self._row(sequence)
        gone = [i for i in slots if row[i] >= 0]
        for i in gone:
            self._drop(row[i])
            row[i] = -1
        if gone:
            self._store(sequence)
        return len(gone)

    def trim(self, sequence: int, position: int) -> int:
        """Take back the pages that no token from ``position`` on sees under the window; returns their number. Groups last as
        long as their members still have some of the pages in common. Calls in flight on other streams must have ended."""
        if self.window == 0:
            return 0
        first = min(max(0, position - self.window + 1) // self.page_size, self.max_pages)
        sinks = -(-self.sinks // self.page_size)
        gone = self._take_back(sequence, range(sinks, first))
        if gone and sinks < self._common[sequence]:
            self._reorder(sequence)
        return gone

    def release(self, sequence: int) -> int:
        """Take back all pages of a sequence (those that others share stay theirs); returns their number. Calls in flight on
        other streams must have ended."""
        gone = self._take_back(sequence, range(self.max_pages))
        if self._forked[sequence]:
            self._branch(sequence, [], 0)
            self._regroup()
        return gone

    def fork(self, source: int, targets, length: int) -> None:
        """The sequences ``targets``, which have no pages, get the first ``length`` positions of ``source``: its whole pages as
        they are, shared from now on, and a copy each of the page that ``length`` ends in. What is shared is only read: see
        ``own``. RuntimeError, and no change, where the pool has too few pages left."""
        row, targets = self._row(source), list(targets)
        if not 0 <= length <= self.max_len:
            raise ValueError(f"{length} positions do not fit max_len {self.max_len}")
        if len(set(targets)) != len(targets) or source in targets or any(page >= 0 for b in targets for page in self._row(b)):
            raise ValueError(f"sequences {targets} must be others than {source}, named once and without pages")
        whole = length // self.page_size
        split = length % self.page_size > 0 and row[whole] >= 0
        if split and len(targets) > len(self._free):
            raise RuntimeError(f"the paged cache has {len(self._free)} pages left, {len(targets)} forks need one each")
        moves = []
        pages = [self._free[-1 - i] for i in range(len(targets))] if split else []  # those that will be taken
        if pages:
            self._copy([(row[whole], page) for page in pages])
        for b in targets:
            self._host[b][:whole] = row[:whole]
            for page in row[:whole]:
                if page >= 0:
                    self._owners[page] += 1
            if split:
                self._host[b][whole] = self._take()
            self._store(b)
            self._branch(b, self._lines[source], whole)
        if targets:
            self._forked[source] = max(self._forked[source], whole)
        self._regroup()

    def own(self, sequence: int, length: int, start: int) -> int:
        """Pages of the sequence alone, with the same contents, in place of those of positions ``start`` to ``length - 1`` that
        others have too, so that it may write there (a sequence set back before the position that it was forked at); returns
        their number. RuntimeError, and no change, where the pool has too few pages left."""
        row = self._row(sequence)
        if not 0 <= start <= length <= self.max_len:
            raise ValueError(f"positions {start} to {length} do not fit max_len {self.max_len}")
        slots = range(start // self.page_size, -(-length // self.page_size))
        shared = [i for i in slots if row[i] >= 0 and self._owners[row[i]] > 1]
        if len(shared) > len(self._free):
            raise RuntimeError(f"the paged cache has {len(self._free)} pages left, sequence {sequence} needs {len(shared)}")
        if shared:
            self._copy([(row[i], self._free[-1 - k]) for k, i in enumerate(shared)])  # those that will be taken
            for i in shared:
                page = self._take()
                self._drop(row[i])
                row[i] = page
            self._store(sequence)
            self._branch(sequence, self._lines[sequence], shared[0])
            self._regroup()
        return len(shared)

    def compact(self) -> int:
        """Move the pages that are in use to the front of the pools; returns their number, which is the first page that is not.
        Calls in flight on other streams must have ended."""
        used = self.pages - len(self._free)
        holes = [page for page in range(used) if self._owners[page] == 0]
        moved = dict(zip((page for page in range(used, self.pages) if self._owners[page]), holes))
        if moved:
            self._copy(list(moved.items()))
            for page, to in moved.items():
                self._owners[to], self._owners[page] = self._owners[page], 0
            for row in self._host:
                row[:] = [moved.get(page, page) for page in row]
            self._free = list(range(self.pages - 1, used - 1, -1))
            self.table.copy_(torch.tensor(self._host, dtype=torch.int32))
        return used


def _alike(line, other) -> int:
    """How many leading slots two of ``PagedKVCache._lines`` have in common."""
    common = 0
    for (stretch, end), (other_stretch, other_end) in zip(line, other):
        if stretch != other_stretch:
            break
        common = min(end, other_end)
        if end != other_end:
            break
    return common


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


def paged_shared_attention(q, k_pages, v_pages, table, positions, members, shared, window: int = 0, sinks: int = 0,
                           scale: float | None = None):
    """:func:`paged_attention` of sequences of which groups have their leading pages in common (answers to one prompt):
    ``members`` int32 [groups, most] are the sequences of each group (entries outside the batch, as -1, are nobody), whose rows
    of the table begin with the same ``shared`` (int32 [groups]) entries; see :meth:`PagedKVCache.fork`. Those pages are read
    once a group. A sequence in no group is on its own; of one that is named twice the last place counts. Where members' rows
    do not begin alike, their results mean nothing; but a row may lack pages that its window is past (-1), and then stands
    behind those of the group that have them.

    Other arguments and the result, but for rounding, are :func:`paged_attention`'s, which also takes the calls that the kernel
    does not: those that run torch ops, small ones, many tokens a sequence (prompts), and batches past about a thousand sequences
    (``nq_paged_shared_attention`` says where). It pays from about 100 MB of keys and values that are not read again."""
    what = "paged_shared_attention"
    given = (q, k_pages, v_pages, table, positions, members, shared)
    if _native_shared is not None and q.is_cuda and _only_eager(*given):
        out = _native_shared(*given, window, sinks, scale)
        if out is not None:
            return out
    if members.dim() != 2 or shared.dim() != 1 or members.shape[0] != shared.shape[0]:
        raise ValueError(f"{what}: members must be [groups, most] and shared [groups], got {tuple(members.shape)} and "
                         f"{tuple(shared.shape)}")
    if members.dtype != torch.int32 or shared.dtype != torch.int32:
        raise TypeError(f"{what}: members and shared must be int32, got {members.dtype} and {shared.dtype}")
    for t in (members, shared):
        if t.device != q.device:
            raise ValueError(f"{what}: tensors on {t.device} and {q.device}")
    B, T, N, KV, S, D = _check_pages(what, k_pages, v_pages, table, positions, q.dtype, q.device)
    if q.dim() != 3 or q.shape[:2] != positions.shape or q.shape[2] % (KV * D) or q.shape[2] == 0:
        raise ValueError(f"{what}: q {tuple(q.shape)} does not fit {B} x {T} tokens and pages of {KV} heads of {D}")
    if window < 0 or sinks < 0:
        raise ValueError(f"{what}: negative window ({window}) or sinks ({sinks})")
    if (q.is_cuda and q.dtype in _HALF and (D == 128 or D == 64) and S % 16 == 0 and members.numel() and q.numel()
            and _only_eager(*given) and _pool_fits(k_pages, v_pages) and table.shape[1] * S <= 1 << 30):
        lib = _lib.load()
        nbytes = lib.nq_paged_shared_attention_workspace_bytes(B, T, q.shape[2] // D, KV, D, table.shape[1], S, *members.shape)
        if nbytes:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            q, qs = _rows(q, B, T)
            table, positions = _table_rows(table), positions.contiguous()
            members, shared = members.contiguous(), shared.contiguous()
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            _launch(what, lib.nq_paged_shared_attention, q, _lib.dtype_code(q.dtype), q.data_ptr(), qs, k_pages.data_ptr(),
                    v_pages.data_ptr(), N, S, table.data_ptr(), table.stride(0), table.shape[1], positions.data_ptr(),
                    members.data_ptr(), shared.data_ptr(), *members.shape, out.data_ptr(), B, T, q.shape[2] // D, KV, D, window,
                    sinks, D ** -0.5 if scale is None else scale, ws.data_ptr(), nbytes)
            return out
    return paged_attention(q, k_pages, v_pages, table, positions, window, sinks, scale)


def copy_pages(pools, source, target) -> None:
    """Copy page ``source[i]`` over page ``target[i]`` in each of ``pools``, tensors [pages, ...] alike in shape and type (the
    keys' and values' of every layer). source and target are int32 [moves] on the pools' device; a pair with a page that is not
    there (-1) is passed over. No page may be the target of two pairs, or the target of one and the source of another."""
    what = "copy_pages"
    pools = list(pools)
    eager = _only_eager_many(pools, source, target)
    if _native_copy is not None and eager and source.is_cuda and _native_copy(pools, source, target):
        return
    if source.dim() != 1 or target.shape != source.shape:
        raise ValueError(f"{what}: source and target must be [moves], got {tuple(source.shape)} and {tuple(target.shape)}")
    if source.dtype != torch.int32 or target.dtype != torch.int32:
        raise TypeError(f"{what}: source and target must be int32, got {source.dtype} and {target.dtype}")
    for t in (target, *pools):
        if t.device != source.device:
            raise ValueError(f"{what}: tensors on {t.device} and {source.device}")
    for pool in pools:
        if pool.dim() == 0 or pool.shape != pools[0].shape or pool.dtype != pools[0].dtype:
            raise ValueError(f"{what}: pools must be alike, got {tuple(pool.shape)} of {pool.dtype} and "
                             f"{tuple(pools[0].shape)} of {pools[0].dtype}")
    if not pools or pools[0].numel() == 0 or source.numel() == 0:
        return
    pages = pools[0].shape[0]
    if source.is_cuda and eager and all(pool.is_contiguous() for pool in pools):
        source, target = source.contiguous(), target.contiguous()
        at = (ctypes.c_void_p * len(pools))(*(pool.data_ptr() for pool in pools))
        _launch(what, _lib.load().nq_copy_pages, source, at, len(pools), pages, pools[0].nbytes // pages, source.data_ptr(),
                target.data_ptr(), source.shape[0])
        return
    there = ((source >= 0) & (source < pages) & (target >= 0) & (target < pages)).nonzero()[:, 0]
    source, target = source[there].long(), target[there].long()
    for pool in pools:
        pool[target] = pool[source]


# Bytes that groups save in a layer, from which the attention over shared pages is the faster one. Its beginning and its join take
# up to 10 us more, and what the plain one reads again comes in part from caches. Captured steps over many layers, us with and
# without groups, 64 heads of 8 kv heads of 128: 2 sequences in 16000 shared keys (66 MB) 28.9 and 23.5, 100 in 250 (97) 29.4 and
# 22.8, 8 in 4000 (115) 24.8 and 29.2, 16 in 4000 (246) 26.5 and 43.4; heads of 64, 40 in 1000 (79) 19.1 and 16.6, 16 in 4000 (123)
# 19.4 and 26.1; 32 kv heads, 2 in 4000 (66) 24.8 and 29.7, 8 in 1000 (114) 18.2 and 19.7. Past it still slower: 40 in 1000 (158)
# 25.1 and 21.4, 4 in 16000 (197) 32.4 and 28.4.
_WORTH_SHARING = 100 << 20


def paged_rotary_attention(shape, layer: int, q, k, v, cos, sin, positions, cache: PagedKVCache):
    """A layer's attention between the q, k and v projections and o_proj: rotary embedding, write into the pages and
    attention over them under the cache's window and sinks, shared pages read once a group. Arguments as
    :func:`paged_rope_write`; returns [B, T, H * D]."""
    k_pages, v_pages = cache.k[layer], cache.v[layer]
    dtype = k_pages.dtype
    q = paged_rope_write(q.to(dtype), k.to(dtype), v.to(dtype), cos, sin, positions, k_pages, v_pages, cache.table)
    if cache.groups and cache.saved >= _WORTH_SHARING:
        return paged_shared_attention(q, k_pages, v_pages, cache.table, positions, cache.members, cache.shared, cache.window,
                                      cache.sinks, shape.head_dim ** -0.5)
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


# ------------------------------------------------------------------------------------- scored tokens

_TEMPERATURES = (2.0 ** -64, 2.0 ** 64)  # that float32 exponents have room for


def token_logprobs(logits, tokens, top: int = 0, temperature: float = 1.0):
    """What p = softmax(logits / temperature) says of given tokens.

    logits [rows, vocab] or [B, T, vocab] (any strides with the vocabulary's elements side by side, as of ``logits[:, :-1]``;
    float32, float16, bfloat16, or float64 by torch ops), tokens int64 [rows] or [B, T]. Returns ``(logprobs, entropy,
    top_tokens, top_logprobs)``: log p of the given token, 0 for one outside the vocabulary (-1 for padding); -sum p log p; the
    ``top`` largest logits' indexes [..., top], the lowest first of equal ones, and their log p. In float32 (float64 for float64
    logits). A logit of -inf has no part in the sums. In a row with a NaN, or whose largest logit is infinite, log p and the
    entropy are NaN, and a NaN counts as the largest logit."""
    what = "token_logprobs"
    if _native_score is not None and logits.is_cuda and _only_eager(logits, tokens):
        out = _native_score(logits, tokens, top, temperature)
        if out:
            return tuple(out)
    if logits.dim() not in (2, 3) or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: logits must be [rows, vocab] or [B, T, vocab] and tokens like them without vocab, got "
                         f"{tuple(logits.shape)} and {tuple(tokens.shape)}")
    if logits.dtype not in (torch.float32, torch.float64, *_HALF) or tokens.dtype != torch.int64:
        raise TypeError(f"{what}: logits float32, float64, float16 or bfloat16 and tokens int64, got {logits.dtype} and "
                        f"{tokens.dtype}")
    if tokens.device != logits.device:
        raise ValueError(f"{what}: tensors on {tokens.device} and {logits.device}")
    V = logits.shape[-1]
    if V == 0 or not 0 <= top <= V:
        raise ValueError(f"{what}: {top} alternatives of {V} tokens")
    if not 0.0 < temperature < math.inf:
        raise ValueError(f"{what}: the temperature must be a finite number above 0, got {temperature}")
    shape, kind = tokens.shape, torch.promote_types(logits.dtype, torch.float32)
    usual = _TEMPERATURES[0] <= temperature <= _TEMPERATURES[1]
    if (logits.is_cuda and kind == torch.float32 and top <= 64 and V <= 1 << 30 and usual and 0 < tokens.numel() < 1 << 23
            and _only_eager(logits, tokens)):
        rows = logits if logits.dim() == 3 else logits.unsqueeze(0)
        B, T = rows.shape[:2]
        if (V > 1 and rows.stride(2) != 1) or (T > 1 and rows.stride(1) < V) or (B > 1 and rows.stride(0) < V):
            rows = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device).copy_(rows)
        at = tokens if tokens.dim() == 2 else tokens.unsqueeze(0)
        lib = _lib.load()
        nbytes = lib.nq_token_logprobs_workspace_bytes(B, T, V, top)
        logprobs, entropy = torch.empty(2, *shape, dtype=kind, device=logits.device).unbind(0)
        top_tokens = torch.empty(*shape, top, dtype=torch.int64, device=logits.device)
        top_logprobs = torch.empty(*shape, top, dtype=kind, device=logits.device)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=logits.device) if nbytes else None
        code = _lib.NQ_F32 if logits.dtype == torch.float32 else _lib.dtype_code(logits.dtype)
        _launch(what, lib.nq_token_logprobs, logits, code, rows.data_ptr(), rows.stride(0), rows.stride(1), at.data_ptr(),
                at.stride(0), at.stride(1), temperature, top, logprobs.data_ptr(), entropy.data_ptr(), top_tokens.data_ptr(),
                top_logprobs.data_ptr(), B, T, V, _lib.ptr(ws), nbytes)
        return logprobs, entropy, top_tokens, top_logprobs
    x = logits.to(kind if usual else torch.float64)
    d = (x - x.detach().amax(dim=-1, keepdim=True)) / temperature
    e = torch.exp(d)
    total = e.sum(dim=-1)
    log_total = torch.log(total)
    there = (tokens >= 0) & (tokens < V)
    given = d.gather(-1, torch.where(there, tokens, 0).unsqueeze(-1))[..., 0] - log_total
    entropy = log_total - (e * torch.where(d == -math.inf, 0.0, d)).sum(dim=-1) / total
    # an order that is stable gives the lowest index of equal logits, and a NaN comes first in it
    order = torch.sort(logits.detach(), dim=-1, descending=True, stable=True).indices[..., :top].contiguous()
    best = d.gather(-1, order) - log_total.unsqueeze(-1)
    return torch.where(there, given, 0.0).to(kind), entropy.to(kind), order, best.to(kind)
