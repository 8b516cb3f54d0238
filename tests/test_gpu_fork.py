"""Page copies, attention over shared pages and scored tokens against plain 64-bit forms (needs a gfx950 GPU)."""
import math

import pytest
import torch

import fork_oracle
import serve_oracle as oracle
from nanoquant_amd import (PagedKVCache, _lib, copy_pages, paged_attention, paged_shared_attention, serve, token_logprobs)
from nanoquant_amd.decode import LlamaShape, random_llama
from test_fork_host import odd_rows

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
IDS = ["f16", "bf16"]

# (heads, kv_heads, head_dim, page_size, groups, alone, tokens, window, sinks)
SHARED = [
    # two answers a few tokens in; a prompt of one page; answers that end around a tile and a page
    (4, 4, 128, 16, [(1, [1, 2])], [], 1, 0, 0),
    (8, 1, 128, 16, [(1, [1, 15, 16, 17]), (3, [31, 32, 33])], [1], 1, 0, 0),
    (5, 5, 64, 48, [(2, [1, 47, 49, 96])], [5, 300], 1, 0, 0),
    # prompts whose pages end inside a tile, many members, many query heads a kv head
    (16, 1, 64, 16, [(7, list(range(1, 34)))], [], 1, 0, 0),
    (8, 2, 128, 16, [(63, [3] * 40)], [1000], 1, 0, 0),
    (64, 2, 64, 16, [(5, [9, 40, 2])], [], 1, 0, 0),
    (20, 1, 128, 48, [(11, [100, 1, 7]), (1, [5, 5])], [], 1, 0, 0),
    (12, 4, 128, 64, [(30, [70, 300, 5, 5, 5]), (2, [1500, 1]), (17, [9])], [40, 600], 1, 0, 0),
    # a group of one member, and groups that share nothing
    (8, 2, 128, 32, [(4, [10])], [33], 1, 0, 0),
    (8, 2, 64, 32, [(0, [40, 50]), (2, [1, 1])], [], 1, 0, 0),
    # drafted tokens
    (4, 4, 128, 16, [(9, [5, 6, 7])], [3], 2, 0, 0),
    (8, 1, 128, 32, [(6, [5, 40, 9, 5])], [2], 5, 0, 0),
    (24, 1, 64, 64, [(8, [4, 9])], [], 3, 0, 0),
    (6, 2, 128, 16, [(20, [21, 22, 23, 24, 25, 26])], [], 8, 0, 0),
    (8, 4, 64, 16, [(3, [80, 90])], [], 33, 0, 0),
    # the most rows of a sequence that this kernel takes
    (24, 1, 64, 64, [(8, [4, 9])], [], 2, 0, 0),
    (8, 4, 64, 16, [(3, [80, 90])], [], 32, 0, 0),
    # windows: over the prompt's end, past it, with sinks in the prompt, through all of it, and behind it
    (8, 2, 128, 16, [(20, [5, 60, 140])], [90], 1, 100, 4),
    (4, 4, 64, 32, [(10, [33, 1, 200])], [], 1, 33, 40),
    (8, 1, 128, 48, [(2, [300, 20, 1])], [50], 1, 60, 100),
    (8, 2, 64, 16, [(3, [400, 390])], [], 1, 70, 60),
    (8, 2, 128, 16, [(13, [40, 7, 60])], [], 9, 60, 3),
    (4, 2, 128, 16, [(6, [1, 2])], [], 1, 1, 0),
]
ids = lambda c: "x".join(str(len(e) if isinstance(e, list) else e) for e in c)  # noqa: E731


def _check(y, ref, spread, dtype, keys):
    bound = oracle.attention_bound(ref, spread, dtype, keys)
    off = ((y.double().cpu() - ref).abs() / bound).max().item()
    assert off <= 1.0, f"{off:.2f} times the bound"


def _keys(table, k):
    """The most keys of a sequence."""
    return int((table >= 0).sum(dim=1).max()) * k.shape[2]


def shared_case(*sizes, **kw):
    """A case whose table is wide enough for the kernel of shared pages: smaller calls are the plain attention's."""
    return fork_oracle.shared_case(*sizes, **kw, read=1 << 27)


def attend(q, k, v, table, pos, members, shared, *args, **kw):
    """paged_shared_attention, of a call that its kernel takes unless a sequence has more than 64 rows a kv head."""
    B, T = pos.shape
    KV, S, D = k.shape[1:]
    H = q.shape[2] // D
    nbytes = _lib.load().nq_paged_shared_attention_workspace_bytes(B, T, H, KV, D, table.shape[1], S, *members.shape)
    assert (nbytes > 0) == (T * H // KV <= 64)
    return paged_shared_attention(q, k, v, table, pos, members, shared, *args, **kw)


@pytest.mark.parametrize("dtype", HALF, ids=IDS)
@pytest.mark.parametrize("case", SHARED, ids=ids)
def test_attention(case, dtype):
    *sizes, window, sinks = case
    q, k, v, table, pos, members, shared = shared_case(*sizes, dtype, "cuda")
    y = attend(q, k, v, table, pos, members, shared, window, sinks)
    ref, spread = oracle.attention(q, k, v, table, pos, window, sinks)
    _check(y, ref, spread, dtype, _keys(table, k))
    assert torch.equal(y[pos < 0], torch.zeros_like(y[pos < 0]))
    again = attend(q, k, v, table, pos, members, shared, window, sinks)
    assert torch.equal(y, again)


# long enough that several blocks share a group's keys, and a sequence's
@pytest.mark.parametrize("case", [(8, 2, 128, 16, [(500, [30, 700])], [], 1), (16, 2, 64, 64, [(90, [2000] + [11] * 20)], [4000], 1),
                                  (8, 8, 128, 32, [(100, [900, 40, 7]), (40, [3, 3])], [], 4)], ids=ids)
def test_attention_over_long_prompts(case):
    q, k, v, table, pos, members, shared = shared_case(*case, torch.bfloat16, "cuda")
    y = attend(q, k, v, table, pos, members, shared)
    ref, spread = oracle.attention(q, k, v, table, pos)
    _check(y, ref, spread, torch.bfloat16, _keys(table, k))


# (members, heads, kv_heads, head_dim, page_size, prompt, steps, tokens, window, sinks)
TRIMMED = [
    (40, 8, 2, 128, 16, 400, 30, 1, 150, 5),   # 160 rows a group
    (70, 8, 2, 64, 32, 700, 40, 1, 333, 0),    # 280, no sinks
    (9, 8, 2, 128, 16, 300, 6, 4, 100, 20),    # 144, drafted tokens
    (7, 8, 2, 64, 16, 500, 20, 1, 200, 0),     # 28: one kernel for groups and sequences
]


@pytest.mark.parametrize("dtype", HALF, ids=IDS)
@pytest.mark.parametrize("case", TRIMMED, ids=ids)
def test_forks_that_trim_behind_their_windows(case, dtype):
    """Answers at lengths of their own, each trimmed at its position while they grow: what they see is in the row of the member
    that has the most. Row groups' windows begin in many tiles. Against the table as it was without any trim."""
    members, heads, kv, dim, page, prompt, steps, tokens, window, sinks = case
    shape = LlamaShape(hidden=heads * dim, layers=1, heads=heads, kv_heads=kv, ffn=64, vocab=64)
    g = torch.Generator(device="cuda").manual_seed(members)
    room = prompt + 3 * members + steps * tokens
    keys = -(-(1 << 27) // (members * kv * dim * 4))
    cache = PagedKVCache(shape, members, prompt // page + members * (3 * members // page + steps * tokens // page + 4), page,
                         max(room, keys), "cuda", dtype, window=window, sinks=sinks)
    cache.k[0].normal_(generator=g), cache.v[0].normal_(generator=g)
    first = members // 2  # not the one that trims least
    cache.reserve(first, prompt)
    others = [b for b in range(members) if b != first]
    cache.fork(first, others, prompt)
    shared = int(cache.shared[0])
    assert shared == prompt // page
    length = [prompt + 3 * ((11 * b + 5) % members) + tokens for b in range(members)]
    whole = torch.full_like(cache.table, -1)
    apart = False
    for step in range(steps):
        for b in range(members):
            cache.reserve(b, length[b], length[b] - tokens if step else prompt)
        whole = torch.where(cache.table >= 0, cache.table, whole)
        for b in range(members):
            cache.trim(b, length[b] - tokens)
        if step % (steps // 2 - 1) == 1:
            assert cache.groups == 1 and int(cache.shared[0]) == shared and cache.saved > 0
            trimmed = (cache.table < 0)[:, :shared].sum(1)
            apart |= bool(trimmed.max() > trimmed.min())
            q = torch.randn(members, tokens, heads * dim, device="cuda", generator=g).to(dtype) * 1.5
            pos = torch.tensor(length, device="cuda").unsqueeze(1) - tokens + torch.arange(tokens, device="cuda")
            pos[3] = -1  # has no token in this step
            y = attend(q, cache.k[0], cache.v[0], cache.table, pos, cache.members, cache.shared, window, sinks)
            used = whole[:, :-(-room // page)]
            ref, spread = oracle.attention(q, cache.k[0], cache.v[0], used, pos, window, sinks)
            _check(y, ref, spread, dtype, window + sinks)
            again = paged_attention(q, cache.k[0], cache.v[0], cache.table, pos, window, sinks)
            _check(again, ref, spread, dtype, window + sinks)
        length = [n + tokens for n in length]
    assert apart


def test_groups_as_a_caller_may_give_them():
    """Members named twice, in two groups, that are nobody; counts below zero and past the table; tables without padding."""
    q, k, v, table, pos, members, shared = shared_case(8, 2, 128, 16, [(6, [5, 40, 9])], [30, 7], 1, torch.float16, "cuda")
    ref, spread = oracle.attention(q, k, v, table, pos)
    of = [b for b in members[0].tolist() if b >= 0]
    no = [b for b in range(5) if b not in of]
    rows = [
        ([[of[0], of[1], of[1], of[2]]], [6]),
        ([[of[0], of[1], -7, 99], [of[2], of[1], of[0], 1 << 30]], [6, 4]),
        ([[of[0], of[1], of[2], -1], [of[1], -1, -1, -1]], [6, 6]),
        ([[-1, -1, -1, -1], [-1, of[0], of[2], -1]], [3, 2]),
        ([[of[0], of[2], -1, -1], [no[0], no[1], -1, -1]], [1, 0]),
        ([[of[0], of[2], of[1], -1], [no[0], no[1], -1, -1]], [-5, -(1 << 31)]),
        ([[no[0], -1, -1, -1], [no[1], -1, -1, -1]], [1 << 30, (1 << 31) - 1]),  # alone in a group: all of its table
        ([[-1]], [4]),
    ]
    for lists, counts in rows:
        y = attend(q, k, v, table, pos, torch.tensor(lists, dtype=torch.int32, device="cuda"),
                                   torch.tensor(counts, dtype=torch.int32, device="cuda"))
        _check(y, ref, spread, torch.float16, _keys(table, k))
    strided = torch.stack((members, members), 2)[..., 0]
    assert not strided.is_contiguous()
    first = attend(q, k, v, table, pos, members, shared)
    assert torch.equal(attend(q, k, v, table, pos, strided, torch.stack((shared, shared), 1)[:, 0]), first)
    none = members[:, :0]
    assert torch.equal(paged_shared_attention(q, k, v, table, pos, none, shared), paged_attention(q, k, v, table, pos))


def test_tokens_before_the_end_of_the_shared_pages():
    """Set back into the prompt, not yet begun, past the table; pages that are not there in the prompt and behind it."""
    q, k, v, table, pos, members, shared = shared_case(8, 2, 128, 16, [(6, [5, 40, 9, 20])], [30], 2, torch.bfloat16, "cuda")
    of = [b for b in members[0].tolist() if b >= 0]
    pos[of[0]] = torch.tensor([3, 90], device="cuda")
    pos[of[1]] = torch.tensor([-1, 17], device="cuda")
    pos[of[2]] = torch.tensor([table.shape[1] * 16, 1 << 40], device="cuda")
    table[of, 2] = -1
    table[of, 4] = 1 << 30
    table[of[3], 7] = -1
    for window, sinks in ((0, 0), (20, 5)):
        y = attend(q, k, v, table, pos, members, shared, window, sinks)
        ref, spread = oracle.attention(q, k, v, table, pos, window, sinks)
        _check(y, ref, spread, torch.bfloat16, _keys(table, k))
    table[of] = -1
    y = attend(q, k, v, table, pos, members, shared)
    assert torch.equal(y[of], torch.zeros_like(y[of]))


@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_that_a_token_does_not_see_do_not_reach_it(dim, tokens):
    """An infinity or NaN in shared pages for the members that see it and no others, whatever rows are computed together."""
    q, k, v, table, pos, members, shared = shared_case(8, 2, dim, 16, [(6, [30, 40, 29])], [30], tokens, torch.bfloat16, "cuda")
    of = [b for b in members[0].tolist() if b >= 0]
    page = int(table[of[0], 3])  # positions 48 to 63
    v[page, 0, 5] = math.inf
    v[page, 1, 6] = math.nan
    k[page, 1, 7] = math.nan
    own = int(table[of[1], 7])   # positions 112 to 127
    v[own, :, 3] = -math.inf
    pos[of[2]] = 52              # sees none of them
    window, sinks = 70, 0        # member 0 is past the first with 126 - 69 = 57 on, member 1 with 67 on
    for w in (0, window):
        y = attend(q, k, v, table, pos, members, shared, w, sinks)
        ref, spread = oracle.attention(q, k, v, table, pos, w, sinks)
        odd = ~torch.isfinite(ref)
        assert odd.any() and not odd[of[2]].any()
        y = y.double().cpu()
        assert torch.equal(y.isnan(), ref.isnan())
        assert torch.equal(y[odd].nan_to_num(1.0), ref[odd].nan_to_num(1.0))
        _check(torch.where(odd, 0.0, y), torch.where(odd, 0.0, ref), torch.where(odd, 0.0, spread), torch.bfloat16, _keys(table, k))


def test_attention_of_large_scores():
    q, k, v, table, pos, members, shared = shared_case(8, 2, 128, 16, [(9, [30, 4])], [3], 1, torch.float16, "cuda")
    q, k = q * 20, k.nan_to_num(0.0) * 20  # scores of thousands: one key takes all
    y = attend(q, k, v, table, pos, members, shared)
    ref, _ = oracle.attention(q, k, v, table, pos)
    # scores up to 9000 in fp32 are off by 128 * 9000 * 2^-24 = 0.07 at most: weights by 15% where two are near
    top = (y.double().cpu() - ref).abs()
    assert torch.isfinite(y).all() and top.max() < 0.5 and top.mean() < 0.01


def test_attention_takes_strided_tensors_and_a_scale():
    q, k, v, table, pos, members, shared = shared_case(8, 2, 128, 16, [(4, [5, 9])], [70], 3, torch.float16, "cuda")
    want = attend(q, k, v, table, pos, members, shared, scale=0.05)
    ref, spread = oracle.attention(q, k, v, table, pos, scale=0.05)
    _check(want, ref, spread, torch.float16, _keys(table, k))
    wide = torch.full((3, 3, q.shape[2] + 24), math.nan, dtype=q.dtype, device="cuda")
    wide[..., 8:8 + q.shape[2]] = q
    broad = torch.full((3, table.shape[1] + 3), 1 << 29, dtype=torch.int32, device="cuda")
    broad[:, 1:1 + table.shape[1]] = table
    odd = torch.empty(q.numel() + 3, dtype=q.dtype, device="cuda")[3:].view(q.shape).copy_(q)
    for qq, tt, pp in ((wide[..., 8:8 + q.shape[2]], broad[:, 1:1 + table.shape[1]], pos), (odd, table.t().contiguous().t(), pos),
                       (q.transpose(0, 1).contiguous().transpose(0, 1), table, torch.stack((pos, pos), 2)[..., 0])):
        assert torch.equal(attend(qq, k, v, tt, pp, members, shared, scale=0.05), want)
    spread_out = torch.stack((k, k), 1)[:, 0]  # pools that are not contiguous run torch ops
    y = attend(q, spread_out, v, table, pos, members, shared, scale=0.05)
    _check(y, ref, spread, torch.float16, _keys(table, k))


@pytest.mark.parametrize("scale", [0.0, -0.07])
@pytest.mark.parametrize("members", [3, 20])
def test_attention_with_scales_that_are_not_positive(members, scale):
    q, k, v, table, pos, lists, shared = shared_case(8, 2, 128, 16, [(9, [30, 4, 70][:members] + [5] * (members - 3))], [40],
                                                                 1, torch.bfloat16, "cuda")
    y = attend(q, k, v, table, pos, lists, shared, scale=scale)
    ref, spread = oracle.attention(q, k, v, table, pos, scale=scale)
    _check(y, ref, spread, torch.bfloat16, _keys(table, k))


@pytest.mark.parametrize("members", [3, 20])
def test_members_that_have_ended(members):
    """A sequence without tokens whose row of the table is gone leaves the others theirs, wherever it stands."""
    case = shared_case(8, 2, 64, 16, [(5, [9] * members)], [], 1, torch.float16, "cuda")
    q, k, v, table, pos, lists, shared = case
    for gone in (0, 1, members - 1):
        pos[gone], table[gone] = -1, -1
        y = attend(q, k, v, table, pos, lists, shared)
        ref, spread = oracle.attention(q, k, v, table, pos)
        _check(y, ref, spread, torch.float16, _keys(table, k))
    pos[:], table[:] = -1, -1
    assert not attend(q, k, v, table, pos, lists, shared).any()


def test_attention_of_nothing_and_of_other_types():
    q, k, v, table, pos, members, shared = fork_oracle.shared_case(4, 2, 128, 16, [(4, [5, 9])], [], 1, torch.float16, "cuda")
    assert paged_shared_attention(q[:0], k, v, table[:0], pos[:0], members, shared).shape == (0, 1, 512)
    wide = [t.float() for t in (q, k, v)]
    y = paged_shared_attention(*wide, table, pos, members, shared)
    ref, _ = oracle.attention(*wide, table, pos)
    assert y.dtype == torch.float32 and (y.double().cpu() - ref).abs().max() < 1e-5
    q.requires_grad_(True)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    y = paged_shared_attention(q, k, v, table, pos, members, shared)
    y.float().sum().backward()
    assert q.grad is not None and torch.isfinite(q.grad).all()


def test_calls_that_are_the_plain_attentions():
    """Past the kernel's list of work, with many tokens a sequence, and small."""
    q, k, v, table, pos, members, shared = fork_oracle.shared_case(2, 1, 64, 16, [(2, [1] * 1100)], [], 1, torch.float16, "cuda", spare=1, read=1 << 28)
    assert torch.equal(paged_shared_attention(q, k, v, table, pos, members, shared), paged_attention(q, k, v, table, pos))
    some = torch.arange(900, device="cuda")
    keep = torch.where((members >= 0) & (members < 900), members, -1)
    y = attend(q[some], k, v, table[some], pos[some], keep, shared)
    ref, spread = oracle.attention(q[some], k, v, table[some], pos[some])
    _check(y, ref, spread, torch.float16, _keys(table, k))
    for case in (shared_case(8, 1, 64, 16, [(2, [9, 30])], [], 9, torch.float16, "cuda"),
                 fork_oracle.shared_case(8, 1, 64, 16, [(2, [9, 30])], [], 1, torch.float16, "cuda")):
        assert torch.equal(paged_shared_attention(*case), paged_attention(*case[:5]))


def test_attention_past_32_bit_offsets():
    pages, KV, S, D = 2 * 8193, 8, 16, 128  # 2^28 elements, past 2^32 bytes with values behind
    k = torch.zeros(2 * pages, KV, S, D, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator(device="cuda").manual_seed(1)
    far = 2 * pages - 4
    k[far:].normal_(generator=g)
    v[far:].normal_(generator=g)
    table = torch.full((2, 1024), -1, dtype=torch.int32, device="cuda")
    table[:, :3] = torch.tensor([[far, far + 1, far + 2], [far, far + 1, far + 3]])
    pos = torch.tensor([[40], [45]], device="cuda")
    q = torch.randn(2, 1, 8 * D, device="cuda", generator=g).half()
    y = attend(q, k, v, table, pos, torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"),
                               torch.tensor([2], dtype=torch.int32, device="cuda"))
    ref, spread = oracle.attention(q, k[far:], v[far:], torch.where(table >= 0, table - far, -1), pos)
    _check(y, ref, spread, torch.float16, 48)


@pytest.mark.parametrize("native", [True, False])
def test_captured_calls_follow_their_tensors(native, monkeypatch):
    """Two graphs of calls, replayed in turn with eager work between, the groups, the table and the positions changed."""
    if not native:
        for name in ("_native_shared", "_native_copy", "_native_score"):
            monkeypatch.setattr(serve, name, None)
    cases = [shared_case(8, 2, 128, 16, [(30, [5, 40, 9])], [100, 7], 1, torch.float16, "cuda", seed=i) for i in range(2)]
    logits = torch.randn(5, 5001, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).half()
    tokens = torch.arange(5, device="cuda")
    source, target = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, 1))
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    for case in cases:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(2):
                attend(*case)
                token_logprobs(logits, tokens, 4)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = attend(*case)
            s = token_logprobs(logits, tokens, 4)
        graphs.append(graph)
        outs.append((y, s))
    spare = torch.zeros(4, 100, device="cuda")
    copier = torch.cuda.CUDAGraph()
    copy_pages([spare], source, source)
    with torch.cuda.graph(copier):
        copy_pages([spare], source, target)
    for step in range(4):
        for graph, (y, s), case in zip(graphs, outs, cases):
            q, k, v, table, pos, members, shared = case
            q.normal_()
            if step == 1:
                shared.fill_(20)
            elif step == 2:
                members[0, 0] = -1
            elif step == 3:
                shared.zero_()
                pos.sub_(pos.clamp(max=1))
            logits.normal_()
            spare.normal_()
            source.fill_(step % 4)
            target.fill_((step + 1) % 4)
            graph.replay()
            copier.replay()
            torch.cuda.synchronize()
            ref, spread = oracle.attention(q, k, v, table, pos)
            _check(y, ref, spread, torch.float16, _keys(table, k))
            fork_oracle.check_score(s, fork_oracle.score(logits, tokens, 4, 1.0))
            assert torch.equal(spare[step % 4], spare[(step + 1) % 4])
            assert torch.equal(y, attend(*case))


def test_calls_on_two_streams():
    cases = [shared_case(8, 2, 128, 16, [(30, [5, 40, 9])], [600, 7], 1, torch.bfloat16, "cuda", seed=i) for i in range(2)]
    logits = [torch.randn(40, 20011, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)) for i in range(2)]
    tokens = torch.arange(40, device="cuda")
    want = [(attend(*c), token_logprobs(x, tokens, 5)) for c, x in zip(cases, logits)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append((attend(*cases[i]), token_logprobs(logits[i], tokens, 5)))
    torch.cuda.synchronize()
    for i in range(2):
        for y, s in got[i]:
            assert torch.equal(y, want[i][0]) and all(torch.equal(a, b) for a, b in zip(s, want[i][1]))


def test_calls_through_python_equal_those_through_the_library_of_operators(monkeypatch):
    assert None not in (serve._native_shared, serve._native_copy, serve._native_score)
    case = shared_case(8, 2, 128, 16, [(30, [5, 40, 9])], [100, 7], 2, torch.float16, "cuda")
    logits, tokens = torch.randn(2, 7, 3001, device="cuda").bfloat16(), torch.randint(-1, 3001, (2, 7), device="cuda")
    pools = [torch.randn(9, 33, device="cuda") for _ in range(3)]
    source, target = torch.tensor([[0, 3, 8, 9], [1, 2, -1, 4]], dtype=torch.int32, device="cuda").unbind(0)

    def everything():
        mine = [p.clone() for p in pools]
        copy_pages(mine, source, target)
        return [attend(*case), *token_logprobs(logits[:, :-1], tokens[:, 1:], 6, 0.9), *mine]

    native = everything()
    for name in ("_native_shared", "_native_copy", "_native_score"):
        monkeypatch.setattr(serve, name, None)
    assert all(torch.equal(a, b) for a, b in zip(native, everything()))


# ---------------------------------------------------------------------------------------- pages

@pytest.mark.parametrize("shape,dtype", [((5, 2, 16, 64), torch.bfloat16), ((40, 8, 32, 128), torch.float16), ((9, 7), torch.uint8),
                                         ((6, 3, 5), torch.float32), ((7, 1), torch.float64), ((4, 5000), torch.int8),
                                         ((3, 2, 2), torch.bool), ((300, 4096), torch.float32)])
def test_copy_pages(shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    pools = [torch.randint(0, 2 if dtype == torch.bool else 100, shape, device="cuda", generator=g).to(dtype) for _ in range(3)]
    n = shape[0] // 2
    order = torch.randperm(shape[0], device="cuda", generator=g).int()
    source, target = order[:n].clone(), order[n:2 * n].clone()
    want = [p.clone() for p in pools]
    for p in want:
        p[target.long()] = p[source.long()]
    nobody = torch.tensor([-1, shape[0], 1 << 30, -(1 << 31)], dtype=torch.int32, device="cuda")
    source = torch.cat((source, nobody, source[:1].expand(4)))
    target = torch.cat((target, order[2 * n:2 * n + 1].expand(4) if shape[0] % 2 else target[:1].expand(4), nobody))
    copy_pages(pools, source, target)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_copy_pages_of_many_pools_and_of_odd_places():
    """More pools than a launch takes; pools that begin at an odd element; strided numbers; a page over itself."""
    flat = torch.randn(300, 1 + 6 * 12, device="cuda")
    for lead in (0, 1):
        pools = [row[lead:lead + 72].view(6, 12) for row in flat]
        want = [p.clone() for p in pools]
        for p in want:
            p[1], p[5] = p[4], p[0]
        numbers = torch.tensor([[4, 1], [0, 5], [2, 2]], dtype=torch.int32, device="cuda")
        copy_pages(pools, numbers[:, 0], numbers[:, 1])
        assert all(torch.equal(a, b) for a, b in zip(pools, want))
    spread = [torch.randn(6, 12, 2, device="cuda")[..., 0] for _ in range(2)]  # not contiguous: torch ops
    want = [p.clone() for p in spread]
    for p in want:
        p[1] = p[4]
    copy_pages(spread, numbers[:1, 0], numbers[:1, 1])
    assert all(torch.equal(a, b) for a, b in zip(spread, want))


def test_copy_pages_past_32_bit_offsets():
    pool = torch.zeros(5, 1 << 30, dtype=torch.uint8, device="cuda")
    pool[4, -16:] = 7
    pool[4, :16] = 9
    copy_pages([pool], *torch.tensor([[4], [2]], dtype=torch.int32, device="cuda").unbind(0))
    assert torch.equal(pool[2], pool[4]) and not pool[1].any() and not pool[3].any()


# ---------------------------------------------------------------------------------------- scores

@pytest.mark.parametrize("dtype", [torch.float32, *HALF], ids=["f32", *IDS])
@pytest.mark.parametrize("shape,V,top,temperature", [
    ((1,), 1, 1, 1.0), ((3,), 5, 5, 1.0), ((7,), 64, 64, 0.5), ((2, 3), 1000, 5, 1.0), ((1,), 32000, 20, 0.8), ((5,), 8191, 1, 1.0),
    ((3, 2), 8193, 33, 1.3), ((2,), 100003, 64, 1.0), ((300,), 777, 3, 1.0), ((700,), 257, 0, 2.0), ((1, 1), 128256, 8, 1.0),
    ((40,), 16385, 32, 1.0)])
def test_score(shape, V, top, temperature, dtype):
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = (torch.randn(*shape, V, device="cuda", generator=g) * 3).to(dtype)
    tokens = torch.randint(0, V, shape, device="cuda", generator=g)
    tokens.view(-1)[2::5] = -1
    tokens.view(-1)[4::7] = V
    got = token_logprobs(logits, tokens, top, temperature)
    fork_oracle.check_score(got, fork_oracle.score(logits, tokens, top, temperature))


@pytest.mark.parametrize("dtype", [torch.float32, *HALF], ids=["f32", *IDS])
@pytest.mark.parametrize("rows,V,top", [(70, 100003, 3), (37, 128000, 64), (129, 70001, 2), (256, 8192, 1), (257, 8192, 4), (1280, 4097, 2),
                                        (1281, 8193, 5), (1301, 20011, 40), (1500, 3000, 0)])
def test_score_of_rows_in_parts(rows, V, top, dtype):
    """Parts that end with a row and those that do not, rows whole, on both sides of where the kernel cuts otherwise."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    logits = (torch.randn(rows, V, device="cuda", generator=g) * 3).to(dtype)
    tokens = torch.randint(0, V, (rows,), device="cuda", generator=g)
    fork_oracle.check_score(token_logprobs(logits, tokens, top), fork_oracle.score(logits, tokens, top, 1.0))


@pytest.mark.parametrize("dtype", [torch.float32, *HALF], ids=["f32", *IDS])
@pytest.mark.parametrize("V", [41, 9001, 70000])
def test_score_of_odd_rows(V, dtype):
    logits, tokens = odd_rows(V, dtype)
    for top in (0, 3, 40):
        got = token_logprobs(logits.cuda(), tokens.cuda(), top)
        fork_oracle.check_score(got, fork_oracle.score(logits, tokens, top, 1.0))


@pytest.mark.parametrize("dtype", [torch.float32, *HALF], ids=["f32", *IDS])
def test_the_largest_wherever_they_lie(dtype):
    """Ascending and descending rows, the largest side by side, a stride apart, at the ends; equal ones over the whole row."""
    V = 30011
    ramp = torch.linspace(-8, 8, V)
    rows = [ramp, ramp.flip(0), torch.where(torch.arange(V) % 256 == 17, 9.0, ramp), torch.where(torch.arange(V) % 8192 < 40, 10.0, 0.0),
            torch.full((V,), -3.0), torch.where(torch.arange(V) >= V - 30, 5.0, -5.0), torch.where(torch.arange(V) < 30, 5.0, -5.0),
            (torch.arange(V) % 7).float(), -(torch.arange(V) % 5).float().abs() - 100, torch.where(torch.arange(V) == 12345, 1.0, -math.inf)]
    logits = torch.stack(rows).to(dtype)
    tokens = torch.arange(len(rows))
    for top in (1, 20, 64):
        got = token_logprobs(logits.cuda(), tokens.cuda(), top)
        fork_oracle.check_score(got, fork_oracle.score(logits, tokens, top, 1.0))


def test_score_of_one_long_row():
    """More parts with more alternatives than the join keeps at hand."""
    g = torch.Generator(device="cuda").manual_seed(6)
    logits = torch.randn(2, 1 << 22, device="cuda", generator=g).half()
    logits[1, 5::7] = -math.inf
    tokens = torch.tensor([7, -1], device="cuda")
    for top in (2, 64):
        fork_oracle.check_score(token_logprobs(logits, tokens, top), fork_oracle.score(logits, tokens, top, 1.0))


def test_score_takes_strided_rows():
    g = torch.Generator(device="cuda").manual_seed(8)
    whole = torch.randn(3, 6, 1003, device="cuda", generator=g).bfloat16()
    tokens = torch.randint(0, 1003, (3, 6), device="cuda", generator=g)
    views = [(whole[:, :-1], tokens[:, 1:]), (whole[:, ::2, 1:900], tokens[:, ::2].clamp(max=898)), (whole.transpose(0, 1), tokens.t()),
             (whole[1:2, 3:4], tokens[1:2, 3:4]), (whole[..., ::3], tokens % 335), (whole[1, :, 5:], tokens[1] % 998),
             (whole[:1].expand(3, 6, 1003), tokens), (whole[0, 0].expand(4, 1003), tokens[0, :4])]
    for x, t in views:
        fork_oracle.check_score(token_logprobs(x, t, 5), fork_oracle.score(x, t, 5, 1.0))


@pytest.mark.parametrize("temperature", [1e-300, 2.0 ** -65, 2.0 ** -64, 1e-3, 1e4, 2.0 ** 64, 1e300])
def test_score_at_extreme_temperatures(temperature):
    g = torch.Generator(device="cuda").manual_seed(9)
    logits = torch.randn(4, 3000, device="cuda", generator=g)
    logits[0, 5:900] = -math.inf
    logits[1, ::3] = torch.finfo(torch.float32).min
    tokens = torch.tensor([1, 2, 3, -1], device="cuda")
    fork_oracle.check_score(token_logprobs(logits, tokens, 3, temperature), fork_oracle.score(logits, tokens, 3, temperature))


def test_score_of_large_logits():
    """fp32 logits near the type's ends."""
    logits = torch.tensor([[3e38, 2.9e38, -3e38, 0.0], [-3e38, -3.1e38, -math.inf, -3.4e38], [1e30, 1e30, -1e30, 1e30]], device="cuda")
    tokens = torch.tensor([0, 0, 3], device="cuda")
    fork_oracle.check_score(token_logprobs(logits, tokens, 1), fork_oracle.score(logits, tokens, 1, 1.0))


def test_score_of_nothing_and_of_other_types():
    x, t = torch.randn(4, 50, device="cuda"), torch.tensor([1, 2, 3, -1], device="cuda")
    assert [tuple(y.shape) for y in token_logprobs(x[:0], t[:0], 2)] == [(0,), (0,), (0, 2), (0, 2)]
    fork_oracle.check_score(token_logprobs(x.double(), t, 2), fork_oracle.score(x.double(), t, 2, 1.0))
    many = torch.randn(3, 200, device="cuda")
    fork_oracle.check_score(token_logprobs(many, t[:3], 100), fork_oracle.score(many, t[:3], 100, 1.0))
    x.requires_grad_(True)
    given, entropy, _, _ = token_logprobs(x, t, 2)
    (given.sum() + entropy.sum()).backward()
    assert torch.isfinite(x.grad).all()


def test_score_past_32_bit_offsets():
    rows, V = 33, 1 << 27  # 2^32 elements and more
    logits = torch.zeros(rows, V, dtype=torch.float16, device="cuda")
    logits[-1, -1], logits[-1, 5], logits[-2, 0] = 20.0, 12.0, 30.0
    tokens = torch.full((rows,), V - 1, device="cuda")
    given, entropy, order, best = token_logprobs(logits, tokens, 3)
    assert order[-1].tolist() == [V - 1, 5, 0] and order[-2].tolist() == [0, 1, 2] and order[0].tolist() == [0, 1, 2]
    total = math.exp(20.0) + math.exp(12.0) + V - 2
    # sums of 2^27 terms, up to 2^21 in a lane one after the other: 2^21 * 2^-24 of them at the very most
    for got, want in ((given[-1], 20.0 - math.log(total)), (given[-2], -30.0 - math.log1p((V - 1) * math.exp(-30.0))),
                      (given[0], -27 * math.log(2.0)), (best[-1, 1], 12.0 - math.log(total)), (entropy[0], 27 * math.log(2.0))):
        assert abs(got.item() - want) < 0.13


# ---------------------------------------------------------------------------------------- together

def test_a_model_answers_a_prompt_several_times(monkeypatch):
    """A prompt, its forks, their tokens decoded together in a captured step and scored; pages written after a fork are each
    sequence's own, and the cache moved together keeps what it holds."""
    shape = LlamaShape(hidden=1024, layers=3, heads=8, kv_heads=2, ffn=1408, vocab=1003)
    model = random_llama(shape, bpw=1.0, device="cuda", dtype=torch.float16).eval()
    model.prepare_kernels("gemv", torch.float16)
    g = torch.Generator(device="cuda").manual_seed(5)
    answers, P, page, more = 5, 75, 16, 8
    prompt = torch.randint(0, shape.vocab, (P,), device="cuda", generator=g)
    texts = torch.randint(0, shape.vocab, (answers, more), device="cuda", generator=g)
    calls = []
    monkeypatch.setattr(serve, "_WORTH_SHARING", 1)
    monkeypatch.setattr(serve, "paged_shared_attention", lambda *x: calls.append(1) or attend(*x))
    with torch.no_grad():
        caches = [PagedKVCache(shape, answers, 60, page, 40000, "cuda", torch.float16) for _ in range(2)]
        alone, forked = caches
        for b in range(answers):
            alone.reserve(b, P + more)
        model(prompt.expand(answers, -1), torch.arange(P, device="cuda").expand(answers, -1), alone)
        forked.reserve(2, P)
        pos = torch.full((answers, P), -1, device="cuda")
        pos[2] = torch.arange(P, device="cuda")
        model(prompt.expand(answers, -1), pos, forked)
        forked.fork(2, [0, 1, 3, 4], P)
        for b in range(answers):
            forked.reserve(b, P + more, P)
        assert forked.groups == 1 and int(forked.shared[0]) == 4
        ids, at = torch.zeros(answers, 1, dtype=torch.int64, device="cuda"), torch.zeros(answers, 1, dtype=torch.int64, device="cuda")
        ids.copy_(texts[:, :1])
        at.fill_(P)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            model(ids, at, forked)  # the same keys again at the first replay
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model(ids, at, forked)
            scores = token_logprobs(logits, ids, 4)
        for t in range(more):
            if t == 4:
                forked.release(1)  # one answer has ended; its place stays, without pages
                at[1], texts[1] = -1, 0
                forked.compact()
            live = torch.tensor([b for b in range(answers) if t < 4 or b != 1], device="cuda")
            ids.copy_(texts[:, t:t + 1])
            at[live] = P + t
            want = model(ids, torch.full_like(at, P + t), alone)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.isfinite(logits[live]).all()
            # the two ways round the probabilities' sums apart: fp16 steps of the hidden states, some layers of them
            assert (logits[live] - want[live]).abs().max() < 0.05 * want.abs().max()
            fork_oracle.check_score([s[live] for s in scores], fork_oracle.score(logits[live], ids[live], 4, 1.0))
    assert len(calls) >= 2 * shape.layers and forked.saved == 3 * 4 * page * 2 * 2 * 128 * 2  # of four members, four pages


def test_a_model_answers_under_a_window(monkeypatch):
    """Answers of lengths of their own whose pages are taken back behind their windows between the replays of a captured step."""
    shape = LlamaShape(hidden=1024, layers=2, heads=8, kv_heads=2, ffn=1408, vocab=1003)
    model = random_llama(shape, bpw=1.0, device="cuda", dtype=torch.float16).eval()
    model.prepare_kernels("gemv", torch.float16)
    g = torch.Generator(device="cuda").manual_seed(7)
    answers, P, page, more, window, sinks = 6, 100, 16, 40, 70, 5
    prompt = torch.randint(0, shape.vocab, (P,), device="cuda", generator=g)
    begin = [17, 0, 5, 30, 11, 24]  # tokens of each answer before the others' first
    texts = torch.randint(0, shape.vocab, (answers, more + max(begin)), device="cuda", generator=g)
    calls = []
    monkeypatch.setattr(serve, "_WORTH_SHARING", 1)
    monkeypatch.setattr(serve, "paged_shared_attention", lambda *x: calls.append(1) or attend(*x))
    with torch.no_grad():
        alone, forked = caches = [PagedKVCache(shape, answers, 120, page, 40000, "cuda", torch.float16, window=window, sinks=sinks)
                                  for _ in range(2)]
        every = torch.arange(P, device="cuda").expand(answers, -1)
        for b in range(answers):
            alone.reserve(b, P + begin[b] + more)
        model(prompt.expand(answers, -1), every, alone)
        forked.reserve(3, P)
        model(prompt.expand(answers, -1), torch.where(torch.arange(answers, device="cuda").unsqueeze(1) == 3, every, -1), forked)
        forked.fork(3, [b for b in range(answers) if b != 3], P)
        for b in range(answers):
            forked.reserve(b, P + begin[b] + 1, P)
        head = max(begin)
        at = torch.arange(P, P + head, device="cuda").expand(answers, -1)
        at = torch.where(at < P + torch.tensor(begin, device="cuda").unsqueeze(1), at, -1)
        for cache in caches:
            model(texts[:, :head], at, cache)
        place = P + torch.tensor(begin, device="cuda").unsqueeze(1)
        ids, pos = texts.gather(1, place - P), place.clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            model(ids, pos, forked)  # the same keys again at the first replay
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model(ids, pos, forked)
        lead = set()
        for t in range(more):
            for b in range(answers):
                forked.reserve(b, P + begin[b] + t + 1, P + begin[b] + t)
                forked.trim(b, P + begin[b] + t)
            lead.add(int(forked.members[0, 0]))
            pos.copy_(place + t)
            ids.copy_(texts.gather(1, pos - P))
            graph.replay()
            want = model(ids, pos, alone)
            torch.cuda.synchronize()
            # as above: the two ways round the probabilities' sums apart
            assert (logits - want).abs().max() < 0.05 * want.abs().max()
        assert forked.trim(0, 0) == 0 and (forked.table[:, 1:] >= 0).sum() < answers * 7 and lead == {0, 1}
    assert len(calls) >= 2 * shape.layers
