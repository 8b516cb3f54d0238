"""The paged cache's kernels and draft verification against plain 64-bit forms (needs a gfx950 GPU)."""
import math

import pytest
import torch

import serve_oracle as oracle
from nanoquant_amd import PagedKVCache, _lib, paged_attention, paged_rope_write, verify_drafts
from nanoquant_amd.decode import LlamaShape, random_llama

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
IDS = ["f16", "bf16"]

# (heads, kv_heads, head_dim, page_size, lengths, tokens, window, sinks)
ATTENTION = [
    # one token: a single key; lengths around a tile and a page; many query heads a kv head; no grouping; odd head counts
    (4, 4, 128, 16, [1], 1, 0, 0),
    (8, 1, 128, 16, [15, 16, 17, 31, 32, 33, 64, 65], 1, 0, 0),
    (16, 1, 64, 32, [100, 1, 257], 1, 0, 0),
    (20, 1, 128, 48, [70, 300], 1, 0, 0),
    (64, 2, 64, 16, [130], 1, 0, 0),
    (5, 5, 64, 48, [47, 49, 96, 500], 1, 0, 0),
    (6, 2, 128, 256, [255, 256, 257], 1, 0, 0),
    (8, 2, 128, 64, [2300, 40, 1500], 1, 0, 0),
    (2, 2, 128, 16, [n * 7 % 90 + 1 for n in range(40)], 1, 0, 0),
    # a window, with sinks inside a page, past it, inside the window, and none
    (8, 2, 128, 16, [400, 20, 129], 1, 100, 4),
    (4, 4, 64, 32, [333, 1000], 1, 33, 40),
    (8, 1, 128, 48, [50, 51, 700], 1, 49, 0),
    (4, 2, 128, 16, [90], 1, 1, 1),
    (4, 2, 64, 16, [200], 1, 150, 100),
    # drafted tokens: rows below, at and past a tile of rows
    (4, 4, 128, 16, [2, 90], 2, 0, 0),
    (8, 1, 128, 32, [40, 300, 5], 5, 0, 0),
    (16, 2, 64, 16, [257], 8, 0, 0),
    (8, 2, 128, 16, [1100, 64], 9, 60, 3),
    (24, 1, 128, 64, [500], 3, 0, 0),
    # prompts and chunks: ragged ends, contexts before them, windows that start inside a tile
    (4, 4, 128, 16, [33], 33, 0, 0),
    (8, 2, 128, 32, [200, 64, 1], 200, 0, 0),
    (2, 2, 64, 16, [129, 128], 129, 0, 0),
    (6, 2, 128, 48, [700, 301], 300, 0, 0),
    (8, 1, 64, 64, [900], 257, 0, 0),
    (4, 2, 128, 16, [600, 350], 300, 70, 5),
    (4, 1, 64, 32, [500], 400, 128, 64),
    (5, 5, 128, 16, [1030], 260, 0, 0),
]
ids = lambda c: "x".join(str(len(e) if isinstance(e, list) else e) for e in c)  # noqa: E731


def _check(y, ref, spread, dtype, keys):
    bound = oracle.attention_bound(ref, spread, dtype, keys)
    off = ((y.double().cpu() - ref).abs() / bound).max().item()
    assert off <= 1.0, f"{off:.2f} times the bound"


@pytest.mark.parametrize("dtype", HALF, ids=IDS)
@pytest.mark.parametrize("case", ATTENTION, ids=ids)
def test_attention(case, dtype):
    """Rows and pages that hold nothing are NaN, and pages that the window hides are not there."""
    print("\n[case] paged attention", case, dtype, flush=True)
    heads, kv, dim, page, lengths, tokens, window, sinks = case
    q, k, v, table, pos = oracle.paged_case(heads, kv, dim, page, lengths, tokens, dtype, "cuda", window=window, sinks=sinks)
    y = paged_attention(q, k, v, table, pos, window, sinks)
    ref, spread = oracle.attention(q, k, v, table, pos, window, sinks)
    assert y.shape == q.shape and y.dtype == dtype and y.is_contiguous()
    _check(y, ref, spread, dtype, max(lengths))
    assert torch.equal(y, paged_attention(q, k, v, table, pos, window, sinks))  # the same bits again
    assert (y[pos < 0] == 0).all()


# (heads, kv_heads, head_dim, page_size, lengths, tokens, window, sinks, columns of the table), every kernel with every number
# of row tiles, those that share the work of all sequences out over the card and those that do not
KERNELS = {
    "few": [
        (4, 2, 64, 32, [650], 10, 0, 0, 0),
        (8, 1, 128, 16, [700, 90], 3, 0, 0, 0),
        (8, 1, 64, 16, [720], 5, 0, 0, 0),
        (6, 2, 128, 48, [800, 333], 13, 0, 0, 0),
        (16, 2, 128, 16, [700], 8, 0, 0, 0),
        (4, 4, 64, 64, [900, 20], 50, 0, 0, 0),
        (8, 1, 128, 16, [1500, 700], 7, 600, 20, 0),
        (8, 1, 64, 16, [1100, 650, 9], 6, 100, 0, 0),
        # more sequences than one launch takes, and a table much wider than the lengths
        (2, 1, 64, 16, [n % 45 + 1 for n in range(600)], 1, 0, 0, 300),
        (3, 3, 128, 16, [50, 7, 33], 15, 0, 0, 400),
        (4, 2, 128, 16, [3000, 2500], 1, 2000, 40, 0),
        # under windows that leave a block little to read
        (4, 2, 128, 16, [3000, 2500, 4], 1, 100, 4, 0),
        (8, 2, 64, 32, [2000, 5], 2, 33, 0, 0),
    ],
    "shares": [
        (4, 2, 128, 64, [4100, 700], 50, 0, 0, 0),
        (8, 2, 64, 16, [3300], 30, 0, 0, 0),
        (8, 1, 128, 32, [4000, 2900], 32, 0, 0, 0),
        (4, 4, 64, 48, [3500], 250, 0, 0, 0),
        (8, 1, 128, 16, [5000], 32, 4000, 70, 0),
        (8, 2, 64, 16, [5000, 300], 100, 200, 1, 0),
        (2, 2, 128, 16, [200, 150], 130, 0, 0, 200),
        (8, 1, 64, 16, [n % 70 + 9 for n in range(1030)], 9, 0, 0, 125),
    ],
    "groups": [
        (4, 4, 128, 16, [1, 17, 300], 1, 0, 0, 0),
        (8, 1, 64, 32, [600, 64], 2, 0, 0, 0),
        (4, 2, 128, 16, [600, 31, 2], 3, 100, 5, 0),
        (16, 1, 64, 16, [500, 33], 1, 33, 40, 0),
        (8, 2, 128, 48, [n * 9 % 600 + 1 for n in range(70)], 1, 0, 0, 0),
        (2, 2, 64, 16, [n * 61 % 1900 + 1 for n in range(130)], 1, 0, 0, 0),
        (8, 2, 128, 16, [300, 90], 9, 0, 0, 0),
        (3, 3, 64, 16, [20, 64], 20, 0, 0, 0),
        (4, 2, 128, 64, [333], 200, 0, 0, 0),
        (4, 2, 64, 64, [333], 200, 90, 3, 0),
        (64, 8, 128, 16, [n * 37 % 270 + 1 for n in range(56)], 32, 0, 0, 0),
        (64, 8, 64, 32, [n * 53 % 330 + 32 for n in range(56)], 32, 100, 5, 0),
        (32, 32, 64, 16, [257, 300, 511, 256], 1000, 0, 0, 0),
        (16, 16, 128, 48, [600, 250, 333, 577, 100, 512, 511], 1020, 0, 0, 0),
    ],
}


@pytest.mark.parametrize("kernel,case", [(k, c) for k, cases in KERNELS.items() for c in cases],
                         ids=lambda e: e if isinstance(e, str) else "x".join(str(len(x) if isinstance(x, list) else x) for x in e))
def test_attention_kernels(kernel, case):
    heads, kv, dim, page, lengths, tokens, window, sinks, columns = case
    dtype = HALF[len(lengths) % 2]
    print("\n[case] paged attention", kernel, heads, kv, dim, page, len(lengths), tokens, window, sinks, dtype, flush=True)
    q, k, v, table, pos = oracle.paged_case(heads, kv, dim, page, lengths, tokens, dtype, "cuda", window=window, sinks=sinks)
    if columns:
        table = torch.nn.functional.pad(table, (0, columns - table.shape[1]), value=-1)
    # only row groups that blocks have for themselves need no workspace
    bytes_ = _lib.load().nq_paged_attention_workspace_bytes(len(lengths), tokens, heads, kv, dim, table.shape[1], page)
    assert (bytes_ == 0) == (kernel == "groups")
    y = paged_attention(q, k, v, table, pos, window, sinks)
    ref, spread = oracle.attention(q, k, v, table, pos, window, sinks)
    _check(y, ref, spread, dtype, max(lengths))
    assert torch.equal(y, paged_attention(q, k, v, table, pos, window, sinks))
    assert (y[pos < 0] == 0).all()


@pytest.mark.parametrize("length,tokens", [(40, 1), (700, 1), (700, 9), (700, 40), (40, 40), (300, 150), (3000, 100)])
def test_keys_that_are_not_finite_reach_the_tokens_that_see_them(length, tokens):
    q, k, v, table, pos = oracle.paged_case(4, 2, 128, 16, [length], tokens, torch.bfloat16, "cuda")
    want = paged_attention(q, k, v, table, pos).view(tokens, 2, 2, 128)
    k[int(table[0, 0]), 1, 5, 3] = math.nan
    y = paged_attention(q, k, v, table, pos).view(tokens, 2, 2, 128)
    seen = (pos[0] >= 5).cpu()
    assert y[seen, 1].isnan().all() and torch.equal(y[:, 0], want[:, 0])
    assert torch.equal(y[~seen], want[~seen])


@pytest.mark.parametrize("tokens", [1, 5, 100])
def test_calls_through_python_equal_those_through_the_library_of_operators(tokens, monkeypatch):
    from nanoquant_amd import serve
    q, k, v, table, pos = oracle.paged_case(8, 2, 128, 16, [300, 120], tokens, torch.float16, "cuda")
    cos, sin = torch.randn(2, 2, tokens, 128, device="cuda").unbind(0)
    logits, drafts, u, probs = _drafts(3, tokens, 700, False, torch.float32, seed=tokens)

    def all_calls():
        pools = k.clone(), v.clone()
        heads = q[..., :256].contiguous()
        return (paged_attention(q, k, v, table, pos, 64, 2), paged_rope_write(q, heads, heads, cos, sin, pos, *pools, table),
                *(p.nan_to_num(7.0) for p in pools), *verify_drafts(logits, drafts, u, probs, 0.7))

    natives = (serve._native_attention, serve._native_write, serve._native_verify)
    assert None not in natives
    assert natives[0](q, k, v, table, pos, 64, 2, None) is not None  # it takes the call
    want = all_calls()
    for name in ("_native_attention", "_native_write", "_native_verify"):
        monkeypatch.setattr(serve, name, None)
    assert all(torch.equal(a, b) for a, b in zip(all_calls(), want))


@pytest.mark.parametrize("case", ATTENTION, ids=ids)
def test_attention_counts_its_keys(case):
    """Queries of zero make every probability 1, so with values of 0 and 1 the sums are whole numbers and the result their
    quotient, rounded once: a key too many or too few shows (2 ulp of fp32 for the division)."""
    print("\n[case] paged attention, equal scores", case, flush=True)
    heads, kv, dim, page, lengths, tokens, window, sinks = case
    q, k, v, table, pos = oracle.paged_case(heads, kv, dim, page, lengths, tokens, torch.float16, "cuda", window=window,
                                            sinks=sinks)
    q.zero_()
    v = torch.where(v.isnan(), v, (v > 0.3).to(v.dtype))
    y = paged_attention(q, k, v, table, pos, window, sinks)
    ref, _ = oracle.attention(q, k, v, table, pos, window, sinks)
    assert ((y.double().cpu() - ref).abs() <= ref * (2.0 ** -11 + 2.0 ** -22)).all()


@pytest.mark.parametrize("tokens", [1, 4, 150])
def test_attention_rows_and_pages_that_are_not_there(tokens):
    """Pages missing in the middle, entries that name no page, positions outside the table and in another order, and a
    sequence of padding alone."""
    q, k, v, table, pos = oracle.paged_case(8, 2, 128, 16, [400, 300, 310], tokens, torch.bfloat16, "cuda")
    table[0, 3], table[0, 20], table[1, 5:9] = -1, 1 << 30, k.shape[0]
    table[2] = -(1 << 31)
    pos = pos[:, torch.randperm(tokens, generator=torch.Generator().manual_seed(0)).cuda()]
    if tokens > 1:
        pos[0, 0], pos[0, 1], pos[1, 2] = table.shape[1] * 16, 1 << 40, -(1 << 60)
    else:
        pos[1, 0] = table.shape[1] * 16
    y = paged_attention(q, k, v, table, pos)
    ref, spread = oracle.attention(q, k, v, table, pos)
    _check(y, ref, spread, torch.bfloat16, 400)
    assert (y[2] == 0).all() and (ref == 0).any()


@pytest.mark.parametrize("dtype", HALF, ids=IDS)
@pytest.mark.parametrize("group,tokens", [(1, 4), (4, 4), (2, 40), (4, 100)])
def test_values_that_a_token_does_not_see_do_not_reach_it(group, tokens, dtype):
    """NaN and infinities in the keys and values of later tokens, and in what the window has left behind."""
    length, window, sinks = 200, 64, 3
    q, k, v, table, pos = oracle.paged_case(2 * group, 2, 128, 16, [length], tokens, dtype, "cuda", window=window, sinks=sinks)
    first = length - tokens
    for p, x in ((length - 1, math.nan), (length - 2, math.inf), (first - window + 1, -math.inf)):
        page, row = int(table[0, p // 16]), p % 16
        k[page, 1, row, 5] = x if x != math.inf else 0.0
        v[page, 1, row, 7] = x
    y = paged_attention(q, k, v, table, pos, window, sinks).view(tokens, 2, group, 128)
    clean = [t for t in range(tokens) if not (t >= tokens - 2 or t == 0)]
    qc, kc, vc = q, k.nan_to_num(0.0, 0.0, 0.0), v.nan_to_num(0.0, 0.0, 0.0)
    ref, spread = (r.view(tokens, 2, group, 128) for r in oracle.attention(qc, kc, vc, table, pos, window, sinks))
    _check(y[clean], ref[clean], spread[clean], dtype, length)
    _check(y[:, 0], ref[:, 0], spread[:, 0], dtype, length)  # the other kv head
    assert y[-1, 1].isnan().any()


@pytest.mark.parametrize("dim,tokens,group", [(128, 4, 1), (64, 3, 4), (128, 16, 1)])
def test_values_that_a_token_does_not_see_in_blocks_without_shares(dim, tokens, group):
    """Sequences of two to five tiles of 32 keys, whose last one each of a block's four waves has in turn: a value there that
    is not finite and that the last token alone sees leaves the others what they are without it."""
    lengths = [60, 90, 120, 160]
    q, k, v, table, pos = oracle.paged_case(2 * group, 2, dim, 16, lengths, tokens, torch.bfloat16, "cuda")
    assert _lib.load().nq_paged_attention_workspace_bytes(4, tokens, 2 * group, 2, dim, table.shape[1], 16) == 0
    ref, spread = oracle.attention(q, k, v, table, pos)
    for bad in (math.nan, math.inf, -math.inf):
        for b, n in enumerate(lengths):
            v[int(table[b, (n - 1) // 16]), :, (n - 1) % 16] = bad
        y = paged_attention(q, k, v, table, pos)
        _check(y[:, :-1], ref[:, :-1], spread[:, :-1], torch.bfloat16, 160)
        assert not torch.isfinite(y[:, -1]).any()


def test_attention_of_large_scores():
    """Scores of some hundreds, of both signs, and a last key that beats all before it."""
    q, k, v, table, pos = oracle.paged_case(4, 1, 128, 16, [300, 150], 1, torch.float16, "cuda")
    q *= 12
    k[table[0, 18].long(), 0, 11] = (q[0, 0, :128] * 0.5).to(k.dtype)
    for scale in (None, -0.09, 0.0, 1.0):
        y = paged_attention(q, k, v, table, pos, scale=scale)
        ref, spread = oracle.attention(q, k, v, table, pos, scale=scale)
        # scores are off by 128 roundings of their summed |products|, up to 128 * 18 * 3.5 * scale here: 2^-24 of that, twice
        s = abs(scale if scale is not None else 128 ** -0.5)
        u = 2.0 ** -11
        bound = u * ref.abs() + (2 * u + 2 * 128 * 128 * 18 * 3.5 * s * 2.0 ** -24 / 8) * (spread + ref.abs()) + 1e-6
        assert ((y.double().cpu() - ref).abs() <= bound).all(), scale


def test_attention_takes_strided_queries_and_tables():
    q, k, v, table, pos = oracle.paged_case(4, 2, 128, 16, [90, 130], 3, torch.float16, "cuda")
    want = paged_attention(q, k, v, table, pos)
    wide = torch.full((2, 3, 900), math.nan, dtype=q.dtype, device="cuda")
    for at in (0, 8, 3):  # aligned rows, and rows that have to be copied
        wide[..., at:at + 512] = q
        assert torch.equal(paged_attention(wide[..., at:at + 512], k, v, table, pos), want)
    assert torch.equal(paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, table, pos), want)
    odd = torch.full((2, 2 * table.shape[1]), -7, dtype=torch.int32, device="cuda")
    odd[:, ::2] = table
    assert torch.equal(paged_attention(q, k, v, odd[:, ::2], pos), want)
    odd[:, :table.shape[1]] = table
    assert torch.equal(paged_attention(q, k, v, odd[:, :table.shape[1]], pos), want)
    assert torch.equal(paged_attention(q, k, v, table, pos.t().contiguous().t()), want)
    one = q[:, 1:2]  # one token a row, rows 3 apart
    ref, spread = oracle.attention(one, k, v, table, pos[:, 1:2])
    _check(paged_attention(one, k, v, table, pos[:, 1:2]), ref, spread, torch.float16, 130)


def test_one_sequence_takes_a_table_of_any_stride():
    q, k, v, table, pos = oracle.paged_case(4, 2, 128, 16, [90], 3, torch.float16, "cuda")
    close = table.view(-1, 1).t()
    assert close.shape == table.shape and close.stride() == (1, 1)
    assert torch.equal(paged_attention(q, k, v, close, pos), paged_attention(q, k, v, table, pos))
    cos, sin = torch.randn(2, 1, 3, 128, device="cuda").unbind(0)
    heads, pools = q[..., :256].contiguous(), [(k.clone(), v.clone()) for _ in range(2)]
    out = [paged_rope_write(q, heads, heads, cos, sin, pos, *pool, t) for pool, t in zip(pools, (close, table))]
    assert torch.equal(*out) and all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(*pools))


def test_attention_of_nothing():
    q, k, v, table, pos = oracle.paged_case(4, 2, 128, 16, [20], 1, torch.float16, "cuda")
    assert paged_attention(q[:0], k, v, table[:0], pos[:0]).shape == (0, 1, 512)
    assert paged_attention(q[:, :0], k, v, table, pos[:, :0]).shape == (1, 0, 512)


def test_attention_past_32_bit_offsets():
    """A pool of 4.3 GB whose last pages a sequence uses: offsets in elements and bytes pass 2^31."""
    pages, kv, page, dim = 8200, 4, 512, 128
    k = torch.zeros(pages, kv, page, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    q, ks, vs, table, pos = oracle.paged_case(8, kv, dim, page, [700, 513], 1, torch.bfloat16, "cuda", spare=0)
    want = paged_attention(q, ks, vs, table, pos)
    n = ks.shape[0]
    k[-n:], v[-n:] = ks, vs
    moved = torch.where(table >= 0, table + (pages - n), -1)
    assert torch.equal(paged_attention(q, k, v, moved, pos), want)


def test_attention_of_more_blocks_than_a_launch_takes():
    """2^17 sequences of 17 tokens and 64 kv heads are 2^23 blocks of 512 threads, one launch's threads and one more."""
    batch, tokens, heads, dim = 1 << 17, 17, 64, 64
    print("\n[case] paged attention", batch, tokens, heads, dim, flush=True)
    k, v = (torch.randn(3, heads, 32, dim, device="cuda").half() for _ in range(2))
    table = (torch.arange(batch, device="cuda") % 3).int().view(batch, 1)
    pos = torch.arange(tokens, device="cuda").expand(batch, tokens).contiguous()
    some = torch.randn(3, tokens, heads * dim, device="cuda").half()
    q = torch.empty(batch, tokens, heads * dim, dtype=torch.float16, device="cuda")
    q.view(-1)[:3 * (batch // 3) * tokens * heads * dim].view(batch // 3, 3, -1).copy_(some.view(1, 3, -1))
    q[3 * (batch // 3):] = some[:batch % 3]
    y = paged_attention(q, k, v, table, pos)
    ref, spread = oracle.attention(some, k, v, table[:3], pos[:3])
    _check(y[:3], ref, spread, torch.float16, tokens)
    whole = y[:3 * (batch // 3)].view(batch // 3, 3, -1)
    assert all(bool((part == whole[:1]).all()) for part in whole.split(2048))
    assert torch.equal(y[3 * (batch // 3):], y[:batch % 3])


WRITE = [(4, 4, 128, 16, [1, 17], 1), (8, 2, 64, 48, [100, 3, 50], 7), (5, 5, 128, 16, [65], 64), (4, 1, 32, 8, [20, 9], 12),
         (6, 3, 16, 5, [23], 11)]


@pytest.mark.parametrize("dtype", HALF, ids=IDS)
@pytest.mark.parametrize("wide", [False, True], ids=["tables16", "tables32"])
@pytest.mark.parametrize("case", WRITE, ids=ids)
def test_write(case, wide, dtype):
    """Two products and a sum in fp32, three roundings of 2^-24 each, then one to the type; the rest of the pages stays."""
    print("\n[case] paged write", case, wide, dtype, flush=True)
    heads, kv, dim, page, lengths, tokens = case
    _, k_pages, v_pages, table, pos = oracle.paged_case(heads, kv, dim, page, lengths, tokens, dtype, "cuda")
    B = len(lengths)
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn(B, tokens, (heads + 2 * kv) * dim, generator=g).to(dtype).cuda()
    q, k, v = qkv.split([heads * dim, kv * dim, kv * dim], -1)
    angle = torch.randn(B, tokens, dim, generator=g) * 3
    cos, sin = (t.cuda() if wide else t.to(dtype).cuda() for t in (angle.cos(), angle.sin()))
    if page > 5:
        table[0, 0] = -1
    ref = oracle.write(q, k, v, cos, sin, pos, k_pages, v_pages, table)
    out = paged_rope_write(q, k, v, cos, sin, pos, k_pages, v_pages, table)
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for y, r in ((out, ref[0]), (k_pages, ref[1])):
        assert torch.allclose(y.double().cpu(), r, rtol=u, atol=3 * 2.0 ** -24 * 10 + tiny, equal_nan=True)
    assert torch.equal(v_pages.double().cpu().nan_to_num(123.0), ref[2].nan_to_num(123.0))
    assert (out[pos < 0] == 0).all()


def _drafts(B, n, V, greedy, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(B, n + 1, V, generator=g) * 2.5
    probs = torch.softmax(base[:, :n] + 0.6 * torch.randn(B, n, V, generator=g), -1)
    drafts = probs.argmax(-1) if greedy else torch.multinomial(probs.view(-1, V), 1, generator=g).view(B, n)
    if n and B > 1:
        drafts[::3, n // 2:] = -1
    u = torch.rand(B, n + 1, generator=g)
    return base.to(dtype).cuda(), drafts.cuda(), u.cuda(), None if greedy else probs.cuda()


VERIFY = [(1, 4, 32000), (5, 1, 1), (3, 2, 7), (64, 3, 257), (9, 0, 4096), (4, 5, 4097), (7, 7, 10001), (2, 17, 8192), (3, 2, 70001)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("temperature", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("case", VERIFY, ids=ids)
def test_verify(case, temperature, dtype):
    print("\n[case] verify", case, temperature, dtype, flush=True)
    for greedy in (False, True):
        logits, drafts, u, probs = _drafts(*case, greedy, dtype, seed=sum(case))
        want = oracle.verify(logits, drafts, u, probs, temperature)
        got = verify_drafts(logits, drafts, u, probs, temperature)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@pytest.mark.parametrize("temperature", [1e-37, 1e-20, 1e-9, 1e-3, 50.0, 1e30])
def test_verify_at_extreme_temperatures(temperature):
    for dtype in (torch.float32, torch.bfloat16):
        logits, drafts, u, probs = _drafts(7, 3, 5001, False, dtype, seed=12)
        drafts[:3] = logits[:3, :3].argmax(-1)
        for q in (probs, None):
            want = oracle.verify(logits, drafts, u, q, torch.tensor(temperature, dtype=torch.float32).item())
            got = verify_drafts(logits, drafts, u, q, temperature)
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_verify_rows_without_a_distribution():
    logits, drafts, u, probs = _drafts(8, 2, 9001, False, torch.float32, seed=3)
    drafts[:] = 4000
    logits[0, 0, 5000], logits[0, 0, 8000] = math.nan, math.nan
    logits[1, 0, 9000] = math.inf
    logits[2, 0] = -math.inf
    logits[3, 0, 4096:] = -math.inf
    logits[4, 0, :8192] = -math.inf
    logits[5, 0, 17] = logits[5, 0, 6000] = 50.0
    logits[6, 0] = -3.0e38  # far from 0, all alike
    drafts[7, 0] = 1 << 40
    for temperature in (0.0, 1.0):
        for q in (probs, None):
            want = oracle.verify(logits, drafts, u, q, temperature)
            got = verify_drafts(logits, drafts, u, q, temperature)
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert got[1][:3, 0].tolist() == [5000, 9000, 0]


@pytest.mark.parametrize("case", [(300, 3, 16390), (90, 7, 12300), (2100, 0, 4100), (700, 2, 30)], ids=ids)
def test_verify_of_many_rows(case):
    """Chunks of several parts: rows alike in number to what the card holds, and more."""
    print("\n[case] verify", case, flush=True)
    B, n, V = case
    logits, drafts, u, probs = _drafts(B, n, V, False, torch.bfloat16, seed=V)
    logits[0, 0, V - 1] = logits[1, 0, V // 2] = math.nan
    logits[2, 0, V - 2] = math.inf
    logits[3, 0, 1:] = -math.inf
    logits[4, 0, :V - 1] = -math.inf
    logits[5, 0] = -math.inf
    want = oracle.verify(logits, drafts, u, probs)
    got = verify_drafts(logits, drafts, u, probs)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_verify_at_the_ends_of_the_random_numbers():
    """0 and the largest number below 1; drafter and model alike, so that nothing is left of a turned-down draft's row."""
    logits, drafts, u, probs = _drafts(6, 2, 5000, False, torch.float32, seed=8)
    logits[:, :, 4990:] = -math.inf
    u[:3], u[3:] = 0.0, 1.0 - 2.0 ** -24
    probs[:] = torch.softmax(logits[:, :2], -1) * (1 + 1e-3)
    probs[5] = 1.0
    want = oracle.verify(logits, drafts, u, probs)
    got = verify_drafts(logits, drafts, u, probs)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert int(got[1].max()) < 4990


@pytest.mark.parametrize("dtype,mask", [(torch.float32, -1e4), (torch.float32, torch.finfo(torch.float32).min),
                                        (torch.float16, -65504.0), (torch.bfloat16, -1e4)], ids=str)
def test_verify_never_takes_a_token_masked_with_a_finite_number(dtype, mask):
    """exp is 0 in float64 that far below the largest: at a random number of 0 neither the first index nor a draft is taken for
    it, and where the drafter's probabilities cover the model's there is nothing left but p itself."""
    logits, drafts, u, probs = _drafts(6, 2, 5000, False, dtype, seed=15)
    logits[:, :, :10] = mask
    logits[:, :, 4990:] = mask
    u[:3] = 0.0
    drafts[0], drafts[1] = 3, 4995   # masked drafts
    u[3:, :2] = 1.0 - 2.0 ** -24
    probs[:] = torch.softmax(logits[:, :2].float(), -1) * (1 + 1e-3)  # q > p wherever p is positive
    for q in (probs, None):
        for temperature in (1.0, 0.7):
            want = oracle.verify(logits, drafts, u, q, temperature)
            got = verify_drafts(logits, drafts, u, q, temperature)
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
            kept = got[0].view(-1, 1) > torch.arange(3, device="cuda")
            extra = got[1][(got[1] >= 0) & ~kept]
            assert int(extra.min()) >= 10 and int(extra.max()) < 4990


def test_verify_where_exponentials_are_subnormal():
    """Weights down to 2^-1074 are weights, and those below are none: exponents of -728 and -768, whose exponentials are near
    1e-316 and 1e-334, and the same by a small temperature."""
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.full((4, 2, 3000), -768.0, dtype=dtype, device="cuda")
        logits[:, :, 2000] = 0.0
        logits[1:, :, 700] = -728.0
        drafts = torch.tensor([[5], [700], [1], [2000]], device="cuda")
        u = torch.zeros(4, 2, device="cuda")
        for x, temperature in ((logits, 1.0), (logits / 1024, 2.0 ** -10)):
            got = verify_drafts(x, drafts, u, None, temperature)
            want = oracle.verify(x, drafts, u, None, temperature)
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
            assert got[1][:3, 0].tolist() == [2000, 700, 700]
    x = torch.tensor([[[0.0, -10.0, 5.0]]], device="cuda")
    got = verify_drafts(x, torch.zeros(1, 0, dtype=torch.int64, device="cuda"), torch.zeros(1, 1, device="cuda"), None, 0.005)
    assert got[1].tolist() == [[2]]


@pytest.mark.parametrize("temperature", [0.6, 0.7, 1.3])
def test_verify_takes_the_temperature_as_given(temperature):
    """Accept tests u q < p whose two sides differ by less than rounding the temperature to float32 moves p, and by more than
    1e-13 of it: float64's exponential and quotient are off by some 1e-15."""
    g = torch.Generator().manual_seed(16)
    logits = torch.randn(4000, 2, 3, generator=g) * 4
    drafts = torch.randint(0, 3, (4000, 1), generator=g)
    rounded = torch.tensor(temperature).double()  # float32
    p, near = (torch.softmax(logits[:, 0].double() / t, -1).gather(1, drafts)[:, 0] for t in (temperature, rounded))
    u = torch.rand(4000, 2, generator=g) * 0.5 + 0.5
    q = ((p + near) / 2 / u[:, 0].double()).float()
    sides = torch.stack((p, near)) - u[:, 0].double() * q.double()
    pick = (sides[0] * sides[1] < 0) & (sides.abs() > 1e-13 * p).all(0)
    assert int(pick.sum()) > 50
    logits, drafts, u, q = logits[pick], drafts[pick], u[pick], q[pick]
    probs = torch.zeros(len(q), 1, 3).scatter_(2, drafts.unsqueeze(1), q.view(-1, 1, 1))
    want = oracle.verify(logits, drafts, u, probs, temperature)
    assert 0 < int(want[0].sum()) < len(q)
    for device in ("cpu", "cuda"):
        got = verify_drafts(*(t.to(device) for t in (logits, drafts, u, probs)), temperature)
        assert torch.equal(got[0].cpu(), want[0])


@pytest.mark.parametrize("temperature", [1e-310, 5e-324, 1e-46, 1e-40, 1e300])
def test_verify_at_temperatures_that_no_float32_holds(temperature):
    """A positive temperature is not greedy, however small, and no finite one too large."""
    logits = torch.tensor([1.0, 1.0, 0.0], device="cuda").expand(4, 2, 3)
    u = torch.tensor([[0.9, 0.3], [0.9, 0.7], [0.3, 0.99], [0.1, 0.0]], device="cuda")
    for draft in (0, 1, 2):
        drafts = torch.full((4, 1), draft, device="cuda")
        for probs in (None, torch.tensor([0.9, 0.1, 0.0], device="cuda").expand(4, 1, 3)):
            want = oracle.verify(logits, drafts, u, probs, temperature)
            got = verify_drafts(logits, drafts, u, probs, temperature)
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_verify_takes_strided_rows():
    logits, drafts, u, probs = _drafts(4, 3, 5003, False, torch.bfloat16, seed=9)
    want = verify_drafts(logits, drafts, u, probs)
    for shift in (0, 1, 5):
        wide = torch.full((4, 4, 5100), 60.0, dtype=torch.bfloat16, device="cuda")
        wide[..., shift:shift + 5003] = logits
        got = verify_drafts(wide[..., shift:shift + 5003], drafts, u, probs)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = verify_drafts(logits, drafts.t().contiguous().t(), u, probs.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(got[1], want[1])


def test_verify_takes_single_rows_whatever_their_strides():
    """No drafts: one row a sequence, as a view whose strides of dimensions of one element are any."""
    logits, drafts, u, _ = _drafts(6, 0, 3001, True, torch.float32, seed=14)
    want = verify_drafts(logits, drafts, u)
    across = logits.view(1, 6, 3001).transpose(0, 1)
    assert across.stride() == (3001, 18006, 1)
    wide = torch.full((6, 2, 3100), 60.0, device="cuda")
    wide[:, 1, :3001] = logits[:, 0]
    close = torch.as_strided(logits, (1, 1, 3001), (1, 1, 1))
    for x, n in ((across, 6), (wide[:, 1:, :3001], 6), (close, 1)):
        got = verify_drafts(x, drafts[:n], u[:n])
        assert torch.equal(got[0], want[0][:n]) and torch.equal(got[1], want[1][:n])


def _together(cache, shape, tokens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda n: torch.randn(cache.batch, tokens, n * 128, device="cuda", generator=g).half()  # noqa: E731
    return draw(shape.heads), draw(shape.kv_heads), draw(shape.kv_heads)


def test_captured_steps_follow_the_table_and_the_positions():
    """Two graphs (one token, three tokens), captured one after the other and replayed in turn between eager calls and
    synchronizations, while positions and pages move: every replay equals the eager call."""
    shape = LlamaShape(hidden=1024, layers=1, heads=8, kv_heads=2, ffn=64, vocab=64)
    cache = PagedKVCache(shape, 3, pages=64, page_size=16, max_len=600, device="cuda", dtype=torch.float16, window=0)
    cache.k[0].normal_()
    cache.v[0].normal_()
    for b in range(3):
        cache.reserve(b, 20 + 90 * b)
    stream, graphs = torch.cuda.Stream(), []
    for tokens in (1, 3):
        q, _, _ = _together(cache, shape, tokens, tokens)
        pos = torch.zeros(3, tokens, dtype=torch.int64, device="cuda")
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            paged_attention(q, cache.k[0], cache.v[0], cache.table, pos)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = paged_attention(q, cache.k[0], cache.v[0], cache.table, pos)
        graphs.append((graph, q, pos, out, tokens))
    for step in range(4):
        for graph, q, pos, out, tokens in graphs:
            base = torch.tensor([3 + step, 100 + step, 190 + 2 * step], device="cuda")
            pos.copy_(base.view(3, 1) + torch.arange(tokens, device="cuda"))
            graph.replay()
            got = out.clone()
            assert torch.equal(got, paged_attention(q, cache.k[0], cache.v[0], cache.table, pos))
        torch.cuda.synchronize()
        cache.release(1)
        cache.reserve(1, 110 + 60 * step)


def test_captured_steps_that_share_their_work():
    """The same for calls with a workspace (one token, drafts, a chunk; long tables), each graph holding two calls in a row."""
    k, v = (torch.randn(400, 2, 16, 128, device="cuda").bfloat16() for _ in range(2))
    table = torch.randperm(400, device="cuda")[:390].view(2, 195).int()
    stream, graphs = torch.cuda.Stream(), []
    for tokens in (1, 9, 40):
        assert _lib.load().nq_paged_attention_workspace_bytes(2, tokens, 8, 2, 128, 195, 16) > 0
        q = torch.randn(2, 2, tokens, 1024, device="cuda").bfloat16()
        pos = torch.zeros(2, tokens, dtype=torch.int64, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = [paged_attention(x, k, v, table, pos) for x in q]
        graphs.append((graph, q, pos, out))
    for step in range(4):
        for graph, q, pos, out in graphs:
            base = torch.tensor([[700 * step], [3000 - 900 * step]], device="cuda")
            pos.copy_(base + torch.arange(pos.shape[1], device="cuda"))
            graph.replay()
            got = [o.clone() for o in out]
            assert all(torch.equal(g, paged_attention(x, k, v, table, pos)) for g, x in zip(got, q))
        torch.cuda.synchronize()
        table.copy_(table.flip(0) if step % 2 else table.flip(1))


def test_captured_verification():
    logits, drafts, u, probs = _drafts(5, 3, 9000, False, torch.float32, seed=10)
    verify_drafts(logits, drafts, u, probs)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        out = verify_drafts(logits, drafts, u, probs)
    for step in range(3):
        fresh = _drafts(5, 3, 9000, False, torch.float32, seed=20 + step)
        for kept, new in zip((logits, drafts, u, probs), fresh):
            kept.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want = oracle.verify(logits, drafts, u, probs)
        assert torch.equal(out[0].cpu(), want[0]) and torch.equal(out[1].cpu(), want[1])


def test_calls_on_two_streams():
    """Calls at once on two streams, each with its own workspace, equal the calls one after the other."""
    made = [oracle.paged_case(8, 2, 128, 16, lengths, tokens, torch.float16, "cuda", seed=s)
            for s, (lengths, tokens) in enumerate([([900, 1200], 1), ([700, 300], 4)])]
    want = [paged_attention(*m) for m in made]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, m in zip(streams, made):
            with torch.cuda.stream(s):
                got.append(paged_attention(*m))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_gradients_and_other_types_run_torch_ops():
    q, k, v, table, pos = oracle.paged_case(4, 2, 32, 8, [12, 20], 3, torch.float32, "cuda")
    ref, _ = oracle.attention(q, k, v, table, pos)
    assert (paged_attention(q, k, v, table, pos).double().cpu() - ref).abs().max() < 1e-5
    q, k, v, table, pos = oracle.paged_case(4, 2, 64, 16, [12, 20], 3, torch.float16, "cuda")
    q.requires_grad_(True)
    y = paged_attention(q, k, v, table, pos)
    assert y.requires_grad and (y.detach().float() - paged_attention(q.detach(), k, v, table, pos).float()).abs().max() < 4e-3


def test_a_model_serves_two_sequences():
    """Prompts of two lengths in one padded batch, drafted tokens of both in one pass, their verification, and a single token:
    the tokens that a model alone on each sequence takes greedily."""
    shape = LlamaShape(hidden=512, layers=2, heads=4, kv_heads=2, ffn=768, vocab=1000)
    model = random_llama(shape, device="cuda", kernel_type="gemv", dtype=torch.float16, seed=5)
    g = torch.Generator().manual_seed(6)
    lengths = [70, 33]
    cache = PagedKVCache(shape, 2, pages=30, page_size=16, max_len=200, device="cuda", dtype=torch.float16)
    ids, positions = torch.zeros(2, 70, dtype=torch.int64), torch.full((2, 70), -1)
    for b, n in enumerate(lengths):
        ids[b, :n] = torch.randint(0, 1000, (n,), generator=g)
        positions[b, :n] = torch.arange(n)
        cache.reserve(b, n + 12)
    ids, positions = ids.cuda(), positions.cuda()

    def alone(b, tokens, upto):  # float32 logits of a whole sequence on a paged cache of its own, run as one prompt
        own = PagedKVCache(shape, 1, pages=12, page_size=16, max_len=192, device="cuda", dtype=torch.float16)
        own.reserve(0, upto)
        return model(tokens[:upto].view(1, -1), torch.arange(upto, device="cuda"), own)[0]

    with torch.no_grad():
        logits = model(ids, positions, cache)
        seqs = []
        for b, n in enumerate(lengths):
            seqs.append(torch.cat((ids[b, :n], logits[b, n - 1].argmax().view(1))))
            want = alone(b, seqs[b], n)
            assert (logits[b, :n] - want).abs().max() <= 0.02 * want.abs().max()
        for _ in range(3):
            # three drafts each: the greedy ones of sequence 0, of sequence 1 the second one wrong
            drafts = []
            for b in range(2):
                s = seqs[b]
                for i in range(3):
                    nxt = alone(b, s, s.numel())[-1].argmax().view(1)
                    s = torch.cat((s, (nxt + 1) % 1000 if b == 1 and i == 1 else nxt))
                drafts.append(s[-3:])
            drafts = torch.stack(drafts)
            pos = torch.stack([torch.arange(s.numel() - 1, s.numel() + 3, device="cuda") for s in seqs])
            logits = model(torch.cat((torch.stack([s[-1:] for s in seqs]), drafts), 1), pos, cache)
            accepted, tokens = verify_drafts(logits, drafts, torch.rand(2, 4, device="cuda"), temperature=0.0)
            for b in range(2):
                cache.reserve(b, seqs[b].numel() + 12)
                kept = int(accepted[b])
                whole = alone(b, torch.cat((seqs[b], drafts[b])), seqs[b].numel() + 3)[-4:]
                # the pass over the drafts sees what one prompt sees
                assert (logits[b] - whole).abs().max() <= 0.02 * whole.abs().max()
                greedy = logits[b].argmax(-1)
                assert kept == int((greedy[:3] == drafts[b]).long().cumprod(0).sum())
                assert tokens[b, :kept + 1].tolist() == greedy[:kept + 1].tolist() and (tokens[b, kept + 1:] == -1).all()
                seqs[b] = torch.cat((seqs[b], tokens[b, :kept + 1]))
            assert int(accepted[1]) <= 1
