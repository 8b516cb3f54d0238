"""The paged cache and draft verification on the CPU (the torch ops), their refusals, and the C ABI's."""
import math

import pytest
import torch

import serve_oracle as oracle
from nanoquant_amd import PagedKVCache, _lib, paged_attention, paged_rope_write, verify_drafts
from nanoquant_amd.decode import LlamaShape, StaticKVCache, random_llama

TINY = LlamaShape(hidden=128, layers=2, heads=4, kv_heads=2, ffn=320, vocab=500)


@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 0), (7, 2), (1, 1)])
@pytest.mark.parametrize("lengths,tokens", [([1], 1), ([17, 3, 40], 1), ([9, 31], 5), ([4, 33], 12)])
def test_attention_against_the_definition(lengths, tokens, window, sinks):
    """float32: what is left is summation, far below 1e-5."""
    q, k, v, table, pos = oracle.paged_case(4, 2, 32, 8, lengths, tokens, torch.float32, "cpu", window=window, sinks=sinks)
    y = paged_attention(q, k, v, table, pos, window, sinks)
    ref, _ = oracle.attention(q, k, v, table, pos, window, sinks)
    assert (y.double() - ref).abs().max() < 1e-5
    assert torch.equal(y[pos < 0], torch.zeros_like(y[pos < 0]))


def test_attention_rows_that_see_nothing():
    q, k, v, table, pos = oracle.paged_case(2, 1, 32, 8, [10, 20], 1, torch.float32, "cpu")
    pos[0, 0] = table.shape[1] * 8  # past the table
    table[1] = 1000                 # no such page
    assert torch.equal(paged_attention(q, k, v, table, pos), torch.zeros_like(q))


def test_values_that_a_token_does_not_see_do_not_reach_it():
    q, k, v, table, pos = oracle.paged_case(2, 1, 32, 8, [12], 4, torch.float32, "cpu")
    page = int(table[0, 1])
    k[page, 0, 3], v[page, 0, 3] = math.inf, math.nan  # position 11, which the last token alone sees
    v[page, 0, 2] = math.inf                           # position 10
    y = paged_attention(q, k, v, table, pos)
    ref, _ = oracle.attention(q, k, v, table, pos)
    assert torch.isfinite(y[0, :2]).all() and (y[0, :2].double() - ref[0, :2]).abs().max() < 1e-5
    assert (y[0, 2] == math.inf).all()
    assert y[0, 3].isnan().all()


def test_rows_of_the_table_whatever_the_strides():
    """A table of one sequence has any stride between its rows, and is not refused for it."""
    from nanoquant_amd.serve import _table_rows
    x = torch.arange(24, dtype=torch.int32).view(4, 6)
    for t in (x, x[:, 1:3], x[1:2], x[:, 2:3], x[:, 3:4].t(), x[0, :, None].t(), x.t(), x[2].expand(5, 6), x[:, ::2],
              torch.as_strided(x, (1, 6), (0, 1))):
        rows = _table_rows(t)
        assert rows.stride(0) >= t.shape[1] and (rows.stride(1) == 1 or t.shape[1] == 1) and torch.equal(rows, t)
    assert _table_rows(x[:, 1:3]).data_ptr() == x[:, 1:3].data_ptr()  # read in place


def _gradients(q, k_pages, v_pages, table, positions, w, window=0, sinks=0):
    """Of sum w out by q and the pages, from the formula in float64, and how far float32 ones may be off.

    A score is off by (D + 1) u times its summed |q k| scale at most (u = 2^-24), so a probability by a factor of 1 +- e with e
    twice the largest of that, and 8 u for the exponential and the division. With a_j = |w| . |v_j| the gradient of score j,
    p_j (w . v_j - sum_i p_i w . v_i), is off by e p_j (a_j + 2 sum_i p_i a_i), and those of q, k and v by what that makes of
    their terms, and half as much again for the sums' own roundings."""
    q, k_pages, v_pages, w = (t.double() for t in (q, k_pages, v_pages, w))
    N, KV, S, D = k_pages.shape
    dq, dk, dv = (torch.zeros(2, *t.shape, dtype=torch.float64) for t in (q, k_pages, v_pages))
    for b in range(q.shape[0]):
        page = table[b].long().repeat_interleave(S)
        row = torch.arange(page.shape[0]) % S
        for t in range(q.shape[1]):
            seen = oracle.visible(int(positions[b, t]), page.shape[0], window, sinks) & (page >= 0) & (page < N)
            if not seen.any():
                continue
            at = (page[seen], slice(None), row[seen])
            k, v = k_pages[at].transpose(0, 1), v_pages[at].transpose(0, 1)  # [KV, keys, D]
            qt, wt = (x[b, t].view(KV, -1, D) for x in (q, w))
            p = torch.softmax(qt @ k.transpose(1, 2) * D ** -0.5, -1)
            e = 1.5 * (2 * (D + 1) * 2.0 ** -24 * float((qt.abs() @ k.abs().transpose(1, 2)).max()) * D ** -0.5 + 8 * 2.0 ** -24)
            for i, (dp, sign, s, kk, qq, ww) in enumerate((
                    (wt @ v.transpose(1, 2), -1.0, 1.0, k, qt, wt),
                    (wt.abs() @ v.abs().transpose(1, 2), 2.0, e, k.abs(), qt.abs(), wt.abs()))):
                ds = s * p * (dp + sign * (p * dp).sum(-1, keepdim=True)) * D ** -0.5
                dq[i, b, t] += (ds @ kk).reshape(-1)
                dk[i][at] += (ds.transpose(1, 2) @ qq).transpose(0, 1)
                dv[i][at] += (s * p.transpose(1, 2) @ ww).transpose(0, 1)
    return dq, dk, dv


def _leaves(*tensors):
    return [t.clone().requires_grad_(True) for t in tensors]


@pytest.mark.parametrize("window,sinks", [(0, 0), (7, 2)])
def test_gradients_of_tokens_that_all_see_something(window, sinks):
    """No padding, whole pages: the torch ops' gradients against the formula's and, in one direction, against differences."""
    q, k, v, table, pos = oracle.paged_case(4, 2, 32, 8, [16, 32], 5, torch.float32, "cpu", window=window, sinks=sinks, spare=0)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    w = torch.randn(q.shape, generator=torch.Generator().manual_seed(11))
    leaves = _leaves(q, k, v)
    (paged_attention(*leaves, table, pos, window, sinks) * w).sum().backward()
    along = 0.0
    step = [torch.randn(x.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64) for i, x in enumerate((q, k, v))]
    for leaf, want, d in zip(leaves, _gradients(q, k, v, table, pos, w, window, sinks), step):
        assert ((leaf.grad.double() - want[0]).abs() <= want[1]).all()
        along += float((want[0] * d).sum())
    h = 1e-4  # the third derivative's part of the quotient is h^2 / 6 times it, far below 1e-4 of the sum
    ends = [(oracle.attention(*(x.double() + f * h * d for x, d in zip((q, k, v), step)), table, pos, window, sinks)[0] * w).sum()
            for f in (1.0, -1.0)]
    assert abs(float(ends[0] - ends[1]) / (2 * h) - along) < 1e-4 * (1 + abs(along))


@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 2)])
def test_gradients_beside_tokens_that_see_nothing(window, sinks):
    """Padding, a sequence without pages and a position past the table have no gradient and leave the others theirs."""
    q, k, v, table, pos = oracle.paged_case(4, 2, 32, 8, [16, 3, 32], 5, torch.float32, "cpu", window=window, sinks=sinks)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    pos[0, 1] = table.shape[1] * 8
    table[2, :] = -1
    q[pos < 0] = math.nan
    w = torch.randn(q.shape, generator=torch.Generator().manual_seed(12))
    leaves = _leaves(q, k, v)
    y = paged_attention(*leaves, table, pos, window, sinks)
    (y * w).sum().backward()
    assert (y[pos < 0] == 0).all() and (y[2] == 0).all()
    for leaf, want in zip(leaves, _gradients(q, k, v, table, pos, w, window, sinks)):
        assert ((leaf.grad.double() - want[0]).abs() <= want[1]).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_gradients_beside_keys_that_are_not_finite(bad):
    """Rows of the pages that hold nothing yet, or keys of later tokens, have no part in a token's gradient."""
    q, k, v, table, pos = oracle.paged_case(4, 2, 32, 8, [9, 21], 3, torch.float32, "cpu")
    k, v = torch.where(k.isnan(), bad, k), torch.where(v.isnan(), bad, v)
    w = torch.randn(q.shape, generator=torch.Generator().manual_seed(13))
    want = _gradients(q, k, v, table, pos, w)
    leaves = _leaves(q, k, v)
    (paged_attention(*leaves, table, pos) * w).sum().backward()
    for leaf, (grad, bound) in zip(leaves, want):
        assert ((leaf.grad.double() - grad).abs() <= bound).all()
    k[int(table[1, 2]), :, 4, 3] = math.nan  # position 20 of sequence 1, which its last token alone sees
    leaves = _leaves(q, k, v)
    y = paged_attention(*leaves, table, pos)
    (y * w).sum().backward()
    assert y[1, 2].isnan().all()
    early = torch.tensor([[True, True, True], [True, True, False]])
    assert ((leaves[0].grad.double() - want[0][0])[early].abs() <= want[0][1][early]).all()


def test_float64_stays_float64():
    """Results and gradients: differences of float64 results need them."""
    q, k, v, table, pos = oracle.paged_case(2, 1, 8, 4, [3, 7], 3, torch.float64, "cpu", window=4, sinks=1)
    ref, _ = oracle.attention(q, k, v, table, pos, 4, 1)
    assert (paged_attention(q, k, v, table, pos, 4, 1) - ref).abs().max() < 1e-13
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    pos[0, 2] = -1
    assert torch.autograd.gradcheck(lambda *x: paged_attention(*x, table, pos, 4, 1), _leaves(q, k, v))
    g = torch.Generator().manual_seed(17)
    q, heads = torch.randn(2, 3, 16, generator=g).double(), torch.randn(2, 3, 8, generator=g).double()
    cos, sin = torch.randn(2, 2, 3, 8, generator=g).double().unbind(0)
    want = oracle.write(q, heads, heads, cos, sin, pos, k, v, table)
    out = paged_rope_write(q, heads, heads, cos, sin, pos, k, v, table)
    assert all((a - b).abs().max() < 1e-13 for a, b in zip((out, k, v), want))


def test_torch_ops_keep_their_precision_under_autocast():
    q, k, v, table, pos = oracle.paged_case(4, 2, 32, 8, [17, 30], 3, torch.float32, "cpu")
    leaves = _leaves(q, k, v)
    want = paged_attention(*leaves, table, pos)
    want.sum().backward()
    again = _leaves(q, k, v)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = paged_attention(*again, table, pos)
    got.sum().backward()
    assert torch.equal(got, want) and all(torch.equal(a.grad, b.grad) for a, b in zip(again, leaves))


def test_write_against_the_definition():
    _, k_pages, v_pages, table, pos = oracle.paged_case(4, 2, 32, 8, [9, 30, 3], 5, torch.float32, "cpu")
    g = torch.Generator().manual_seed(1)
    B, T = pos.shape
    q, k, v = (torch.randn(B, T, n * 32, generator=g) for n in (4, 2, 2))
    angle = torch.randn(B, T, 32, generator=g)
    cos, sin = angle.cos(), angle.sin()
    table[1, 3] = -1  # the page of position 25 on
    ref = oracle.write(q, k, v, cos, sin, pos, k_pages, v_pages, table)
    y = paged_rope_write(q, k, v, cos, sin, pos, k_pages, v_pages, table)
    for a, b in zip((y, k_pages, v_pages), ref):
        assert torch.allclose(a.double(), b, rtol=0, atol=1e-6, equal_nan=True)


@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
@pytest.mark.parametrize("greedy", [False, True])
def test_verify_against_the_definition(greedy, temperature):
    logits, drafts, probs, u = _drafts(40, 3, 50, greedy, seed=2)
    want = oracle.verify(logits, drafts, u, probs, temperature)
    got = verify_drafts(logits, drafts, u, probs, temperature)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if temperature:
        assert 0 < int(want[0].sum()) < want[0].numel() * 3  # both ways were taken


def _drafts(B, n, V, greedy, seed):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, n + 1, V, generator=g) * 2
    probs = torch.softmax(logits[:, :n] + 0.5 * torch.randn(B, n, V, generator=g), -1)
    drafts = probs.argmax(-1) if greedy else torch.multinomial(probs.view(B * n, V), 1, generator=g).view(B, n)
    drafts[::5, n // 2:] = -1
    drafts[3::7, 0] = V
    return logits, drafts, None if greedy else probs, torch.rand(B, n + 1, generator=g)


def test_verify_rows_without_a_distribution():
    logits, drafts, probs, u = _drafts(6, 2, 20, False, seed=3)
    drafts[:] = 4
    logits[0, 0, 7] = math.nan
    logits[1, 0, 9] = math.inf
    logits[2, 0] = -math.inf
    logits[3, 0, 11:] = -math.inf  # fine: those tokens cannot come
    want = oracle.verify(logits, drafts, u, probs)
    got = verify_drafts(logits, drafts, u, probs)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert got[1][:3, 0].tolist() == [7, 9, 0]


def test_rows_of_logits_whatever_the_strides():
    """The rows that a kernel would read are the tensor's, also where a dimension has one element and any stride."""
    from nanoquant_amd.serve import _logit_rows
    x = torch.arange(4 * 7 * 10).view(4, 7, 10).float()
    for t in (x, x[..., 1:9], x[:, :3], x[:, ::2], x[:, 2:3], x[2:3], x[2:3, 4:5], x[1:2].transpose(0, 1), x[..., 3:4], x[:1, :1, :1],
              x.transpose(0, 1), x[:, 3].unsqueeze(1).expand(4, 5, 10), x[0, :, :1].t()[None], x[0, :, :1].t().unsqueeze(1)):
        rows, stride = _logit_rows(t)
        B, R, V = t.shape
        at = rows.storage_offset() + (B * R - 1) * stride + V
        assert stride >= V and at <= rows.untyped_storage().nbytes() // 4
        assert torch.equal(torch.as_strided(rows, (B * R, V), (stride, 1), rows.storage_offset()).reshape(t.shape), t)
    assert _logit_rows(x[1:2].transpose(0, 1))[0].data_ptr() == x[1:2].data_ptr()  # read in place


def test_verified_tokens_have_the_models_distribution():
    """Over a fine grid of random numbers the first token's frequencies are the model's probabilities: of 400 x 400 pairs
    (accept, pick) a border moves a count by at most one a row of the grid, so each is within 2 / 400 of p."""
    n, V = 400, 6
    g = torch.Generator().manual_seed(5)
    logits, probs = torch.randn(1, 2, V, generator=g), torch.softmax(torch.randn(1, 1, V, generator=g), -1)
    p = torch.softmax(logits[0, 0].double(), -1)
    grid = (torch.arange(n) + 0.5) / n
    u = torch.stack(torch.meshgrid(grid, grid, indexing="ij"), -1).view(-1, 2)
    count = torch.zeros(V, dtype=torch.float64)
    for d in range(V):
        drafts = torch.full((n * n, 1), d)
        _, tokens = verify_drafts(logits.expand(n * n, 2, V), drafts, u, probs.expand(n * n, 1, V))
        count += probs[0, 0, d].double() * torch.bincount(tokens[:, 0], minlength=V)
    assert ((count / (n * n)) - p).abs().max() < 2.0 / n


@pytest.mark.parametrize("temperature", [1e-310, 5e-324, 1e-46, 1e300])
def test_verify_at_temperatures_whose_reciprocal_or_float_is_none(temperature):
    """A positive temperature is not greedy, however small: two tokens that are equally likely share the draws."""
    logits = torch.tensor([1.0, 1.0, 0.0]).expand(1, 2, 3)
    for draft in (0, 1, 2):
        for u in ([0.9, 0.3], [0.9, 0.7], [0.3, 0.99], [0.1, 0.0]):
            drafts, us = torch.tensor([[draft]]), torch.tensor([u])
            for probs in (None, torch.tensor([[[0.9, 0.1, 0.0]]])):
                want = oracle.verify(logits, drafts, us, probs, temperature)
                got = verify_drafts(logits, drafts, us, probs, temperature)
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_paged_model_equals_the_static_cache():
    """Prompts of two lengths in one padded batch, then single tokens, against each sequence alone on a static cache."""
    model = random_llama(TINY, device="cpu", seed=3)
    g = torch.Generator().manual_seed(4)
    lengths = [11, 5]
    ids = torch.randint(0, TINY.vocab, (2, 14), generator=g)
    cache = PagedKVCache(TINY, 2, pages=12, page_size=4, max_len=24, device="cpu", dtype=torch.float32)
    positions = torch.full((2, 11), -1)
    for b, n in enumerate(lengths):
        cache.reserve(b, n + 3)
        positions[b, :n] = torch.arange(n)
    with torch.no_grad():
        first = model(ids[:, :11], positions, cache)
        steps = []
        for i in range(3):
            tok = torch.stack([ids[b, n + i] for b, n in enumerate(lengths)]).view(2, 1)
            steps.append(model(tok, torch.tensor([[n + i] for n in lengths]), cache))
        for b, n in enumerate(lengths):
            alone = StaticKVCache(TINY, 1, 24, "cpu", torch.float32)
            want = model(ids[b:b + 1, :n], torch.arange(n), alone)
            assert torch.allclose(first[b, :n], want[0], atol=1e-4)
            for i in range(3):
                want = model(ids[b:b + 1, n + i:n + i + 1], torch.tensor([n + i]), alone)
                assert torch.allclose(steps[i][b], want[0], atol=1e-4)


def test_pages_are_handed_out_and_taken_back():
    cache = PagedKVCache(TINY, 2, pages=6, page_size=4, max_len=40, device="cpu", dtype=torch.float32, window=8, sinks=3)
    cache.reserve(0, 17)
    assert (cache.table[0, :5] >= 0).all() and (cache.table[0, 5:] == -1).all()
    with pytest.raises(RuntimeError, match="1 pages left, sequence 1 needs 2"):
        cache.reserve(1, 5)
    assert (cache.table[1] == -1).all()
    assert cache.trim(0, 15) == 1  # positions 8 .. and the first 3: page 1 (4 .. 7) goes
    assert cache.table[0, :5].lt(0).tolist() == [False, True, False, False, False]
    cache.reserve(1, 5)
    used = cache.table[cache.table >= 0]
    assert used.unique().numel() == used.numel() == 6
    assert cache.trim(0, 1000) == 3 and cache.release(0) == 1 and cache.release(0) == 0
    cache.reserve(0, 40, start=28)
    assert (cache.table[0] >= 0).nonzero().flatten().tolist() == [7, 8, 9]
    with pytest.raises(ValueError, match="max_len"):
        cache.reserve(0, 41)
    with pytest.raises(IndexError):
        cache.reserve(2, 1)
    with pytest.raises(ValueError, match="bad sizes"):
        PagedKVCache(TINY, 1, 1, 0, 1, "cpu", torch.float32)


def test_refusals():
    q, k, v, table, pos = oracle.paged_case(4, 2, 32, 8, [9, 12], 2, torch.float32, "cpu")
    kv, cs = torch.zeros(2, 2, 64), torch.zeros(2, 2, 32)
    with pytest.raises(ValueError, match="does not fit"):
        paged_attention(q[:, :1], k, v, table, pos)
    with pytest.raises(ValueError, match="does not fit"):
        paged_attention(q[..., :96], k, v, table, pos)  # 3 heads over 2
    with pytest.raises(ValueError, match="alike"):
        paged_attention(q, k, v[:1], table, pos)
    with pytest.raises(ValueError, match="table"):
        paged_attention(q, k, v, table[:1], pos)
    with pytest.raises(TypeError, match="int32"):
        paged_attention(q, k, v, table.long(), pos)
    with pytest.raises(TypeError, match="pages are"):
        paged_attention(q.half(), k, v, table, pos)
    with pytest.raises(ValueError, match="negative"):
        paged_attention(q, k, v, table, pos, window=-1)
    with pytest.raises(ValueError, match="do not fit"):
        paged_rope_write(q, kv[:, :1], kv, cs, cs, pos, k, v, table)
    with pytest.raises(ValueError, match="cos"):
        paged_rope_write(q, kv, kv, cs[:1], cs[:1], pos, k, v, table)
    with pytest.raises(TypeError, match="one type"):
        paged_rope_write(q, kv, kv, cs.double(), cs.double(), pos, k, v, table)
    logits, drafts, u = torch.zeros(2, 3, 5), torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 3)
    with pytest.raises(ValueError, match="drafts"):
        verify_drafts(logits[:, :2], drafts, u)
    with pytest.raises(ValueError, match="uniforms"):
        verify_drafts(logits, drafts, u[:, :2])
    with pytest.raises(ValueError, match="draft_probs"):
        verify_drafts(logits, drafts, u, torch.zeros(2, 2, 4))
    with pytest.raises(TypeError, match="int64"):
        verify_drafts(logits, drafts.int(), u)
    for bad in (-1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            verify_drafts(logits, drafts, u, temperature=bad)


def test_c_abi_argument_errors_need_no_gpu():
    lib = _lib.load()
    p = 256  # a pointer that is never followed: every call below ends before its launch

    def attn(dtype=0, q=p, stride=128 * 4, pages=4, page_size=16, table_stride=8, table_pages=8, batch=1, tokens=1, heads=4, kv=2,
             dim=128, window=0, sinks=0, ws=p, nbytes=1 << 30, k=p):
        return lib.nq_paged_attention(dtype, q, stride, k, p, pages, page_size, p, table_stride, table_pages, p, p, batch, tokens,
                                      heads, kv, dim, window, sinks, 1.0, ws, nbytes, None)

    assert attn(dtype=2) == _lib.NQ_ERR_DTYPE
    assert attn(batch=0) == attn(tokens=0) == 0
    assert attn(batch=-1) == attn(pages=0) == attn(window=-1) == attn(sinks=-1) == attn(heads=0) == _lib.NQ_ERR_INVALID_ARGUMENT
    assert attn(q=None) == attn(k=None) == _lib.NQ_ERR_INVALID_ARGUMENT
    assert attn(heads=3) == attn(table_stride=7) == attn(stride=504) == attn(stride=516) == _lib.NQ_ERR_SHAPE
    assert attn(dim=96, stride=4096) == attn(page_size=24) == attn(table_pages=1 << 27, table_stride=1 << 27) == \
        _lib.NQ_ERR_UNSUPPORTED
    assert attn(q=p + 8) == attn(k=p + 2) == _lib.NQ_ERR_ALIGNMENT
    assert attn(batch=1 << 20, tokens=1 << 20) == _lib.NQ_ERR_UNSUPPORTED

    def write(dtype=1, stride=512, kv_stride=256, dim=128, q=p, batch=1, heads=4):
        return lib.nq_paged_rope_write(dtype, q, stride, p, kv_stride, p, kv_stride, p, p, 1, p, p, 8, 8, p, p, 4, 16, p, batch, 1,
                                       heads, 2, dim, None)

    assert write(dtype=7) == _lib.NQ_ERR_DTYPE
    assert write(batch=0) == 0
    assert write(dim=72, stride=4096, kv_stride=4096) == _lib.NQ_ERR_UNSUPPORTED
    assert write(stride=504) == write(kv_stride=248) == write(stride=516) == _lib.NQ_ERR_SHAPE
    assert write(q=None) == _lib.NQ_ERR_INVALID_ARGUMENT
    assert write(q=p + 4) == _lib.NQ_ERR_ALIGNMENT

    def verify(dtype=2, stride=100, temperature=1.0, batch=2, drafts=3, vocab=100, ws=p, nbytes=1 << 30, logits=p):
        return lib.nq_verify_drafts(dtype, logits, stride, p, None, p, temperature, p, p, batch, drafts, vocab, ws, nbytes, None)

    assert verify(dtype=3) == _lib.NQ_ERR_DTYPE
    assert verify(batch=0) == 0
    assert verify(stride=99) == _lib.NQ_ERR_SHAPE
    assert verify(temperature=-1.0) == verify(temperature=math.nan) == verify(temperature=math.inf) == \
        verify(vocab=0) == verify(logits=None) == verify(ws=None) == _lib.NQ_ERR_INVALID_ARGUMENT
    assert verify(batch=1 << 30, drafts=1 << 20) == verify(vocab=1 << 32, stride=1 << 32) == _lib.NQ_ERR_UNSUPPORTED
    assert verify(logits=p + 2) == verify(ws=p + 8) == _lib.NQ_ERR_ALIGNMENT
    assert verify(nbytes=lib.nq_verify_drafts_workspace_bytes(2, 3, 100) - 1) == _lib.NQ_ERR_WORKSPACE


def test_c_abi_limits_of_the_verification_need_no_gpu():
    """A launch has fewer than 2^32 threads, 1024 for a part of a row in float32 and 512 in the 16-bit types. Every call below
    ends before its launch, for its workspace of no bytes if not for its size."""
    lib, p = _lib.load(), 256

    def verify(dtype, batch, vocab=4):
        return lib.nq_verify_drafts(dtype, p, vocab, p, None, p, 1.0, p, p, batch, 0, vocab, p, 0, None)

    assert verify(_lib.NQ_F32, 1 << 22) == verify(_lib.NQ_F16, 1 << 23) == verify(_lib.NQ_BF16, 1 << 23) == _lib.NQ_ERR_UNSUPPORTED
    assert verify(_lib.NQ_F32, (1 << 22) - 1) == verify(_lib.NQ_F16, (1 << 23) - 1) == _lib.NQ_ERR_WORKSPACE
    three = 2 * 4096 + 1  # logits, which lie in up to three parts
    assert verify(_lib.NQ_F32, (1 << 22) // 3 + 1, three) == verify(_lib.NQ_BF16, (1 << 23) // 3 + 1, three) == _lib.NQ_ERR_UNSUPPORTED
    assert verify(_lib.NQ_F32, (1 << 22) // 3, three) == verify(_lib.NQ_BF16, (1 << 23) // 3, three) == _lib.NQ_ERR_WORKSPACE
