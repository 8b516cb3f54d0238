"""Forked sequences, attention over shared pages and scored tokens on the CPU (the torch ops), their refusals, and the C ABI's."""
import math

import pytest
import torch

import fork_oracle
import serve_oracle as oracle
from nanoquant_amd import (PagedKVCache, _lib, copy_pages, paged_attention, paged_shared_attention, serve, token_logprobs)
from nanoquant_amd.decode import LlamaShape, random_llama

TINY = LlamaShape(hidden=128, layers=2, heads=4, kv_heads=2, ffn=320, vocab=500)


def test_shared_attention_is_attention():
    case = fork_oracle.shared_case(4, 2, 32, 8, [(3, [1, 9, 4]), (1, [2, 30])], [5, 17], 3, torch.float32, "cpu")
    q, k, v, table, pos, members, shared = case
    ref, _ = oracle.attention(q, k, v, table, pos, 9, 2)
    y = paged_shared_attention(*case, window=9, sinks=2)
    assert (y.double() - ref).abs().max() < 1e-5
    assert torch.equal(y, paged_attention(q, k, v, table, pos, 9, 2))


def test_copy_pages():
    pools = [torch.randn(7, 2, 3, 5) for _ in range(3)]
    want = [p.clone() for p in pools]
    source, target = torch.tensor([0, 5, -1, 2, 9, 3], dtype=torch.int32), torch.tensor([4, 1, 6, 7, 0, -2], dtype=torch.int32)
    for p in want:
        p[4], p[1] = p[0], p[5]
    copy_pages(pools, source, target)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    copy_pages(pools, source[:0], target[:0])
    copy_pages([], source, target)
    copy_pages((p for p in pools), source, target)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def _cache(batch=6, pages=12, page=4, max_len=30, **kw):
    cache = PagedKVCache(TINY, batch, pages, page, max_len, "cpu", torch.float32, **kw)
    for pool in (*cache.k, *cache.v):
        pool.normal_()
    return cache


def _contents(cache, b, length):
    """What the sequence's positions hold, by the device's table."""
    j = torch.arange(length)
    page = cache.table[b].long()[j // cache.page_size]
    assert (page >= 0).all()
    return [pool[page, :, j % cache.page_size].clone() for pool in (*cache.k, *cache.v)]


def _sound(cache):
    """Every page is free, or counted as often as rows of the table have it; the table is what the host has."""
    assert cache.table.tolist() == cache._host
    held = [0] * cache.pages
    for row in cache._host:
        for page in row:
            if page >= 0:
                held[page] += 1
    assert held == cache._owners
    assert sorted(cache._free) == [p for p in range(cache.pages) if held[p] == 0]
    if cache.members is None:
        return
    for i in range(cache.members.shape[0]):
        sequences = [b for b in cache.members[i].tolist() if b >= 0]
        n = int(cache.shared[i])
        assert (len(sequences) > 1 and n > 0) if i < cache.groups else (not sequences and n == 0)
        assert len({tuple(cache._host[b][:n]) for b in sequences}) <= 1


def test_forks_share_whole_pages_and_copy_the_last():
    cache = _cache()
    cache.reserve(0, 10)
    want = _contents(cache, 0, 10)
    cache.fork(0, [2, 5], 10)
    _sound(cache)
    assert cache._host[2][:2] == cache._host[0][:2] == cache._host[5][:2] and len({cache._host[b][2] for b in (0, 2, 5)}) == 3
    assert cache.groups == 1 and sorted(b for b in cache.members[0].tolist() if b >= 0) == [0, 2, 5] and int(cache.shared[0]) == 2
    assert cache.saved == 2 * 2 * 4 * (2 * 2 * 32 * 4)  # twice two pages of four positions' keys and values
    cache.window, cache.sinks = 4, 1
    cache._regroup()
    assert cache.saved == 2 * 5 * (2 * 2 * 32 * 4)
    assert len(cache._free) == 12 - 5
    for b in (0, 2, 5):
        assert all(torch.equal(x, y) for x, y in zip(_contents(cache, b, 10), want))
    cache.reserve(2, 20)
    cache.fork(2, [1], 17)  # a fork of a fork
    _sound(cache)
    assert cache.release(0) == 3 and len(cache._free) == 12 - 5 - 2 - 1 + 1
    _sound(cache)
    assert all(torch.equal(x, y) for x, y in zip(_contents(cache, 5, 10), want))
    for b in (1, 2, 5):
        cache.release(b)
        _sound(cache)
    assert cache.groups == 0 and len(cache._free) == 12


def test_forks_at_the_end_of_a_page_and_of_nothing():
    cache = _cache()
    cache.reserve(0, 8)
    cache.fork(0, [1], 8)   # no page to copy
    assert cache._host[1] == cache._host[0]
    cache.fork(0, [2], 0)   # nothing in common
    assert cache._host[2] == [-1] * cache.max_pages
    cache.fork(0, [3], 6)
    cache.fork(0, [], 8)
    _sound(cache)
    assert cache._host[3][0] == cache._host[0][0] and cache._host[3][1] not in cache._host[0]
    assert int(cache.shared[0]) == 1  # what all three begin with
    cache.fork(2, [4], 20)  # of a sequence without pages
    _sound(cache)


def test_pages_of_its_own_before_a_sequence_writes():
    cache = _cache()
    cache.reserve(0, 12)
    cache.fork(0, [1, 2], 12)
    want = _contents(cache, 0, 12)
    assert cache.own(1, 11, 5) == 2
    _sound(cache)
    assert cache._host[1][0] == cache._host[0][0] and not set(cache._host[1][1:3]) & set(cache._host[0])
    assert cache.own(1, 11, 5) == 0
    assert int(cache.shared[0]) == 1
    for pool in (*cache.k, *cache.v):
        pool[cache._host[1][1]] = 7.0
    for b in (0, 2):
        assert all(torch.equal(x, y) for x, y in zip(_contents(cache, b, 12), want))
    cache.release(0), cache.release(1)
    assert cache.own(2, 12, 0) == 0  # nobody else has them any more
    _sound(cache)


def test_compaction_keeps_what_sequences_hold():
    cache = _cache(pages=15)
    for b, n in enumerate((9, 20, 5)):
        cache.reserve(b, n)
    cache.fork(1, [3, 4], 18)
    cache.release(0)
    held = {b: _contents(cache, b, n) for b, n in ((1, 20), (2, 5), (3, 18), (4, 18))}
    used = cache.compact()
    _sound(cache)
    assert used == 15 - len(cache._free) == 9 and max(map(max, cache._host)) == used - 1
    for b, want in held.items():
        assert all(torch.equal(x, y) for x, y in zip(_contents(cache, b, want[0].shape[0]), want))
    assert cache.compact() == used
    cache.reserve(0, 24)
    _sound(cache)
    assert _cache().compact() == 0


def test_groups_under_a_window():
    """Sequences that have dropped pages of the prompt: grouped by what their rows still begin with."""
    cache = _cache(window=6, sinks=2, pages=20)
    cache.reserve(0, 20)
    cache.fork(0, [1, 2], 20)
    cache.reserve(1, 28)
    cache.trim(1, 27)
    _sound(cache)
    assert int(cache.shared[0]) == 1  # the sinks' page
    cache.trim(0, 27), cache.trim(2, 27)
    _sound(cache)
    assert cache.groups == 1 and int(cache.shared[0]) == 1


def _groups_hold(cache):
    """The groups are those that the rows make when asked anew, and what a member has, those before it in its group have too."""
    state = [cache.members.tolist(), cache.shared.tolist(), cache.groups, cache.saved]
    cache._regroup()
    assert state == [cache.members.tolist(), cache.shared.tolist(), cache.groups, cache.saved]
    for sequences, n in zip(cache.members.tolist(), cache.shared.tolist()):
        rows = [cache._host[b][:n] for b in sequences if b >= 0]
        for row, later in zip(rows, rows[1:]):
            assert all(page == other or other == -1 for page, other in zip(row, later))


@pytest.mark.parametrize("sinks", [0, 2])
def test_members_that_trim_one_after_the_other_stay_a_group(sinks):
    """At one position, partly into the prompt: the rows are alike again when the last has trimmed."""
    cache = _cache(window=20, sinks=sinks, pages=60, max_len=80)
    cache.reserve(0, 32)
    cache.fork(0, [1, 2, 3], 32)
    for b in range(4):
        cache.reserve(b, 37, 32)
    for b in (0, 2, 1, 3):
        assert cache.trim(b, 36) == 4 - bool(sinks)
        _groups_hold(cache)
        assert cache.groups == 1 and int(cache.shared[0]) == 8 and set(cache.members[0].tolist()) == {0, 1, 2, 3}
    _sound(cache)
    assert cache.members.tolist()[0] == [0, 1, 2, 3]
    assert cache.saved == 3 * (4 + bool(sinks)) * 4 * (2 * 2 * 32 * 4)  # of eight pages, those that are left


def test_pages_that_windows_are_past_save_nothing():
    """Each member's own pages count, and those of the one that has the most are read anyway."""
    position = 2 * 2 * 32 * 4
    cache = _cache(window=40, sinks=4, pages=60, max_len=80)
    cache.reserve(0, 32)
    cache.fork(0, [1, 2], 32)
    assert cache.saved == 2 * 32 * position
    for b, at, left in ((0, 47, 28 + 32), (1, 51, 28 + 24), (2, 59, 24 + 16), (0, 70, 16 + 8)):
        cache.reserve(b, at + 1, 32)
        cache.trim(b, at)  # sees positions at - 39 on, and the first page's
        assert cache.saved == left * position
        _groups_hold(cache)
    for b in (0, 1, 2):
        cache.reserve(b, 80, 72)
        cache.trim(b, 79)
        _groups_hold(cache)
    assert cache.groups == 1 and cache.saved == 2 * 4 * position  # the sinks' page


@pytest.mark.parametrize("sinks", [0, 2])
def test_members_that_trim_at_positions_of_their_own_stay_a_group(sinks):
    """Answers at different lengths have the prompt's last pages in common, and differ in what is behind their windows."""
    cache = _cache(window=30, sinks=sinks, pages=90, max_len=120)
    cache.reserve(0, 64)
    cache.fork(0, [1, 2, 3], 64)
    at = [74, 66, 78, 70]
    for b in range(4):
        cache.reserve(b, at[b], 64)
        cache.trim(b, at[b])
        _groups_hold(cache)
    assert cache.groups == 1 and int(cache.shared[0]) == 16
    assert cache.members.tolist()[0] == [1, 3, 0, 2]  # the one that has the most comes first
    cache.trim(1, 86)  # further than the others
    _groups_hold(cache)
    assert cache.members.tolist()[0] == [3, 0, 2, 1] and int(cache.shared[0]) == 16
    cache.reserve(4, 9)
    cache.release(3)
    _groups_hold(cache)
    assert cache.members.tolist()[0] == [0, 2, 1, -1]
    cache.fork(2, [5], 78)  # the fork of one that has trimmed lacks the same pages
    _groups_hold(cache)
    assert cache.members.tolist()[0] == [0, 2, 5, 1]
    cache.compact()
    _groups_hold(cache)
    cache.reserve(0, 78, 0)  # pages of its own where it had trimmed: its row begins otherwise now
    _groups_hold(cache)
    assert int(cache.shared[0]) == (1 if sinks else 16) and (0 in cache.members.tolist()[0]) == (sinks > 0)
    for b in range(6):
        cache.release(b)
        _groups_hold(cache)
    assert cache.groups == 0 and len(cache._free) == 90


WIDE = LlamaShape(hidden=1024, layers=1, heads=8, kv_heads=8, ffn=64, vocab=64)  # 8 KB a position


def _groups(cache):
    return [([b for b in x if b >= 0], n) for x, n in zip(cache.members.tolist(), cache.shared.tolist()) if n]


def test_a_short_fork_leaves_the_others_their_pages():
    """Seven answers to a prompt of a thousand tokens, and one that branches off after twenty."""
    cache = PagedKVCache(WIDE, 12, 120, 16, 1040, "cpu", torch.float32)
    cache.reserve(0, 1000)
    cache.fork(0, range(1, 8), 1000)
    saved = 7 * 62 * 16 * 8192
    assert _groups(cache) == [([*range(8)], 62)] and cache.saved == saved
    cache.fork(0, [8], 20)
    assert _groups(cache) == [([*range(8)], 62)] and cache.saved == saved
    cache.fork(3, [9, 10], 20)  # the short ones have a page in common with each other
    assert _groups(cache) == [([*range(8)], 62), ([8, 9, 10], 1)] and cache.saved == saved + 2 * 16 * 8192
    for b in range(1, 8):
        cache.release(b)
    assert _groups(cache) == [([0, 8, 9, 10], 1)]
    _sound(cache)


def test_groups_of_a_tree_of_forks():
    """Second prompts behind a first one: groups of their own where they are long, one group where they are short."""
    for second, want in ((30, [([0, 2, 4, 6], 70), ([1, 3, 5, 7], 70)]), (2, [([*range(8)], 40)])):
        cache = PagedKVCache(WIDE, 8, 160, 16, 1280, "cpu", torch.float32)
        cache.reserve(0, 40 * 16)
        cache.fork(0, [1], 40 * 16)
        for b in (0, 1):
            cache.reserve(b, (40 + second) * 16)
            cache.fork(b, [b + 2, b + 4, b + 6], (40 + second) * 16)
        assert _groups(cache) == want
        _sound(cache)
    # each fork a little earlier than the one before: together while that saves more
    cache = PagedKVCache(WIDE, 11, 100, 16, 1280, "cpu", torch.float32)
    cache.reserve(0, 64 * 16)
    for b, n in enumerate((60, 58, 56, 54, 52, 50, 9, 8, 1), 1):
        cache.fork(0, [b], n * 16)
    assert _groups(cache) == [([*range(7)], 50), ([7, 8], 8)]
    _sound(cache)


def test_a_member_past_the_prompt_leaves_the_others_their_pages():
    for sinks in (0, 16):
        cache = PagedKVCache(WIDE, 5, 240, 16, 1600, "cpu", torch.float32, window=600, sinks=sinks)
        cache.reserve(0, 800)
        cache.fork(0, [1, 2, 3], 800)
        cache.reserve(2, 1500, 800)
        cache.trim(2, 1499)
        assert _groups(cache) == [([0, 1, 3], 50)] and cache.saved == 2 * (600 + sinks) * 8192
        _groups_hold(cache)
        for b in (0, 3, 1):
            cache.reserve(b, 1500, 800)
            cache.trim(b, 1499)
            _groups_hold(cache)
        assert _groups(cache) == ([([0, 1, 2, 3], 1)] if sinks else [])


@pytest.mark.parametrize("answers,prompt,heads,dim,faster", [
    (100, 250, 8, 128, False), (2, 16000, 8, 128, False), (40, 1000, 8, 64, False), (16, 4000, 8, 128, True), (16, 4000, 8, 64, True),
    (8, 1000, 32, 128, True)])
def test_a_layer_reads_groups_where_that_was_measured_to_be_faster(answers, prompt, heads, dim, faster, monkeypatch):
    shape = LlamaShape(hidden=heads * dim, layers=1, heads=heads, kv_heads=heads, ffn=64, vocab=64)
    cache = PagedKVCache(shape, answers, prompt // 16 + answers + 1, 16, prompt + 32, "cpu", torch.bfloat16)
    cache.reserve(0, prompt // 16 * 16)
    cache.fork(0, range(1, answers), prompt // 16 * 16)
    for b in range(answers):
        cache.reserve(b, prompt // 16 * 16 + 1)
    took = []
    monkeypatch.setattr(serve, "paged_shared_attention", lambda *x: took.append(True))
    monkeypatch.setattr(serve, "paged_attention", lambda *x: took.append(False))
    x = torch.zeros(answers, 1, heads * dim, dtype=torch.bfloat16)
    angles = torch.zeros(answers, 1, dim)
    serve.paged_rotary_attention(shape, 0, x, x, x, angles, angles, torch.full((answers, 1), prompt // 16 * 16), cache)
    assert took == [faster]


def test_forks_and_trims_at_random():
    import random
    rng = random.Random(9)
    cache = _cache(batch=7, pages=70, max_len=64, window=18, sinks=3)
    length = [0] * 7
    grouped = 0
    for step in range(400):
        b = rng.randrange(7)
        try:
            what = rng.choice(["reserve", "reserve", "trim", "trim", "trim", "fork", "release", "own", "compact"])
            if what == "reserve" and length[b] < 64:
                n = rng.randint(length[b], min(64, length[b] + 20))
                cache.reserve(b, n, rng.choice([length[b], length[b], 0]))
                length[b] = n
            elif what == "trim" and length[b]:
                cache.trim(b, rng.randint(length[b] // 2, length[b]))
            elif what == "fork":
                targets = [c for c in range(7) if c != b and cache._host[c] == [-1] * cache.max_pages][:rng.randint(1, 3)]
                n = rng.randint(length[b] // 2, length[b])
                cache.fork(b, targets, n)
                for c in targets:
                    length[c] = n
            elif what == "release" and rng.random() < 0.5:
                cache.release(b)
                length[b] = 0
            elif what == "own":
                cache.own(b, length[b], rng.randint(length[b] // 2, length[b]))
            elif what == "compact":
                cache.compact()
        except RuntimeError:
            assert len(cache._free) < 18
        held = [0] * cache.pages
        for row in cache._host:
            for page in row:
                if page >= 0:
                    held[page] += 1
        assert held == cache._owners and cache.table.tolist() == cache._host
        if cache.members is not None:
            grouped += cache.groups > 0
            if rng.random() < 0.3:
                _groups_hold(cache)
    assert grouped > 200


def test_many_forks_at_random():
    import random
    rng = random.Random(4)
    cache = _cache(batch=7, pages=30, max_len=32)
    length, text = [0] * 7, [None] * 7
    for step in range(300):
        b = rng.randrange(7)
        try:
            what = rng.choice(["reserve", "fork", "release", "own", "compact"])
            if what == "reserve":
                n = rng.randint(length[b], 32)
                cache.reserve(b, n)
                length[b] = n
            elif what == "fork":
                targets = [c for c in range(7) if c != b and cache._host[c] == [-1] * cache.max_pages][:rng.randint(1, 3)]
                cache.fork(b, targets, rng.randint(0, length[b]))
                for c in targets:
                    length[c] = sum(page >= 0 for page in cache._host[c]) * 4
            elif what == "release":
                cache.release(b)
                length[b] = 0
            elif what == "own":
                start = rng.randint(0, length[b])
                cache.own(b, length[b], start)
                assert all(cache._owners[p] == 1 for p in cache._host[b][start // 4:-(-length[b] // 4)] if p >= 0)
            else:
                text = [_contents(cache, c, length[c]) for c in range(7)]
                cache.compact()
                for c in range(7):
                    assert all(torch.equal(x, y) for x, y in zip(_contents(cache, c, length[c]), text[c]))
        except RuntimeError:
            assert len(cache._free) < 9
        _sound(cache)


def _score_case(shape, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(*shape, V, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, V, shape, generator=g)
    tokens.view(-1)[1::4] = torch.tensor([-1, V, 1 << 40]).repeat(tokens.numel())[:tokens.view(-1)[1::4].numel()]
    return logits, tokens


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("shape,V,top,temperature", [((5,), 33, 4, 1.0), ((2, 3), 500, 7, 0.7), ((4,), 1, 1, 1.0), ((3, 1), 9, 9, 2.5),
                                                     ((6,), 200, 0, 1.0)])
def test_score_against_the_definition(shape, V, top, temperature, dtype):
    logits, tokens = _score_case(shape, V, dtype)
    got = token_logprobs(logits, tokens, top, temperature)
    assert got[0].dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
    fork_oracle.check_score(got, fork_oracle.score(logits, tokens, top, temperature))


def odd_rows(V, dtype):
    """Rows with masks, equal logits, infinities and NaN, and a token for each."""
    x = torch.randn(12, V, generator=torch.Generator().manual_seed(5)).to(dtype)
    x[0, 1:] = -math.inf                  # one token left: log p 0, no entropy
    x[1, ::2] = -math.inf
    x[2] = 1.5                            # all alike
    x[3] = -math.inf
    x[4, V // 2] = math.nan
    x[5, 3], x[5, V - 1] = math.inf, math.nan
    x[6, 4] = math.inf
    x[7, V // 3:] = torch.finfo(dtype).min
    x[8, V - 2:] = 60.0                   # two far above the others
    x[9, :] = 0.0
    x[9, 1::2] = -0.0
    x[10, 2], x[10, 5] = math.nan, -math.nan
    x[11, :] = -20000.0
    return x, torch.tensor([0, 0, V - 1, 1, 0, 3, 4, V - 1, V - 1, 2, 0, 7])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_score_of_odd_rows(dtype):
    logits, tokens = odd_rows(41, dtype)
    for top in (0, 3, 41):
        fork_oracle.check_score(token_logprobs(logits, tokens, top), fork_oracle.score(logits, tokens, top, 1.0))


@pytest.mark.parametrize("temperature", [5e-324, 1e-300, 1e-30, 1e30, 1e300])
def test_score_at_extreme_temperatures(temperature):
    logits, tokens = _score_case((6,), 50, torch.float32)
    logits[0, 3:9] = -math.inf
    fork_oracle.check_score(token_logprobs(logits, tokens, 3, temperature), fork_oracle.score(logits, tokens, 3, temperature))


def test_gradients_of_scores():
    """log p's and the entropy's, against the formulas: (1[j = token] - p_j) / T, and -p_j (log p_j + H) / T."""
    logits, tokens = _score_case((5,), 30, torch.float32)
    logits[1, 4:9] = -math.inf
    w, z = torch.randn(2, 5, generator=torch.Generator().manual_seed(1))
    T = 0.8
    x = logits.clone().requires_grad_(True)
    given, entropy, _, best = token_logprobs(x, tokens, 2, T)
    (given * w + entropy * z).sum().backward()
    d = logits.double()
    logp = torch.log_softmax(d / T, -1)
    p = logp.exp()
    there = (tokens >= 0) & (tokens < 30)
    one = torch.nn.functional.one_hot(torch.where(there, tokens, 0), 30).double()
    H = -(p * torch.where(p > 0, logp, 0.0)).sum(-1, keepdim=True)
    want = torch.where(there, w, 0.0).double().unsqueeze(1) * (one - p) / T
    want -= z.double().unsqueeze(1) * p * (torch.where(p > 0, logp, 0.0) + H) / T
    # every factor is a float32 result off by a few of its roundings, of sums over 30 terms: 2^-24 * 64 of terms up to 10
    assert (x.grad.double() - want).abs().max() < 64 * 2.0 ** -24 * 10
    assert torch.autograd.gradcheck(lambda y: token_logprobs(y, tokens[2:], 0, T)[:2], (logits[2:].double().requires_grad_(True),))


def test_a_model_answers_a_prompt_several_times():
    """Forked, then decoded together: every answer is what a sequence of its own says, and its score what its logits say."""
    torch.manual_seed(0)
    model = random_llama(TINY, bpw=2.0, device="cpu", dtype=torch.float32).eval()
    answers, P, page = 3, 11, 4
    prompt = torch.randint(0, TINY.vocab, (P,))
    texts = torch.randint(0, TINY.vocab, (answers, 6))
    with torch.no_grad():
        alone = PagedKVCache(TINY, answers, 40, page, 40, "cpu", torch.float32)
        forked = PagedKVCache(TINY, answers, 40, page, 40, "cpu", torch.float32)
        for b in range(answers):
            alone.reserve(b, P + 6)
        model(prompt.expand(answers, -1), torch.arange(P).expand(answers, -1), alone)
        forked.reserve(0, P)
        ids, pos = torch.zeros(answers, P, dtype=torch.int64), torch.full((answers, P), -1)
        ids[0], pos[0] = prompt, torch.arange(P)
        model(ids, pos, forked)
        forked.fork(0, [1, 2], P)
        for b in range(answers):
            forked.reserve(b, P + 6, P)
        assert forked.groups == 1 and int(forked.shared[0]) == 2
        for t in range(6):
            at = torch.full((answers, 1), P + t)
            want, got = model(texts[:, t:t + 1], at, alone), model(texts[:, t:t + 1], at, forked)
            assert torch.allclose(got, want, rtol=0, atol=1e-4)
            chosen = texts[:, t + 1:t + 2] if t < 5 else texts[:, :1]
            a, b = token_logprobs(want, chosen, 3), token_logprobs(got, chosen, 3)
            assert torch.allclose(a[0], b[0], rtol=0, atol=1e-3) and a[3].shape == (answers, 1, 3)
        forked.compact()


def test_refusals():
    case = fork_oracle.shared_case(4, 2, 32, 8, [(3, [1, 9])], [5], 1, torch.float32, "cpu")
    q, k, v, table, pos, members, shared = case
    with pytest.raises(ValueError, match="members"):
        paged_shared_attention(*case[:5], members[0], shared)
    with pytest.raises(ValueError, match="members"):
        paged_shared_attention(*case[:5], members, torch.cat((shared, shared)))
    with pytest.raises(TypeError, match="int32"):
        paged_shared_attention(*case[:5], members.long(), shared)
    with pytest.raises(TypeError, match="int32"):
        paged_shared_attention(*case[:5], members, shared.long())
    with pytest.raises(ValueError, match="window"):
        paged_shared_attention(*case, window=-1)
    with pytest.raises(ValueError, match="does not fit"):
        paged_shared_attention(q[..., :24], *case[1:])
    pools = [torch.zeros(4, 2, 3), torch.zeros(4, 2, 3)]
    one = torch.tensor([1], dtype=torch.int32)
    with pytest.raises(ValueError, match="alike"):
        copy_pages([pools[0], torch.zeros(4, 3, 2)], one, one)
    with pytest.raises(ValueError, match="alike"):
        copy_pages([pools[0], pools[1].half()], one, one)
    with pytest.raises(ValueError, match="moves"):
        copy_pages(pools, one, torch.cat((one, one)))
    with pytest.raises(TypeError, match="int32"):
        copy_pages(pools, one.long(), one)
    cache = _cache(pages=4)
    cache.reserve(0, 10)
    with pytest.raises(RuntimeError, match="pages left"):
        cache.fork(0, [1, 2], 10)
    _sound(cache)
    for targets in ([0], [1, 1]):
        with pytest.raises(ValueError, match="without pages"):
            cache.fork(0, targets, 8)
    cache.fork(0, [1], 8)
    with pytest.raises(ValueError, match="without pages"):
        cache.fork(0, [1], 8)
    with pytest.raises(IndexError):
        cache.fork(0, [6], 8)
    with pytest.raises(ValueError, match="max_len"):
        cache.fork(0, [2], 31)
    with pytest.raises(ValueError, match="max_len"):
        cache.own(0, 4, 5)
    with pytest.raises(RuntimeError, match="pages left"):
        cache.own(1, 8, 0)
    _sound(cache)
    logits, tokens = _score_case((5,), 30, torch.float32)
    with pytest.raises(ValueError, match="vocab"):
        token_logprobs(logits, tokens[:4])
    with pytest.raises(ValueError, match="vocab"):
        token_logprobs(logits[0], tokens[0])
    with pytest.raises(TypeError, match="int64"):
        token_logprobs(logits, tokens.int())
    with pytest.raises(TypeError, match="float32"):
        token_logprobs(logits.int(), tokens)
    for top in (-1, 31):
        with pytest.raises(ValueError, match="alternatives"):
            token_logprobs(logits, tokens, top)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            token_logprobs(logits, tokens, temperature=bad)
    assert [tuple(x.shape) for x in token_logprobs(logits[:0], tokens[:0], 2)] == [(0,), (0,), (0, 2), (0, 2)]


def test_groups_that_outgrow_their_tensors_leave_nobody_in_the_old_ones():
    """A graph captured before reads the old tensors on."""
    cache = _cache()
    cache.reserve(0, 9)
    cache.fork(0, [1], 9)
    members, shared = cache.members, cache.shared
    assert members.tolist() == [[0, 1]] and shared.tolist() == [2]
    cache.release(1)
    cache.fork(0, [3], 9)
    assert cache.members is members and members.tolist() == [[0, 3]]
    cache.fork(0, [4, 5], 9)
    assert cache.members is not members and cache.members.tolist() == [[0, 3, 4, 5]]
    assert members.tolist() == [[-1, -1]] and shared.tolist() == [0]
    assert any(a is members and b is shared for a, b in cache._outgrown)  # their memory is nobody else's


def test_groups_made_in_inference_mode_change_outside_it():
    cache = _cache()
    with torch.inference_mode():
        cache.reserve(0, 9)
        cache.fork(0, [1], 9)
    cache.fork(0, [2, 3], 9)
    assert cache.members.tolist() == [[0, 1, 2, 3]]
    cache.release(1)
    with torch.inference_mode():
        cache.release(2)
    assert cache.members.tolist() == [[0, 3, -1, -1]]
    _sound(cache)


def test_c_abi_limits_of_shared_pages_need_no_gpu():
    """What a launch lists: row groups of groups and of sequences, and a wave for each row of the output in 32-bit threads; and
    what is left to the plain attention."""
    lib, p = _lib.load(), 256

    def nbytes(batch, tokens=1, heads=8, kv=2, groups=1, most=9, keys=1 << 24, page=16):
        return lib.nq_paged_shared_attention_workspace_bytes(batch, tokens, heads, kv, 128, keys // page, page, groups, most)

    assert nbytes(1023) > 0 and nbytes(1024) == 0                      # 36 rows a group: one entry, and one a sequence
    assert nbytes(1015, most=32 * 9) > 0 and nbytes(1016, most=32 * 9) == 0  # 1152 rows, nine entries
    assert nbytes(511, most=8) > 0 and nbytes(512, most=8) == 0        # up to 32 rows
    assert nbytes(500, tokens=16) > 0 and nbytes(512, tokens=16) == 0  # 64 rows a sequence, two entries
    assert nbytes(100, tokens=17) == 0                                 # 68
    assert nbytes(500, heads=65536, kv=65536, most=64) > 0 and nbytes(600, heads=65536, kv=65536, most=64) == 0
    assert nbytes(0) == nbytes(4, groups=0) == nbytes(4, most=0) == nbytes(4, heads=7) == nbytes(4, most=1 << 31) == 0
    assert nbytes(4, keys=1 << 31) == nbytes(4, page=0x7FFFFFFF) == nbytes(4, keys=0) == 0
    assert nbytes(1000, keys=1 << 25) > 0 and nbytes(1000, keys=1 << 27) == 0  # 2^31 tiles of 32
    # 2^27 bytes of the tables' keys and values, 2^26 with few rows a group: 8 sequences of 2 kv heads of 128, 8 KB a position
    assert nbytes(8, keys=1 << 14) > 0 and nbytes(8, keys=(1 << 14) - 16) == 0
    assert nbytes(8, keys=1 << 13, most=8) > 0 and nbytes(8, keys=(1 << 13) - 16, most=8) == 0
    assert lib.nq_paged_shared_attention(0, p, 1024, p, p, 4, 16, p, 1 << 20, 1 << 20, p, p, p, 1, 9, p, 1024, 1, 8, 2, 128, 0, 0, 1.0, p,
                                         1 << 40, None) == _lib.NQ_ERR_UNSUPPORTED
    assert lib.nq_paged_shared_attention(0, p, 1024, p, p, 4, 16, p, 1 << 20, 1 << 20, p, p, p, 1, 9, p, 10, 1, 8, 2, 128, 0, 0, 1.0, p,
                                         nbytes(10) - 1, None) == _lib.NQ_ERR_WORKSPACE
    assert lib.nq_token_logprobs_workspace_bytes(1, 1, 1000, 5) == 0 < lib.nq_token_logprobs_workspace_bytes(1, 64, 100003, 5)
    assert lib.nq_token_logprobs(2, p, 0, 100003, p, 0, 1, 1.0, 3, p, p, p, p, 1, 64, 100003, p, 100, None) == _lib.NQ_ERR_WORKSPACE


def test_c_abi_argument_errors_need_no_gpu():
    import ctypes
    lib = _lib.load()
    p = 256  # a pointer that is never followed: every call below ends before its launch

    def attn(dtype=0, q=p, stride=128 * 4, pages=4, page_size=16, table_stride=8, table_pages=8, members=p, groups=2, most=3, batch=1,
             tokens=1, heads=4, kv=2, dim=128, window=0, sinks=0, ws=p, nbytes=1 << 40, k=p):
        return lib.nq_paged_shared_attention(dtype, q, stride, k, p, pages, page_size, p, table_stride, table_pages, p, members, p,
                                             groups, most, p, batch, tokens, heads, kv, dim, window, sinks, 1.0, ws, nbytes, None)

    assert attn(dtype=2) == _lib.NQ_ERR_DTYPE
    assert attn(batch=0) == attn(tokens=0) == 0
    assert attn(batch=-1) == attn(pages=0) == attn(window=-1) == attn(sinks=-1) == attn(groups=-1) == attn(most=-1) == \
        attn(q=None) == attn(k=None) == attn(members=None) == _lib.NQ_ERR_INVALID_ARGUMENT
    assert attn(heads=3) == attn(table_stride=7) == attn(stride=504) == attn(stride=516) == _lib.NQ_ERR_SHAPE
    assert attn(dim=96, stride=4096) == attn(page_size=24) == attn(batch=1 << 20, tokens=1 << 20) == _lib.NQ_ERR_UNSUPPORTED
    assert attn(q=p + 8) == attn(k=p + 2) == attn(members=p + 2) == attn(ws=p + 8) == _lib.NQ_ERR_ALIGNMENT

    def copy(pools=(p, p), pages=4, nbytes=64, source=p, moves=2):
        at = (ctypes.c_void_p * 2)(*pools)
        return lib.nq_copy_pages(at, 2, pages, nbytes, source, p, moves, None)

    assert copy(moves=0) == 0
    assert copy(moves=-1) == copy(pages=0) == copy(nbytes=0) == copy(source=None) == copy(pools=(p, None)) == \
        _lib.NQ_ERR_INVALID_ARGUMENT
    assert copy(source=p + 2) == _lib.NQ_ERR_ALIGNMENT
    assert copy(pages=1 << 31) == copy(nbytes=(1 << 33) + 1) == _lib.NQ_ERR_UNSUPPORTED

    def score(dtype=2, row=100, batch_stride=300, temperature=1.0, top=3, batch=2, rows=3, vocab=100, ws=p, nbytes=1 << 40, logits=p,
              best=p):
        return lib.nq_token_logprobs(dtype, logits, batch_stride, row, p, 3, 1, temperature, top, p, p, best, p, batch, rows, vocab,
                                     ws, nbytes, None)

    assert score(dtype=3) == _lib.NQ_ERR_DTYPE
    assert score(batch=0) == score(rows=0) == 0
    assert score(row=99) == score(batch_stride=99) == _lib.NQ_ERR_SHAPE
    assert score(temperature=0.0) == score(temperature=math.nan) == score(temperature=math.inf) == score(vocab=0) == \
        score(top=-1) == score(top=101) == score(logits=None) == score(best=None) == _lib.NQ_ERR_INVALID_ARGUMENT
    assert score(batch=1 << 20, rows=1 << 20) == score(vocab=1 << 31, row=1 << 31, batch_stride=1 << 33) == score(top=65) == \
        score(temperature=2.0 ** -65) == score(temperature=2.0 ** 65) == _lib.NQ_ERR_UNSUPPORTED
    assert score(logits=p + 2) == score(best=p + 4) == _lib.NQ_ERR_ALIGNMENT
