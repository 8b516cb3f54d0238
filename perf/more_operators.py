"""Performance cases of what a server of several answers to one prompt has the framework do next to the paged cache's writes
and attention.

The kinds of cases, and the entry point each one times:

* ``copy``    ``copy_pages``: pages of a cache copied within every layer's pools, for a fork or a compaction;
* ``shared``  ``paged_shared_attention``: attention over pages of which groups of sequences have the leading ones in common;
* ``score``   ``token_logprobs``: given tokens' log probabilities, the entropy, the largest alternatives.

Sequences have lengths of their own, and their pages lie anywhere in the pool; a group's members are spread over the batch.
Queries are N(0, 1.5), keys and values N(0, 1) as after a norm; logits are N(0, 2.5) with some tokens well above, the given
tokens drawn from them, every eleventh a padding's -1.

``run`` with ``own`` false computes the operators in elementary torch operations, in float32; with ``own`` true it calls the
framework.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one answer more: the page that the prompt ends in, in all 32 layers (7B heads)
        dict(name="copy_fork_1", kind="copy", layers=32, kv_heads=32, dim=128, page=16, pages=24, moves=1, dtype="fp16"),
        # five new answers of a prompt, grouped heads
        dict(name="copy_fork_5", kind="copy", layers=32, kv_heads=8, dim=128, page=48, pages=37, moves=5, dtype="bf16"),
        # the cache moved together after many requests have ended
        dict(name="copy_compact_61", kind="copy", layers=32, kv_heads=8, dim=128, page=32, pages=150, moves=61, dtype="bf16"),
        # four answers to a prompt of a thousand tokens (7B heads)
        dict(name="shared_4_mha", kind="shared", heads=32, kv_heads=32, dim=128, page=16, groups=1, members=4, alone=0,
             prefix=1000, low=1, high=130, tokens=1, window=0, sinks=0, dtype="fp16"),
        # sixteen answers about one document (70B heads)
        dict(name="shared_16_gqa", kind="shared", heads=64, kv_heads=8, dim=128, page=32, groups=1, members=16, alone=0,
             prefix=8000, low=20, high=700, tokens=1, window=0, sinks=0, dtype="bf16"),
        # a full server: users of five system prompts, some with none, conversations of their own behind
        dict(name="shared_60_server", kind="shared", heads=64, kv_heads=8, dim=128, page=64, groups=5, members=11, alone=5,
             prefix=6000, low=100, high=4000, tokens=1, window=0, sinks=0, dtype="bf16"),
        # eleven answers, five drafted tokens each, small heads
        dict(name="shared_11x5_draft", kind="shared", heads=32, kv_heads=8, dim=64, page=48, groups=1, members=11, alone=1,
             prefix=5000, low=5, high=900, tokens=5, window=0, sinks=0, dtype="fp16"),
        # very many samples of one long prompt, a wide window with sinks (70B heads)
        dict(name="shared_128_window", kind="shared", heads=64, kv_heads=8, dim=128, page=64, groups=1, members=128, alone=0,
             prefix=14000, low=1, high=1500, tokens=1, window=12011, sinks=16, dtype="bf16"),
        # the next token of one sequence with five alternatives (7B vocabulary, float32 logits)
        dict(name="score_1_top5", kind="score", rows=1, vocab=32000, top=5, temperature=1.0, dtype="fp32"),
        # the next tokens of 64 sequences with twenty alternatives, a large odd vocabulary
        dict(name="score_64_top20", kind="score", rows=64, vocab=100003, top=20, temperature=0.8, dtype="bf16"),
        # a prompt scored token by token
        dict(name="score_777", kind="score", rows=777, vocab=32000, top=0, temperature=1.0, dtype="fp16"),
        # a batch of answers ranked under a large vocabulary, with the largest alternative
        dict(name="score_2111_top1", kind="score", rows=2111, vocab=100003, top=1, temperature=1.0, dtype="bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["copy", "shared", "shared", "shared", "shared", "score", "score"])
    c = dict(kind=kind, dtype=rng.choice(["fp16", "bf16"]))
    if kind == "score":
        c.update(vocab=_spread(rng, 1000, 128000), top=rng.choice([0, 0, 1, 2, 5, 8, 20, 32]),
                 temperature=rng.choice([0.7, 1.0, 1.0, 1.3]), dtype=rng.choice(["fp32", "fp16", "bf16"]))
        c["rows"] = _spread(rng, 1, min(2500, int((1.0e8 if c["dtype"] == "fp32" else 2.0e8) // c["vocab"])))
        return c
    heads, kv_heads = rng.choice([(32, 32), (16, 16), (64, 8), (64, 8), (32, 8), (24, 8), (20, 4), (8, 1), (5, 5)])
    c.update(kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), page=rng.choice([16, 16, 32, 48, 64, 128]))
    if kind == "copy":
        c["layers"] = _spread(rng, 2, 32)
        most = int(2.4e8 // (c["layers"] * 4 * kv_heads * c["dim"] * c["page"]))  # no costlier than the listed ones
        c["moves"] = _spread(rng, 1, max(1, min(100, most)))
        c["pages"] = 2 * c["moves"] + _spread(rng, 2, 30)
        return c
    windowed = rng.random() < 0.25
    c.update(heads=heads, window=_spread(rng, 300, 12000) if windowed else 0,
             sinks=rng.choice([0, 1, 4, 16, 100]) if windowed else 0, tokens=rng.choice([1, 1, 1, 1, 2, 5, 8]),
             groups=rng.choice([1, 1, 1, 2, 3, 7]), alone=rng.choice([0, 0, 1, 5]))
    c["members"] = _spread(rng, 2, 128 // (c["groups"] * c["tokens"]))
    c["prefix"] = _spread(rng, max(100, c["page"]), 14000)
    rows = (c["groups"] * c["members"] + c["alone"]) * kv_heads
    most = max(c["tokens"] + 1, min(4000, int(9e5 // rows)))
    c["high"] = _spread(rng, c["tokens"] + 1, most)
    c["low"] = max(1, int(c["high"] * rng.choice([0.02, 0.3, 1.0])))
    return c


# ------------------------------------------------------------------------------ inputs from a seed

def _batch(case):
    return case["groups"] * case["members"] + case["alone"]


def _plan(case):
    """What `work` has to know, so the same for every seed: (each sequence's group or -1, each sequence's length with its new
    tokens, each group's pages). Members are dealt out in turn, the groups' prompts get shorter by a ninth each, and a sequence
    that has none is as long as the longest prompt and a conversation."""
    B, low, high, S = _batch(case), case["low"], case["high"], case["page"]
    group = [(i % case["groups"]) if i < case["groups"] * case["members"] else -1 for i in range(B)]
    group = group[::-1] if case["alone"] else group
    shared = [max(1, int(case["prefix"] * (1 - g / 9)) // S) for g in range(case["groups"])]
    mine = [high] + [low + int((high - low) * ((i * 0.6180339887) % 1.0)) for i in range(1, B)]
    lengths = [(shared[g] * S if g >= 0 else case["prefix"]) + n for g, n in zip(group, mine)]
    return group, lengths, shared


def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, device=DEVICE, generator=g, dtype=dtype).mul_(scale)


def _prepare_shared(case, s, g, dt):
    B, T, S, KV, D = _batch(case), case["tokens"], case["page"], case["kv_heads"], case["dim"]
    group, lengths, shared = _plan(case)
    used = [-(-n // S) for n in lengths]
    own_pages = [u - (shared[i] if i >= 0 else 0) for u, i in zip(used, group)]
    total = sum(shared) + sum(own_pages)
    pool = total + 3
    order = torch.randperm(pool, device=DEVICE, generator=g).tolist()
    prompts = [[order.pop() for _ in range(n)] for n in shared]
    table = torch.full((B, max(used) + 1), -1, dtype=torch.int32)
    for b in range(B):
        row = (prompts[group[b]] if group[b] >= 0 else []) + [order.pop() for _ in range(own_pages[b])]
        table[b, :used[b]] = torch.tensor(row, dtype=torch.int32)
    lists = [[b for b in range(B) if group[b] == i] for i in range(case["groups"])]
    most = max(len(x) for x in lists)
    s["members"] = torch.tensor([x + [-1] * (most - len(x)) for x in lists], dtype=torch.int32).to(DEVICE)
    s["shared"] = torch.tensor(shared, dtype=torch.int32).to(DEVICE)
    s["table"] = table.to(DEVICE)
    positions = [[n - min(T, n) + i if i < min(T, n) else -1 for i in range(T)] for n in lengths]
    s["positions"] = torch.tensor(positions, dtype=torch.int64).to(DEVICE)
    s["k_pages"] = _normal(g, (pool, KV, S, D), dt)
    s["v_pages"] = _normal(g, (pool, KV, S, D), dt)
    s["q"] = _normal(g, (B, T, case["heads"] * D), dt, 1.5)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["kind"] == "score":
        R, V = case["rows"], case["vocab"]
        logits = torch.randn(R, V, device=DEVICE, generator=g) * 2.5
        tall = torch.randint(0, V, (R, 7), device=DEVICE, generator=g)
        logits.scatter_add_(1, tall, 6.0 + 3.0 * torch.randn(R, 7, device=DEVICE, generator=g))
        tokens = torch.multinomial(torch.softmax(logits, -1), 1, generator=g)[:, 0]
        if R > 1:
            tokens[10::11] = -1
        s["logits"], s["tokens"] = logits.to(dt), tokens
    elif case["kind"] == "copy":
        shape = (case["pages"], case["kv_heads"], case["page"], case["dim"])
        s["pools"] = [_normal(g, shape, dt) for _ in range(2 * case["layers"])]
        order = torch.randperm(case["pages"], device=DEVICE, generator=g).to(torch.int32)
        s["source"], s["target"] = order[:case["moves"]].clone(), order[case["moves"]:2 * case["moves"]].clone()
    else:
        _prepare_shared(case, s, g, dt)
    return s


# -------------------------------------------------------------------------------------------- a pass

def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    with torch.no_grad():
        if own:
            from nanoquant_amd.serve import copy_pages, paged_shared_attention, token_logprobs
            if kind == "copy":
                copy_pages(s["pools"], s["source"], s["target"])
                return s["pools"]
            if kind == "score":
                return token_logprobs(s["logits"], s["tokens"], top=case["top"], temperature=case["temperature"])
            return paged_shared_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["positions"], s["members"],
                                          s["shared"], window=case["window"], sinks=case["sinks"])
        if kind == "copy":
            source, target = s["source"].long(), s["target"].long()
            for pool in s["pools"]:
                pool[target] = pool[source]
            return s["pools"]
        if kind == "score":
            return _plain_score(s)
        return _plain_attention(s)


def _plain_score(s):
    case, tokens = s["case"], s["tokens"]
    x = s["logits"].float()
    d = (x - x.amax(-1, keepdim=True)) / case["temperature"]
    e = torch.exp(d)
    total = e.sum(-1)
    log_total = torch.log(total)
    given = d.gather(1, tokens.clamp(min=0).unsqueeze(1))[:, 0] - log_total
    given = torch.where(tokens >= 0, given, 0.0)
    entropy = log_total - (e * d).sum(-1) / total
    order = tokens.new_empty(x.shape[0], case["top"])
    left = x.clone() if case["top"] else x
    for i in range(case["top"]):
        order[:, i] = left.argmax(-1)  # the first of equal ones
        left.scatter_(1, order[:, i:i + 1], -math.inf)
    return given, entropy, order, d.gather(1, order) - log_total.unsqueeze(1)


def _plain_attention(s):
    case = s["case"]
    B, T, D, S, H, KV = _batch(case), case["tokens"], case["dim"], case["page"], case["heads"], case["kv_heads"]
    G, window, sinks = H // KV, case["window"], case["sinks"]
    out = torch.empty(B, T, H, D, device=DEVICE, dtype=s["q"].dtype)
    for b, n in enumerate(_plan(case)[1]):
        used = s["table"][b, :-(-n // S)].long()
        key = torch.arange(used.shape[0] * S, device=DEVICE).view(1, 1, 1, -1)
        k = s["k_pages"][used].float().transpose(0, 1).reshape(KV, -1, D)
        v = s["v_pages"][used].float().transpose(0, 1).reshape(KV, -1, D)
        p = s["positions"][b].view(1, 1, -1, 1)
        q = s["q"][b].view(T, KV, G, D).permute(1, 2, 0, 3).float()  # [KV, G, T, D]
        scores = torch.matmul(q.reshape(KV, -1, D), k.transpose(1, 2).contiguous()).view(KV, G, T, -1) * D ** -0.5
        seen = key <= p
        if window:
            seen = seen & ((key > p - window) | (key < sinks))
        scores = scores.masked_fill(~seen, -math.inf)
        e = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
        o = torch.matmul(e.view(KV, G * T, -1), v).view(KV, G, T, D) / e.sum(-1, keepdim=True).clamp(min=1e-30)
        out[b] = o.permute(2, 0, 1, 3).reshape(T, H, D).to(out.dtype)
    return out.view(B, T, H * D)


# --------------------------------------------------------------------- what a pass cannot do without

def _visible(case, p):
    """(first, last + 1) of the window's keys and the number of sinks before it, of a token at p."""
    start = max(0, p - case["window"] + 1) if case["window"] else 0
    return start, p + 1, min(case["sinks"], start)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "copy":
        page = case["kv_heads"] * case["page"] * case["dim"] * size
        return {"bytes": 2 * case["moves"] * 2 * case["layers"] * page, "flops": 0}
    if case["kind"] == "score":
        return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 12 * case["top"]), "flops": 0}
    H, KV, D, T, S = case["heads"], case["kv_heads"], case["dim"], case["tokens"], case["page"]
    group, lengths, shared = _plan(case)
    keys = pairs = 0
    first_of = {}  # a group's first visible shared key
    for b, n in enumerate(lengths):
        end = shared[group[b]] * S if group[b] >= 0 else 0
        positions = range(n - min(T, n), n)
        for p in positions:
            start, stop, sinks = _visible(case, p)
            pairs += stop - start + sinks
        start, _, sinks = _visible(case, positions[0])
        keys += n - max(start, end) + max(0, sinks - end)
        if group[b] >= 0:
            first, most = first_of.get(group[b], (end, 0))
            first_of[group[b]] = min(first, start), max(most, min(sinks, end))
    for g, (first, sinks) in first_of.items():
        keys += shared[g] * S - first + min(sinks, first)
    real = sum(min(T, n) for n in lengths)
    return {"bytes": 2 * keys * KV * D * size + 2 * real * H * D * size, "flops": 4.0 * pairs * H * D}


# ----------------------------------------------------------------------------------- 64-bit reference

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        moves = list(zip(s["source"].tolist(), s["target"].tolist()))
        pools = [pool.double() for pool in s["pools"]]
        for pool in pools:
            for a, b in moves:
                pool[b].copy_(pool[a])
        return pools
    if case["kind"] == "score":
        return _exact_score(case, s)
    B, D, S, H, KV, T = _batch(case), case["dim"], case["page"], case["heads"], case["kv_heads"], case["tokens"]
    out = torch.zeros(B, T, H, D, device=DEVICE, dtype=torch.float64)
    for b in range(B):
        p = s["positions"][b]
        p = p[p >= 0]
        j = torch.arange(int(p.max()) + 1, device=DEVICE)
        page = s["table"][b].long()[j // S]
        hidden = j.view(1, -1) > p.view(-1, 1)
        if case["window"]:
            hidden |= (p.view(-1, 1) - j.view(1, -1) >= case["window"]) & (j.view(1, -1) >= case["sinks"])
        for kv in range(KV):
            k, v = s["k_pages"][page, kv, j % S].double(), s["v_pages"][page, kv, j % S].double()
            for h in range(kv * (H // KV), (kv + 1) * (H // KV)):
                scores = (s["q"][b, :len(p), h * D:(h + 1) * D].double() @ k.T) / math.sqrt(D)
                out[b, :len(p), h] = torch.softmax(scores.masked_fill_(hidden, -math.inf), -1) @ v
    return out.view(B, T, H * D)


def _exact_score(case, s):
    given, entropy, chosen, worth = [], [], [], []
    for logits, tokens in zip(s["logits"].split(128), s["tokens"].split(128)):
        x = logits.double()
        logp = torch.log_softmax(x / case["temperature"], -1)
        at = logp[torch.arange(len(tokens), device=DEVICE), tokens.clamp(min=0)]
        given.append(torch.where(tokens < 0, 0.0, at))
        entropy.append(-(logp.exp() * logp).sum(-1))
        index = torch.arange(x.shape[1], device=DEVICE)
        picks = []
        for _ in range(case["top"]):
            best = torch.where(x == x.amax(-1, keepdim=True), index, x.shape[1]).amin(-1, keepdim=True)
            picks.append(best)
            x.scatter_(1, best, -math.inf)
        order = torch.cat(picks, -1) if picks else torch.empty(len(tokens), 0, dtype=torch.int64, device=DEVICE)
        chosen.append(order)
        worth.append(logp.gather(1, order))
    return tuple(torch.cat(x) for x in (given, entropy, chosen, worth))
