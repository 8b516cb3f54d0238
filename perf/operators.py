"""Performance cases of the paged cache's operators: what a server of many sequences has the framework do in one
layer of a step, and at its end.

The kinds of cases, and the entry point each one times:

* ``write``   ``paged_rope_write``: the new tokens' queries rotated, their rotated keys and their values into the pages;
* ``decode``  ``paged_attention`` of one new token a sequence over its pages;
* ``chunk``   ``paged_attention`` of several tokens a sequence: drafted tokens, prompts, chunks after a context;
* ``verify``  ``verify_drafts``: drafted tokens against the model's logits, from given random numbers.

Sequences have lengths of their own, and their pages lie anywhere in the pool. A sliding window with a few first
tokens that stay visible drops the pages between them (their table entries are -1). Queries are N(0, 1.5), keys and
values N(0, 1) as after a norm; logits are N(0, 2.5) with some tokens well above, the drafter's the same with noise.

``run`` with ``own`` false computes the operators in elementary torch operations, in float32 (``verify`` in float64:
a token is chosen where a running sum passes a number); with ``own`` true it calls the framework.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
THETA = 10000.0


# ------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one token of one sequence: the smallest write of a step (7B heads)
        dict(name="write_1", kind="write", heads=32, kv_heads=32, dim=128, page=16, batch=1, tokens=1, low=500, high=500,
             dtype="fp16"),
        # the prompts of a batch of four going in at once, ragged ends padded (70B heads)
        dict(name="write_prompt_4x777", kind="write", heads=64, kv_heads=8, dim=128, page=64, batch=4, tokens=777, low=300,
             high=777, dtype="bf16"),
        # a chat's next token: one sequence in a 1000-token context (7B heads)
        dict(name="decode_1_mha", kind="decode", heads=32, kv_heads=32, dim=128, page=16, batch=1, low=1000, high=1000,
             window=0, sinks=0, dtype="fp16"),
        # 17 users of grouped-query layers (70B heads), contexts from a greeting to a document
        dict(name="decode_17_gqa", kind="decode", heads=64, kv_heads=8, dim=128, page=32, batch=17, low=20, high=8000,
             window=0, sinks=0, dtype="bf16"),
        # a full server: 64 users with long contexts
        dict(name="decode_64_gqa", kind="decode", heads=64, kv_heads=8, dim=128, page=64, batch=64, low=4000, high=16000,
             window=0, sinks=0, dtype="bf16"),
        # streaming over endless text: 48 sequences, the last 1021 tokens and four sinks, small heads
        dict(name="decode_48_window", kind="decode", heads=32, kv_heads=8, dim=64, page=16, batch=48, low=500, high=30000,
             window=1021, sinks=4, dtype="fp16"),
        # five drafted tokens of nine sequences, to be verified in one pass (70B heads)
        dict(name="chunk_draft_9x5", kind="chunk", heads=64, kv_heads=8, dim=128, page=32, batch=9, tokens=5, low=300,
             high=6000, window=0, sinks=0, dtype="bf16"),
        # a prompt of a thousand tokens (7B heads)
        dict(name="chunk_prompt_1000", kind="chunk", heads=32, kv_heads=32, dim=128, page=16, batch=1, tokens=1000, low=1000,
             high=1000, window=0, sinks=0, dtype="fp16"),
        # a chunk of a long prompt under a window with sinks (70B heads)
        dict(name="chunk_window_4001", kind="chunk", heads=64, kv_heads=8, dim=128, page=64, batch=1, tokens=4001, low=12345,
             high=12345, window=2047, sinks=16, dtype="bf16"),
        # two sequences' chunks after contexts of their own, small heads
        dict(name="chunk_2x700_past", kind="chunk", heads=32, kv_heads=8, dim=64, page=48, batch=2, tokens=700, low=1500,
             high=9000, window=0, sinks=0, dtype="fp16"),
        # four drafted tokens of one sequence against float32 logits (7B vocabulary)
        dict(name="verify_1x4", kind="verify", batch=1, drafts=4, vocab=32000, greedy=False, temperature=0.8, dtype="fp32"),
        # up to seven drafts of 64 sequences, bf16 logits of a large odd vocabulary
        dict(name="verify_64x7", kind="verify", batch=64, drafts=7, vocab=100003, greedy=False, temperature=1.0, dtype="bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["write", "decode", "decode", "decode", "chunk", "chunk", "chunk", "verify"])
    c = dict(kind=kind, dtype=rng.choice(["fp16", "bf16"]))
    if kind == "verify":
        c.update(batch=_spread(rng, 1, 64), drafts=_spread(rng, 1, 8), vocab=_spread(rng, 1000, 128000),
                 greedy=rng.random() < 0.25, temperature=rng.choice([0.0, 0.7, 1.0, 1.3]),
                 dtype=rng.choice(["fp32", "fp16", "bf16"]))
        return c
    heads, kv_heads = rng.choice([(32, 32), (16, 16), (64, 8), (32, 8), (24, 8), (20, 4), (8, 1), (5, 5)])
    c.update(heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), page=rng.choice([16, 16, 32, 48, 64, 128, 256]))
    if kind != "write":
        windowed = rng.random() < 0.4
        c.update(window=_spread(rng, 100, 4000) if windowed else 0, sinks=rng.choice([0, 1, 4, 16, 100]) if windowed else 0)
    if kind == "decode":
        c["batch"] = _spread(rng, 1, 64)
        most = max(64, min(16000, int(5e6 // (c["batch"] * kv_heads))))  # no costlier than the listed ones
        c["high"] = _spread(rng, 64, most)
        c["low"] = max(1, int(c["high"] * rng.choice([0.02, 0.3, 1.0])))
        return c
    c["batch"] = rng.choice([1, 1, 2, 3, 8])
    if kind == "write":
        c["tokens"] = _spread(rng, 1, 3000 // c["batch"])
        c["low"] = max(1, c["tokens"] - rng.choice([0, 0, c["tokens"] // 2]))
        c["high"] = c["low"] + _spread(rng, 1, 2000)
        return c
    c["tokens"] = _spread(rng, 2, 2000 // c["batch"])
    most = max(c["tokens"], min(16000, int(6e8 // (c["batch"] * c["tokens"] * heads))))
    c["high"] = min(most, c["tokens"] + _spread(rng, 1, 12000))
    c["low"] = max(1, int(c["high"] * rng.choice([0.3, 0.6, 1.0])))
    return c


# ------------------------------------------------------------------------------ inputs from a seed

def _lengths(case):
    """Each sequence's length with its new tokens: from ``low`` to ``high``, the first the longest."""
    B, low, high = case["batch"], case["low"], case["high"]
    if B == 1:
        return [high]
    # a low-discrepancy spread, the same for every seed, so that `work` knows it
    return [high] + [low + int((high - low) * ((i * 0.6180339887) % 1.0)) for i in range(1, B)]


def _positions(case):
    """[batch, tokens]: the last tokens of each sequence; a sequence shorter than the chunk has its tokens at the front and
    -1 behind them."""
    T, rows = case.get("tokens", 1), []
    for n in _lengths(case):
        real = min(T, n)
        rows.append([n - real + i for i in range(real)] + [-1] * (T - real))
    return torch.tensor(rows, dtype=torch.int64)


def _pages(case, g):
    """The page table [batch, most pages of a sequence] (int32, -1 where there is none) and the pool's size."""
    S, T, lengths = case["page"], case.get("tokens", 1), _lengths(case)
    most = max(math.ceil(n / S) for n in lengths) + 1
    keep = torch.zeros(len(lengths), most, dtype=torch.bool)
    for b, n in enumerate(lengths):
        keep[b, :math.ceil(n / S)] = True
        if case.get("window"):  # pages that no new token sees are gone
            first = max(0, n - min(T, n) - case["window"] + 1)  # the first token's first key
            keep[b, math.ceil(case["sinks"] / S):first // S] = False
    used = int(keep.sum())
    pool = used + 3
    order = torch.randperm(pool, device=DEVICE, generator=g)[:used].to(torch.int32)
    table = torch.full(keep.shape, -1, dtype=torch.int32, device=DEVICE)
    table[keep.to(DEVICE)] = order
    return table, pool


def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, device=DEVICE, generator=g, dtype=dtype).mul_(scale)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B = case["batch"]
    s = dict(case=case)
    if case["kind"] == "verify":
        n, V = case["drafts"], case["vocab"]
        base = torch.randn(B, n + 1, V, device=DEVICE, generator=g) * 2.5
        tall = torch.randint(0, V, (B, n + 1, 5), device=DEVICE, generator=g)
        base.scatter_add_(2, tall, 6.0 + 3.0 * torch.randn(B, n + 1, 5, device=DEVICE, generator=g))
        drafter = base[:, :n] + 0.7 * torch.randn(B, n, V, device=DEVICE, generator=g)
        s["logits"] = base.to(dt)
        probs = torch.softmax(drafter, -1)
        if case["greedy"]:
            s["drafts"], s["draft_probs"] = probs.argmax(-1), None
        else:
            s["drafts"] = torch.multinomial(probs.view(B * n, V), 1, generator=g).view(B, n)
            s["draft_probs"] = probs
        if n > 1 and B > 1:  # every third sequence has fewer drafts
            s["drafts"][::3, n // 2:] = -1
        s["uniforms"] = torch.rand(B, n + 1, device=DEVICE, generator=g)
        return s
    H, KV, D, S, T = case["heads"], case["kv_heads"], case["dim"], case["page"], case.get("tokens", 1)
    s["positions"] = _positions(case).to(DEVICE)
    s["table"], pool = _pages(case, g)
    s["k_pages"] = _normal(g, (pool, KV, S, D), dt)
    s["v_pages"] = _normal(g, (pool, KV, S, D), dt)
    if case["kind"] == "write":
        qkv = _normal(g, (B, T, (H + 2 * KV) * D), dt, 1.5)  # one projection's output
        s["q"], s["k"], s["v"] = qkv.split([H * D, KV * D, KV * D], dim=-1)
        angle = s["positions"].double().view(B, T, 1) / THETA ** (torch.arange(0, D, 2, device=DEVICE).double() / D)
        angle = torch.cat((angle, angle), -1)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = _normal(g, (B, T, H * D), dt, 1.5)
    return s


# -------------------------------------------------------------------------------------------- a pass

def run(state):
    case = state["case"]
    kind = case["kind"]
    with torch.no_grad():
        if own:
            from nanoquant_amd.serve import paged_attention, paged_rope_write, verify_drafts
            s = state
            if kind == "write":
                q = paged_rope_write(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["k_pages"], s["v_pages"],
                                     s["table"])
                return q, s["k_pages"], s["v_pages"]
            if kind == "verify":
                return verify_drafts(s["logits"], s["drafts"], s["uniforms"], draft_probs=s["draft_probs"],
                                     temperature=case["temperature"])
            return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["positions"], window=case["window"],
                                   sinks=case["sinks"])
        if kind == "write":
            return _plain_write(state)
        if kind == "verify":
            return _plain_verify(state)
        return _plain_attention(state)


def _plain_write(s):
    case = s["case"]
    B, T, D, S, H = case["batch"], case["tokens"], case["dim"], case["page"], case["heads"]
    cos, sin = s["cos"].view(B, T, 1, D), s["sin"].view(B, T, 1, D)

    def rotate(x):
        x = x.reshape(B, T, -1, D).float()
        half = torch.cat((-x[..., D // 2:], x[..., :D // 2]), -1)
        return x * cos + half * sin

    pos = s["positions"]
    real = pos >= 0
    q = torch.where(real.view(B, T, 1, 1), rotate(s["q"]), 0.0).to(s["q"].dtype).view(B, T, H * D)
    at = pos.clamp(min=0)
    page = torch.gather(s["table"].long(), 1, at // S)
    ok = (real & (page >= 0)).nonzero(as_tuple=True)
    rows, offs = page[ok], (at % S)[ok]
    s["k_pages"][rows, :, offs] = rotate(s["k"])[ok].to(s["k_pages"].dtype)
    s["v_pages"][rows, :, offs] = s["v"].reshape(B, T, -1, D)[ok]
    return q, s["k_pages"], s["v_pages"]


def _plain_attention(s):
    case = s["case"]
    B, T, D, S, H, KV = (case.get(k, 1) for k in ("batch", "tokens", "dim", "page", "heads", "kv_heads"))
    G, window, sinks = H // KV, case["window"], case["sinks"]
    table, pos = s["table"], s["positions"]
    out = torch.empty(B, T, H, D, device=DEVICE, dtype=s["q"].dtype)
    step = max(1, int(1.5e8 // (H * table.shape[1] * S)))
    for b, n in enumerate(_lengths(case)):
        used = table[b, :math.ceil(n / S)]
        key = torch.arange(used.shape[0] * S, device=DEVICE).view(-1, S)
        there = used >= 0
        key = key[there].view(1, 1, 1, -1)
        k = s["k_pages"][used[there].long()].float().transpose(0, 1).reshape(KV, -1, D)
        v = s["v_pages"][used[there].long()].float().transpose(0, 1).reshape(KV, -1, D)
        kt = k.transpose(1, 2).contiguous()
        for t in range(0, T, step):
            p = pos[b, t:t + step].view(1, 1, -1, 1)
            q = s["q"][b, t:t + step].view(-1, KV, G, D).permute(1, 2, 0, 3).float()  # [KV, G, t, D]
            scores = torch.matmul(q.reshape(KV, -1, D), kt).view(KV, G, q.shape[2], -1) * D ** -0.5
            seen = key <= p
            if window:
                seen = seen & ((key > p - window) | (key < sinks))
            scores = scores.masked_fill(~seen, -math.inf)
            e = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
            o = torch.matmul(e.view(KV, -1, e.shape[-1]), v).view(KV, G, -1, D) / e.sum(-1, keepdim=True).clamp(min=1e-30)
            out[b, t:t + step] = o.permute(2, 0, 1, 3).reshape(-1, H, D).to(out.dtype)
    return out.view(B, T, H * D)


def _plain_verify(s):
    case, drafts, u = s["case"], s["drafts"], s["uniforms"].double()
    B, n = drafts.shape
    x = s["logits"].double()
    if case["temperature"] == 0.0:
        p = torch.zeros_like(x).scatter_(2, x.argmax(-1, keepdim=True), 1.0)
    else:
        x = x / case["temperature"]
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    at = drafts.clamp(min=0).unsqueeze(-1)
    if s["draft_probs"] is None or case["temperature"] == 0.0:
        q = torch.zeros_like(p[:, :n]).scatter_(2, at, 1.0)
    else:
        q = s["draft_probs"].double()
    q = torch.where((drafts >= 0).unsqueeze(-1), q, 0.0)
    keep = (drafts >= 0) & (u[:, :n] * q.gather(2, at)[..., 0] < p[:, :n].gather(2, at)[..., 0])
    accepted = keep.long().cumprod(1).sum(1)
    row = accepted.view(B, 1, 1).expand(B, 1, p.shape[2])
    chosen = p.gather(1, row)[:, 0]
    q = torch.cat((q, torch.zeros_like(q[:, :1])), 1).gather(1, row)[:, 0]  # zeros behind the last draft
    left = (chosen - q).clamp(min=0.0)
    left = torch.where(left.sum(-1, keepdim=True) > 0.0, left, chosen)
    sums = left.cumsum(-1)
    token = torch.searchsorted(sums, u[:, n:] * sums[:, -1:], right=True).clamp(max=p.shape[2] - 1)
    index = torch.arange(n + 1, device=DEVICE)
    tokens = torch.nn.functional.pad(drafts, (0, 1), value=-1)
    tokens = torch.where(index < accepted.view(B, 1), tokens, torch.where(index == accepted.view(B, 1), token, -1))
    return accepted, tokens


# --------------------------------------------------------------------- what a pass cannot do without

def _seen(case):
    """(keys that some token of a sequence sees, (token, key) pairs that are seen), summed over the sequences."""
    T, window, sinks = case.get("tokens", 1), case["window"], case["sinks"]
    keys = pairs = 0
    for n in _lengths(case):
        first = n - min(T, n)
        for p in range(first, n):
            full = p + 1
            if window and full > window:
                start = p - window + 1
                full = window + min(sinks, start)
            pairs += full
        start = max(0, first - window + 1) if window else 0
        keys += n - start + min(sinks, start)
    return keys, pairs


def work(case):
    B = case["batch"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "verify":
        # every row of logits once, and of the drafter's probabilities those of the chosen rows (one a sequence)
        rows = B * (case["drafts"] + 1)
        draft_rows = 0 if case["greedy"] or case["temperature"] == 0.0 else B
        return {"bytes": rows * case["vocab"] * size + draft_rows * case["vocab"] * 4 + B * (case["drafts"] + 1) * 20,
                "flops": 0}
    H, KV, D, T = case["heads"], case["kv_heads"], case["dim"], case.get("tokens", 1)
    real = sum(min(T, n) for n in _lengths(case))
    if case["kind"] == "write":
        return {"bytes": real * (2 * (H + 2 * KV) * D * size + 8 * D + 8), "flops": 3.0 * real * (H + KV) * D}
    keys, pairs = _seen(case)
    return {"bytes": 2 * keys * KV * D * size + 2 * real * H * D * size, "flops": 4.0 * pairs * H * D}


# ----------------------------------------------------------------------------------- 64-bit reference

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(case, s)
    B, D, S, H, KV, T = (case.get(k, 1) for k in ("batch", "dim", "page", "heads", "kv_heads", "tokens"))
    if case["kind"] == "write":
        return _exact_write(s, B, T, D, S)
    if _seen(case)[1] * H > 3e9:
        return None
    out = torch.zeros(B, T, H, D, device=DEVICE, dtype=torch.float64)
    for b in range(B):
        real = [t for t in range(T) if s["positions"][b, t] >= 0]
        p = s["positions"][b, real]
        last = int(p.max())
        j = torch.arange(last + 1, device=DEVICE)
        page = s["table"][b].long()[j // S]
        j, page = j[page >= 0], page[page >= 0]
        mask = j.view(1, -1) > p.view(-1, 1)
        if case["window"]:
            mask |= (p.view(-1, 1) - j.view(1, -1) >= case["window"]) & (j.view(1, -1) >= case["sinks"])
        for h in range(H):
            k = s["k_pages"][page, h * KV // H, j % S].double()
            v = s["v_pages"][page, h * KV // H, j % S].double()
            scores = (s["q"][b, real, h * D:(h + 1) * D].double() @ k.T) / math.sqrt(D)
            out[b, real, h] = torch.softmax(scores.masked_fill_(mask, -math.inf), -1) @ v
    return out.view(B, T, H * D)


def _exact_write(s, B, T, D, S):
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    q = torch.zeros(s["q"].shape, device=DEVICE, dtype=torch.float64)
    for b in range(B):
        real = int((s["positions"][b] >= 0).sum())
        pos = s["positions"][b, :real]
        c, sn = s["cos"][b, :real, None, :D // 2].double(), s["sin"][b, :real, None, :D // 2].double()

        def turn(x):
            x = x[b, :real].double().reshape(real, -1, D)
            lo, hi = x[..., :D // 2], x[..., D // 2:]
            return torch.cat((lo * c - hi * sn, hi * c + lo * sn), -1)

        q[b, :real] = turn(s["q"]).reshape(real, -1)
        page = s["table"][b].long()[pos // S]
        k_pages[page, :, pos % S] = turn(s["k"])
        v_pages[page, :, pos % S] = s["v"][b, :real].double().reshape(real, -1, D)
    return q, k_pages, v_pages


def _exact_verify(case, s):
    B, n = s["drafts"].shape
    accepted = torch.zeros(B, dtype=torch.int64)
    tokens = torch.full((B, n + 1), -1, dtype=torch.int64)
    for b in range(B):
        x, u = s["logits"][b].double().cpu(), s["uniforms"][b].double().cpu()
        drafts = [int(t) for t in s["drafts"][b]]
        drafts = drafts[:drafts.index(-1)] if -1 in drafts else drafts
        if case["temperature"] == 0.0:
            best = x.argmax(-1)
            p = torch.nn.functional.one_hot(best, x.shape[1]).double()
        else:
            p = torch.softmax(x / case["temperature"], -1)
        i, rest = 0, None
        while i < len(drafts):
            if s["draft_probs"] is None:
                q = torch.zeros_like(p[i])
                q[drafts[i]] = 1.0
            else:
                q = s["draft_probs"][b, i].double().cpu()
            if not u[i] * q[drafts[i]] < p[i, drafts[i]]:
                rest = (p[i] - q).clamp(min=0.0)
                if case["temperature"] == 0.0 or not rest.sum() > 0.0:
                    rest = p[i]
                break
            tokens[b, i] = drafts[i]
            i += 1
        rest = p[i] if rest is None else rest
        sums = rest.cumsum(0)
        tokens[b, i] = min(int((sums <= u[n] * sums[-1]).sum()), x.shape[1] - 1)
        accepted[b] = i
    return accepted.to(DEVICE), tokens.to(DEVICE)
