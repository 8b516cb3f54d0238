"""Plain 64-bit forms of the paged cache's operators, a token at a time on the CPU, and inputs for their tests."""
import math

import torch


def visible(p, length, window, sinks):
    """The positions that a token at p sees, of a table that holds ``length``."""
    j = torch.arange(length)
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    return seen if 0 <= p < length else torch.zeros_like(seen)


def attention(q, k_pages, v_pages, table, positions, window=0, sinks=0, scale=None):
    """(out [B, T, H * D], sum_j p_j |v_j| of the same shape) in float64."""
    q, k_pages, v_pages, table, positions = (t.detach().cpu() for t in (q, k_pages, v_pages, table, positions))
    N, KV, S, D = k_pages.shape
    B, T = positions.shape
    H = q.shape[2] // D
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    spread = torch.zeros_like(out)
    L = table.shape[1] * S
    for b in range(B):
        page = table[b].long().repeat_interleave(S)
        row = torch.arange(L) % S
        there = (page >= 0) & (page < N)
        for t in range(T):
            seen = visible(int(positions[b, t]), L, window, sinks) & there
            if not seen.any():
                continue
            k = k_pages[page[seen], :, row[seen]].double().transpose(0, 1)  # [KV, keys, D]
            v = v_pages[page[seen], :, row[seen]].double().transpose(0, 1)
            s = q[b, t].double().view(KV, H // KV, D) @ k.transpose(1, 2) * scale
            p = torch.softmax(s, -1)
            out[b, t] = (p @ v).view(H, D)
            spread[b, t] = (p @ v.abs()).view(H, D)
    return out.view(B, T, H * D), spread.view(B, T, H * D)


def attention_bound(ref, spread, dtype, keys):
    """How far a result may be from ``ref``. With u the half step of the type: the output's rounding u |o|; every
    probability rounded, p_j (1 + d_j) with |d_j| <= u both in the products and in their sum, so sum_j p_j d_j (v_j - o), at most
    u (sum_j p_j |v_j| + |o|); float16 probabilities below 2^-14 of the largest are off by 2^-25 at most, ``keys`` of them; and
    2^-11 of the same for fp32 scores (128 products of up to 13 in sum |q k| scale: 128 * 13 * 2^-24 = 2^-13.3, into both the
    products and their sum, and exp2's own error far below)."""
    u = torch.finfo(dtype).eps / 2
    weight = u + 2.0 ** -11 + (keys * 2.0 ** -25 if dtype == torch.float16 else 0.0)
    return u * ref.abs() + weight * (spread + ref.abs()) * (1 + u) + 1e-12


def rotate(x, cos, sin):
    """x [..., D] float64 under the rotate-half convention."""
    h = x.shape[-1] // 2
    return torch.cat((x[..., :h] * cos[..., :h] - x[..., h:] * sin[..., :h],
                      x[..., h:] * cos[..., h:] + x[..., :h] * sin[..., h:]), -1)


def write(q, k, v, cos, sin, positions, k_pages, v_pages, table):
    """(rotated queries, key pages, value pages) in float64."""
    q, k, v, cos, sin, positions, k_pages, v_pages, table = (
        t.detach().cpu() for t in (q, k, v, cos, sin, positions, k_pages, v_pages, table))
    N, KV, S, D = k_pages.shape
    B, T = positions.shape
    out = torch.zeros(q.shape, dtype=torch.float64)
    k_pages, v_pages = k_pages.double(), v_pages.double()
    cos, sin = cos.double().view(B, T, D), sin.double().view(B, T, D)
    for b in range(B):
        for t in range(T):
            p = int(positions[b, t])
            if not 0 <= p < table.shape[1] * S:
                continue
            turn = lambda x: rotate(x[b, t].double().view(-1, D), cos[b, t], sin[b, t])  # noqa: E731
            out[b, t] = turn(q).view(-1)
            page = int(table[b, p // S])
            if 0 <= page < N:
                k_pages[page, :, p % S] = turn(k)
                v_pages[page, :, p % S] = v[b, t].double().view(KV, D)
    return out, k_pages, v_pages


def verify(logits, drafts, uniforms, draft_probs=None, temperature=1.0):
    """([accepted], [[tokens]]) by the definition, a sequence at a time."""
    B, n = drafts.shape
    V = logits.shape[2]
    kept, out = [], []
    for b in range(B):
        x, u = logits[b].detach().cpu().double(), uniforms[b].detach().cpu().double()
        best = [next((i for i, e in enumerate(r.tolist()) if math.isnan(e)), int(r.argmax())) for r in x]
        sound = [math.isfinite(float(r.max())) and not bool(r.isnan().any()) for r in x]

        def dist(i):
            if temperature == 0.0 or not sound[i]:
                return torch.nn.functional.one_hot(torch.tensor(best[i]), V).double()
            e = torch.exp((x[i] - x[i].max()) / temperature)
            return e / e.sum()

        tokens, w = [], None
        for i in range(n):
            d = int(drafts[b, i])
            if not 0 <= d < V:
                break
            p = dist(i)
            if draft_probs is None or temperature == 0.0:
                q = torch.nn.functional.one_hot(torch.tensor(d), V).double()
            else:
                q = draft_probs[b, i].detach().cpu().double()
            if sound[i] and bool(u[i] * q[d] < p[d]):
                tokens.append(d)
                continue
            w = (p - q).clamp(min=0.0)
            if not sound[i] or temperature == 0.0 or float(w.sum()) == 0.0:
                w = p
            break
        kept.append(len(tokens))
        w = dist(len(tokens)) if w is None else w
        sums = w.cumsum(0)
        passed = ((sums > u[n] * sums[-1]) & (w > 0)).nonzero()
        tokens.append(int(passed[0]) if len(passed) else int((w > 0).nonzero()[-1]))
        out.append(tokens + [-1] * (n + 1 - len(tokens)))
    return torch.tensor(kept), torch.tensor(out)


def paged_case(heads, kv, dim, page, lengths, tokens, dtype, device, seed=0, window=0, sinks=0, spare=2):
    """(q, k_pages, v_pages, table, positions) of sequences of ``lengths`` whose last ``tokens`` are new (front-aligned,
    -1 behind those of a sequence that has fewer), pages in random order; pages that a window hides are not there. Rows of the
    pages that hold no position, and pages of nobody, are NaN."""
    g = torch.Generator().manual_seed(seed)
    B = len(lengths)
    slots = max(-(-n // page) for n in lengths) + 1
    keep = torch.zeros(B, slots, dtype=torch.bool)
    positions = torch.full((B, tokens), -1, dtype=torch.int64)
    for b, n in enumerate(lengths):
        real = min(tokens, n)
        positions[b, :real] = torch.arange(n - real, n)
        keep[b, :-(-n // page)] = True
        if window:
            keep[b, -(-sinks // page):max(0, n - real - window + 1) // page] = False
    used = int(keep.sum())
    pool = used + spare
    table = torch.full((B, slots), -1, dtype=torch.int32)
    table[keep] = torch.randperm(pool, generator=g)[:used].int()
    k = torch.full((pool, kv, page, dim), math.nan)
    v = torch.full((pool, kv, page, dim), math.nan)
    for b, n in enumerate(lengths):
        for s in range(-(-n // page)):
            if keep[b, s]:
                rows = min(page, n - s * page)
                k[table[b, s], :, :rows] = torch.randn(kv, rows, dim, generator=g)
                v[table[b, s], :, :rows] = torch.randn(kv, rows, dim, generator=g)
    q = torch.randn(B, tokens, heads * dim, generator=g) * 1.5
    return (q.to(dtype).to(device), k.to(dtype).to(device), v.to(dtype).to(device), table.to(device), positions.to(device))
