"""Inputs for the tests of what several answers to one prompt need, and plain 64-bit forms beside those of serve_oracle."""
import math

import torch


def shared_case(heads, kv, dim, page, groups, alone, tokens, dtype, device, seed=0, spare=2, read=0):
    """(q, k_pages, v_pages, table, positions, members, shared): ``groups`` are (pages in common, [positions of each member
    behind them]), ``alone`` lengths of sequences in no group. Sequences come in random order, pages too; rows of the pages that
    hold no position, and pages of nobody, are NaN. The last ``tokens`` positions of a sequence are new, -1 behind them. The
    table is as wide as ``read`` bytes of keys and values in all its rows would take: calls are told apart by that."""
    g = torch.Generator().manual_seed(seed)
    whole = [(i, n, n * page + own) for i, (n, owns) in enumerate(groups) for own in owns] + [(-1, 0, n) for n in alone]
    B = len(whole)
    place = torch.randperm(B, generator=g).tolist()
    slots = max(max(-(-n // page) for _, _, n in whole) + 1, -(-read // (B * page * kv * dim * 4)))
    prompts = [n for n, _ in groups]
    used = sum(prompts) + sum(-(-n // page) - m for _, m, n in whole)
    pool = used + spare
    order = torch.randperm(pool, generator=g).tolist()
    k, v = (torch.full((pool, kv, page, dim), math.nan) for _ in range(2))
    random = lambda rows: torch.randn(kv, rows, dim, generator=g)  # noqa: E731
    pages = [[order.pop() for _ in range(n)] for n in prompts]
    for at in (at for list_ in pages for at in list_):
        k[at], v[at] = random(page), random(page)
    table = torch.full((B, slots), -1, dtype=torch.int32)
    positions = torch.full((B, tokens), -1, dtype=torch.int64)
    most = max((len(owns) for _, owns in groups), default=1) + 1
    members = torch.full((max(1, len(groups)), most), -1, dtype=torch.int32)
    for b, (i, m, n) in zip(place, whole):
        row = pages[i][:] if i >= 0 else []
        for slot in range(m, -(-n // page)):
            row.append(order.pop())
            rows = min(page, n - slot * page)
            k[row[-1], :, :rows], v[row[-1], :, :rows] = random(rows), random(rows)
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        real = min(tokens, n)
        positions[b, :real] = torch.arange(n - real, n)
        if i >= 0:
            free = (members[i] < 0).nonzero()[:, 0]
            members[i, free[int(torch.randint(0, len(free), (1,), generator=g))]] = b
    shared = torch.tensor(prompts or [0], dtype=torch.int32)
    q = torch.randn(B, tokens, heads * dim, generator=g) * 1.5
    return (q.to(dtype).to(device), k.to(dtype).to(device), v.to(dtype).to(device),
            *(t.to(device) for t in (table, positions, members, shared)))


def score(logits, tokens, top, temperature):
    """(logprobs, entropy, top tokens, their logprobs, bound of logprobs, of the entropy, of the top's), in float64.

    With u = 2^-24, d = (x - max) / temperature and weights p: a float32 d is off by 3 u |d| at most (the scale's rounding, the
    difference's or product's, and that of the sum with the largest, in which a shift that all d share cancels), its exponential
    by that and 2 u, a sum over the vocabulary by a rounding for each of the V / 64 terms that one lane adds in turn and 32 for
    the lanes' and the blocks' sums. So the total is off by a factor of 1 +- e, e = u (3 E|d| + V / 64 + 34), its logarithm by e
    and its own rounding of 4 u, and log p by those and the roundings of d and the difference. The sum of p d takes the same e
    and d's own error, E|d| (e + 3 u) + 3 u E d^2, divided by the total."""
    x = logits.detach().cpu().double()
    t = tokens.detach().cpu()
    V = x.shape[-1]
    d = (x - x.amax(-1, keepdim=True)) / temperature
    e = torch.exp(d)
    total = e.sum(-1)
    log_total = total.log()
    p = e / total.unsqueeze(-1)
    dz = torch.where(e > 0, d, 0.0)
    there = (t >= 0) & (t < V)
    given = torch.where(there, d.gather(-1, torch.where(there, t, 0).unsqueeze(-1))[..., 0] - log_total, 0.0)
    entropy = log_total - (p * dz).sum(-1)
    key = torch.where(x.isnan(), math.inf, x)
    picks = []
    flat, nan = key.reshape(-1, V).clone(), x.isnan().reshape(-1, V).clone()
    taken = torch.zeros_like(nan)
    for _ in range(top):
        row = []
        for r in range(flat.shape[0]):
            left = (nan[r] & ~taken[r]).nonzero()[:, 0]
            if len(left) == 0:
                rest = torch.where(taken[r], -math.inf, flat[r])
                left = ((flat[r] == rest.max()) & ~taken[r]).nonzero()[:, 0]
            row.append(int(left[0]))
            taken[r, left[0]] = True
        picks.append(row)
    order = torch.tensor(picks, dtype=torch.int64).view(top, flat.shape[0]).t().reshape(*t.shape, top)
    best = d.gather(-1, order) - log_total.unsqueeze(-1)
    u = 2.0 ** -24
    mean, square = (p * dz.abs()).sum(-1), (p * dz * dz).sum(-1)
    off = u * (3 * mean + V / 64 + 34)
    own = lambda y: off.view(*off.shape, *[1] * (y.dim() - off.dim())) + u * (  # noqa: E731
        8 * y.abs().nan_to_num(0.0, posinf=0.0) + 8 * log_total.abs().view(*off.shape, *[1] * (y.dim() - off.dim())) + 4)
    entropy_bound = off + 4 * u * (log_total.abs() + 1) + mean * (2 * off + 8 * u) + 3 * u * square + 4 * u * entropy.abs()
    return given, entropy, order, best, own(given), entropy_bound, own(best)


def check_score(got, want):
    """``token_logprobs``' results against ``score``'s: whole numbers equal, the others within their bounds, and NaN and
    infinities where they have to be."""
    given, entropy, order, best = (x.detach().cpu() for x in got)
    assert given.dtype == entropy.dtype == best.dtype and order.dtype == torch.int64
    assert torch.equal(order, want[2])
    for x, y, bound in ((given, want[0], want[4]), (entropy, want[1], want[5]), (best, want[3], want[6])):
        assert x.shape == y.shape
        held = y.to(x.dtype).double()  # infinite too where the result's type holds no such number
        x = x.double()
        odd = ~torch.isfinite(held)
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x[odd].nan_to_num(1.0), held[odd].nan_to_num(1.0))
        off = ((x - y).abs() / bound)[~odd]
        assert off.numel() == 0 or off.max() <= 1.0, f"{off.max().item():.2f} times the bound"
