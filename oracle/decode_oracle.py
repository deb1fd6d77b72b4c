"""Plain 64-bit implementations of rotary positions, beam selection, shared pages and page copies for the tests: Python loops and lists."""
import math

import torch


def rotate(x, positions, inv_freq, axes=None, interleaved=False, inverse=False):
    """[batch, heads, tokens, channels] turned, in 64 bits; positions [batch, tokens] or [axes, batch, tokens]."""
    at = positions.cpu().long().view(-1, *positions.shape[-2:])
    y = x.detach().cpu().double().clone()
    pairs = inv_freq.numel()
    for i, f in enumerate(inv_freq.cpu().double().tolist()):
        a = at[0 if axes is None else min(max(int(axes[i]), 0), at.shape[0] - 1)].double() * f
        cos, sin = torch.cos(a)[:, None], torch.sin(a)[:, None] * (-1.0 if inverse else 1.0)
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        x1, x2 = x.detach().cpu().double()[..., lo], x.detach().cpu().double()[..., hi]
        y[..., lo], y[..., hi] = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    return y


def select(logits, scores, count, finished=None, end_token=0):
    """(scores [groups, count] in 64 bits, rows, tokens); NaN ranks first, ties go to the lowest place."""
    G, K = scores.shape
    V = logits.shape[1]
    values, rows, tokens = [], [], []
    for g in range(G):
        c = torch.empty(K, V, dtype=torch.float64)
        for k in range(K):
            s, x = float(scores[g, k]), logits[g * K + k].cpu().double()
            if finished is not None and bool(finished[g, k]):
                c[k] = -math.inf
                c[k, end_token] = s
            elif s == -math.inf or bool((x == -math.inf).all()):
                c[k] = -math.inf
            else:
                c[k] = torch.where(x == -math.inf, -math.inf, s + (x - torch.logsumexp(x, 0)) if not bool((x.isnan() | (x == math.inf)).any()) else math.nan)
        flat = c.view(-1)
        key = torch.where(flat.isnan(), math.inf, flat)
        # NaN before +inf, then descending, stable
        order = torch.tensor(sorted(range(K * V), key=lambda n: (not bool(flat[n].isnan()), -float(key[n]), n))[:count]) if K * V <= 4096 else \
            flat.sort(stable=True, descending=True).indices[:count]
        values.append(flat[order])
        rows.append(g * K + order // V)
        tokens.append(order % V)
    return torch.stack(values), torch.stack(rows), torch.stack(tokens)


def _let_go(entries, shared, stack):
    """entries: pages whose holder lets go of them, in the order of rows and blocks; `shared`: counts beyond one before anything is let go of.  The pages that nobody holds
    then go on the stack, the first on top."""
    left = dict()
    for q in entries:
        left[q] = left.get(q, shared[q] + 1) - 1
    back = [q for q in dict.fromkeys(entries) if left[q] == 0]
    for q, n in left.items():
        shared[q] = max(n - 1, 0)
    return stack + back[::-1]


def trim_shared(table, held, free, n_free, shared, lens, page):
    """(table, held, stack, shared)."""
    table, held, shared = [list(r) for r in table], list(held), list(shared)
    entries = []
    for b, c in enumerate(lens):
        keep = min(-(-c // page), len(table[b]))
        for j in range(keep, held[b]):
            if table[b][j] >= 0:
                entries.append(table[b][j])
            table[b][j] = -1
        held[b] = min(held[b], keep)
    return table, held, _let_go(entries, shared, list(free[:n_free])), shared


def fork(table, held, free, n_free, shared, lens, parents, page):
    """(table, held, stack, shared, missing, lens, copies): copies a list of (source, target, rows)."""
    B, old, stack = len(table), [list(r) for r in table], list(free[:n_free])
    lens = [min(c, h * page) for c, h in zip(lens, held)]
    shared, before = list(shared), list(shared)
    new, now, out, copies, missing = [], [], [], [], 0
    kept = set()  # rows whose begun page stays with the first child
    first, count = {}, {}
    for b, r in enumerate(parents):
        first.setdefault(r, b)
        count[r] = count.get(r, 0) + 1
    for b, r in enumerate(parents):
        if not 0 <= r < B:
            new.append([])
            now.append(0)
            out.append(0)
            continue
        whole, rest = divmod(lens[r], page)
        row, tokens = old[r][:whole], lens[r]
        if rest > 0:
            q = old[r][whole]
            if q < 0:
                tokens = whole * page
            elif before[q] == 0 and r not in kept and first[r] == b:
                kept.add(r)
                row.append(q)
            elif stack:
                row.append(stack.pop())
                copies.append((q, row[-1], rest))
            else:
                missing += 1
                tokens = whole * page
        new.append(row)
        now.append(len(row))
        out.append(tokens)
    entries = []
    for r in range(B):
        children = count.get(r, 0)
        whole = lens[r] // page if children else 0
        for q in old[r][:whole]:
            if q >= 0:
                shared[q] += children - 1
        for j in range(whole, held[r]):
            if old[r][j] >= 0 and not (j == whole and r in kept):
                entries.append(old[r][j])
    stack = _let_go(entries, shared, stack)
    width = len(table[0])
    rows = [new[b] + [-1] * (max(held[b], now[b]) - now[b]) + old[b][max(held[b], now[b]):width] for b in range(B)]
    return rows, now, stack, shared, missing, out, copies


def compact(table, held, free, n_free, shared, num_pages):
    """(table, stack, shared, copies): copies a list of (source, target)."""
    stack = set(free[:n_free])
    used = [p for p in range(num_pages) if p not in stack]
    holes = [p for p in range(len(used)) if p in stack]
    high = [p for p in used if p >= len(used)][::-1]
    to = dict(zip(high, holes))
    shared = list(shared)
    for a, b in to.items():
        shared[b], shared[a] = shared[a], 0
    rows = [[to.get(q, q) if j < held[b] else q for j, q in enumerate(r)] for b, r in enumerate(table)]
    return rows, list(range(num_pages - 1, len(used) - 1, -1)), shared, list(zip(high, holes))
