"""Plain 64-bit implementation of the paged-cache operators for the tests: Python loops over requests, sets for trees."""
import torch

from .attention_oracle import builtin_mask_dense


def reserve(table, held, free, n_free, lens, new_lens, max_new, page, parents=None):
    """(table, held, n_free, missing, slots, positions, ancestor sets) as Python lists; nothing is changed in place."""
    table, held, free, n_free = [list(r) for r in table], list(held), list(free), n_free
    missing = 0
    for b, (c, n) in enumerate(zip(lens, new_lens)):
        n = min(max(n, 0), max_new)
        need = min(-(-(c + n) // page), len(table[b]))
        while held[b] < need:
            if n_free == 0:
                missing += need - held[b]
                break
            n_free -= 1
            table[b][held[b]] = free[n_free]
            held[b] += 1
    slots, positions, sets = [], [], []
    for b, (c, n) in enumerate(zip(lens, new_lens)):
        n = min(max(n, 0), max_new)
        slot, pos, family = [], [], []
        for i in range(max_new):
            block = (c + i) // page
            p = table[b][block] if block < len(table[b]) else -1
            slot.append(p * page + (c + i) % page if i < n and p >= 0 else -1)
            up = parents[b][i] if parents is not None else i - 1
            family.append(({i} | (family[up] if 0 <= up < i else set())) if i < n else set())
            pos.append(c + len(family[i]) - 1 if i < n else 0)
        slots.append(slot)
        positions.append(pos)
        sets.append(family)
    return table, held, n_free, missing, slots, positions, sets


def trim(table, held, free, n_free, lens, page):
    """(table, held, free stack as far as it is used)."""
    table, held, stack = [list(r) for r in table], list(held), list(free[:n_free])
    back = []
    for b, c in enumerate(lens):
        keep = min(-(-c // page), len(table[b]))
        for j in range(keep, held[b]):
            back.append(table[b][j])
            table[b][j] = -1
        held[b] = min(held[b], keep)
    return table, held, stack + back[::-1]


def attention(q, k_cache, v_cache, table, lens, new_lens, positions, sets, mask, scale, chain):
    """O, LSE (log2) and, for error bounds, per row: the sum of p |v|, the largest |scale q . k| taken over absolute values, the
    number of keys.  Everything on the CPU; q and the caches hold the rounded inputs."""
    B, H, N, D = q.shape
    pages, Hkv, page, _ = k_cache.shape
    qd, kd, vd = q.double(), k_cache.double(), v_cache.double()
    o = torch.zeros(B, H, N, D, dtype=torch.float64)
    lse = torch.zeros(B, H, N, dtype=torch.float64)
    size, most, keys = (torch.zeros(B, H, N, D, dtype=torch.float64), torch.zeros(B, H, N, dtype=torch.float64),
                        torch.zeros(B, H, N, dtype=torch.float64))
    for b in range(B):
        c, n = int(lens[b]), min(max(int(new_lens[b]), 0), N)
        total = min(c + n, table.shape[1] * page)
        place = [(int(table[b, t // page]), t % page) for t in range(total)]
        here = [t for t in range(total) if 0 <= place[t][0] < pages]
        if n == 0:
            continue
        lse[b, :, :n] = -torch.inf
        if not here:
            continue
        pi, ri = torch.tensor([place[t][0] for t in here]), torch.tensor([place[t][1] for t in here])
        k_pos = torch.tensor([t if t < c else (t if chain else int(positions[b][t - c])) for t in here])
        q_pos = torch.tensor([c + i if chain else int(positions[b][i]) for i in range(n)])
        seen = builtin_mask_dense(mask.name, mask.constargs, q_pos, k_pos)
        if not chain:
            related = torch.tensor([[t < c or (t - c) in sets[b][i] for t in here] for i in range(n)])
            seen = seen & related
        for h in range(H):
            hk = h // (H // Hkv)
            k, v = kd[pi, hk, ri], vd[pi, hk, ri]
            x = (qd[b, h, :n] @ k.T) * scale
            x = x.masked_fill(~seen, -torch.inf)
            top = x.amax(1, keepdim=True)
            safe = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
            w = torch.exp(x - safe)
            w = torch.where(seen, w, torch.zeros_like(w))
            s = w.sum(1, keepdim=True)
            w = w / s.clamp(min=1e-300)
            v = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))  # a key that nobody sees may hold anything
            k = torch.where(seen.any(0)[:, None], k, torch.zeros_like(k))
            o[b, h, :n] = w @ v
            lse[b, h, :n] = (safe + torch.log(s))[:, 0] / torch.log(torch.tensor(2.0, dtype=torch.float64))
            lse[b, h, :n] = torch.where(seen.any(1), lse[b, h, :n], torch.full_like(lse[b, h, :n], -torch.inf))
            size[b, h, :n] = w @ v.abs()
            most[b, h, :n] = ((qd[b, h, :n].abs() @ k.abs().T) * scale).amax(1)
            keys[b, h, :n] = seen.sum(1)
    return o, lse, size, most, keys
