"""Serving from a paged cache, as cases that can be timed: pages and slots for new tokens, storing their keys and values,
attention of new tokens (one each, a chunk, or a tree of drafts) over the cache, and keeping the accepted path of a tree.

    own                   False: run() computes the operators in elementary torch operations; True: it calls the framework
    listed()              the cases
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   what a serving program holds before the call
    run(state)            one pass through an operator
    exact(case, seed)     what run() returns, from the definition in 64 bits
    work(case)            bytes and floating-point operations a pass cannot do without

Import it with the repository's root as the working folder.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
#: mask name -> (class of the framework, names of its constants in a case)
_MASKS = {
    "full": ("FullChillMask", ()),
    "causal": ("CausalChillMask", ()),
    "window": ("SlidingWindowChillMask", ("left", "right")),
    "chunkwise": ("ChunkwiseChillMask", ("context", "back")),
    "prefix_lm": ("PrefixLMChillMask", ("prefix",)),
}


def _framework():
    path = os.path.join(os.getcwd(), "chill-attention_b200")
    if path not in sys.path:
        sys.path.insert(1, path)
    import chill_attention

    return chill_attention


def _attend(name, dtype, B, H, Hkv, D, ctx, N, page, mask="causal", tree=False, idle=0, **constants):
    c = {"op": "attend", "dtype": dtype, "B": B, "H": H, "kv_heads": Hkv, "D": D, "ctx": ctx, "new": N, "page": page,
         "mask": mask, "tree": tree, "idle": idle, **constants}
    return c if name is None else {"name": name, **c}


def _pages(name, B, ctx, N, page, tree, idle=0):
    c = {"op": "reserve", "B": B, "ctx": ctx, "new": N, "page": page, "tree": tree, "idle": idle}
    return c if name is None else {"name": name, **c}


def _store(name, op, dtype, B, Hkv, D, ctx, N, page, path=0, idle=0):
    c = {"op": op, "dtype": dtype, "B": B, "kv_heads": Hkv, "D": D, "ctx": ctx, "new": N, "page": page, "path": path,
         "tree": op == "commit", "idle": idle}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # The next token of two short conversations with a small model in the default precision: all latency.
        _attend("decode_small_fp32", "fp32", 2, 8, 4, 64, 300, 1, 16),
        # The ordinary serving step: one token for each of many requests of different lengths, grouped-query heads.
        _attend("decode_batch_gqa_bf16", "bf16", 64, 32, 8, 128, 8192, 1, 64),
        # One request with a very long context: few rows, the keys have to be split over the whole GPU.
        _attend("decode_long_bf16", "bf16", 1, 32, 8, 128, 131072, 1, 128),
        # Verification of a tree of drafted tokens for a batch of requests.
        _attend("tree_gqa_bf16", "bf16", 16, 32, 8, 128, 8000, 64, 64, tree=True),
        # The same for a model with a sliding window and as many kv heads as heads, small pages.
        _attend("tree_window_fp16", "fp16", 32, 12, 12, 64, 5000, 24, 16, mask="window", tree=True, left=1024, right=0),
        # Chunked prompts: a chunk of a long prompt against what is in the cache already.
        _attend("chunk_prompt_bf16", "bf16", 4, 32, 8, 128, 8192, 1024, 64),
        # Pages between two steps (what the last drafts took goes back, the next ones are placed): one token for a few requests.
        _pages("pages_decode", 8, 2000, 1, 16, False),
        # The same for a large batch with draft trees, whose ancestors are worked out too.
        _pages("pages_tree", 256, 32768, 64, 16, True),
        # Keys and values of drafted tokens into the cache.
        _store("append_drafts_fp16", "append", "fp16", 32, 12, 64, 5000, 24, 16),
        # Those of a batch of prompts, tensors as the projections leave them.
        _store("append_prompt_bf16", "append", "bf16", 16, 8, 128, 4096, 2048, 64),
        # Drafts stored and, after their verification, the accepted ones moved together: a small model in the default precision.
        _store("commit_small_fp32", "commit", "fp32", 2, 4, 64, 300, 8, 16, path=4),
        # The same for a large batch with wide trees.
        _store("commit_tree_bf16", "commit", "bf16", 128, 8, 128, 2000, 64, 64, path=9),
    ]


def _log_int(rng, lo, hi):
    return min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1e-9))))), lo), hi)


def _draw_attend(rng):
    dtype, D = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice([32, 64, 64, 128, 128, 128, 256])
    Hkv, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 6, 8])
    kind = rng.choice(["one", "tree", "tree", "chunk"])
    N = 1 if kind == "one" else _log_int(rng, 2, 128) if kind == "tree" else _log_int(rng, 16, 1000)
    ctx, B = _log_int(rng, 1, 100000), _log_int(rng, 1, 64)
    mask = rng.choice(list(_MASKS))
    constants = {"full": {}, "causal": {}, "window": {"left": _log_int(rng, 16, 4096), "right": rng.choice([0, 0, 5])},
                 "chunkwise": {"context": _log_int(rng, 16, 512), "back": rng.randint(0, 8)},
                 "prefix_lm": {"prefix": _log_int(rng, 1, 1000)}}[mask]
    c = _attend(None, dtype, B, Hkv * group, Hkv, D, ctx, N, rng.choice([16, 16, 32, 48, 64, 128]), mask, kind == "tree",
                rng.choice([0, 0, 3]), **constants)
    # no more than the largest listed case costs, in either form
    keys = lambda: c["B"] * (c["ctx"] + c["new"]) * Hkv * D * _BYTES[dtype]  # noqa: E731
    pairs = lambda: c["B"] * c["H"] * c["new"] * (c["ctx"] + c["new"]) * (8 if dtype == "fp32" else 1)  # noqa: E731
    while c["B"] > 1 and (keys() > 2.6e8 or pairs() * D > 5e10 or pairs() > 5e8):
        c["B"] -= 1
    while c["ctx"] > 1 and (keys() > 2.6e8 or pairs() * D > 5e10 or pairs() > 5e8):
        c["ctx"] = c["ctx"] * 3 // 4
    return c


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "reserve", "append", "commit"])
    if op == "attend":
        return _draw_attend(rng)
    page, idle = rng.choice([16, 32, 48, 64, 128]), rng.choice([0, 3])
    if op == "reserve":
        tree = rng.random() < 0.5
        return _pages(None, _log_int(rng, 1, 256), _log_int(rng, 1, 32768), _log_int(rng, 1, 64 if tree else 128), page, tree, idle)
    dtype, Hkv, D = rng.choice(list(_DTYPES)), rng.choice([1, 2, 5, 8, 12]), rng.choice([32, 64, 128, 256])
    if op == "append":
        B, N = _log_int(rng, 1, 64), _log_int(rng, 1, 500)
        N = max(1, min(N, int(6e7) // (B * Hkv * D * _BYTES[dtype])))
        return _store(None, op, dtype, B, Hkv, D, _log_int(rng, 1, 1000), N, page, idle=idle)
    N = _log_int(rng, 2, 64)
    return _store(None, op, dtype, _log_int(rng, 1, 64), Hkv, D, _log_int(rng, 1, 1000), N, page, rng.randint(1, min(N, 12)), idle)


# ------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """(cached, new) tokens of every request, the same ones for every seed (in an order of its own)."""
    B, ctx, N, idle = case["B"], case["ctx"], case["new"], case["idle"]
    rows = []
    for b in range(B):
        share = 1.0 if b == 0 else (b * 0.6180339887) % 1.0
        new = N if b == 0 or N == 1 else N - (7 * b) % (N // 4 + 1)
        rows.append((max(ctx // 8, int(ctx * share)), 0 if idle and b % idle == 2 else new))
    return rows


def _normal(shape, dtype, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, N, P = case["B"], case["new"], case["page"]
    rows = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[torch.randperm(B, generator=g, device="cuda")]
    lens, new = rows[:, 0].contiguous(), rows[:, 1].contiguous()
    held = ((lens + new + P - 1) // P).to(torch.int32)
    width = max((c + n + P - 1) // P for c, n in _lengths(case)) + 1
    total = sum((c + n + P - 1) // P for c, n in _lengths(case))
    spare = total // 8 + 4
    order = torch.randperm(total + spare, generator=g, device="cuda").to(torch.int32)  # pages in the order they were handed out
    first = torch.cumsum(held, 0) - held
    block = torch.arange(width, device="cuda")
    at = (first[:, None] + block).clamp(max=total + spare - 1)
    table = torch.where(block < held[:, None], order[at], -1).to(torch.int32)
    s = {"case": case, "lens": lens, "new": new, "table": table}
    if case["tree"]:  # parent of every drafted token: one of the few before it, or the last cached token (-1)
        back = torch.empty(B, N, device="cuda").exponential_(0.4, generator=g).to(torch.int64)
        node = torch.arange(N, device="cuda")
        s["parents"] = (node - 1 - back).clamp(min=-1).to(torch.int32)
    if case["op"] == "reserve":
        s["held"], s["n_free"] = held, torch.tensor([spare], dtype=torch.int32, device="cuda")
        s["missing"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["free"] = torch.cat([order[total:], torch.full((total,), -1, dtype=torch.int32, device="cuda")])
        return s
    dtype, Hkv, D = _DTYPES[case["dtype"]], case["kv_heads"], case["D"]
    s["k_cache"], s["v_cache"] = (_normal((total + spare, Hkv, P, D), dtype, g) for _ in range(2))
    s["slots"], s["positions"], s["ancestors"] = _plan(table, lens, new, N, P, s.get("parents"))
    if case["op"] == "attend":
        s["q"] = _normal((B, N, case["H"], D), dtype, g).transpose(1, 2)  # as the projection leaves it
        s["scale"] = D ** -0.5
        return s
    s["k"], s["v"] = (_normal((B, N, Hkv, D), dtype, g).transpose(1, 2) for _ in range(2))
    if case["op"] == "commit":  # the accepted drafts: an increasing run of tokens
        A = case["path"]
        s["accepted"] = (torch.rand(B, generator=g, device="cuda") * (A + 1)).to(torch.int32).minimum(new)
        picked = torch.rand(B, N, generator=g, device="cuda").masked_fill(torch.arange(N, device="cuda") >= new[:, None], 2.0)
        chosen = picked.argsort(1).argsort(1) < s["accepted"][:, None]
        s["path"] = torch.where(chosen, torch.arange(N, device="cuda"), N).sort(1).values[:, :A].to(torch.int32)
    return s


# -------------------------------------------------------------------------------------------------- the plain forms
def _plan(table, lens, new, N, P, parents):
    """Slots, positions and ancestor bits of the new tokens."""
    B, width = table.shape
    i = torch.arange(N, device=lens.device)
    real = i < new[:, None]
    t = lens[:, None].long() + i
    page = torch.gather(table, 1, (t // P).clamp(max=width - 1)).long()
    slots = torch.where(real & (page >= 0) & (t // P < width), page * P + t % P, -1).to(torch.int32)
    if parents is None:
        return slots, torch.where(real, t, 0).to(torch.int32), None
    rooted = (parents < 0) | (parents >= i)
    edge = ((parents[:, :, None] == i) & ~rooted[:, :, None]) | (i[:, None] == i)
    twice = lambda m: ((m @ m) > 0).float()  # noqa: E731
    reach = twice(twice(twice(twice(twice(twice(twice(edge.float()))))))) > 0  # up to 128 tokens deep
    positions = torch.where(real, lens[:, None] + reach.sum(2) - 1, 0).to(torch.int32)
    words = (N + 31) // 32
    bits = torch.nn.functional.pad((reach & real[:, :, None]).long(), (0, words * 32 - N)).view(B, N, words, 32)
    word = (bits << torch.arange(32, device=lens.device)).sum(3)
    return slots, positions, torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)


def _reserve(s):
    table, held, free, n_free, lens, new = (s[n] for n in ("table", "held", "free", "n_free", "lens", "new"))
    N, P = s["case"]["new"], s["case"]["page"]
    block = torch.arange(table.shape[1], device=lens.device)
    # pages behind the cached tokens go back, the first request's on top
    keep = (lens + P - 1) // P
    give = (held - keep).clamp(min=0)
    at = n_free + give.sum() - 1 - ((torch.cumsum(give, 0) - give)[:, None] + block - keep[:, None])
    back = (block >= keep[:, None]) & (block < held[:, None])
    spill = torch.cat([free, free.new_empty(1)])
    spill.scatter_(0, torch.where(back, at, free.numel()).flatten(), table.flatten())
    free.copy_(spill[:-1])
    table.masked_fill_(back, -1)
    held.copy_(torch.minimum(held, keep))
    n_free += give.sum().int()
    # and the new tokens' pages are taken from there
    need = ((lens + new + P - 1) // P).clamp(max=table.shape[1])
    take = (need - held).clamp(min=0)
    at = n_free - 1 - ((torch.cumsum(take, 0) - take)[:, None] + block - held[:, None])
    got = (block >= held[:, None]) & (block < need[:, None]) & (at >= 0)
    table.copy_(torch.where(got, free[at.clamp(min=0)], table))
    held += got.sum(1).int()
    s["missing"].copy_((take.sum() - n_free).clamp(min=0))
    n_free -= got.sum().int()
    return _plan(table, lens, new, N, P, s.get("parents"))


def _append(s):
    P = s["case"]["page"]
    slots = s["slots"].long()
    rows = (slots >= 0).nonzero()
    page, row = slots[rows[:, 0], rows[:, 1]] // P, slots[rows[:, 0], rows[:, 1]] % P
    s["k_cache"][page, :, row] = s["k"].transpose(1, 2)[rows[:, 0], rows[:, 1]]
    s["v_cache"][page, :, row] = s["v"].transpose(1, 2)[rows[:, 0], rows[:, 1]]


def _commit(s):
    P, lens = s["case"]["page"], s["lens"].long()
    j = torch.arange(s["path"].shape[1], device=lens.device)
    rows = (j < s["accepted"][:, None]).nonzero()
    b, j = rows[:, 0], rows[:, 1]
    source, target = lens[b] + s["path"][b, j], lens[b] + j
    p0, p1 = s["table"][b, source // P].long(), s["table"][b, target // P].long()
    s["k_cache"][p1, :, target % P] = s["k_cache"][p0, :, source % P]
    s["v_cache"][p1, :, target % P] = s["v_cache"][p0, :, source % P]
    return s["lens"] + s["accepted"]


def _visible(case, p, t):
    """Whether a query at position p may see a key at position t."""
    if case["mask"] == "full":
        return (t == t) & (p == p)
    if case["mask"] == "causal":
        return p >= t
    if case["mask"] == "window":
        return (t >= p - case["left"]) & (t <= p + case["right"])
    if case["mask"] == "chunkwise":
        back = p // case["context"] - t // case["context"]
        return (back >= 0) & (back <= case["back"])
    return (t < case["prefix"]) | (p >= t)


def _attention(s):
    case, lens, new, q = s["case"], s["lens"].long(), s["new"].long(), s["q"]
    B, H, N, D = q.shape
    Hkv, P = case["kv_heads"], case["page"]
    T = s["table"].shape[1] * P
    k, v = (s[n][s["table"].clamp(min=0).long()].transpose(1, 2).reshape(B, Hkv, T, D).float() for n in ("k_cache", "v_cache"))
    t = torch.arange(T, device=q.device)
    node = t - lens[:, None]  # number of a key among the new tokens
    there = node < new[:, None]
    if s["ancestors"] is None:
        seen = _visible(case, s["positions"][:, :, None], t) & there[:, None, :]
    else:
        i = node.clamp(0, N - 1)
        key_at = torch.where(node < 0, t, torch.gather(s["positions"].long(), 1, i))
        word = torch.gather(s["ancestors"], 2, (i // 32)[:, None, :].expand(B, N, T))
        related = (node < 0)[:, None, :] | ((word >> (i % 32)[:, None, :]) & 1).bool()
        seen = _visible(case, s["positions"][:, :, None], key_at[:, None, :]) & related & there[:, None, :]
    real = torch.arange(N, device=q.device) < new[:, None]
    seen = (seen & real[:, :, None])[:, None, None]
    x = q.reshape(B, Hkv, H // Hkv, N, D).float().flatten(2, 3) @ k.transpose(2, 3)
    x = (x.view(B, Hkv, H // Hkv, N, T) * (s["scale"] * math.log2(math.e))).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x = torch.exp2(x.sub_(top))
    total = x.sum(-1, keepdim=True)
    o = (x.flatten(2, 3) @ v).view(B, Hkv, H // Hkv, N, D) / total.clamp(min=1e-30)
    lse = torch.where(real[:, None, None], (top + torch.log2(total)).squeeze(-1), 0.0)
    return o.view(B, H, N, D).to(q.dtype), lse.view(B, H, N)


# -------------------------------------------------------------------------------------------------------- one pass
def _step(s, ca):
    return ca.ChillStep(s["lens"], s["new"], s["slots"], s["positions"], s["ancestors"])


def run(s):
    case, op = s["case"], s["case"]["op"]
    ca = _framework() if own else None
    if op == "reserve":
        if own:
            pages = ca.ChillPages(s["table"], s["held"], s["free"], s["n_free"], s["missing"])
            ca.chill_pages_trim(pages, s["lens"], case["page"])
            step = ca.chill_pages_reserve(pages, s["lens"], s["new"], case["new"], case["page"], parents=s.get("parents"))
            slots, positions, ancestors = step.slots, step.positions, step.ancestors
        else:
            slots, positions, ancestors = _reserve(s)
        return {"table": s["table"], "held": s["held"], "free": s["free"], "n_free": s["n_free"], "missing": s["missing"],
                "slots": slots, "positions": positions, "ancestors": ancestors}
    if op == "attend":
        if own:
            cls, names = _MASKS[case["mask"]]
            mask = getattr(ca, cls)(*[case[n] for n in names])
            return ca.chill_attention_cached(s["q"], s["k_cache"], s["v_cache"], s["table"], _step(s, ca), mask,
                                             sm_scale=s["scale"], return_lse=True)
        return _attention(s)
    out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if own:
        ca.chill_cache_append(s["k_cache"], s["v_cache"], s["k"], s["v"], s["slots"])
        if op == "commit":
            out["lens"] = ca.chill_cache_commit(s["k_cache"], s["v_cache"], s["table"], _step(s, ca), s["path"], s["accepted"])
    else:
        _append(s)
        if op == "commit":
            out["lens"] = _commit(s)
    return out


# ------------------------------------------------------------------------------------------- 64 bits, from the definition
def _family(parents, n):
    """Ancestors of every drafted token with itself, as sets, one request."""
    sets = []
    for i in range(n):
        p = parents[i]
        sets.append({i} | (sets[p] if 0 <= p < i else set()))
    return sets


def exact(case, seed):
    if case["op"] == "reserve":
        return None  # whole numbers
    s = prepare(case, seed)
    lens, new, table = s["lens"].tolist(), s["new"].tolist(), s["table"].tolist()
    P, N = case["page"], case["new"]
    place = lambda b, t: (table[b][t // P], t % P)  # noqa: E731
    if case["op"] != "attend":
        pools = {}
        for name in ("k", "v"):
            pool, rows = s[name + "_cache"].double(), s[name].double()
            where, what = [], []
            for b, (c, n) in enumerate(zip(lens, new)):
                order = list(range(n))
                if case["op"] == "commit":  # after the drafts are stored, row j takes what draft path[j] has
                    a = s["accepted"][b].item()
                    order[:a] = s["path"][b, :a].tolist()
                where += [place(b, c + j) for j in range(n)]
                what += [(b, j) for j in order]
            if where:
                where, what = torch.tensor(where, device=pool.device), torch.tensor(what, device=pool.device)
                pool[where[:, 0], :, where[:, 1]] = rows[what[:, 0], :, what[:, 1]]
            pools[name + "_cache"] = pool
        return {**pools, **({"lens": None} if case["op"] == "commit" else {})}
    B, H, _, D = s["q"].shape
    Hkv = case["kv_heads"]
    o = torch.zeros(B, H, N, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, H, N, dtype=torch.float64, device="cuda")
    for b, (c, n) in enumerate(zip(lens, new)):
        if n == 0:
            continue
        slot = torch.tensor([place(b, t) for t in range(c + n)], device="cuda")
        k, v = (s[m][slot[:, 0], :, slot[:, 1]].transpose(0, 1).double() for m in ("k_cache", "v_cache"))
        where = torch.arange(c + n, device="cuda")
        related = None
        if case["tree"]:
            family = _family(s["parents"][b].tolist(), n)
            depth = torch.tensor([len(f) - 1 for f in family], device="cuda")
            where = torch.cat([where[:c], c + depth])
            related = torch.zeros(n, c + n, dtype=torch.bool)
            related[:, :c] = True
            for i, f in enumerate(family):
                related[i, [c + j for j in f]] = True
            related = related.cuda()
        seen = _visible(case, where[c:, None], where[None, :])
        seen = seen if related is None else seen & related
        for h in range(Hkv):  # the heads that share a kv head
            heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
            x = torch.einsum("gid,td->git", s["q"][b, heads, :n].double(), k[h]) * s["scale"]
            x = x.masked_fill(~seen, -math.inf)
            lse[b, heads, :n] = torch.logsumexp(x, -1) / math.log(2.0)
            o[b, heads, :n] = torch.softmax(x, -1).nan_to_num(0.0) @ v[h]
    return o, lse


# ------------------------------------------------------------------------------------------------------------ floors
def work(case):
    rows, N, P = _lengths(case), case["new"], case["page"]
    tokens = sum(n for _, n in rows)
    B = case["B"]
    if case["op"] == "reserve":
        turned = sum((c + n + P - 1) // P - (c + P - 1) // P for c, n in rows)  # pages given back and taken again
        per_token = 4 * (2 + (1 + (N + 31) // 32 if case["tree"] else 0))
        return {"bytes": B * (4 * 5 + N * per_token) + turned * 16, "flops": 0}
    row = case["kv_heads"] * case["D"] * _BYTES[case["dtype"]]  # K or V of one token
    if case["op"] == "append":
        return {"bytes": 4 * tokens * row + 4 * B * N, "flops": 0}
    if case["op"] == "commit":
        return {"bytes": 4 * (tokens + B * case["path"] / 2) * row + 4 * B * (N + case["path"] + 4), "flops": 0}
    keys = pairs = 0
    for c, n in rows:
        if n == 0:
            continue
        first = 0  # first cached key that the new tokens see
        if case["mask"] == "window":
            first = max(0, c - case["left"])
        elif case["mask"] == "chunkwise":
            first = max(0, (c // case["context"] - case["back"]) * case["context"])
        keys += c - min(first, c) + n
        among = min(n, 8) if case["tree"] else (n + 1) / 2
        pairs += n * (c - min(first, c) + among)
    es = _BYTES[case["dtype"]]
    return {"bytes": 2 * keys * row + tokens * case["H"] * (2 * case["D"] * es + 4) + 4 * B * (2 + N),
            "flops": 4 * case["D"] * case["H"] * pairs}
