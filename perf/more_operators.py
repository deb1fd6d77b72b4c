"""Generation with beams from a paged cache, as cases that can be timed: rotary positions (forward and backward, and fused with storing
keys and values in the cache), selection over beams and vocabulary, forking of the beams' pages, and turnover of requests with
compaction of the pages.

    own                   False: run() computes the operators in elementary torch operations; True: it calls the framework
    listed()              the cases
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   what a program holds before the call
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


def _framework():
    path = os.path.join(os.getcwd(), "chill-attention_b200")
    if path not in sys.path:
        sys.path.insert(1, path)
    import chill_attention

    return chill_attention


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _rotate(name, dtype, B, H, Hkv, D, L, rotary, axes=1, interleaved=False):
    return _named(name, {"op": "rotate", "dtype": dtype, "B": B, "H": H, "kv_heads": Hkv, "D": D, "len": L, "rotary": rotary, "axes": axes,
                         "interleaved": interleaved})


def _append(name, dtype, B, H, Hkv, D, ctx, N, page, rotary, axes=1, interleaved=False, idle=0):
    return _named(name, {"op": "append", "dtype": dtype, "B": B, "H": H, "kv_heads": Hkv, "D": D, "ctx": ctx, "new": N, "page": page,
                         "rotary": rotary, "axes": axes, "interleaved": interleaved, "idle": idle})


def _select(name, dtype, groups, beams, count, vocab, finished=0.0, first=False):
    return _named(name, {"op": "select", "dtype": dtype, "groups": groups, "beams": beams, "count": count, "vocab": vocab,
                         "finished": finished, "first": first})


def _fork(name, dtype, groups, beams, ctx, page, Hkv, D, layers):
    return _named(name, {"op": "fork", "dtype": dtype, "groups": groups, "beams": beams, "ctx": ctx, "page": page, "kv_heads": Hkv, "D": D,
                         "layers": layers})


def _turnover(name, dtype, B, prompt, ctx, page, Hkv, D, layers):
    return _named(name, {"op": "turnover", "dtype": dtype, "B": B, "prompt": prompt, "ctx": ctx, "page": page, "kv_heads": Hkv, "D": D,
                         "layers": layers})


def listed():
    return [
        # A training step's rotation of a small model in the default precision, forward and backward: all latency.
        _rotate("rotate_small_fp32", "fp32", 1, 4, 2, 64, 257, 64),
        # The same in the framework's benchmark shape.
        _rotate("rotate_train_bf16", "bf16", 8, 16, 16, 128, 4096, 128),
        # Images and text in one sequence: positions of time, height and width, part of the channels turned, neighbouring pairs.
        _rotate("rotate_axes_fp16", "fp16", 3, 32, 8, 128, 5003, 96, axes=3, interleaved=True),
        # The ordinary serving step: one token for each of many requests.
        _append("append_decode_bf16", "bf16", 64, 32, 8, 128, 8192, 1, 64, 128),
        # Chunks of prompts with images.
        _append("append_prompt_fp16", "fp16", 6, 24, 8, 128, 2048, 1000, 16, 128, axes=3, idle=3),
        # The next token of four beams of one request, scores in the default precision.
        _select("select_small_fp32", "fp32", 1, 4, 4, 32000),
        # A batch of requests, twice as many candidates as beams, some beams at their end.
        _select("select_batch_bf16", "bf16", 32, 8, 16, 128000, finished=0.1),
        # Wide beams, a vocabulary of odd size.
        _select("select_wide_fp32", "fp32", 4, 32, 64, 50021),
        # Pages of four beams after a selection, a small model's caches of all layers.
        _fork("fork_small_fp32", "fp32", 1, 4, 700, 16, 4, 64, 4),
        # A large batch with long contexts.
        _fork("fork_batch_bf16", "bf16", 16, 16, 16384, 16, 8, 128, 1),
        # Requests end, those that stay move together, new ones come in: a few requests that share a prompt.
        _turnover("turnover_small_fp16", "fp16", 8, 100, 600, 16, 2, 64, 2),
        # The same for a large batch.
        _turnover("turnover_batch_bf16", "bf16", 96, 500, 4000, 32, 8, 128, 1),
    ]


def _log_int(rng, lo, hi):
    return min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1e-9))))), lo), hi)


def _draw_turn(rng, D):
    """Channels that turn, axes, pairing."""
    rotary = D if rng.random() < 0.6 else 2 * rng.randint(1, D // 2)
    return {"rotary": rotary, "axes": rng.choice([1, 1, 2, 3]) if rotary >= 6 else 1, "interleaved": rng.random() < 0.4}


def draw(rng):
    op, dtype = rng.choice(["rotate", "append", "select", "select", "fork", "turnover"]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    es = _BYTES[dtype]
    if op in ("rotate", "append"):
        Hkv, group, D = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([16, 32, 64, 64, 80, 128, 128, 256])
        B, turn = _log_int(rng, 1, 64), _draw_turn(rng, D)
        row = B * Hkv * (group + 1) * D * es
        if op == "rotate":
            return _rotate(None, dtype, B, Hkv * group, Hkv, D, max(1, min(_log_int(rng, 1, 16384), int(2e8) // row)), **turn)
        N = max(1, min(rng.choice([1, _log_int(rng, 2, 1024)]), int(1e8) // row))
        ctx = max(1, min(_log_int(rng, 1, 100000), int(4e8) // (B * Hkv * D * es)))
        return _append(None, dtype, B, Hkv * group, Hkv, D, ctx, N, rng.choice([8, 16, 16, 32, 48, 64]), idle=rng.choice([0, 0, 3]), **turn)
    if op == "select":
        beams, vocab = _log_int(rng, 1, 32), _log_int(rng, 100, 131072)
        groups = max(1, min(_log_int(rng, 1, 64), int(3e7) // (beams * vocab)))
        return _select(None, dtype, groups, beams, rng.choice([beams, 2 * beams]), vocab, rng.choice([0.0, 0.0, 0.2]), rng.random() < 0.2)
    page, Hkv, D = rng.choice([8, 16, 16, 32, 48, 64]), rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 128])
    page_bytes = page * Hkv * D * es
    if op == "fork":
        groups, beams, ctx = _log_int(rng, 1, 32), rng.randint(2, 16), _log_int(rng, 1, 16384)
        layers = rng.randint(1, 4)
        while groups > 1 and 2 * layers * page_bytes * groups * (ctx // page + 4 * beams) > 5e8:
            groups -= 1
        while ctx > 1 and 2 * layers * page_bytes * groups * (ctx // page + 4 * beams) > 5e8:
            ctx = ctx * 3 // 4
        return _fork(None, dtype, groups, beams, ctx, page, Hkv, D, layers)
    B, ctx, layers = _log_int(rng, 2, 96), _log_int(rng, 16, 8000), rng.randint(1, 3)
    while B > 2 and 2 * layers * page_bytes * B * (ctx // page + 2) > 4e8:
        B -= 1
    while ctx > 16 and 2 * layers * page_bytes * B * (ctx // page + 2) > 4e8:
        ctx = ctx * 3 // 4
    return _turnover(None, dtype, B, rng.randint(0, ctx // 3), ctx, page, Hkv, D, layers)


# ------------------------------------------------------------------------------------------------------------- inputs
def _blocks(tokens, page):
    return (tokens + page - 1) // page


def _spread(count, most):
    """Lengths of `count` requests, the same ones for every seed (in an order of its own)."""
    return [most if b == 0 else max(most // 8, int(most * ((b * 0.6180339887) % 1.0)), 1) for b in range(count)]


def _new_tokens(case):
    return [0 if case["idle"] and b % case["idle"] == 2 else case["new"] - ((7 * b) % (case["new"] // 4 + 1)) for b in range(case["B"])]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(shape, dtype, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _axes(case):
    """Axis of every pair: the pairs in as many runs as there are axes, or with `interleaved` pairs in turn."""
    pairs, A = case["rotary"] // 2, case["axes"]
    return [i % A if case["interleaved"] else i * A // pairs for i in range(pairs)]


def _grid_positions(case, start, count):
    """[axes, batch, count] positions behind `start` [batch] tokens: pictures of 3 frames, 16 x 24 patches each, between stretches of text."""
    A, i = case["axes"], torch.arange(count, device="cuda")
    t = start[:, None].long() + i
    if A == 1:
        return t[None].int()
    picture, inside = t // 2000, t % 2000
    patch = (inside - 400).clamp(0, 3 * 16 * 24 - 1)
    seen = (inside >= 400) & (inside < 400 + 3 * 16 * 24)
    base = picture * 2000 + 400
    parts = (patch // (16 * 24), patch // 24 % 16, patch % 24)
    return torch.stack([torch.where(seen, base + parts[a], t) for a in range(A)]).int()


def _prepare_turn(case, s):
    s["inv_freq"] = (10000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])).float().cuda()
    s["axes"] = _ints(_axes(case)) if case["axes"] > 1 else None


def _prepare_rotate(case, g):
    dtype, B, L, D = _DTYPES[case["dtype"]], case["B"], case["len"], case["D"]
    s = {"case": case}
    _prepare_turn(case, s)
    start = (torch.rand(B, generator=g, device="cuda") * 5000).int()  # packed documents: a batch row begins anywhere
    s["positions"] = _grid_positions(case, start, L) if case["axes"] > 1 else (start[:, None] + torch.arange(L, device="cuda")).int()
    for name, heads in (("q", case["H"]), ("k", case["kv_heads"])):
        s[name] = _normal((B, L, heads, D), dtype, g).transpose(1, 2).requires_grad_()  # as the projection leaves it
        s["g" + name] = _normal((B, heads, L, D), dtype, g)  # as attention's backward leaves it
    return s


def _prepare_append(case, g):
    dtype, B, N, P, Hkv, D = _DTYPES[case["dtype"]], case["B"], case["new"], case["page"], case["kv_heads"], case["D"]
    rows = list(zip(_spread(B, case["ctx"]), _new_tokens(case)))
    width, total = max(_blocks(c + n, P) for c, n in rows) + 1, sum(_blocks(c + n, P) for c, n in rows)
    rows = _ints(rows)[torch.randperm(B, generator=g, device="cuda")]
    lens, new = rows[:, 0].contiguous(), rows[:, 1].contiguous()
    pages = total + total // 8 + 4
    table = _fill_table(_blocks(lens + new, P), width, torch.randperm(pages, generator=g, device="cuda"))
    t = lens[:, None].long() + torch.arange(N, device="cuda")
    page = torch.gather(table, 1, (t // P).clamp(max=width - 1)).long()
    real = torch.arange(N, device="cuda") < new[:, None]
    s = {"case": case, "lens": lens, "new": new, "slots": torch.where(real, page * P + t % P, -1).int(), "chain": torch.where(real, t, 0).int()}
    s["positions"] = torch.where(real, _grid_positions(case, lens, N), 0).int() if case["axes"] > 1 else s["chain"]
    _prepare_turn(case, s)
    s["q"], s["k"], s["v"] = (_normal((B, N, heads, D), dtype, g).transpose(1, 2) for heads in (case["H"], Hkv, Hkv))
    s["k_cache"], s["v_cache"] = (_normal((pages, Hkv, P, D), dtype, g) for _ in range(2))
    return s


def _prepare_select(case, g):
    G, K, V = case["groups"], case["beams"], case["vocab"]
    x = torch.randn((G * K, V), generator=g, device="cuda") * 2.5
    x.masked_fill_(torch.rand((G * K, V), generator=g, device="cuda") < 0.02, -math.inf)  # tokens that may not come
    scores = -40 * torch.rand((G, K), generator=g, device="cuda")
    if case["first"]:
        scores[:, 1:] = -math.inf  # the beams of a request are still one
    s = {"case": case, "logits": x.to(_DTYPES[case["dtype"]]), "scores": scores}
    s["finished"] = torch.rand((G, K), generator=g, device="cuda") < case["finished"] if case["finished"] else None
    s["end"] = V // 3
    return s


def _fill_table(held, width, order):
    """Rows of `held` pages each, taken from `order`."""
    block, first = torch.arange(width, device="cuda"), torch.cumsum(held, 0) - held
    at = (first[:, None] + block).clamp(max=order.numel() - 1)
    return torch.where(block < held[:, None], order[at], -1).int()


def _prepare_pages(s, lens, first, prefix, width, spare, g):
    """Integer tensors of requests of `lens` tokens, whose `prefix` first blocks are those of request `first`, and caches."""
    P = s["case"]["page"]
    B, block = lens.numel(), torch.arange(width, device="cuda")
    held = _blocks(lens, P)
    whose = torch.where(block < prefix[:, None], first[:, None], torch.arange(B, device="cuda")[:, None])  # whose page a block is
    is_own = (whose == torch.arange(B, device="cuda")[:, None]) & (block < held[:, None])
    total = s["total"]
    order = torch.randperm(total + spare, generator=g, device="cuda").int()  # pages in the order they were handed out
    number = (torch.cumsum(is_own.flatten(), 0) - 1).view(B, width).clamp(min=0)
    mine = torch.where(is_own, order[number], -1)
    table = torch.where(block < held[:, None], mine[whose, block], -1).int()
    used = is_own.sum()
    free_at = torch.arange(total + spare, device="cuda")
    shared = torch.zeros(total + spare + 1, dtype=torch.int32, device="cuda")
    shared.scatter_add_(0, torch.where(table >= 0, table, total + spare).flatten().long(), torch.ones(B * width, dtype=torch.int32, device="cuda"))
    n_free = total + spare - used
    s.update(table=table, held=held.int(), n_free=n_free.int().view(1), missing=torch.zeros(1, dtype=torch.int32, device="cuda"),
             free=torch.where(free_at < n_free, order[(free_at + used).clamp(max=total + spare - 1)], -1).int(),
             shared=(shared[:-1] - 1).clamp(min=0))
    Hkv, D, layers = (s["case"][n] for n in ("kv_heads", "D", "layers"))
    s["k_cache"], s["v_cache"] = (_normal((layers, total + spare, Hkv, P, D), _DTYPES[s["case"]["dtype"]], g) for _ in range(2))


def _prepare_fork(case, g):
    G, K, P = case["groups"], case["beams"], case["page"]
    lens = _ints(_spread(G, case["ctx"]))[torch.randperm(G, generator=g, device="cuda")].repeat_interleave(K)
    s = {"case": case, "lens": lens.contiguous(), "total": sum(_blocks(c, P) + 4 * K for c in _spread(G, case["ctx"]))}
    b = torch.arange(G * K, device="cuda")
    apart = (torch.rand(G, generator=g, device="cuda") * 3).long().repeat_interleave(K)  # blocks since the beams parted
    _prepare_pages(s, lens.long(), b // K * K, (lens.long() // P - apart).clamp(min=0), _blocks(case["ctx"], P) + 2, G * K + 8, g)
    s["parents"] = (b // K * K + (torch.rand(G * K, generator=g, device="cuda") * K).long()).int()
    return s


def _prepare_turnover(case, g):
    B, P = case["B"], case["page"]
    lens = _ints(_spread(B, case["ctx"]))[torch.randperm(B, generator=g, device="cuda")]
    s = {"case": case, "total": sum(_blocks(c, P) for c in _spread(B, case["ctx"])), "turn": 0}
    b = torch.arange(B, device="cuda")
    first = b // 4 * 4  # four requests at a time share a prompt
    prefix = torch.minimum(lens, lens[first]).clamp(max=case["prompt"]).long() // P
    _prepare_pages(s, lens.long(), first, prefix, _blocks(case["ctx"], P) + 1, 4, g)
    leaves = [b % 2 == 0, b % 2 == 1]  # the two halves end in turn, and as many requests come in their place
    s["stay"], s["come"] = [torch.where(x, 0, lens) for x in leaves], [torch.where(x, lens, 0) for x in leaves]
    s["stored"] = torch.empty_like(lens)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = {"rotate": _prepare_rotate, "append": _prepare_append, "select": _prepare_select, "fork": _prepare_fork, "turnover": _prepare_turnover}
    return make[case["op"]](case, g)


# -------------------------------------------------------------------------------------------------- the plain forms
def _angles(s):
    """cos and sin, [batch, 1, tokens, pairs]; angles in 64 bits, far positions have large ones."""
    at = s["positions"].double()
    at = at[..., None] if s["axes"] is None else at[s["axes"].long()].permute(1, 2, 0)
    a = at * s["inv_freq"].double()
    return a.cos().float()[:, None], a.sin().float()[:, None]


def _turned(case, x, cos, sin):
    R, x32 = case["rotary"], x.float()
    if case["interleaved"]:
        a, b = x32[..., 0:R:2], x32[..., 1:R:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x32[..., :R // 2], x32[..., R // 2:R]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x32[..., R:]], -1).to(x.dtype)


def _plain_rotate(s):
    with torch.no_grad():
        cos, sin = _angles(s)
        return [_turned(s["case"], s["q"], cos, sin), _turned(s["case"], s["k"], cos, sin),
                _turned(s["case"], s["gq"], cos, -sin), _turned(s["case"], s["gk"], cos, -sin)]


def _plain_append(s):
    cos, sin = _angles(s)
    P, slots = s["case"]["page"], s["slots"].long()
    k = _turned(s["case"], s["k"], cos, sin)
    b, i = (slots >= 0).nonzero(as_tuple=True)
    page, row = slots[b, i] // P, slots[b, i] % P
    s["k_cache"][page, :, row] = k.transpose(1, 2)[b, i]
    s["v_cache"][page, :, row] = s["v"].transpose(1, 2)[b, i]
    return _turned(s["case"], s["q"], cos, sin)


def _plain_select(s):
    """In 64 bits: which of two candidates comes first can hang on the last bits."""
    G, K, M, V = (s["case"][n] for n in ("groups", "beams", "count", "vocab"))
    x, scores = s["logits"].double(), s["scores"].double().view(G * K, 1)
    top = x.amax(1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    c = scores + (x - (top + (x - top).exp().sum(1, keepdim=True).log()))
    c = torch.where((x == -math.inf) | (scores == -math.inf), -math.inf, c)
    if s["finished"] is not None:
        over = s["finished"].view(G * K, 1)
        c = torch.where(over, torch.where(torch.arange(V, device=c.device) == s["end"], scores, -math.inf), c)
    value, at = c.view(G, K * V).sort(stable=True, dim=1, descending=True)
    value, at = value[:, :M], at[:, :M]
    return value.float(), (torch.arange(G, device=c.device)[:, None] * K + at // V).int(), (at % V).int()


def _release(s, table, released, kept):
    """Takes `released` entries off their pages' counts, adds `kept`, and puts pages that nobody holds on the stack, the first on top."""
    free, n_free, shared = s["free"], s["n_free"], s["shared"]
    pages = free.numel()
    page = torch.where(released | (kept != 0), table, pages).flatten().long()
    count = torch.cat([shared, shared.new_zeros(1)]).scatter_add_(0, page, (kept - released.int()).flatten().int())
    index = torch.arange(page.numel(), device=page.device)
    first = torch.full((pages + 1,), page.numel(), device=page.device).scatter_reduce_(0, torch.where(released.flatten(), page, pages), index, "amin")
    lets_go = released.flatten() & (first[page] == index) & (count[page] < 0)
    total = lets_go.sum()
    at = torch.where(lets_go, n_free + total - torch.cumsum(lets_go, 0), pages)
    free.copy_(torch.cat([free, free.new_zeros(1)]).scatter_(0, at, table.flatten())[:-1])
    shared.copy_(count[:-1].clamp(min=0))
    n_free += total.int()


def _plain_fork(s, lens, parents):
    table, held, free, n_free = s["table"], s["held"], s["free"], s["n_free"]
    P, (B, width), pages = s["case"]["page"], table.shape, free.numel()
    block, b = torch.arange(width, device=table.device), torch.arange(B, device=table.device)
    lens = torch.minimum(lens, held * P).long()
    whole, rest = lens // P, lens % P
    old, parent = table.clone(), parents.long()
    children = torch.zeros_like(lens).scatter_add_(0, parent, torch.ones_like(lens))
    first = torch.full_like(lens, B).scatter_reduce_(0, parent, b, "amin")
    last = torch.gather(old, 1, whole.clamp(max=width - 1)[:, None])[:, 0]  # page of the block that has begun
    stays = (rest > 0) & (s["shared"][last.clamp(min=0).long()] == 0)
    # new pages
    take = (rest[parent] > 0) & ~(stays[parent] & (first[parent] == b))
    off = torch.cumsum(take, 0) - 1
    got = take & (off < n_free)
    page = free[(n_free - 1 - off).clamp(0, pages - 1)]
    s["missing"].copy_((take.sum() - n_free).clamp(min=0))
    n_free -= got.sum().int()
    # tables
    here = (rest[parent] > 0) & (got | ~take)
    now = (whole[parent] + here).int()
    entry = torch.where((block == whole[parent][:, None]) & take[:, None], page[:, None], old[parent])
    table.copy_(torch.where(block < now[:, None], entry, torch.where(block < held[:, None], -1, table)))
    # counts
    begin = torch.where(children == 0, 0, torch.where(stays | (rest == 0), _blocks(lens, P), whole))
    inside = block < held[:, None]
    kept = torch.where(inside & (block < whole[:, None]) & (children > 0)[:, None], (children - 1)[:, None], 0).int()
    _release(s, old, inside & (block >= begin[:, None]), kept)
    held.copy_(now)
    # what has to be copied
    at = torch.where(got, torch.cumsum(got, 0) - 1, B)
    source, target, rows = (torch.full((B + 1,), v, dtype=torch.int32, device=table.device) for v in (-1, -1, 0))
    source.scatter_(0, at, last[parent])
    target.scatter_(0, at, page)
    rows.scatter_(0, at, rest[parent].int())
    copies = source[:-1], target[:-1], rows[:-1], got.sum().int().view(1)
    return torch.where(take & ~got, whole[parent] * P, lens[parent]).int(), copies


def _plain_copy(s, copies):
    n = copies[3].item()
    source, target, rows = (x[:n].long() for x in copies[:3])
    fits = torch.arange(s["case"]["page"], device=source.device)[:, None] < rows[:, None, None, None]
    for cache in (s["k_cache"], s["v_cache"]):
        cache[:, target] = torch.where(fits, cache[:, source], cache[:, target])


def _plain_trim(s, lens):
    block, need = torch.arange(s["table"].shape[1], device=lens.device), _blocks(lens, s["case"]["page"])
    back = (block >= need[:, None]) & (block < s["held"][:, None])
    _release(s, s["table"], back, torch.zeros_like(s["table"]))
    s["table"].masked_fill_(back, -1)
    s["held"].copy_(torch.minimum(s["held"], need))


def _plain_compact(s):
    table, free, n_free, shared = s["table"], s["free"], s["n_free"], s["shared"]
    pages = free.numel()
    p = torch.arange(pages, device=free.device)
    is_free = torch.zeros(pages + 1, dtype=torch.bool, device=free.device).scatter_(0, torch.where(p < n_free, free, pages).long(), True)[:-1]
    used = pages - is_free.sum()
    hole, moves = is_free & (p < used), ~is_free & (p >= used)
    room = max(pages // 2, 1)
    source, target, rows = (torch.full((room + 1,), v, dtype=torch.int32, device=free.device) for v in (-1, -1, 0))
    target.scatter_(0, torch.where(hole, torch.cumsum(hole, 0) - 1, room), p.int())
    from_top = torch.cumsum(moves.flip(0), 0).flip(0) - 1
    source.scatter_(0, torch.where(moves, from_top, room), p.int())
    rows.scatter_(0, torch.where(moves, from_top, room), s["case"]["page"])
    to = torch.where(moves, target[from_top.clamp(0, room)], p)
    inside = (torch.arange(table.shape[1], device=free.device) < s["held"][:, None]) & (table >= 0)
    table.copy_(torch.where(inside, to[table.clamp(min=0).long()].int(), table))
    count = torch.cat([torch.where(is_free | moves, 0, shared), shared.new_zeros(1)])
    shared.copy_(count.scatter_(0, torch.where(moves, to, pages), shared)[:-1])
    free.copy_(torch.where(p < pages - used, pages - 1 - p, free).int())
    n_free.copy_((pages - used).int().view(1))
    return source[:-1], target[:-1], rows[:-1], moves.sum().int().view(1)


def _plain_reserve(s, lens, new, N):
    table, held, free, n_free = s["table"], s["held"], s["free"], s["n_free"]
    P, block = s["case"]["page"], torch.arange(table.shape[1], device=lens.device)
    need = _blocks(lens + new, P).clamp(max=table.shape[1])
    take = (need - held).clamp(min=0)
    at = n_free - 1 - ((torch.cumsum(take, 0) - take)[:, None] + block - held[:, None])
    got = (block >= held[:, None]) & (block < need[:, None]) & (at >= 0)
    table.copy_(torch.where(got, free[at.clamp(min=0)], table))
    held += got.sum(1).int()
    s["missing"].copy_((take.sum() - n_free).clamp(min=0))
    n_free -= got.sum().int()
    t = lens[:, None].long() + torch.arange(N, device=lens.device)
    page = torch.gather(table, 1, (t // P).clamp(max=table.shape[1] - 1)).long()
    real = torch.arange(N, device=lens.device) < new[:, None]
    return torch.where(real & (page >= 0), page * P + t % P, -1).int()


# -------------------------------------------------------------------------------------------------------- one pass
def _rotary(s, ca):
    return ca.ChillRotary(s["inv_freq"], s["axes"], s["case"]["interleaved"])


def _held_state(s):
    return {n: s[n] for n in ("table", "held", "free", "n_free", "missing", "shared", "k_cache", "v_cache")}


def run(s):
    case, op = s["case"], s["case"]["op"]
    ca = _framework() if own else None
    if op == "rotate":
        if own:
            out = ca.chill_rotate(s["q"], s["k"], s["positions"], _rotary(s, ca))
            return [*out, *torch.autograd.grad(out, (s["q"], s["k"]), (s["gq"], s["gk"]))]
        return _plain_rotate(s)
    if op == "append":
        if own:
            step = ca.ChillStep(s["lens"], s["new"], s["slots"], s["chain"], None)
            q = ca.chill_rotate_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], step, _rotary(s, ca), s["positions"])
        else:
            q = _plain_append(s)
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "select":
        if own:
            scores, parents, tokens = ca.chill_beam_select(s["logits"], s["scores"], case["count"], finished=s["finished"], end_token=s["end"])
        else:
            scores, parents, tokens = _plain_select(s)
        return {"scores": scores, "parents": parents, "tokens": tokens}
    pages = ca.ChillPages(s["table"], s["held"], s["free"], s["n_free"], s["missing"]) if own else None
    if op == "fork":
        if own:
            lens, copies = ca.chill_pages_fork(pages, s["shared"], s["lens"], s["parents"], case["page"])
            ca.chill_cache_copy(s["k_cache"], s["v_cache"], copies)
        else:
            lens, copies = _plain_fork(s, s["lens"], s["parents"])
            _plain_copy(s, copies)
        return {**_held_state(s), "lens": lens, "copies": list(copies)}
    stay, come = s["stay"][s["turn"]], s["come"][s["turn"]]
    s["turn"] = 1 - s["turn"]
    if own:
        ca.chill_pages_trim(pages, stay, case["page"], shared=s["shared"])
        copies = ca.chill_pages_compact(pages, case["page"], shared=s["shared"])
        ca.chill_cache_copy(s["k_cache"], s["v_cache"], copies)
        slots = ca.chill_pages_reserve(pages, stay, come, case["ctx"], case["page"]).slots
    else:
        _plain_trim(s, stay)
        copies = _plain_compact(s)
        _plain_copy(s, copies)
        slots = _plain_reserve(s, stay, come, case["ctx"])
    return {**_held_state(s), "slots": slots, "copies": list(copies)}


# ------------------------------------------------------------------------------------------- 64 bits, from the definition
def _by_complex(case, x, angle):
    """Channels as complex numbers, times e^(i angle); angle: [batch, tokens, pairs]."""
    R, x = case["rotary"], x.detach().double()
    pairs = [(2 * i, 2 * i + 1) if case["interleaved"] else (i, i + R // 2) for i in range(R // 2)]
    re, im = ([p[n] for p in pairs] for n in (0, 1))
    z = torch.complex(x[..., re], x[..., im]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    y = x.clone()
    y[..., re], y[..., im] = z.real, z.imag
    return y


def _exact_angle(case, s):
    at = s["positions"].view(-1, *s["positions"].shape[-2:])
    freq = s["inv_freq"].double().tolist()
    return torch.stack([at[a].double() * freq[i] for i, a in enumerate(_axes(case))], -1)


def _exact_select(s):
    G, K, M, V = (s["case"][n] for n in ("groups", "beams", "count", "vocab"))
    scores = torch.empty(G, M, dtype=torch.float64, device="cuda")
    for g in range(G):
        best = []
        for k in range(K):
            base, row = s["scores"][g, k].double(), s["logits"][g * K + k].double()
            if s["finished"] is not None and s["finished"][g, k]:
                c = torch.full_like(row, -math.inf)
                c[s["end"]] = base
            elif base == -math.inf or (row == -math.inf).all():
                c = torch.full_like(row, -math.inf)
            else:
                c = base + torch.log_softmax(row, 0)
            best.append(c.sort(descending=True).values[:M])
        scores[g] = torch.cat(best).sort(descending=True).values[:M]
    return {"scores": scores, "parents": None, "tokens": None}


def exact(case, seed):
    if case["op"] in ("fork", "turnover"):
        return None  # whole numbers, and rows that move as they are
    s = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(s)
    angle = _exact_angle(case, s)
    if case["op"] == "rotate":
        return [_by_complex(case, s[n], a) for n, a in (("q", angle), ("k", angle), ("gq", -angle), ("gk", -angle))]
    k_cache, v_cache, P = s["k_cache"].double(), s["v_cache"].double(), case["page"]
    k, slots = _by_complex(case, s["k"], angle), s["slots"].tolist()
    rows = [(b, i, slot) for b, line in enumerate(slots) for i, slot in enumerate(line) if slot >= 0]
    if rows:
        b, i, slot = torch.tensor(rows, device="cuda").T
        k_cache[slot // P, :, slot % P] = k[b, :, i]
        v_cache[slot // P, :, slot % P] = s["v"].double()[b, :, i]
    return {"q": _by_complex(case, s["q"], angle), "k_cache": k_cache, "v_cache": v_cache}


# ------------------------------------------------------------------------------------------------------------ floors
def work(case):
    op, es = case["op"], _BYTES[case["dtype"]]
    if op == "select":
        K, V = case["beams"], case["vocab"]
        values = case["groups"] * K * V * (1 - case["finished"])
        return {"bytes": values * es + case["groups"] * (5 * K + 12 * case["count"]), "flops": 4 * values}
    row = case["kv_heads"] * case["D"] * es  # K or V of one token
    if op == "rotate":
        tokens, heads = case["B"] * case["len"], case["H"] + case["kv_heads"]
        return {"bytes": 4 * tokens * heads * case["D"] * es + 4 * tokens * case["axes"], "flops": 6 * tokens * heads * case["rotary"]}
    if op == "append":
        tokens, heads = sum(_new_tokens(case)), case["H"] + case["kv_heads"]
        return {"bytes": tokens * (2 * case["H"] * case["D"] * es + 4 * row) + 4 * case["B"] * case["new"] * (1 + case["axes"]),
                "flops": 3 * tokens * heads * case["rotary"]}
    P = case["page"]
    if op == "fork":
        G, K = case["groups"], case["beams"]
        blocks = sum(_blocks(c, P) for c in _spread(G, case["ctx"])) * K
        again = G * K * (1 - 1 / K) ** K  # children that are not their parent's first, on average
        rows = sum(c % P for c in _spread(G, case["ctx"])) / G
        return {"bytes": 8 * blocks + 4 * G * K * 8 + 4 * case["layers"] * again * rows * row, "flops": 0}
    lens = _spread(case["B"], case["ctx"])
    halves = [sum(_blocks(c, P) for c in lens[n::2]) for n in (0, 1)]
    return {"bytes": 4 * case["layers"] * min(halves) * P * row + 4 * (4 * sum(halves) + case["B"] * case["ctx"]), "flops": 0}
