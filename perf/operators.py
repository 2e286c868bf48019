"""What the operators of an attention step over a 4-bit paged cache are measured on.

A program that serves a block-quantised model keeps the keys and values of its requests in pages of
Q4_0 blocks.  Each step it works out which pages and slots the new tokens get (`plan`), rotates the
queries and keys (`rope`), quantises the new keys and values into their slots (`store`) and attends
over each request's pages (`attention`).  Head sizes and counts are those of the layers that the
benchmark has (4096 = 32 heads of 128) and generic ones around them.

`own` chooses between the plain forms (elementary torch operations in 32 bits) and the framework.

The cache is a uint8 tensor (pages, kv heads, groups, 18 * D): a page holds 16 * groups tokens, and a
group is 16 tokens of one head.  With nb = D / 32 blocks per row, a group holds
  [0, 8D)    key quants:   word (half, g, t, b) = bytes 4t..4t+3 of block b of token g + 8 * half
  [8D, 16D)  value quants: word (half, g, t, b) = bytes 2g, 2g+1 of block b of token 2t + 8 * half,
                           then the same bytes of the token after it
  [16D, 17D) key scales:   fp16 (token, b)
  [17D, 18D) value scales: fp16 (token, b)
where half < 2, g < 8, t < 4, and a block's byte j holds element j in its low and element j + 16 in its
high nibble, each plus 8: a Q4_0 block's 16 quant bytes.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _tc():
    import importlib

    return importlib.import_module("tianchen-rv_b200")


def listed():
    return [
        # Decode for eight requests: queries and keys of one token each are rotated in one call.
        {"name": "rope_decode_8", "op": "rope", "tokens": 8, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "halves": False, "scaling": "none", "far": 4096, "inverse": False, "type": "f32"},
        # A prompt batch of a long-context model: positions of up to a million, frequencies blended for it.
        {"name": "rope_prompt_8192_far", "op": "rope", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "halves": True, "scaling": "yarn", "far": 1 << 20, "inverse": False, "type": "bf16"},
        # Fine-tuning: the gradient of a rotation of half of each head, over sequences of 2047 tokens.
        {"name": "rope_gradient_2047_partial", "op": "rope", "tokens": 2047, "heads": 32, "kv_heads": 32, "dim": 128,
         "rot": 64, "halves": False, "scaling": "none", "far": 2047, "inverse": True, "type": "f32"},
        # A decode step of 64 requests: one slot each, now and then a new page.
        {"name": "plan_decode_64", "op": "plan", "requests": 64, "page": 32, "context": 4096, "new": 1, "idle": 0.0},
        # A mixed step of 1000 requests, some with a prompt, most with a token, some with nothing to add.
        {"name": "plan_mixed_1000", "op": "plan", "requests": 1000, "page": 16, "context": 8192, "new": 512, "idle": 0.2},
        # The new keys and values of a decode step of 64 requests.
        {"name": "store_decode_64", "op": "store", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 32, "run": 1,
         "type": "f32"},
        # Those of a batch of prompts: runs of neighbouring slots that begin and end anywhere.
        {"name": "store_prompt_8191", "op": "store", "tokens": 8191, "kv_heads": 8, "dim": 128, "page": 32, "run": 700,
         "type": "bf16"},
        # One request, a short context: what one user alone waits for.
        {"name": "attention_single_777", "op": "attention", "requests": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "context": 777, "ragged": False, "new": 1, "window": 0, "type": "f32"},
        # A full decode batch, contexts of all lengths up to 8191.
        {"name": "attention_decode_64", "op": "attention", "requests": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "context": 8191, "ragged": True, "new": 1, "window": 0, "type": "bf16"},
        # Two very long contexts: the work has to be split along them.
        {"name": "attention_long_131072", "op": "attention", "requests": 2, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "context": 131072, "ragged": False, "new": 1, "window": 0, "type": "f16"},
        # Five drafted tokens of each of 16 requests are scored in one pass.
        {"name": "attention_draft_16x5", "op": "attention", "requests": 16, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "context": 4095, "ragged": True, "new": 5, "window": 0, "type": "f32"},
        # A batch of prompts of up to 2048 tokens behind contexts of up to 2048.
        {"name": "attention_prompt_4x2048", "op": "attention", "requests": 4, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "context": 4096, "ragged": True, "new": 2048, "window": 0, "type": "bf16"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("rope", "plan", "store", "attention", "attention", "attention"))
    kind = rng.choice(("f32", "f16", "bf16"))
    if op == "rope":
        dim = rng.choice((64, 96, 128, 256))
        kv = rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 2, 4, 7))
        most = max(1, (8192 * 40 * 128) // (dim * (heads + kv)) // (2 if kind == "f32" else 1))
        return {"op": op, "tokens": _log(rng, 1, min(8192, most)), "heads": heads, "kv_heads": kv, "dim": dim,
                "rot": rng.choice((dim, dim, dim // 2, dim // 4)), "halves": rng.random() < 0.5,
                "scaling": rng.choice(("none", "linear", "yarn", "bands")), "far": _log(rng, 64, 1 << 20),
                "inverse": rng.random() < 0.4, "type": kind}
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 1000), "page": rng.choice((16, 32, 64)),
                "context": _log(rng, 16, 8192), "new": _log(rng, 1, 512), "idle": rng.choice((0.0, 0.1, 0.5))}
    if op == "store":
        dim, kv = rng.choice((64, 96, 128, 256)), rng.choice((1, 2, 4, 8, 32))
        return {"op": op, "tokens": _log(rng, 1, min(8191, 8191 * 8 * 128 // (2 * dim * kv))), "kv_heads": kv, "dim": dim,
                "page": rng.choice((16, 32, 64)), "run": _log(rng, 1, 1000), "type": kind}
    while True:
        kv = rng.choice((1, 2, 4, 8, 8, 32))
        case = {"op": op, "requests": _log(rng, 1, 96), "heads": kv * rng.choice((1, 2, 4, 4, 7, 8)), "kv_heads": kv,
                "dim": rng.choice((64, 96, 128, 128, 256)), "page": rng.choice((16, 32, 64)),
                "context": _log(rng, 17, 65536), "ragged": rng.random() < 0.7,
                "new": rng.choice((1, 1, 1, 3, 4, _log(rng, 2, 16), _log(rng, 17, 1024))),
                "window": rng.choice((0, 0, 0, 200, 1024)), "type": kind}
        case["new"] = min(case["new"], case["context"])
        w = work(case)
        padded = case["requests"] * case["context"]  # what the plain form has in memory
        if (w["flops"] <= 1.2e11 and w["bytes"] <= 3e8 and padded * kv * case["dim"] <= 1 << 29 and case["heads"] <= 64
                and padded * case["new"] * case["heads"] <= 1 << 29):
            return case


# ------------------------------------------------------------------ what the cases' lengths are


def _lengths(case):
    """[(tokens in the cache before the step, tokens added by it)] of each request: by the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, most, new = case["requests"], case["context"], case["new"]
    if case["op"] == "plan":
        # one request in sixteen brings a prompt; the others go on by one token
        return [(rng.randrange(0, most + 1), 0 if rng.random() < case["idle"] else rng.randint(1, new) if rng.random() < 0.0625 or new < 8 else 1)
                for _ in range(n)]
    out = []
    for i in range(n):
        total = rng.randint(max(new, most // 8), most) if case["ragged"] and i else most
        mine = new if not case["ragged"] or new < 16 else max(1, min(total, rng.randint(new // 2, new) if i else new))
        out.append((total - mine, mine))
    return out


def _row_bytes(case):
    return case["dim"] * 9 // 16


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * SIZE[case["type"]] + 4 * case["tokens"], "flops": 3 * n}
    if op == "plan":
        lens = _lengths(case)
        pages = sum(-(-(c + m) // case["page"]) - -(-c // case["page"]) for c, m in lens)
        return {"bytes": 8 * len(lens) + 8 * len(lens) + 16 * sum(m for _, m in lens) + 8 * pages, "flops": sum(m for _, m in lens)}
    if op == "store":
        n = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": n * (SIZE[case["type"]] + 4) + 2 * n * 9 // 16 + 8 * case["tokens"], "flops": 4 * n}
    keys = pairs = rows = 0
    for c, m in _lengths(case):
        first = c if not case["window"] else min(c, case["window"] - 1)  # what the first new token sees before it
        keys += m + first
        rows += m
        pairs += m * first + m * (m + 1) // 2 if not case["window"] else sum(min(case["window"], c + i + 1) for i in range(m))
    size = SIZE[case["type"]]
    return {"bytes": 2 * keys * case["kv_heads"] * _row_bytes(case) + 2 * rows * case["heads"] * case["dim"] * size,
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, shape, kind, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(TYPES[kind])


def _ints(values, kind=torch.int32):
    return torch.tensor(values, dtype=kind, device="cuda")


def _frequencies(case):
    """Angle per position of each pair, in 64 bits, and the factor on the rotated values.

    linear: all positions 8 times closer.  yarn: pairs that turn more than 32 times within the trained
    8192 positions stay, those that turn less than once are 16 times slower, a ramp over the pair index
    between.  bands: the same idea on the wave length, with a smooth ramp between 8192 / 4 and 8192."""
    rot = case["rot"]
    base = 10000.0
    f = torch.pow(torch.tensor(base, dtype=torch.float64), -torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    magnitude = 1.0
    if case["scaling"] == "linear":
        f = f / 8.0
    elif case["scaling"] == "yarn":
        at = lambda turns: rot * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(0.0, math.floor(at(32.0))), min(rot - 1.0, math.ceil(at(1.0)))
        keep = 1.0 - ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        f = f * keep + f / 16.0 * (1.0 - keep)
        magnitude = 0.1 * math.log(16.0) + 1.0
    elif case["scaling"] == "bands":
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1.0) / 3.0).clamp(0.0, 1.0)
        f = f * keep + f / 8.0 * (1.0 - keep)
    return f.cuda(), magnitude


def _cache(gen, pages, kv_heads, page, dim):
    """Pages as a running program has them: quants and scales of ordinary keys and values everywhere."""
    c = torch.randint(0, 256, (pages, kv_heads, page // 16, 18 * dim), generator=gen, device="cuda", dtype=torch.uint8)
    d = torch.rand((pages, kv_heads, page // 16, dim), generator=gen, device="cuda") * 0.3 + 0.05
    d = torch.where(torch.rand(d.shape, generator=gen, device="cuda") < 0.5, -d, d).to(torch.float16)
    c[..., 16 * dim:] = d.view(torch.uint8)
    return c


def prepare(case, seed):
    gen, op = _gen(seed), case["op"]
    state = dict(case)
    if op == "rope":
        state["freqs"], state["magnitude"] = _frequencies(case)
        state["q"] = _normal(gen, (case["tokens"], case["heads"], case["dim"]), case["type"])
        state["k"] = _normal(gen, (case["tokens"], case["kv_heads"], case["dim"]), case["type"])
        state["positions"] = torch.randint(0, case["far"], (case["tokens"],), generator=gen, device="cuda", dtype=torch.int32)
        return state
    if op == "plan":
        lens = _lengths(case)
        page, n = case["page"], len(lens)
        width = max(1, -(-(case["context"] + case["new"]) // page))
        held = _ints([-(-c // page) for c, _ in lens])
        pages = n * (width + 1)
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        # requests hold the pages at the front of the shuffled order, the free list is the rest
        first = torch.cumsum(held, 0) - held
        column = torch.arange(width, device="cuda")
        table = torch.where(column[None] < held[:, None], order[(first[:, None] + column[None]).clamp(max=pages - 1)], -1)
        used = sum(-(-c // page) for c, _ in lens)
        state.update(context_lens=_ints([c for c, _ in lens]), new_lens=_ints([m for _, m in lens]), width=width,
                     table=table.to(torch.int32).contiguous(), free=order[used:].contiguous(), rows=sum(m for _, m in lens) + 7,
                     free_count=_ints([pages - used]))
        return state
    if op == "store":
        n, page = case["tokens"], case["page"]
        pages = -(-2 * n // page) + 2
        # runs of neighbouring slots, each at a place of its own; a run of one is a decode step
        run, space = case["run"], pages * page
        if run == 1:
            slots = torch.randperm(space, generator=gen, device="cuda")[:n]
        else:
            start = int(torch.randint(0, space - n, (1,), generator=gen, device="cuda"))
            at = torch.arange(n, device="cuda") + start
            blocks = torch.randperm(-(-n // run), generator=gen, device="cuda")  # the runs in another order
            slots = at[torch.argsort(blocks[torch.arange(n, device="cuda") // run], stable=True)]
        slots = slots.to(torch.int64).contiguous()
        slots[n // 2] = -1 if n > 4 else slots[n // 2]  # a padding row
        state.update(slots=slots, cache=_cache(gen, pages, case["kv_heads"], page, case["dim"]),
                     k=_normal(gen, (n, case["kv_heads"], case["dim"]), case["type"]),
                     v=_normal(gen, (n, case["kv_heads"], case["dim"]), case["type"], 0.3))
        return state
    lens = _lengths(case)
    page = case["page"]
    width = -(-case["context"] // page)
    held = [-(-(c + m) // page) for c, m in lens]
    pages = sum(held) + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    h = _ints(held)
    first = torch.cumsum(h, 0) - h
    column = torch.arange(width, device="cuda")
    table = torch.where(column[None] < h[:, None], order[(first[:, None] + column[None]).clamp(max=pages - 1)], 0).to(torch.int32).contiguous()
    rows = [0]
    for _, m in lens:
        rows.append(rows[-1] + m)
    state.update(cache=_cache(gen, pages, case["kv_heads"], page, case["dim"]), table=table,
                 kv_lens=_ints([c + m for c, m in lens]), first_rows=_ints(rows), most=max(m for _, m in lens),
                 q=_normal(gen, (rows[-1], case["heads"], case["dim"]), case["type"]), scale=case["dim"] ** -0.5)
    return state


# ------------------------------------------------------------------ plain forms


def _rotate_plain(x, s):
    rot, half = s["rot"], s["rot"] // 2
    angle = s["positions"].to(torch.float64)[:, None] * s["freqs"][None]
    cos = (torch.cos(angle) * s["magnitude"]).to(torch.float32)[:, None]
    sin = (torch.sin(angle) * (-s["magnitude"] if s["inverse"] else s["magnitude"])).to(torch.float32)[:, None]
    v = x[..., :rot].to(torch.float32)
    a, b = (v[..., :half], v[..., half:]) if s["halves"] else (v[..., 0::2], v[..., 1::2])
    lo, hi = a * cos - b * sin, a * sin + b * cos
    y = torch.cat((lo, hi), -1) if s["halves"] else torch.stack((lo, hi), -1).flatten(-2)
    return torch.cat((y.to(x.dtype), x[..., rot:]), -1)


def _plan_plain(s):
    page, rows, width = s["page"], s["rows"], s["width"]
    ctx, new = s["context_lens"].to(torch.int64), s["new_lens"].to(torch.int64)
    n = ctx.numel()
    kv = ctx + new
    held, need = (ctx + page - 1) // page, (kv + page - 1) // page
    take = need - held
    total, pages, free = new.sum(), take.sum(), s["free_count"][0].to(torch.int64)
    status = torch.where(pages > free, 1, 0)
    status = torch.where((need > width).any(), 2, status)
    status = torch.where(total > rows, 3, status)
    status = torch.where(((ctx < 0) | (new < 0)).any(), 4, status)
    ok = status == 0
    ends = torch.cumsum(new, 0)
    before = torch.cumsum(take, 0) - take
    column = torch.arange(width, device=ctx.device)[None]
    rank = free - 1 - (before[:, None] + column - held[:, None])
    fresh = ok & (column >= held[:, None]) & (column < need[:, None])
    at = rank.clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][at].to(torch.int64), s["table"].to(torch.int64))
    row = torch.arange(rows, device=ctx.device)
    of = torch.searchsorted(ends, row, right=True)
    live = ok & (row < total)
    of = torch.where(live, of, 0).clamp(max=n - 1)
    position = torch.where(live, ctx[of] + row - (ends - new)[of], 0)
    slot = torch.where(live, table[of, (position // page).clamp(max=width - 1)] * page + position % page, -1)
    first = torch.where(ok, torch.cat((ends.new_zeros(1), ends)), 0)
    info = torch.stack((status, torch.where(ok, total, 0), torch.where(ok, pages, 0), free - torch.where(ok, pages, 0)))
    i32 = torch.int32
    return (first.to(i32), torch.where(ok, kv, ctx).to(i32), slot, position.to(i32), torch.where(live, of, -1).to(i32),
            info.to(i32), table.to(i32))


def _unpack_plain(groups, dim):
    """Groups (..., 18 * dim) of bytes -> keys and values (..., 16, dim) in 32 bits."""
    lead, nb = groups.shape[:-1], dim // 32
    k = groups[..., :8 * dim].reshape(*lead, 2, 8, 4, nb, 4).movedim(-3, -2).reshape(*lead, 16, nb, 16)
    v = groups[..., 8 * dim:16 * dim].reshape(*lead, 2, 8, 4, nb, 2, 2)
    m = len(lead)
    v = v.permute(*range(m), m, m + 2, m + 4, m + 3, m + 1, m + 5).reshape(*lead, 16, nb, 16)
    d = groups[..., 16 * dim:].contiguous().view(torch.float16).to(torch.float32).reshape(*lead, 2, 16, nb, 1)
    both = []
    for quants, scale in ((k, d[..., 0, :, :, :]), (v, d[..., 1, :, :, :])):
        values = torch.cat((quants & 15, quants >> 4), -1).to(torch.float32) - 8.0
        both.append((values * scale).reshape(*lead, 16, dim))
    return both


def _quantise_plain(x):
    """(..., dim) -> quant bytes (..., nb, 16) and fp16 scales (..., nb): the scale is the first value of largest magnitude over -8."""
    x = x.to(torch.float32).unflatten(-1, (-1, 32))
    top = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    d = top / -8.0
    inverse = torch.where(d != 0, 1.0 / d, 0.0)
    q = (x * inverse + 8.5).to(torch.int32).clamp(max=15).to(torch.uint8)
    return q[..., :16] | (q[..., 16:] << 4), d[..., 0].to(torch.float16)


def _store_plain(s):
    dim, page, cache, slots = s["dim"], s["page"], s["cache"], s["slots"]
    nb, (n, heads, _) = dim // 32, s["k"].shape
    live = slots >= 0
    slot = slots[live]
    where = (slot // page, slot % page // 16, slot % 16)
    head = torch.arange(heads, device=cache.device)[None, :, None]
    kb, kd = _quantise_plain(s["k"][live])
    vb, vd = _quantise_plain(s["v"][live])
    flat = cache.view(-1)
    start = ((where[0][:, None, None] * heads + head) * (page // 16) + where[1][:, None, None]) * (18 * dim)
    token = where[2][:, None, None]
    b = torch.arange(nb, device=cache.device)[:, None]
    j = torch.arange(16, device=cache.device)[None]
    # byte j of block b of a key: word (half, g, t, b) with t = j / 4
    at = ((token // 8 * 8 + token % 8) * 4 + (j // 4).reshape(1, 1, -1).expand(1, 1, 16))[..., None, :] * nb
    at = (at + b) * 4 + j % 4
    flat[(start[..., None] + at).reshape(-1)] = kb.reshape(-1)
    at = ((token // 8 * 8 + (j // 2).reshape(1, 1, -1)) * 4 + token % 8 // 2)[..., None, :] * nb
    at = (at + b) * 4 + (token % 2)[..., None] * 2 + j % 2 + 8 * dim
    flat[(start[..., None] + at).reshape(-1)] = vb.reshape(-1)
    at = start[..., None] + 16 * dim + (token[..., None] * nb + b.reshape(-1)[None, None, None]).reshape(len(slot), 1, 1, nb) * 2
    scale_at = (at[:, :, 0, :, None] + torch.arange(2, device=cache.device)).reshape(-1)
    flat[scale_at] = kd.view(torch.uint8).reshape(-1)
    flat[scale_at + dim] = vd.view(torch.uint8).reshape(-1)
    # what the slots hold now, as the values that it stands for; a row without a slot reads as zeros
    k, v = _unpack_plain(cache[where[0], :, where[1]], dim)
    pick = where[2][:, None, None, None].expand(-1, heads, 1, dim)
    out = []
    for t in (k, v):
        full = t.new_zeros((n, heads, dim))
        full[live] = t.gather(2, pick)[:, :, 0]
        out.append(full)
    return tuple(out)


def _attention_plain(s):
    dim, page, n = s["dim"], s["page"], s["requests"]
    kv, group, most, q = s["kv_heads"], s["heads"] // s["kv_heads"], s["most"], s["q"]
    pages = s["cache"][s["table"].long()]  # (requests, width, kv heads, groups, 18 dim)
    k, v = _unpack_plain(pages.transpose(1, 2), dim)
    k, v = k.reshape(n, kv, -1, dim), v.reshape(n, kv, -1, dim)
    first, length = s["first_rows"].long(), s["kv_lens"].long()
    count = first[1:] - first[:-1]
    i = torch.arange(most, device=q.device)[None]
    row = (first[:-1, None] + i).clamp(max=q.shape[0] - 1)
    x = q[row].to(torch.float32).reshape(n, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, dim)
    score = torch.matmul(x, k.transpose(-1, -2)).mul_(s["scale"]).reshape(n, kv, group, most, -1)
    position = (length - count)[:, None] + i
    j = torch.arange(score.shape[-1], device=q.device)
    seen = (j <= position[..., None]) & (j < length[:, None, None])
    if s["window"]:
        seen &= j > position[..., None] - s["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = weight.sum(-1, keepdim=True)
    y = torch.matmul(weight.reshape(n, kv, group * most, -1), v).reshape(n, kv, group, most, dim)
    y = torch.where(total > 0, y / total, 0.0)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)[..., 0]
    out = q.new_zeros(q.shape)
    live = i < count[:, None]
    out[row[live]] = y.permute(0, 3, 1, 2, 4).reshape(n, most, kv * group, dim)[live].to(q.dtype)
    full = score.new_zeros(q.shape[:2])
    full[row[live]] = lse.permute(0, 3, 1, 2).reshape(n, most, kv * group)[live]
    return out, full


def run(s):
    op = s["op"]
    if own:
        tc = _tc()
        if op == "rope":
            return tc.rope_qk(s["q"], s["k"], s["positions"], s["freqs"], halves=s["halves"], magnitude=s["magnitude"], inverse=s["inverse"])
        if op == "plan":
            p = tc.kv_plan(s["context_lens"], s["new_lens"], s["table"], s["free"], s["free_count"], s["page"], s["rows"])
            return p.first_rows, p.kv_lens, p.slots, p.positions, p.requests, p.info, s["table"]
        if op == "store":
            tc.kv_store_q4_0(s["cache"], s["k"], s["v"], s["slots"])
            return tc.kv_load_q4_0(s["cache"], s["slots"])
        return tc.attention_q4_0(s["q"], s["cache"], s["table"], s["kv_lens"], first_rows=s["first_rows"], max_new=s["most"],
                                 scale=s["scale"], window=s["window"], with_lse=True)
    if op == "rope":
        return _rotate_plain(s["q"], s), _rotate_plain(s["k"], s)
    if op == "plan":
        return _plan_plain(s)
    if op == "store":
        return _store_plain(s)
    return _attention_plain(s)


# ------------------------------------------------------------------ by definition, in 64 bits


def _exact_rope(case, seed):
    s = prepare(case, seed)
    # each pair as one complex number times exp(i * angle)
    angle = torch.outer(s["positions"].double(), s["freqs"])
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), -angle if case["inverse"] else angle)[:, None]
    out = []
    for x in (s["q"].double(), s["k"].double()):
        y = x.clone()
        rot = case["rot"]
        if case["halves"]:
            z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn
            y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
        else:
            y[..., :rot] = torch.view_as_real(torch.view_as_complex(x[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
        out.append(y)
    return tuple(out)


def _places(dim):
    """Where value d of token t of a group lies: (byte, shift) of its quant in the key part, the same in the value part."""
    nb = dim // 32
    places = []
    for value in (False, True):
        byte, shift = [], []
        for t in range(16):
            for d in range(dim):
                b, e = divmod(d, 32)
                j = e % 16
                if value:
                    word = ((t // 8 * 8 + j // 2) * 4 + t % 8 // 2) * nb + b
                    byte.append(8 * dim + 4 * word + 2 * (t % 2) + j % 2)
                else:
                    word = (t * 4 + j // 4) * nb + b
                    byte.append(4 * word + j % 4)
                shift.append(4 * (e // 16))
        places.append((_ints(byte, torch.int64), _ints(shift, torch.uint8)))
    return places


def _exact_attention(case, seed):
    s = prepare(case, seed)
    dim, page, kv = case["dim"], case["page"], case["kv_heads"]
    group = case["heads"] // kv
    (kb, ks), (vb, vs) = _places(dim)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    row = 0
    for r, (c, m) in enumerate(_lengths(case)):
        total = c + m
        low = max(0, c - case["window"] + 1) if case["window"] else 0
        pages = s["table"][r, :-(-total // page)].long()
        at = torch.arange(c, total, device="cuda")[:, None]
        j = torch.arange(low, total, device="cuda")[None]
        seen = j <= at
        if case["window"]:
            seen = seen & (at - j < case["window"])
        for h in range(kv):
            g = s["cache"][pages, h].flatten(0, 1)  # this head's groups, in order
            scale = g[:, 16 * dim:].contiguous().view(torch.float16).double().reshape(-1, 2, 16, dim // 32).repeat_interleave(32, -1)
            k = (((g[:, kb] >> ks) & 15).double() - 8).reshape(-1, 16, dim) * scale[:, 0]
            v = (((g[:, vb] >> vs) & 15).double() - 8).reshape(-1, 16, dim) * scale[:, 1]
            k, v = k.reshape(-1, dim)[low:total], v.reshape(-1, dim)[low:total]
            for i in range(group):
                x = s["q"][row:row + m, h * group + i].double()
                score = (x @ k.T * s["scale"]).masked_fill(~seen, -math.inf)
                lse[row:row + m, h * group + i] = torch.logsumexp(score, -1)
                out[row:row + m, h * group + i] = torch.softmax(score, -1) @ v
        row += m
    return out, lse


def exact(case, seed):
    if case["op"] == "rope":
        return _exact_rope(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, seed)
    return None  # whole numbers, and 4-bit values that 32-bit arithmetic chooses: that arithmetic is the format's definition
