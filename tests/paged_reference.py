"""Plain restatement, in 64 bits on the CPU, of the paged Q4_0 cache and of what works on it."""
import numpy as np

QK = 32


def places(dim):
    """For token t and element d of a group: (byte of its key quant, of its value quant, shift), each (16, dim), and the
    byte of the key scale and of the value scale of (token, block)."""
    nb = dim // QK
    key, value, shift = (np.zeros((16, dim), np.int64) for _ in range(3))
    for t in range(16):
        for d in range(dim):
            b, e = divmod(d, QK)
            j = e % 16  # byte of the block; elements 16.. are the high nibbles
            key[t, d] = 4 * ((((t // 8) * 8 + t % 8) * 4 + j // 4) * nb + b) + j % 4
            value[t, d] = 8 * dim + 4 * ((((t // 8) * 8 + j // 2) * 4 + t % 8 // 2) * nb + b) + 2 * (t % 2) + j % 2
            shift[t, d] = 4 * (e // 16)
    at = 2 * (np.arange(16)[:, None] * nb + np.arange(nb)[None])
    return key, value, shift, 16 * dim + at, 17 * dim + at


def encode(quants, scales):
    """Group bytes (..., 18 * dim) of quants (2, ..., 16, dim) in 0..15 and float16 scales (2, ..., 16, dim / 32)."""
    dim = quants.shape[-1]
    key, value, shift, kd, vd = places(dim)
    out = np.zeros(quants.shape[1:-2] + (18 * dim,), np.uint8)
    for part, byte in enumerate((key, value)):
        low = shift == 0
        out[..., byte[low]] = quants[part][..., low]
        out[..., byte[~low]] |= quants[part][..., ~low] << 4
    for part, at in enumerate((kd, vd)):
        raw = np.ascontiguousarray(scales[part]).view(np.uint8).reshape(scales[part].shape + (2,))
        out[..., at], out[..., at + 1] = raw[..., 0], raw[..., 1]
    return out


def decode(groups):
    """(keys, values), float64 (..., 16, dim), of group bytes (..., 18 * dim)."""
    dim = groups.shape[-1] // 18
    key, value, shift, kd, vd = places(dim)
    out = []
    for byte, at in ((key, kd), (value, vd)):
        q = ((groups[..., byte] >> shift) & 15).astype(np.float64) - 8
        raw = np.stack((groups[..., at], groups[..., at + 1]), -1)
        d = np.ascontiguousarray(raw).view(np.float16)[..., 0].astype(np.float64)
        out.append(q * np.repeat(d, QK, -1))
    return out


def random_cache(rng, pages, heads, page_tokens, dim, spread=1.0):
    """(pages, heads, groups, 18 * dim) bytes: any quants, scales of either sign."""
    lead = (pages, heads, page_tokens // 16)
    quants = rng.integers(0, 16, (2,) + lead + (16, dim), dtype=np.uint8)
    d = rng.uniform(0.02, 0.3, (2,) + lead + (16, dim // QK)) * rng.choice((-1.0, 1.0), (2,) + lead + (16, dim // QK))
    return encode(quants, (d * spread).astype(np.float16))


def tables(rng, lens, page_tokens, width=None, spare=1):
    """A block table of shuffled pages for the given lengths, -1 where a request has none; (table, pages)."""
    held = [-(-n // page_tokens) for n in lens]
    width = max(held + [1]) if width is None else width
    pages = sum(held) + spare
    order, table, used = rng.permutation(pages), np.full((len(lens), width), -1, np.int32), 0
    for r, n in enumerate(held):
        table[r, :n] = order[used:used + n]
        used += n
    return table, pages


def attention(q, cache, table, lens, first_rows, scale, window=0):
    """(out, lse, weight) in 64 bits; weight is what the error bounds go by: for each row and head the sum of
    |weight * value| of each element, the largest |q| . |k| * scale, and the number of tokens seen.  Rows of
    no request are NaN.  q: float64 (rows, heads, dim)."""
    rows, heads, dim = q.shape
    kv_heads, groups = cache.shape[1], cache.shape[2]
    share, page_tokens = heads // kv_heads, 16 * groups
    out, lse = np.full(q.shape, np.nan), np.full((rows, heads), np.nan)
    size, dot, count = np.zeros(q.shape), np.zeros((rows, heads)), np.zeros((rows, heads))
    for r, n in enumerate(lens):
        n = min(max(int(n), 0), table.shape[1] * page_tokens)
        there = np.arange(n)
        page = table[r, there // page_tokens] if n else np.zeros(0, np.int64)
        alive = (page >= 0) & (page < cache.shape[0])
        new = first_rows[r + 1] - first_rows[r]
        for h in range(kv_heads):
            if n:
                k, v = decode(cache[np.where(alive, page, 0), h, there % page_tokens // 16])
                k, v = k[there, there % 16], v[there, there % 16]
            for i in range(new):
                row, at = first_rows[r] + i, n - new + i
                seen = alive & (there <= at)
                if window:
                    seen &= there > at - window
                if row < 0 or row >= rows:
                    continue
                for x in range(h * share, (h + 1) * share):
                    if not seen.any():
                        out[row, x], lse[row, x] = 0.0, -np.inf
                        continue
                    s = (k[seen] @ q[row, x]) * scale
                    top = s.max()
                    w = np.exp(s - top)
                    lse[row, x] = top + np.log(w.sum())
                    w /= w.sum()
                    out[row, x] = w @ v[seen]
                    size[row, x] = w @ np.abs(v[seen])
                    dot[row, x] = (np.abs(k[seen]) @ np.abs(q[row, x])).max() * abs(scale)
                    count[row, x] = seen.sum()
    return out, lse, (size, dot, count)


HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def attention_bounds(out, lse, weight, kind, largest_scale, prompt=False):
    """How far a result may be from `attention`'s.  Scores: an f32 sum of products, in blocks of 32 and then over at most 8
    blocks (40 additions, each at most one step of 2^-23 where the tensor cores truncate), scaled (2^-23), the query in two fp16
    terms (2^-22).  A weight's relative error is twice the score's (its own, and the sum's) plus that of 2^x and the sum's
    additions (2^-18 allows for them).  16-bit calls round the weight times the value's scale to fp16: half a step, or 2^-25
    absolute below fp16's normal range, times a quant of at most 8.  f32 calls round it to two terms, the second of which is off
    by at most 2^-25 too, after a power of two has lifted the largest scale D to 2^14 or more: 2^-25 / (2^14 / D) = 2^-39 D each.
    (A row whose heaviest tokens have quants of 8, that is values of 0, has nothing else to hide that behind.)  Last, the result's
    own rounding.
    `prompt`: a call whose rows may go to the kernel that rounds every key and value, d * (n - 8), to fp16: half a step of 2^-11 on
    each product and each term, and sums of up to 256 additions in one row of the product."""
    size, dot, count = weight
    score = dot * (41 * 2.0 ** -23 + 2.0 ** -22)
    relative = 2 * score + 2.0 ** -18
    absolute = count[..., None] * 8 * 2.0 ** -39 * largest_scale
    if prompt:
        score = dot * (256 * 2.0 ** -23 + 2.0 ** -22 + 2.0 ** -11)
        relative = 2 * score + 2.0 ** -18 + 2.0 ** -11 + count * 2.0 ** -23
    if kind != "float32":
        relative = relative + 2.0 ** -11
        absolute = count[..., None] * 8 * 2.0 ** -25
    bound = size * relative[..., None] + absolute + np.abs(np.nan_to_num(out)) * HALF_STEP[kind]
    if kind == "float16":
        bound = bound + 2.0 ** -25
    return bound, score + 2.0 ** -18 + np.abs(np.where(np.isfinite(lse), lse, 0.0)) * 2.0 ** -22


def plan(context, new, table, free_pages, free_count, page_tokens, rows):
    """What kv_plan gives, request by request; the table is a changed copy."""
    table = table.copy()
    status, width = 0, table.shape[1]
    take = [-(-(c + m) // page_tokens) - -(-c // page_tokens) if c >= 0 and m >= 0 else 0 for c, m in zip(context, new)]
    if sum(take) > free_count:
        status = 1
    if any(-(-(c + m) // page_tokens) > width for c, m in zip(context, new) if c >= 0 and m >= 0):
        status = 2
    if sum(m for c, m in zip(context, new) if c >= 0 and m >= 0) > rows:
        status = 3
    if any(c < 0 or m < 0 for c, m in zip(context, new)) or not 0 <= free_count <= len(free_pages):
        status = 4
    first, slots, positions, requests = [0], np.full(rows, -1, np.int64), np.zeros(rows, np.int32), np.full(rows, -1, np.int32)
    left = free_count
    lens = list(context)
    for r, (c, m) in enumerate(zip(context, new)):
        if status:
            first.append(0)
            continue
        for i in range(-(-c // page_tokens), -(-(c + m) // page_tokens)):
            left -= 1
            table[r, i] = free_pages[left]
        for i in range(m):
            at, row = c + i, first[-1] + i
            slots[row] = int(table[r, at // page_tokens]) * page_tokens + at % page_tokens
            positions[row], requests[row] = at, r
        first.append(first[-1] + m)
        lens[r] = c + m
    info = [status, first[-1], free_count - left, left]
    return (np.array(first, np.int32), np.array(lens, np.int32), slots, positions, requests, np.array(info, np.int32)), table
