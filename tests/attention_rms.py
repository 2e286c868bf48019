"""Attention over the paged Q4_0 cache by its definition in 64 bits, and how large the error of a result may be on average.

Roundings of different products are independent, so their errors add in squares: where a worst case over n tokens allows n half
steps, the mean square allows sqrt(n) of them, and small values that are lost show."""
import numpy as np

import paged_reference as ref

HALF_STEP = ref.HALF_STEP


def definition(q, cache, table, lens, first_rows, scale, window=0, max_new=None):
    """What each row is by the header: row i of a request's n sits at position kv_len - n + i, whatever the call leaves out, and sees
    the tokens up to there that the table's pages hold.  q: float64 (rows, heads, dim).  Arrays by (row, head) or (row, head, element);
    rows that the call leaves alone are NaN in `out`."""
    rows, heads, dim = q.shape
    kv_heads, groups = cache.shape[1], cache.shape[2]
    share, page_tokens = heads // kv_heads, 16 * groups
    d = {k: np.zeros((rows, heads) + ((dim,) if k in ("out", "size", "rss", "root") else ())) for k in ("out", "lse", "size", "rss", "dot", "spread", "norm", "count", "largest", "root")}
    d["out"][:] = d["lse"][:] = np.nan
    for r, n in enumerate(lens):
        n = max(int(n), 0)
        held = min(n, table.shape[1] * page_tokens)
        first, new = int(first_rows[r]), int(first_rows[r + 1]) - int(first_rows[r])
        mine = min(new, max_new or new, max(0, rows - first)) if first >= 0 else 0
        if mine <= 0:
            continue
        there = np.arange(held)
        page = table[r, there // page_tokens] if held else np.zeros(0, np.int64)
        alive = (page >= 0) & (page < cache.shape[0])
        at = n - new + np.arange(mine)
        seen = alive[:, None] & (there[:, None] <= at)
        if window:
            seen &= there[:, None] > at - window
        for h in range(kv_heads):
            k = v = np.zeros((0, dim))
            if held:
                k, v = ref.decode(cache[np.where(alive, page, 0), h, there % page_tokens // 16])
                k, v = k[there, there % 16], v[there, there % 16]
                k, v = np.where(alive[:, None], k, 0.0), np.where(alive[:, None], v, 0.0)
            for x in range(h * share, (h + 1) * share):
                y = q[first:first + mine, x]
                to = (slice(first, first + mine), x)
                some = seen.any(0)
                s = np.where(seen, k @ y.T * scale, -np.inf)
                top = np.where(some, s.max(0, initial=-np.inf), 0.0)
                w = np.where(seen, np.exp(s - top), 0.0)
                l = w.sum(0)
                w = w / np.where(some, l, 1.0)
                with np.errstate(divide="ignore"):
                    d["lse"][to] = np.where(some, top + np.log(l), -np.inf)
                d["out"][to], d["size"][to], d["rss"][to] = w.T @ v, w.T @ np.abs(v), np.sqrt((w ** 2).T @ v ** 2)
                d["dot"][to] = np.where(seen, np.abs(k) @ np.abs(y).T * abs(scale), 0.0).max(0, initial=0.0)
                d["spread"][to] = np.sqrt(np.where(seen, k ** 2 @ (y ** 2).T * scale ** 2, 0.0).max(0, initial=0.0))
                d["norm"][to], d["count"][to] = np.sqrt((w ** 2).sum(0)), seen.sum(0)
                d["root"][to] = np.sqrt(seen.T @ v ** 2)
                d["largest"][to] = (np.where(seen, np.abs(v).max(1, initial=0.0)[:, None], 0.0)).max(0, initial=0.0)
    return d


def allowed(d, kind, prompt):
    """Mean squares of the errors of `out` and `lse`.
    Sums of scores are f32: 40 additions of a step of 2^-23 in the few-rows kernel, 256 in the prompts', and the scaling; a weight is off
    by twice that, its own and the sum's, and 2^-18 for 2^x and the sum's additions.  These count in full.
    Independent half steps: 16-bit calls of few rows round each weight times its value's scale, 2^-11; prompts round weights, values and
    the elements of keys, 2^-11 each, the last of which moves a score by 2^-11 of the root of its terms' squares.  f32: 2^-22.
    Below fp16's normal range a half step is 2^-25: in few rows of a product that has been lifted so that the largest scale is 2^14 or
    more, times a quant of up to 8, hence 2^-39 of the largest value, sqrt(count) of these; in prompts of a weight, times its value.
    The result's own rounding."""
    few = d["dot"] * (41 * 2.0 ** -23 + 2.0 ** -22)
    score = d["dot"] * (257 * 2.0 ** -23 + 2.0 ** -22) if prompt else few
    step = 2.0 ** -22 if kind == "float32" else 2.0 ** -11
    independent = 2 * step ** 2 + (step * d["spread"]) ** 2 if prompt else np.full(few.shape, step ** 2)
    lost = d["root"] * 2.0 ** -25 if prompt else (np.sqrt(d["count"]) * d["largest"] * 2.0 ** -39)[..., None]
    out = independent[..., None] * d["rss"] ** 2 + ((2 * score + 2.0 ** -18)[..., None] * d["size"]) ** 2 + lost ** 2
    out = out + (HALF_STEP[kind] * d["out"]) ** 2 + (2.0 ** -50 if kind == "float16" else 0.0)
    lse = (score + 2.0 ** -18 + np.abs(np.where(np.isfinite(d["lse"]), d["lse"], 0.0)) * 2.0 ** -22) ** 2
    if prompt:
        lse = lse + (step * d["spread"] * d["norm"]) ** 2
    return out, lse


def check(got, lse, d, kind, prompt=False, where=None):
    """`got` and `lse` (CUDA tensors) against `definition`: mean square error over mean square allowed, element by element.  `where`:
    a mask of (row, head, element) to look at; rows left alone and elements that are no numbers are not looked at."""
    square, lse_square = allowed(d, kind, prompt)
    got = got.double().cpu().numpy()
    look = ~np.isnan(d["out"]) if where is None else where & ~np.isnan(d["out"])
    assert np.isfinite(got[look]).all()
    off = (got[look] - d["out"][look]) ** 2
    zero = square[look] == 0
    assert (off[zero] == 0).all()
    ratio = (off[~zero] / square[look][~zero]).mean() if (~zero).any() else 0.0
    assert ratio <= 1, f"mean square error {ratio:.3g} of the allowed"
    if lse is not None:
        lse = lse.double().cpu().numpy()
        rows = ~np.isnan(d["lse"])
        empty = np.isneginf(d["lse"][rows])
        assert np.array_equal(np.isneginf(lse[rows]), empty)
        off = (lse[rows][~empty] - d["lse"][rows][~empty]) ** 2 / lse_square[rows][~empty]
        assert off.size == 0 or off.mean() <= 1, f"mean square error of lse {off.mean():.3g} of the allowed"
    return ratio
