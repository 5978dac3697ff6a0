"""The paged cache's operators in 64 bits, in plain numpy loops: the cache as
the header defines it, one sequence, page and head at a time."""
import numpy as np

import willamette_hip as wh

EPS = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}


class Step:
    """A step's host arrays: steps [(positions before, new tokens)], pages dealt in a random order."""

    def __init__(self, rng, steps, page, kh, dim, spare=3, extra_stride=1, pad=0):
        self.steps, self.page, self.kh, self.dim = steps, page, kh, dim
        used = [-(-max(c + n, 0) // page) for c, n in steps]
        self.n_pages = sum(used) + spare
        self.stride = max(used) + extra_stride
        perm = rng.permutation(self.n_pages)
        # entries past a sequence's pages are never looked at: no page at all
        self.table = np.full((len(steps), self.stride), -7, np.int32)
        at = 0
        for s, u in enumerate(used):
            self.table[s, :u] = perm[at:at + u]
            at += u
        self.cu = np.concatenate([[0], np.cumsum([n for _, n in steps])]).astype(np.int32)
        self.kv_len = np.array([c + n for c, n in steps], np.int32)
        self.n_tokens = int(self.cu[-1]) + pad
        self.max_new = max(n for _, n in steps)
        self.max_kv = max(1, int(self.kv_len.max()))

    def pool(self, rng):
        """Random codes and scales; scales of pages no sequence has are NaN."""
        shape = (self.n_pages, self.kh, self.page, self.dim)
        k = rng.integers(-127, 128, shape).astype(np.int8)
        v = rng.integers(-127, 128, (self.n_pages, self.kh, self.dim, self.page)).astype(np.int8)
        ks = np.full((self.n_pages, self.kh), np.nan, np.float32)
        vs = ks.copy()
        for s, (c, n) in enumerate(self.steps):
            for lp in range(-(-(c + n) // self.page)):
                ks[self.table[s, lp]] = np.exp(rng.standard_normal(self.kh) * 0.3) / 64
                vs[self.table[s, lp]] = np.exp(rng.standard_normal(self.kh) * 0.3) / 64
        return k, v, ks, vs


def rotate(x, cos, sin, layout):
    """x [.., dim] in 64 bits, cos and sin [pairs]."""
    n = 2 * cos.shape[-1]
    y = x.copy()
    a, b = (slice(0, n // 2), slice(n // 2, n)) if layout == wh.ROPE_HALF else (slice(0, n, 2), slice(1, n, 2))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def quotients(x, s):
    """Rounded half away from zero, within +-127; NaN 0."""
    if not s > 0:
        return np.zeros_like(x)
    with np.errstate(invalid="ignore"):
        q = np.clip(np.trunc(x / s + np.copysign(0.5, x)), -127, 127)
    return np.where(np.isnan(q), 0, q)


def append_block(rows, codes, first, s_old):
    """One head's block: `rows` [n, dim] (f32 values) join at slot `first`; codes [page, dim] in place."""
    s = np.float64(s_old) if first else 0.0
    a = np.abs(rows[np.isfinite(rows)])
    if a.size:
        s = max(s, np.float64(np.float32(a.max() / 127.0)))
    if first and s > s_old:
        codes[:first] = quotients(codes[:first] * np.float64(s_old), s)
    codes[first:first + len(rows)] = quotients(rows, s)
    return np.float32(s)


def append(st, pool, q, k, v, cos, sin, layout):
    """q [tokens, heads, dim], k and v [tokens, kv heads, dim] in 64 bits; the pool in place; rotated q."""
    kc, vc, ks, vs = pool
    q_out = q.copy()
    for s in range(len(st.steps)):
        n, end = int(st.cu[s + 1] - st.cu[s]), int(st.kv_len[s])
        start = end - n
        at = st.cu[s] - start  # packed token of position 0
        kr = {}
        for p in range(max(start, 0), end):
            c, sn = (cos[p], sin[p]) if cos is not None else (np.ones(0), np.zeros(0))
            q_out[at + p] = rotate(q[at + p], c, sn, layout)
            with np.errstate(invalid="ignore", over="ignore"):
                kr[p] = rotate(k[at + p], c, sn, layout).astype(np.float32).astype(np.float64)
        for lp in range(max(start, 0) // st.page, -(-end // st.page)):
            page, lo, hi = st.table[s, lp], max(start, 0, lp * st.page), min(end, (lp + 1) * st.page)
            if lo >= hi:
                continue
            first = lo - lp * st.page
            for h in range(st.kh):
                ks[page, h] = append_block(np.stack([kr[p][h] for p in range(lo, hi)]), kc[page, h], first, ks[page, h])
                vs[page, h] = append_block(np.stack([v[at + p][h] for p in range(lo, hi)]), vc[page, h].T, first,
                                           vs[page, h])
    return q_out


def values(st, pool, s, n, h):
    """K and V of sequence s's first n positions, head h, in 64 bits."""
    kc, vc, ks, vs = pool
    ids = [st.table[s, p // st.page] for p in range(n)]
    k = np.array([kc[i, h, p % st.page] * np.float64(ks[i, h]) for p, i in enumerate(ids)]).reshape(n, st.dim)
    v = np.array([vc[i, h, :, p % st.page] * np.float64(vs[i, h]) for p, i in enumerate(ids)]).reshape(n, st.dim)
    return k, v


def attention(st, pool, q, scale, kind):
    """out, lse and their tolerances for q [tokens, heads, dim] (64 bits).

    The tolerance counts, per row: scores summed in f32 over dim products of
    queries held to 2^-22 (exactly, for half types) against sum |q k|; the
    exponential of a rounded argument; weights held to 2^-22 (f32) or half a
    step of f16; f32 sums over the positions; the output's own rounding."""
    t, heads, dim = q.shape
    out, lse = np.zeros((t, heads, dim)), np.full((t, heads), -np.inf)
    tol, tol_lse = np.zeros((t, heads, dim)), np.zeros((t, heads))
    u, group = 2.0 ** -24, heads // st.kh
    weight = 2.0 ** -22 if kind == "f32" else 2.0 ** -11
    for s in range(len(st.steps)):
        a, b, end = int(st.cu[s]), int(st.cu[s + 1]), int(st.kv_len[s])
        for h in range(st.kh if b > a and end > 0 else 0):
            k, v = values(st, pool, s, end, h)
            for j in range(a, b):
                n = end - (b - a) + (j - a) + 1
                if n <= 0:
                    continue
                for hq in range(h * group, (h + 1) * group):
                    x = k[:n] @ q[j, hq] * scale
                    size = np.abs(k[:n]) @ np.abs(q[j, hq]) * abs(scale)
                    top = x.max()
                    w = np.exp(x - top)
                    total = w.sum()
                    w /= total
                    out[j, hq], lse[j, hq] = w @ v[:n], top + np.log(total)
                    ds = size * ((dim + 8) * u + 2.0 ** -21) + (np.abs(x) + np.abs(top) + 64) * 4 * u
                    mean_ds = w @ ds
                    rel = ds + mean_ds + weight + (n + 64) * 2 * u
                    tol[j, hq] = (w * rel) @ np.abs(v[:n]) + np.abs(out[j, hq]) * EPS[kind] / 2 + 1e-37
                    tol_lse[j, hq] = mean_ds + (n + 64) * 2 * u + abs(lse[j, hq]) * 4 * u
    return out, lse, tol, tol_lse
