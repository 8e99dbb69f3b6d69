"""The paged 8-bit K/V cache, its attention and the sampling operators in 64-bit
numpy, written from their definitions (include/gemma_hip.h)."""
import numpy as np

import gemma_hip as gh

U = 2.0 ** -24  # half a step of f32, relative
NONE = 0xffffffff


def rms(x, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def rope(x, positions, rot, theta):
    """x [rows][heads][D] at the rows' positions, split halves of the first rot dims."""
    h = rot // 2
    a = np.asarray(positions, np.float64)[:, None, None] * theta ** (-2.0 * np.arange(h) / max(rot, 1))
    u, v = x[..., :h], x[..., h:rot]
    return np.concatenate([u * np.cos(a) - v * np.sin(a), u * np.sin(a) + v * np.cos(a), x[..., rot:]], -1)


def power(amax):
    """The least power of two (at least 2^-126) whose 127-fold reaches amax; 0 for 0."""
    if amax == 0:
        return 0.0
    if not np.isfinite(amax):
        return np.nan
    e = int(np.floor(np.log2(amax / 127))) - 1
    while 127 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** max(e, -126)


class Cache:
    """Codes [page][head][token][dim] and scales [page][head][block] of k and v."""

    def __init__(self, pages, page, heads, D, rng=None):
        self.P, self.page, self.H, self.D = pages, page, heads, D
        shape = (pages, heads, page, D)
        if rng is None:
            self.codes = [np.zeros(shape, np.int8) for _ in "kv"]
            self.scales = [np.zeros((pages, heads, page // 16)) for _ in "kv"]
        else:  # something in every page
            self.codes = [rng.integers(-127, 128, shape).astype(np.int8) for _ in "kv"]
            self.scales = [2.0 ** rng.integers(-7, -3, (pages, heads, page // 16)) for _ in "kv"]
        self.near = 0  # codes decided within 1e-6 of a border

    def place(self, table, t):
        """(page, token in it), or None where the table names no page."""
        i = int(t) // self.page
        if i >= len(table) or table[i] >= self.P:
            return None
        return int(table[i]), int(t) % self.page

    def append(self, which, table, past, x):
        """x [rows][heads][D] (64 bits) at tokens past, past + 1, ..."""
        codes, scales = self.codes[which], self.scales[which]
        for b in range(past // 16, (past + len(x) - 1) // 16 + 1):
            lo, hi = max(past, 16 * b), min(past + len(x), 16 * b + 16)
            at = self.place(table, 16 * b)
            if at is None:
                continue
            p, w = at
            for h in range(self.H):
                new = x[lo - past:hi - past, h]
                old = scales[p, h, w // 16] if lo > 16 * b else 0.0
                s = power(np.abs(new).max()) if np.isfinite(new).all() else np.nan
                s = np.nan if np.isnan(s) or np.isnan(old) else max(s, old)
                kept = codes[p, h, w:w + lo - 16 * b]
                if s > old and lo > 16 * b:
                    kept[:] = np.rint(kept * (old / s)).astype(np.int8)
                if s > 0:
                    y = new / s
                    self.near += int((np.abs(np.abs(y - np.floor(y)) - 0.5) < 1e-6).sum())
                    codes[p, h, w + lo - 16 * b:w + hi - 16 * b] = np.rint(y).astype(np.int8)
                elif s == 0:
                    codes[p, h, w + lo - 16 * b:w + hi - 16 * b] = 0
                scales[p, h, w // 16] = s

    def rows(self, which, table, first, n):
        """Values [n][heads][D] of tokens first ..; NaN rows' scales stay; no page: 0, and whether there is one."""
        out, has = np.zeros((n, self.H, self.D)), np.zeros(n, bool)
        for i in range(n):
            at = self.place(table, first + i)
            if at is not None:
                out[i] = self.codes[which][at[0], :, at[1]] * self.scales[which][at[0], :, at[1] // 16][:, None]
                has[i] = True
        return out, has

    # ---- the layout of the device arrays
    def packed(self):
        k, v = (c.reshape(self.P, self.H, self.page // 16, 16, self.D) for c in self.codes)
        k = k.reshape(*k.shape[:4], self.D // 16, 16).swapaxes(3, 4)
        v = v.reshape(*v.shape[:3], 4, 4, self.D).swapaxes(4, 5)
        return [np.ascontiguousarray(a) for a in (k, v)]

    def unpacked(self, k, v):
        k = k.reshape(self.P, self.H, self.page // 16, self.D // 16, 16, 16).swapaxes(3, 4)
        v = v.reshape(self.P, self.H, self.page // 16, 4, self.D, 4).swapaxes(4, 5)
        return [np.ascontiguousarray(a).reshape(self.P, self.H, self.page, self.D) for a in (k, v)]


class Device:
    """The same cache and a batch on the device."""

    def __init__(self, ctx, cache):
        self.ctx, self.c = ctx, cache
        k, v = cache.packed()
        self.k, self.v = ctx.upload(k), ctx.upload(v)
        self.ks, self.vs = (ctx.upload(s.astype(np.float32)) for s in cache.scales)
        self.cache = gh.Kv8Cache(self.k.ptr, self.v.ptr, self.ks.ptr, self.vs.ptr, cache.P, cache.page, cache.H, cache.D)
        assert gh.lib().gh_kv8_code_bytes(self.cache) == k.nbytes
        assert gh.lib().gh_kv8_scale_bytes(self.cache) == cache.scales[0].size * 4

    def batch(self, rows, past, tables, num_rows=None, max_rows=None):
        start = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
        self.held = [self.ctx.upload(a) for a in (start, np.asarray(past, np.uint32), np.asarray(tables, np.uint32))]
        b = gh.Kv8Batch(*[h.ptr for h in self.held], len(rows), np.asarray(tables).shape[1],
                        int(start[-1]) if num_rows is None else num_rows, int(max(rows)) if max_rows is None else max_rows)
        b.held = self.held
        return b

    def codes(self):
        c = self.c
        return c.unpacked(self.k.read(np.int8), self.v.read(np.int8))

    def scales(self):
        return [s.read(np.float32).reshape(self.c.scales[0].shape).astype(np.float64) for s in (self.ks, self.vs)]


def attention(cache, rows, past, tables, q, scale, window):
    """q [rows][nq][D]: (out, bound): the f32 kernel's error bound per element, from the formula.

    A score is a sum that the kernel has exactly, up to q's 31 bits, rounded a handful of times:
    |ds| <= 8 U |s|.  p = exp(s - max): relative error |ds| + |d max| + 4 U |s - max| + 4 U, P's two
    halves 4 U, the sums over n tokens and their joins (n / 4 + 64) U; the quotient has the sum's too.
    The halves are f16 numbers in units of S / 2^10 (few columns: 2^14), S the largest V scale so far: what
    is left of p below half their last step, 2^-25 units, is lost, times a code of up to 127.  What is
    subtracted from the scores is at least the maximum less 4 (log2), so the sum that divides is at least 1.
    """
    out, bound, at = np.zeros_like(q, np.float64), np.zeros_like(q, np.float64), 0
    G = q.shape[1] // cache.H
    for b, n in enumerate(rows):
        k, has = cache.rows(0, tables[b], 0, past[b] + n)
        v, _ = cache.rows(1, tables[b], 0, past[b] + n)
        for i in range(n):
            t = past[b] + i
            seen = has & (np.arange(past[b] + n) <= t)
            if window:
                seen &= np.arange(past[b] + n) > t - window
            if not seen.any():
                continue
            for h in range(q.shape[1]):
                kk, vv = k[seen, h // G], v[seen, h // G]
                s = scale * (kk @ q[at + i, h].astype(np.float64))
                d = s - s.max()
                p = np.exp(d)
                p /= p.sum()
                rel = 8 * U * (np.abs(s) + np.abs(s).max()) + 4 * U * np.abs(d) + (8 + len(p) / 4 + 64) * U
                out[at + i, h] = p @ vv
                bound[at + i, h] = (p * rel) @ np.abs(vv) + (p @ rel) * np.abs(out[at + i, h])
                at_most = np.nan_to_num(cache.scales[1][tables[b][tables[b] < cache.P]]).max()
                bound[at + i, h] += len(p) * 127 * at_most * 2.0 ** -35
        at += n
    return out, bound


def probabilities(x, cap, temperature):
    """(probs, relative bound) of rows x (f32)."""
    x = x.astype(np.float64)
    masked = x == -np.inf
    y = cap * np.tanh(x / cap) if cap else x
    y = np.where(masked, -np.inf, y)
    with np.errstate(all="ignore"):
        m = y.max(1, keepdims=True)
        base = np.where(m == -np.inf, 0, m)
        e = np.where(masked, 0, np.exp((y - base) / temperature))
        total = e.sum(1, keepdims=True)
        p = np.where(total == 0, 0, e / np.where(total == 0, 1, total))
        # tanh to 2 steps, its quotient and product: 6 U |y| of y and of the maximum; the exponent's
        # difference, product and constant: 6 U |y - m|, 2^x to 2 steps; the sum's tree: 64 U
        d = np.where(masked, 0, np.abs(y - base))
        size = np.where(masked, 0, np.abs(y))
        bound = (6 * U * (size + np.abs(base)) * (1 if cap else 0) + 6 * U * d) / temperature
    return p, 2 * bound.max(1, keepdims=True) + 80 * U


def verify(target, draft, tokens, n_draft, u, pick):
    """(out_tokens, accepted) one sequence and one token at a time."""
    B, rows, V = target.shape
    out, accepted = np.full((B, rows), NONE, np.uint32), np.zeros(B, np.uint32)
    for b in range(B):
        n = min(int(n_draft[b]), rows - 1)
        i = 0
        while i < n:
            x = int(tokens[b, i])
            if x >= V:
                break
            q = 1.0 if draft is None else float(draft[b, i, x])
            if not float(u[b, i]) * q < float(target[b, i, x]):
                break
            out[b, i] = x
            i += 1
        p = target[b, i].astype(np.float64)
        full = np.where(p > 0, p, 0)
        w = full
        if i < n:
            q = np.zeros(V) if draft is None else draft[b, i].astype(np.float64)
            if draft is None and tokens[b, i] < V:
                q[tokens[b, i]] = 1.0
            w = p - q
            w = np.where(w > 0, w, 0)
            if not w.sum() > 0:
                w = full
        accepted[b] = i
        total = np.cumsum(w)
        if total[-1] > 0 and np.isfinite(total[-1]):
            goal = max(float(pick[b]), 0.0) * total[-1]
            hit = np.nonzero((total > goal) & (w > 0))[0]
            out[b, i] = hit[0] if len(hit) else np.nonzero(w > 0)[0][-1]
    return out, accepted
