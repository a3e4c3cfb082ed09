"""Plain models, in 64 bits and one step at a time, of the operators over a paged cache (test infrastructure)."""
import numpy as np

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}    # largest relative error of one rounding


def to_bf16(x):
    """f32 -> the nearest bf16, as uint16 bits (ties to even; NaN stays NaN)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r).reshape(np.shape(x))


def from_bf16(b):
    return (np.ascontiguousarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32).reshape(np.shape(b))


def encode(x, dtype):
    return np.ascontiguousarray(x, np.float32) if dtype == "f32" else to_bf16(x)


def decode(b, dtype):
    return b if dtype == "f32" else from_bf16(b)


def rope(x, pos, theta):
    """Rotate-half rope of x [heads, head_dim] at one position."""
    h = x.shape[-1] // 2
    a = pos * theta ** (-2.0 * np.arange(h) / x.shape[-1])
    x0, x1 = x[..., :h].astype(np.float64), x[..., h:].astype(np.float64)
    return np.concatenate([x0 * np.cos(a) - x1 * np.sin(a), x1 * np.cos(a) + x0 * np.sin(a)], -1)


def attention(q, k, v, scale, causal, dtype, p_terms=1):
    """One sequence: q [rows, n_q, d] against k, v [n, n_kv, d] -> (out, tolerance), both [rows, n_q, d].

    The tolerance counts roundings, in units of the element type's half step h and of u = 2^-24 for what is held in f32:
      * a score is a sum of d products: at most (d + 3) u of scale * sum |q_i k_i|, with the factor log2(e) in it; the exponential
        adds 4 u.  Both move a weight by that relative amount d_w (its own and, through the sum, everybody's: twice);
      * a sum of n weights or weighted values adds at most (n + 8) u (additions and rescalings);
      * a weight rounded to bf16 before it meets V: h once (with two terms, h * h);
      * the result's own rounding: h of it.
    """
    rows, n_q, d = q.shape
    n, n_kv = k.shape[0], k.shape[1]
    group, u, h = n_q // n_kv, 2.0 ** -24, HALF[dtype]
    out, tol = np.zeros((rows, n_q, d)), np.zeros((rows, n_q, d))
    for r in range(rows):
        m = min(n, n - rows + 1 + r) if causal else n
        if m <= 0:
            continue
        for a in range(n_q):
            kk, vv = k[:m, a // group].astype(np.float64), v[:m, a // group].astype(np.float64)
            qq = q[r, a].astype(np.float64)
            s = kk @ qq * scale
            w = np.exp(s - s.max())
            p = w / w.sum()
            out[r, a] = p @ vv
            dw = (d + 3) * u * (np.abs(kk) @ np.abs(qq)).max() * abs(scale) + 4 * u
            round_p = 0.0 if dtype == "f32" else h ** p_terms
            tol[r, a] = h * np.abs(out[r, a]) + (2 * dw + 2 * (m + 8) * u + round_p) * (p @ np.abs(vv)) + 1e-37
    return out, tol


class Pages:
    """Tables, lengths and counts of a paged cache, as the calls change them."""

    def __init__(self, seqs, n_pages, width, page):
        self.table = np.full((seqs, width), -1, np.int32)
        self.lens, self.refs = np.zeros(seqs, np.int32), np.zeros(n_pages, np.int32)
        self.page, self.width, self.n_pages = page, width, n_pages

    def held(self, n):
        return -(-int(n) // self.page)

    def used(self):
        return int((self.refs > 0).sum())

    def free_list(self):
        return [i for i in range(self.n_pages) if self.refs[i] <= 0]

    def free(self, seqs):
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.lens) for s in seqs):
            return 2
        for s in seqs:
            for j in range(self.held(self.lens[s])):
                self.refs[self.table[s, j]] -= 1
                self.table[s, j] = -1
            self.lens[s] = 0
        return 0

    def extend(self, seqs, counts):
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.lens) for s in seqs) or min(counts, default=0) < 0:
            return 2
        if any(self.lens[s] + c > self.width * self.page for s, c in zip(seqs, counts)):
            return 3
        for s, c in zip(seqs, counts):
            if c and self.lens[s] % self.page and self.refs[self.table[s, self.lens[s] // self.page]] != 1:
                return 4
        want = sum(self.held(self.lens[s] + c) - self.held(self.lens[s]) for s, c in zip(seqs, counts))
        free = self.free_list()
        if want > len(free):
            return 1
        for s, c in zip(seqs, counts):
            for j in range(self.held(self.lens[s]), self.held(self.lens[s] + c)):
                self.table[s, j] = free.pop(0)
                self.refs[self.table[s, j]] = 1
            self.lens[s] += c
        return 0

    def fork(self, src, dst):
        """-> (status, [(from, to)])"""
        ok = lambda s: 0 <= s < len(self.lens)  # noqa: E731
        if len(set(dst)) < len(dst) or set(src) & set(dst) or not all(ok(s) for s in [*src, *dst]) or any(self.lens[d] for d in dst):
            return 2, []
        free, pairs = self.free_list(), []
        if sum(bool(self.lens[s] % self.page) for s in src) > len(free):
            return 1, []
        for s, d in zip(src, dst):
            full = self.lens[s] // self.page
            for j in range(full):
                self.table[d, j] = self.table[s, j]
                self.refs[self.table[s, j]] += 1
            if self.lens[s] % self.page:
                pairs.append((self.table[s, full], free[0]))
                self.table[d, full] = free.pop(0)
                self.refs[self.table[d, full]] = 1
            self.lens[d] = self.lens[s]
        return 0, pairs

    def compact(self):
        live = self.used()
        moves = [i for i in range(live, self.n_pages) if self.refs[i] > 0]
        holes = [i for i in range(live) if self.refs[i] <= 0]
        to = dict(zip(moves, holes))
        for s, n in enumerate(self.lens):
            for j in range(self.held(n)):
                self.table[s, j] = to.get(self.table[s, j], self.table[s, j])
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        return list(to.items())
