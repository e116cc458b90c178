"""Plain 64-bit implementations of the batched-step operators (numpy), and the
inputs the tests share. Nothing here uses the library."""
import numpy as np

PAGE = 64


def allowed(kind, r, past, n, mask_row=None):
    """Truth value per slot 0 .. past + n - 1: what row r of a sequence attends."""
    ok = np.zeros(past + n, bool)
    if kind == "packed":
        ok[: past + r + 1] = True
    else:
        ok[:past] = True
        for j in range(n):
            if j < 64 * len(mask_row):
                ok[past + j] = (int(mask_row[j // 64]) >> (j % 64)) & 1
    return ok


def attention(kind, q, k, v, table, start, past, n_heads, scale, masks=None, n_pages=None):
    """(out, tol) [rows][n_heads * hd] in float64; rows of no sequence are NaN.
    tol bounds what an implementation with fp32 sums and factors of 22 bits
    may be off by: a product q_d k_d carries 2^-22 for each factor and the
    sum of hd of them hd * 2^-24, so a score is off by at most
    ds = scale * sum_d |q_d k_d| * (2^-21 + hd * 2^-24); a weight exp(s - m)
    by the factor 1 +- (2 ds + 2^-20) (the exponential's own 2^-22 and its
    argument's rounding included for |s| up to 32), a weight's own 22 bits
    and the sums over the keys (blocks of 64 and their chain) 2^-20 more; the
    output is a weighted mean of v, so all of it moves the result by at most
    the relative error times twice the mean of |v|, plus 2^-37 of the largest
    |v| (what the two parts of a factor cannot hold next to it)."""
    n_kv, hd = k.shape[1], k.shape[3]
    G = n_heads // n_kv
    n_pages = k.shape[0] if n_pages is None else n_pages
    rows = q.shape[0]
    out = np.full((rows, n_heads * hd), np.nan)
    tol = np.zeros_like(out)
    for s in range(len(past)):
        n = start[s + 1] - start[s]
        total = past[s] + n
        slots = np.arange(total)
        slots = slots[slots < table.shape[1] * PAGE]
        pages = table[s][slots // PAGE]
        have = (pages >= 0) & (pages < n_pages)
        for h in range(n_kv):
            kk = np.zeros((total, hd))
            vv = np.zeros((total, hd))
            kk[slots[have]] = k[pages[have], h, slots[have] % PAGE]
            vv[slots[have]] = v[pages[have], h, slots[have] % PAGE]
            exist = np.zeros(total, bool)
            exist[slots[have]] = True
            for r in range(n):
                row = start[s] + r
                ok = allowed(kind, r, past[s], n, None if masks is None else masks[row]) & exist
                for g in range(G):
                    col = slice((h * G + g) * hd, (h * G + g + 1) * hd)
                    if not ok.any():
                        out[row, col] = 0.0
                        continue
                    qq = q[row, col].astype(np.float64)
                    sc = kk[ok] @ qq * scale
                    w = np.exp(sc - sc.max())
                    w /= w.sum()
                    out[row, col] = w @ vv[ok]
                    ds = abs(scale) * (np.abs(kk[ok]) @ np.abs(qq)).max() * (2.0 ** -21 + hd * 2.0 ** -24)
                    tol[row, col] = (2 * ds + 2.0 ** -19) * 2 * (w @ np.abs(vv[ok])) + np.abs(vv).max() * 2.0 ** -37
    return out, tol


class Case:
    """Queries, a shuffled page pool and the index arrays of one call."""

    def __init__(self, H, KV, hd, rows, past, seed, spare=2, poison=True):
        rng = np.random.default_rng(seed)
        self.H, self.KV, self.hd = H, KV, hd
        self.rows, self.past = list(rows), list(past)
        S = len(rows)
        need = [-(-(p + r) // PAGE) for p, r in zip(past, rows)]
        self.stride = max(max(need), 1)
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((S, self.stride), -1, np.int32)
        at = 0
        for s in range(S):
            self.table[s, : need[s]] = order[at: at + need[s]]
            at += need[s]
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.T = int(self.start[-1])
        self.q = rng.normal(0, 1.2, (self.T, H * hd)).astype(np.float32)
        self.k = rng.normal(0.3, 1.0, (self.n_pages, KV, PAGE, hd)).astype(np.float32)
        self.v = rng.normal(0, 1.0, (self.n_pages, KV, PAGE, hd)).astype(np.float32)
        if poison:  # what no sequence owns: NaN and infinities
            used = np.zeros((self.n_pages, PAGE), bool)
            for s in range(S):
                for t in range(past[s] + rows[s]):
                    used[self.table[s, t // PAGE], t % PAGE] = True
            bad = np.where(rng.random((self.n_pages, PAGE)) < 0.5, np.nan, np.inf).astype(np.float32)
            for a in (self.k, self.v):
                a[:] = np.where(used[:, None, :, None], a, bad[:, None, :, None])
        self.scale = 1.0 / np.sqrt(hd)


def random_parents(rng, n):
    return [int(rng.integers(-1, i)) if i else -1 for i in range(n)]


def masks_of(parents, words):
    m = np.zeros((len(parents), words), np.uint64)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i // 64] |= np.uint64(1 << (i % 64))
    return m


def sample(logits, temperature, top_k, top_p, min_p, u):
    """One row's token in 64 bits, by sorting."""
    lg = np.asarray(logits, np.float32)
    ids = np.flatnonzero(~np.isnan(lg))
    if ids.size == 0:
        return 0
    ids = ids[np.lexsort((ids, -lg[ids].astype(np.float64)))]
    if not temperature > 0 or not np.isfinite(lg[ids[0]]):
        return int(ids[0])
    n = ids.size if top_k <= 0 else min(int(top_k), ids.size)
    with np.errstate(invalid="ignore"):
        x = (lg[ids[:n]].astype(np.float64) - float(lg[ids[0]])) / float(np.float32(temperature))
    p = np.exp(x)
    mp = min(float(np.float32(min_p)), 1.0) if min_p > 0 else 0.0
    p = p[p >= mp]
    c = np.cumsum(p)
    if top_p < 1:
        c = c[: int(np.searchsorted(c, float(np.float32(top_p)) * c[-1], side="left")) + 1]
    return int(ids[min(int(np.searchsorted(c, float(np.float32(u)) * c[-1], side="left")), c.size - 1)])
