"""The 8-bit KV cache's definitions in 64 bits (numpy, CPU): what the tests of the kernels compare with."""
import numpy as np

DIM = 128


class RefCache:
    """int8 codes, fp32 scales and sums of codes, written row by row as atlas_cuda_kv8_append defines."""

    def __init__(self, nseq, kv_heads, ctx, block, rng=None):
        nblk = -(-ctx // block)
        self.shape = (nseq, kv_heads, ctx, block, nblk)
        r = rng or np.random.default_rng(0)
        # memory that nothing was stored in yet: any bits
        self.k, self.v = (r.integers(-128, 128, (nseq, kv_heads, ctx, DIM)).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (r.standard_normal((nseq, kv_heads, nblk)).astype(np.float32) for _ in range(2))
        self.ksum = r.integers(-9, 9, (nseq, kv_heads, nblk, DIM)).astype(np.int16)

    def append(self, pos0, ntok, k, v):
        """k, v [nseq, tokens, kv_heads, 128]."""
        nseq, heads, ctx, b, _ = self.shape
        for s in range(nseq):
            p, n = int(pos0[s]), min(int(ntok[s]), k.shape[1])
            end = min(p + n, ctx)
            at = p
            while at < end:
                blk, stop = at // b, min(end, (at // b + 1) * b)
                for codes, scales, rows in ((self.k, self.ks, k), (self.v, self.vs, v)):
                    for h in range(heads):
                        self._store(codes[s, h], scales[s, h], blk, at, stop, rows[s, at - p:stop - p, h], b)
                for h in range(heads):
                    self.ksum[s, h, blk] = self.k[s, h, blk * b:stop].astype(np.int64).sum(0)
                at = stop

    @staticmethod
    def _store(codes, scales, blk, at, stop, x, b):
        old = slice(blk * b, at)
        was = scales[blk] if at > blk * b else np.float32(0)
        if not np.isfinite(x).all() or np.isnan(was):
            scales[blk] = np.nan
            codes[at:stop] = 0
            return
        now = max(np.float32(np.float64(np.abs(x).max()) / 127.0), was)
        if now > was and at > blk * b:
            codes[old] = np.rint(codes[old].astype(np.float64) * np.float64(was) / np.float64(now)).astype(np.int8)
        scales[blk] = now
        q = np.zeros_like(x, dtype=np.float64) if now == 0 else np.rint(x.astype(np.float64) / np.float64(now))
        codes[at:stop] = np.clip(q, -127, 127).astype(np.int8)

    def values(self, s, h, n):
        b = self.shape[3]
        blk = np.arange(n) // b
        with np.errstate(invalid="ignore"):
            return (self.k[s, h, :n].astype(np.float64) * self.ks[s, h].astype(np.float64)[blk, None],
                    self.v[s, h, :n].astype(np.float64) * self.vs[s, h].astype(np.float64)[blk, None])


def attend(q, k, v, seen):
    """Rows q [r, 128] over k, v [n, 128] where seen [r, n]: the output and a bound of an fp32-level computation's error.

    The bound counts, with u = 2^-24: q as three int8 planes and its scale, 4 u max|q| per element; the score's own
    roundings, 8 u of the largest score; each weight, exp's argument and value and the two binary16 terms, 16 u; and
    sums of n terms, of which a warp adds every 32nd in order (tensor cores may truncate: 2 u each), (n / 32 + 8) 2 u.
    A score off by E changes a weight by the factor exp(+-E) and the sum likewise."""
    u = 2.0 ** -24
    s = q @ k.T / np.sqrt(DIM)
    s = np.where(seen, s, -np.inf)
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    out = w @ v
    size = np.abs(q).max(1) * np.where(seen, np.abs(k).sum(1)[None], 0).max(1) / np.sqrt(DIM)
    top = np.abs(np.where(seen, s, 0)).max(1)
    e = 4 * u * size + 8 * u * top
    vmax = np.where(seen, np.abs(v).max(1)[None], 0).max(1)
    bound = vmax * (2 * e + 16 * u + (k.shape[0] / 32 + 8) * 2 * u)
    return out, bound[:, None]


def choose(q, cache, s, h, p, n_sel):
    """The blocks that the query rows q [group, 128] of position p select, ascending."""
    b = cache.shape[3]
    own = p // b
    x = q.astype(np.float64).sum(0)
    top = np.abs(x).max()
    c = np.rint(127.0 * x / top) if 0 < top < np.inf else np.zeros(DIM)
    with np.errstate(invalid="ignore"):
        score = (cache.ksum[s, h, :own].astype(np.float64) @ c) * cache.ks[s, h, :own].astype(np.float64)
    score = np.where(np.isnan(score), np.inf, score)
    order = np.argsort(-score, kind="stable")[:n_sel - 1]
    return np.sort(np.append(order, own))
