"""The paged KV cache's definitions, entry by entry and in 64 bits: what the tests of the kernels compare with."""
import math

import torch

DIM = 128
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


class RefPaged:
    """Pools, table and counts on the CPU, changed entry by entry as include/atlas_cuda.h defines."""

    def __init__(self, kind, layers, pages, kv_heads, page, nseq, max_pages, seed=0):
        g = torch.Generator().manual_seed(seed)
        shape = (layers, pages, kv_heads, page, DIM)
        self.k, self.v = (torch.randn(shape, generator=g).to(TYPES[kind]) for _ in range(2))
        self.table = torch.full((nseq, max_pages), -1, dtype=torch.int32)
        self.refs = torch.zeros(pages, dtype=torch.int32)
        self.page, self.nseq, self.pages, self.max_pages = page, nseq, pages, max_pages

    def _has(self, e):
        return 0 <= e < self.pages

    def _count(self):
        self.refs.zero_()
        for e in self.table.flatten().tolist():
            if self._has(e):
                self.refs[e] += 1

    def fork(self, parent, length, first=None):
        old = self.table.clone()
        for s in range(self.nseq):
            for j in range(self.max_pages):
                p, e = int(parent[s]), -1
                if 0 <= p < self.nseq and j * self.page < int(length[s]) and (j + 1) * self.page > (int(first[s]) if first is not None else 0):
                    e = int(old[p, j])
                self.table[s, j] = e if self._has(e) else -1
        self._count()

    def reserve(self, pos0, ntok):
        """The pages lacking."""
        table, refs, copies = self.table.clone(), self.refs.clone(), []
        free = [p for p in range(self.pages) if refs[p] == 0]
        lacking = 0
        # a page is one's own where nobody else names it any more
        for s in range(self.nseq):
            end = min(int(pos0[s]) + int(ntok[s]), self.max_pages * self.page)
            for j in range(int(pos0[s]) // self.page, -(-end // self.page) if end > int(pos0[s]) else 0):
                e = int(table[s, j])
                if self._has(e) and refs[e] <= 1:
                    continue
                if self._has(e):
                    refs[e] -= 1
                if not free:
                    lacking += 1
                    continue
                to = free.pop(0)
                refs[to] = 1
                table[s, j] = to
                if self._has(e) and j * self.page < int(pos0[s]):
                    copies.append((e, to, int(pos0[s]) % self.page))
        if lacking:
            return lacking
        self.table, self.refs = table, refs
        for e, to, rows in copies:
            for x in (self.k, self.v):
                x[:, to, :, :rows] = x[:, e, :, :rows]
        return 0

    def compact(self):
        """The pages in use."""
        used = [p for p in range(self.pages) if self.refs[p] > 0]
        total = len(used)
        moves = dict(zip([p for p in used if p >= total], [p for p in range(total) if self.refs[p] == 0]))
        for a, b in moves.items():
            for x in (self.k, self.v):
                x[:, b] = x[:, a]
        for s in range(self.nseq):
            for j in range(self.max_pages):
                e = int(self.table[s, j])
                self.table[s, j] = moves.get(e, e)
        self._count()
        return total

    def append(self, layer, pos0, ntok, k, v):
        """k, v [nseq, tokens, kv_heads, 128]."""
        for s in range(self.nseq):
            for t in range(min(int(ntok[s]), k.shape[1])):
                p = int(pos0[s]) + t
                if p >= self.max_pages * self.page:
                    continue
                e = int(self.table[s, p // self.page])
                if self._has(e) and self.refs[e] <= 1:
                    self.k[layer, e, :, p % self.page] = k[s, t]
                    self.v[layer, e, :, p % self.page] = v[s, t]


def attend(q, k_pool, v_pool, entries, page, p, one_term):
    """Attention of one token's query rows q [group, 128] of a KV head, at position p, over the pools [pages, page, 128] through
    the sequence's entries: the output in 64 bits, and a bound of the kernels' error.

    The bound counts, with u = 2^-24 and h the output type's half step (eps / 2): a score's 128 products in fp32 sums that
    tensor cores may truncate, 32 u of the sum of their absolute values, and its scaling, 8 u of the largest score; a score off by E
    changes a weight and the sum of weights by the factor exp(+-E); a weight's exponential 16 u and its own rounding for the
    second product, h (`one_term`) or its square (two terms); the sum of n weighted values, of which at most every 16 are
    truncated together, (n / 16 + 64) 2 u; where weights are binary16, steps of 2^-24 under the largest one's 2^6; and
    the output's rounding, h of it and, for subnormal binary16, 2^-25."""
    h, u = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    pos = torch.arange(min(p + 1, entries.numel() * page), device=q.device)
    e = entries.long()[pos // page]
    ok = (e >= 0) & (e < k_pool.shape[0])
    pos, e = pos[ok], e[ok]
    n = pos.numel()
    if n == 0:
        z = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        return z, z
    k, v, q = k_pool[e, pos % page].double(), v_pool[e, pos % page].double(), q.double()
    s = q @ k.T / math.sqrt(DIM)
    w = torch.softmax(s, -1)
    out, size = w @ v, w @ v.abs()
    e_s = 32 * u * (q.abs() @ k.abs().T).amax(-1, keepdim=True) / math.sqrt(DIM) + 8 * u * s.abs().amax(-1, keepdim=True)
    bound = size * (4 * e_s + 16 * u + (h if one_term else h * h) + (n / 16 + 64) * 2 * u)
    bound = bound + n * 2.0 ** -31 * w.amax(-1, keepdim=True) * v.abs().amax(0, keepdim=True)
    return out, bound + h * (out.abs() + bound) + 2.0 ** -25
