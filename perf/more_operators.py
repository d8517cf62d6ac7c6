"""The operators of the paged KV cache, as a user's program calls them, with a plain form and an exact one.

The cache holds the K and V of several layers and sequences in pages of 16, 32, 64 or 128 positions, in binary16 or
bfloat16: [layer][page][kv_head][position in the page][128]. A table [sequence][max_pages] (int32, -1: none) says which page
holds which positions, and `refs` how many entries of the table name a page (0: it is free). Operators:

  append   new rows are stored at their positions' pages (paged_append)
  attn     causal grouped-query attention of a chunk of new tokens over the pages (paged_attn): single tokens and prompts
  fork     a step of forked sequences: each takes over another one's pages up to a length (paged_fork), and gets pages of
           its own for its next tokens, copies of shared ones that it goes on in among them (paged_reserve)
  compact  a change of sequences: the oldest ones' pages are freed (paged_fork), the others move together at the
           pool's start (paged_compact), new sequences get pages (paged_reserve)

Heads have 128 dimensions, as in every model that the framework runs. Positions without a page are not seen.
"""
import math
import os
import sys

import torch

own = False

DIM = 128
# (query heads, KV heads) of the model shapes that the framework's benchmark and tests use
HEADS = [(12, 2), (16, 2), (28, 4), (40, 8)]
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_module = None


def _library():
    global _module
    if _module is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "-1.7-atlas---apollo_b200", "python"))
        import atlas_cuda
        _module = atlas_cuda
    return _module


# What a case says: `tokens` new tokens of each of `nseq` sequences at position `pos` (attn and append: `ragged` ones are at
# other places, with fewer tokens), `page` positions a page; `shared`: the first positions, whose pages all sequences have in
# common; `window`: how many positions before its last a sequence still has pages for (0: all); `layers` of the pool;
# `change`: how many sequences are replaced (compact), or how many there are to fork from (fork)
_BASE = dict(type="bf16", nseq=1, q_heads=28, kv_heads=4, page=64, tokens=1, pos=0, ragged=False, shared=0, window=0, layers=1,
             change=0)


def listed():
    return [dict(_BASE, **c) for c in [
        # a decode step of the 7B shape stores one position: launch latency
        dict(name="append 1 token, 4 heads", op="append", type="fp16", page=16, pos=517, layers=2),
        # the long-context workload's prompt (14B shape) stored at once: memory bandwidth
        dict(name="append 8192 tokens, 8 heads", op="append", q_heads=40, kv_heads=8, tokens=8192),
        # a step of eight beams in four of the 7B shape's layers, behind the benchmark's prompt: latency
        dict(name="fork 8 beams, 639", op="fork", type="fp16", nseq=8, pos=639, layers=4, change=3),
        # 48 answers to one long prompt whose end lies inside a page, in six layers of the 14B shape: copies
        dict(name="fork 48 answers, 8155", op="fork", nseq=48, q_heads=40, kv_heads=8, tokens=257, pos=8155, layers=6, change=1),
        # two of eight short sequences make room for others
        dict(name="compact 8 seqs, 300", op="compact", type="fp16", nseq=8, q_heads=16, kv_heads=2, page=16, tokens=300, layers=2,
             change=2),
        # a quarter of 32 sequences of odd length, four layers of the 14B shape: memory bandwidth
        dict(name="compact 32 seqs, 2001", op="compact", nseq=32, q_heads=40, kv_heads=8, tokens=2001, layers=4, change=8),
        # the middle of the 7B benchmark's decode (512 prompt positions, then 256): latency
        dict(name="decode 7B, 640", op="attn", type="fp16", page=16, pos=640),
        # the eight-sequence workload's decode, sequences of different lengths behind a common prompt
        dict(name="decode 8 seqs, 2303", op="attn", nseq=8, q_heads=40, kv_heads=8, page=32, pos=2303, ragged=True, shared=512),
        # eight sequences at the end of a full context: memory bandwidth
        dict(name="decode 8 seqs, 32767", op="attn", nseq=8, q_heads=40, kv_heads=8, pos=32767),
        # a few proposed tokens of each sequence at a time, whose pages behind a window have been freed
        dict(name="chunk 7 over 8001", op="attn", type="fp16", nseq=4, q_heads=40, kv_heads=8, tokens=7, pos=8001, window=4096),
        # the long-context workload's prompt: the tensor cores
        dict(name="prompt 14B, 8192", op="attn", q_heads=40, kv_heads=8, tokens=8192),
        # a second turn: two prompts of odd lengths over pages that are there already (3B shape)
        dict(name="prompt 333 over 5001", op="attn", type="fp16", nseq=2, q_heads=16, kv_heads=2, page=128, tokens=333, pos=5001,
             ragged=True),
    ]]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    while True:
        q_heads, kv_heads = rng.choice(HEADS + [(rng.randint(1, 8) * 2, 2), (spread(1, 16), 1)])
        c = dict(_BASE, op=rng.choice(["append", "fork", "compact", "attn", "attn", "attn"]), type=rng.choice(["fp16", "bf16"]),
                 q_heads=q_heads, kv_heads=kv_heads, page=rng.choice([16, 32, 64, 128]))
        if c["op"] in ("append", "attn"):
            c.update(nseq=spread(1, 16), pos=spread(1, 32768) - 1, ragged=rng.random() < 0.5, layers=rng.choice([1, 1, 2]))
            if c["op"] == "append" or rng.random() < 0.6:
                c["tokens"] = spread(1, 8192)
            if c["op"] == "attn" and c["nseq"] > 1 and rng.random() < 0.3:
                c["shared"] = rng.randint(0, c["pos"])
            if c["op"] == "attn" and rng.random() < 0.2:
                c["window"] = rng.randint(1, c["pos"] + 1)
            total = c["pos"] + c["tokens"]
            if total > 32768 or c["nseq"] * kv_heads * total * c["layers"] > 64 * 32768:
                continue
            if c["op"] == "append" and c["nseq"] * kv_heads * c["tokens"] > 8 * 8192:
                continue
            if c["op"] == "attn" and c["tokens"] > 1 and c["nseq"] * q_heads * c["tokens"] * total > 40 * 8192 * 8192 // 4:
                continue
        elif c["op"] == "fork":
            c.update(nseq=spread(2, 48), tokens=spread(1, 257), pos=spread(1, 8192), layers=spread(1, 6))
            c["change"] = rng.randint(1, min(4, c["nseq"]))
            if rng.random() < 0.3:
                c["window"] = rng.randint(1, c["pos"])
            if c["layers"] * kv_heads * (c["change"] * c["pos"] + c["nseq"] * (c["tokens"] + 2 * c["page"])) > 6 * 8 * 27000:
                continue
        else:
            c.update(nseq=spread(2, 48), tokens=spread(1, 4096), layers=spread(1, 6))
            c["change"] = rng.randint(1, c["nseq"] // 2)
            if c["layers"] * kv_heads * c["nseq"] * (c["tokens"] + c["page"]) > 4 * 8 * 32 * 2048:
                continue
        return c


def _lengths(case):
    """(first position, tokens) of each sequence: ragged batches end at different places, with pieces of different lengths."""
    n, t, p = case["nseq"], case["tokens"], case["pos"]
    if not case["ragged"]:
        return [(p, t)] * n
    return [(max(0, p - (s * (p // 3 + 1)) // n), max(1, t - (s * (t // 2)) // n)) for s in range(n)]


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    n, kvh, page, t, op = case["nseq"], case["kv_heads"], case["page"], case["tokens"], case["op"]
    kind = TYPES[case["type"]]
    lens = _lengths(case)
    width = -(-(case["pos"] + t) // page) + 1
    rnd = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    s = dict(case=dict(case), page=page, tokens=t, lens=lens, layer=case["layers"] - 1)
    s["pos0"], s["ntok"] = ints([p for p, _ in lens]), ints([m for _, m in lens])
    col = torch.arange(width, device="cuda")
    if op in ("append", "attn"):
        # entry j of a sequence: page number in a random order; the common prefix is the first sequence's
        end = s["pos0"] + s["ntok"]
        there = (col * page < end.view(n, 1))
        common = (col + 1) * page <= min([case["shared"]] + [p for p, _ in lens])
        if case["window"]:   # the pages that end before the window of the sequence's first new token are gone
            there &= (col + 1) * page > (s["pos0"] + 1 - case["window"]).view(n, 1)
        mine = there & (~common | (torch.arange(n, device="cuda") == 0).view(n, 1))
        count = sum(-(-(p + m) // page) for p, m in lens) + 3
        order = torch.randperm(count, generator=g, device="cuda")
        number = order[(mine.view(-1).long().cumsum(0) - 1).clamp(min=0)].view(n, width)
        table = torch.where(common, number[0], number)
        # a common page that the first sequence has freed is nobody's
        there &= ~common | there[0]
    elif op == "fork":
        # `change` sequences of `pos` positions; the others are to be made
        roots = case["change"]
        there = (col * page < case["pos"]) & (torch.arange(n, device="cuda") < roots).view(n, 1)
        pages = -(-case["pos"] // page)
        # room for what they hold, and for the new ends and copies of all
        count = roots * pages + n * (-(-t // page) + 2) + 5
        order = torch.randperm(count, generator=g, device="cuda")
        table = order[(there.view(-1).long().cumsum(0) - 1).clamp(min=0)].view(n, width)
        s["parent"] = torch.randint(0, roots, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["parent"][:roots] = torch.arange(roots, device="cuda", dtype=torch.int32)
        s["length"] = ints([case["pos"]] * n)
        s["first"] = ints([max(0, case["pos"] + 1 - case["window"]) if case["window"] else 0] * n)
        s["short"] = ints([0])
    else:
        # sequences of `tokens` positions; the newest `change` ones have the last pages, as the change before left them
        pages, new = -(-t // page), case["change"]
        there = (col * page < t).expand(n, width)
        count = n * pages + 3
        order = torch.cat([torch.randperm((n - new) * pages, generator=g, device="cuda"),
                           torch.arange((n - new) * pages, n * pages, device="cuda")])
        table = order[(there.reshape(-1).long().cumsum(0) - 1).clamp(min=0)].view(n, width)
        s["parent"] = ints([i + new if i + new < n else -1 for i in range(n)])
        s["length"] = ints([t] * n)
        s["pos0"] = ints([0] * n)
        s["ntok"] = ints([t if i + new >= n else 0 for i in range(n)])
        s["short"], s["used"] = ints([0]), ints([0])
    s["table"] = torch.where(there, table, -1).to(torch.int32).contiguous()
    s["refs"] = _counts(s["table"], count)
    shape = (case["layers"], count, kvh, page, DIM)
    s["k"], s["v"] = torch.empty(shape, dtype=kind, device="cuda"), torch.empty(shape, dtype=kind, device="cuda")
    # keys have a few strong dimensions
    strong = torch.exp(0.5 * rnd(DIM))
    for layer in range(case["layers"]):
        s["k"][layer].copy_(rnd(*shape[1:]).mul_(strong))
        s["v"][layer].copy_(rnd(*shape[1:]))
    if op == "append":
        s["new_k"] = rnd(n, t, kvh, DIM).mul_(strong).to(kind)
        s["new_v"] = rnd(n, t, kvh, DIM).to(kind)
    elif op == "attn":
        s["q"] = rnd(n, t, case["q_heads"], DIM).mul_(0.9).to(kind)
        s["out"] = torch.zeros(n, t, case["q_heads"], DIM, dtype=kind, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        # the descriptor of the cache that a program keeps beside it, with the calls' workspace
        s["cache"] = _library().PagedCache(s["k"], s["v"], s["table"], s["refs"])
    return s


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        lib = _library()
        if op == "append":
            lib.paged_append(s["cache"], s["layer"], s["tokens"], s["pos0"], s["new_k"], s["new_v"], n_tok=s["ntok"])
        elif op == "attn":
            lib.paged_attn(s["cache"], s["layer"], s["case"]["q_heads"], s["tokens"], s["pos0"], s["q"], s["out"],
                           n_tok=s["ntok"])
        elif op == "fork":
            lib.paged_fork(s["cache"], s["parent"], s["length"], first=s["first"])
            lib.paged_reserve(s["cache"], s["tokens"], s["length"], s["short"])
        else:
            lib.paged_fork(s["cache"], s["parent"], s["length"])
            lib.paged_compact(s["cache"], s["used"])
            lib.paged_reserve(s["cache"], s["tokens"], s["pos0"], s["short"], n_tok=s["ntok"])
    elif op == "append":
        _append(s)
    elif op == "attn":
        s["out"] = _attn(s)
    elif op == "fork":
        _fork(s, s["first"])
        _reserve(s, s["length"], torch.full_like(s["length"], s["tokens"]))
    else:
        _fork(s, torch.zeros_like(s["length"]))
        _compact(s)
        _reserve(s, s["pos0"], s["ntok"])
    if op == "attn":
        return s["out"]
    if op == "append":
        return {"k": s["k"], "v": s["v"]}
    return {name: s[name] for name in ("k", "v", "table", "refs", "short", "used") if name in s}


# ------------------------------------------------------------------ the plain forms


def _counts(entries, pages):
    """How many entries name each page."""
    at = torch.where(entries >= 0, entries, pages).long().view(-1)
    return torch.zeros(pages + 1, dtype=torch.int32, device=at.device).index_add_(
        0, at, torch.ones_like(at, dtype=torch.int32))[:pages].contiguous()


def _append(s):
    n, width = s["table"].shape
    t = torch.arange(s["tokens"], device="cuda")
    pos = s["pos0"].view(n, 1).long() + t
    entry = s["table"].gather(1, (pos // s["page"]).clamp(max=width - 1)).long()
    ok = (t < s["ntok"].view(n, 1)) & (pos < width * s["page"]) & (entry >= 0)
    ok &= s["refs"][entry.clamp(min=0)] <= 1
    i, j = ok.nonzero(as_tuple=True)
    where = (s["layer"], entry[i, j], slice(None), pos[i, j] % s["page"])
    s["k"][where] = s["new_k"][i, j]
    s["v"][where] = s["new_v"][i, j]


def _fork(s, first):
    n, width = s["table"].shape
    parent, at = s["parent"].long(), torch.arange(width, device="cuda") * s["page"]
    keep = ((parent >= 0) & (parent < n)).view(n, 1) & (at < s["length"].view(n, 1)) & (at + s["page"] > first.view(n, 1))
    s["table"].copy_(torch.where(keep, s["table"][parent.clamp(0, n - 1)], -1))
    s["refs"].copy_(_counts(s["table"], s["refs"].numel()))


def _reserve(s, pos0, ntok):
    table, refs, page = s["table"], s["refs"], s["page"]
    n, width = table.shape
    pages = refs.numel()
    col = torch.arange(width, device="cuda")
    write = (col >= (pos0 // page).view(n, 1)) & (col * page < (pos0 + ntok).view(n, 1)) & (ntok > 0).view(n, 1)
    has = table >= 0
    at = torch.where(write & has, table, pages).long()
    writers = _counts(torch.where(write & has, table, -1), pages)
    key = torch.arange(n * width, device="cuda").view(n, width)
    last = torch.full((pages + 1,), -1, device="cuda").scatter_reduce_(0, at.view(-1), key.view(-1), "amax")
    # a page that only entries of this call name stays the last one's
    old = table.clamp(min=0).long()
    keeps = has & (refs[old] == writers[old]) & (last[old] == key)
    need = write & ~keeps
    lack = (need.sum() - (refs == 0).sum()).clamp(min=0)
    s["short"].copy_(lack.view(1))
    free = (refs != 0).sort(stable=True).indices
    fresh = free[(need.view(-1).long().cumsum(0) - 1).clamp(0, pages - 1)].view(n, width)
    need &= lack == 0
    # the rows before the first new one move along
    rows = pos0 % page
    copy = need & has & (col == (pos0 // page).view(n, 1)) & (rows > 0).view(n, 1)
    i, j = copy.nonzero(as_tuple=True)
    src, dst = old[i, j], fresh[i, j]
    keep = (torch.arange(page, device="cuda") < rows[i].view(-1, 1)).view(-1, 1, page, 1)
    for name in ("k", "v"):
        s[name][:, dst] = torch.where(keep, s[name][:, src], s[name][:, dst])
    table.copy_(torch.where(need, fresh, table.long()))
    refs.copy_(_counts(table, pages))


def _compact(s):
    table, refs = s["table"], s["refs"]
    number = torch.arange(refs.numel(), device="cuda")
    used = (refs > 0).sum()
    src = ((refs > 0) & (number >= used)).nonzero().view(-1)
    dst = ((refs == 0) & (number < used)).nonzero().view(-1)
    for name in ("k", "v"):
        s[name][:, dst] = s[name][:, src]
    now = number.clone()
    now[src] = dst
    table.copy_(torch.where(table >= 0, now[table.clamp(min=0).long()], -1))
    refs.copy_(_counts(table, refs.numel()))
    s["used"].copy_(used.view(1))


def _attn(s):
    q, page = s["q"], s["page"]
    n, t, qh, _ = q.shape
    kvh = s["k"].shape[2]
    blocks = -(-max(p + m for p, m in s["lens"]) // page)
    table = s["table"][:, :blocks].long()
    length = blocks * page

    def values(pool):   # [n, kvh, length, 128]
        x = pool[s["layer"]].index_select(0, table.clamp(min=0).view(-1)).view(n, blocks, kvh, page, DIM)
        return x.transpose(1, 2).reshape(n, kvh, length, DIM).float()

    rows = q.view(n, t, kvh, qh // kvh, DIM).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, DIM).float()
    score = torch.matmul(rows, values(s["k"]).transpose(2, 3)).mul_(1.0 / math.sqrt(DIM)).view(n, kvh, qh // kvh, t, length)
    at = s["pos0"].view(n, 1) + torch.arange(t, device="cuda")
    hidden = torch.arange(length, device="cuda") > at.view(n, 1, 1, t, 1)
    hidden = hidden | (table < 0).repeat_interleave(page, 1).view(n, 1, 1, 1, length)
    score.masked_fill_(hidden, -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = score.sum(-1)
    out = torch.matmul(score.view(n, kvh, -1, length), values(s["v"])).view(n, kvh, qh // kvh, t, DIM)
    out.div_(torch.where(total > 0, total, torch.ones_like(total)).unsqueeze(-1))   # rows that see nothing: zeros
    out = out.permute(0, 3, 1, 2, 4).reshape(n, t, qh, DIM).to(q.dtype)
    there = torch.arange(t, device="cuda") < s["ntok"].view(n, 1)
    return torch.where(there.view(n, t, 1, 1), out, s["out"])


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    lens, page, kvh, qh, n = _lengths(case), case["page"], case["kv_heads"], case["q_heads"], case["nseq"]
    row = kvh * DIM * 2 * 2   # K and V of a position
    bytes_, flops = 0.0, 0.0
    width = -(-(case["pos"] + case["tokens"]) // page) + 1
    if case["op"] == "append":
        for _, m in lens:
            bytes_ += 2 * m * row + 4 * (m // page + 1)
            flops += m
    elif case["op"] == "attn":
        common = min([case["shared"]] + [p for p, _ in lens]) // page * page
        for i, (p, m) in enumerate(lens):
            gone = max(0, p + 1 - case["window"]) // page * page if case["window"] else 0
            lost = common if i else 0
            bytes_ += max(0, p + m - max(gone, lost)) * row + 2 * m * qh * DIM * 2 + 4 * -(-(p + m) // page)
            flops += 4.0 * DIM * qh * (m * (p - gone) + m * (m + 1) // 2)
    else:
        # the tables before and after, the counts, and the rows that move in every layer
        bytes_ += 2 * 4 * n * width + 2 * 4 * n * -(-(case["pos"] + case["tokens"]) // page)
        if case["op"] == "fork":
            moved = (n - case["change"]) * (case["pos"] % page)
        else:
            moved = case["change"] * -(-case["tokens"] // page) * page
        bytes_ += 2.0 * moved * row * case["layers"]
        flops += n * width
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------ the definitions, in 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "attn":
        return _exact_attn(case, s)
    if case["op"] == "append":
        out = {"k": s["k"].double(), "v": s["v"].double()}
        table = s["table"].tolist()
        refs = s["refs"].tolist()
        for i, (p, m) in enumerate(s["lens"]):
            for j in range(p // case["page"], (p + m - 1) // case["page"] + 1):
                at = table[i][j]
                if at < 0 or refs[at] > 1:
                    continue
                lo, hi = max(p, j * case["page"]), min(p + m, (j + 1) * case["page"])
                to = slice(lo - j * case["page"], hi - j * case["page"])
                for name in ("k", "v"):
                    out[name][s["layer"], at, :, to] = s["new_" + name][i, lo - p:hi - p].double().transpose(0, 1)
        return out
    return _exact_pages(case, s)


def _exact_pages(case, s):
    """The pages' contents after the calls, page by page."""
    page, n = case["page"], case["nseq"]
    rows = {i: [e for e in r] for i, r in enumerate(s["table"].tolist())}
    parent = s["parent"].tolist()
    first = s["first"].tolist() if "first" in s else [0] * n
    pools = [s["k"].double(), s["v"].double()]
    after = {}
    for i in range(n):
        after[i] = [-1] * len(rows[0])
        if 0 <= parent[i] < n:
            for j, e in enumerate(rows[parent[i]]):
                if j * page < int(s["length"][i]) and (j + 1) * page > first[i]:
                    after[i][j] = e
    pages = s["refs"].numel()

    def names():
        count = [0] * pages
        for r in after.values():
            for e in r:
                if e >= 0:
                    count[e] += 1
        return count

    if case["op"] == "compact":
        count = names()
        total = sum(1 for x in count if x)
        holes = [p for p in range(total) if not count[p]]
        high = [p for p in range(total, pages) if count[p]]
        to = dict(zip(high, holes))
        for p in pools:
            for a, b in to.items():
                p[:, b] = p[:, a]
        after = {i: [to.get(e, e) for e in r] for i, r in after.items()}
    pos0 = s["length"].tolist() if case["op"] == "fork" else s["pos0"].tolist()
    ntok = [case["tokens"]] * n if case["op"] == "fork" else s["ntok"].tolist()
    # one entry after the other: a page is left while someone else names it, so the last of its writers keeps it
    count = names()
    free = [p for p in range(pages) if not count[p]]
    for i in range(n):
        for j in range(pos0[i] // page, -(-(pos0[i] + ntok[i]) // page) if ntok[i] else 0):
            e = after[i][j]
            if e >= 0 and count[e] == 1:
                continue
            if not free:
                return None
            to = free.pop(0)
            if e >= 0:
                count[e] -= 1
                if j * page < pos0[i]:
                    for p in pools:
                        p[:, to, :, :pos0[i] % page] = p[:, e, :, :pos0[i] % page]
            count[to] += 1
            after[i][j] = to
    return {"k": pools[0], "v": pools[1], "table": None, "refs": None, "short": None, "used": None}


def _exact_attn(case, s):
    out = s["out"].double().clone()
    page, group = case["page"], case["q_heads"] // case["kv_heads"]
    for i, (p, m) in enumerate(s["lens"]):
        entry = s["table"][i, torch.arange(p + m, device="cuda") // page].long()
        seen = (entry >= 0).nonzero().view(-1)                      # the positions that have a page
        for h in range(case["kv_heads"]):
            k = s["k"][s["layer"], entry[seen], h, seen % page].double()
            v = s["v"][s["layer"], entry[seen], h, seen % page].double()
            for t0 in range(0, m, 1024):
                t1 = min(m, t0 + 1024)
                w = torch.einsum("tgd,ld->tgl", s["q"][i, t0:t1, h * group:(h + 1) * group].double(), k) / math.sqrt(DIM)
                after = seen.view(1, 1, -1) > torch.arange(p + t0, p + t1, device="cuda").view(-1, 1, 1)
                w = torch.softmax(w.masked_fill(after, -math.inf), -1).nan_to_num(0.0)
                out[i, t0:t1, h * group:(h + 1) * group] = w @ v
    return out
