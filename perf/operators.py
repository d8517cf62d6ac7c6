"""The operators of the 8-bit KV cache, as a user's program calls them, with a plain form and an exact one.

The cache holds K and V as int8 codes [seq][kv_head][max_context][128] with one fp32 scale for each block of
positions and KV head (values are code * scale), and for each block the sums of its K codes. Four operators:

  append   new fp32 rows are quantised into the cache (kv8_append), and the touched blocks are read back as the
           values that they now stand for (kv8_read)
  attn     causal grouped-query attention over the cache (kv8_attn): single tokens and prompts
  sparse   the same over the blocks that a cheap score selects for each token and KV head (kv8_attn_sparse)

Heads have 128 dimensions, as in every model that the framework runs.
"""
import math
import os
import sys

import torch

own = False

DIM = 128
# (query heads, KV heads) of the model shapes that the framework's benchmark and tests use
HEADS = [(12, 2), (16, 2), (28, 4), (40, 8)]
_module = None


def _library():
    global _module
    if _module is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "-1.7-atlas---apollo_b200", "python"))
        import atlas_cuda
        _module = atlas_cuda
    return _module


def listed():
    return [
        # a decode step of the 7B shape stores one position: launch latency
        dict(name="append 1 token, 4 heads", op="append", nseq=1, q_heads=28, kv_heads=4, block=64, tokens=1, pos=517,
             ragged=False, select=0),
        # the long-context workload's prompt (14B shape) stored at once: memory bandwidth
        dict(name="append 8192 tokens, 8 heads", op="append", nseq=1, q_heads=40, kv_heads=8, block=64, tokens=8192,
             pos=0, ragged=False, select=0),
        # prompt pieces of eight sequences of odd lengths behind caches that end inside a block
        dict(name="append 8 ragged pieces", op="append", nseq=8, q_heads=40, kv_heads=8, block=32, tokens=257,
             pos=2047, ragged=True, select=0),
        # the middle of the 7B benchmark's decode (512 prompt positions, then 256): launch latency
        dict(name="decode 7B, 640", op="attn", nseq=1, q_heads=28, kv_heads=4, block=64, tokens=1, pos=640,
             ragged=False, select=0),
        # the long-context workload's decode
        dict(name="decode 14B, 8447", op="attn", nseq=1, q_heads=40, kv_heads=8, block=64, tokens=1, pos=8447,
             ragged=False, select=0),
        # the eight-sequence workload's decode, sequences of different lengths
        dict(name="decode 8 seqs, 2303", op="attn", nseq=8, q_heads=40, kv_heads=8, block=32, tokens=1, pos=2303,
             ragged=True, select=0),
        # eight sequences at the end of a full context: memory bandwidth
        dict(name="decode 8 seqs, 32767", op="attn", nseq=8, q_heads=40, kv_heads=8, block=64, tokens=1, pos=32767,
             ragged=False, select=0),
        # the 7B benchmark's prompt
        dict(name="prompt 7B, 512", op="attn", nseq=1, q_heads=28, kv_heads=4, block=64, tokens=512, pos=0,
             ragged=False, select=0),
        # the long-context workload's prompt: the tensor cores
        dict(name="prompt 14B, 8192", op="attn", nseq=1, q_heads=40, kv_heads=8, block=64, tokens=8192, pos=0,
             ragged=False, select=0),
        # a second turn: two prompts of odd lengths over caches that are there already (3B shape)
        dict(name="prompt 333 over 5001", op="attn", nseq=2, q_heads=16, kv_heads=2, block=128, tokens=333, pos=5001,
             ragged=True, select=0),
        # one token against 32 of the 512 blocks of a full context
        dict(name="sparse decode, 32767", op="sparse", nseq=1, q_heads=40, kv_heads=8, block=64, tokens=1, pos=32767,
             ragged=False, select=32),
        # a piece of a prompt, each token with blocks of its own
        dict(name="sparse 129 over 8001", op="sparse", nseq=2, q_heads=28, kv_heads=4, block=32, tokens=129, pos=8001,
             ragged=True, select=16),
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    while True:
        q_heads, kv_heads = rng.choice(HEADS + [(rng.randint(1, 8) * 2, 2), (spread(1, 8), 1)])
        c = dict(op=rng.choice(["append", "attn", "attn", "attn", "sparse"]), nseq=spread(1, 8), q_heads=q_heads,
                 kv_heads=kv_heads, block=rng.choice([16, 32, 64, 128]), tokens=1, pos=spread(1, 32768) - 1,
                 ragged=rng.random() < 0.5, select=0)
        if c["op"] == "append" or rng.random() < 0.5:
            c["tokens"] = spread(1, 8192 if c["op"] != "sparse" else 256)
        if c["op"] == "sparse":
            c["select"] = spread(1, 64)
        total = c["pos"] + c["tokens"]
        if total > 32768:
            continue
        if c["op"] == "append" and c["nseq"] * c["kv_heads"] * c["tokens"] > 8 * 8192:
            continue
        if c["op"] == "attn" and c["tokens"] > 1 and c["nseq"] * q_heads * c["tokens"] * total > 40 * 8192 * 8192 // 4:
            continue
        if c["op"] == "sparse" and c["nseq"] * kv_heads * c["tokens"] * c["select"] * c["block"] > 1 << 22:
            continue
        return c


def _lengths(case):
    """(first position, tokens) of each sequence: ragged batches end at different places, with pieces of different lengths."""
    n, t, p = case["nseq"], case["tokens"], case["pos"]
    if not case["ragged"]:
        return [(p, t)] * n
    return [(max(0, p - (s * (p // 3 + 1)) // n), max(1, t - (s * (t // 2)) // n)) for s in range(n)]


def _context(case):
    return case["pos"] + case["tokens"] + 13


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    n, kvh, b, t, ctx = case["nseq"], case["kv_heads"], case["block"], case["tokens"], _context(case)
    nblk = -(-ctx // b)
    lens = _lengths(case)
    rnd = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731

    def codes():
        # a Gaussian whose block maximum, about four deviations, is at the end of the code range; blocks have means of their own
        c = rnd(n, kvh, nblk, b, DIM).mul_(28.0).add_(rnd(n, kvh, nblk, 1, DIM).mul_(12.0))
        return c.round_().clamp_(-127, 127).to(torch.int8).view(n, kvh, nblk * b, DIM)

    s = dict(case=dict(case), block=b, tokens=t, lens=lens)
    k, v = codes(), codes()
    s["k_scale"] = torch.exp(0.25 * rnd(n, kvh, nblk)).mul_(0.035)
    s["v_scale"] = torch.exp(0.5 * rnd(n, kvh, nblk)).mul_(0.01)
    pos0 = torch.tensor([p for p, _ in lens], dtype=torch.int32, device="cuda")
    ntok = torch.tensor([m for _, m in lens], dtype=torch.int32, device="cuda")
    end = pos0 if case["op"] == "append" else pos0 + ntok
    live = torch.arange(nblk * b, device="cuda") < end.view(n, 1)
    s["k_sum"] = (k * live.view(n, 1, -1, 1)).view(n, kvh, nblk, b, DIM).sum(3, dtype=torch.int32).to(torch.int16)
    s["k"], s["v"] = k[:, :, :ctx].contiguous(), v[:, :, :ctx].contiguous()
    s["pos0"], s["ntok"] = pos0, ntok
    if case["op"] == "append":
        # keys have a few strong dimensions; some rows raise the scale of the block that they join
        strong = torch.exp(0.6 * rnd(DIM))
        s["new_k"] = rnd(n, t, kvh, DIM).mul_(strong).mul_(torch.exp(0.3 * rnd(n, t, kvh, 1)))
        s["new_v"] = rnd(n, t, kvh, DIM).mul_(torch.exp(0.3 * rnd(n, t, kvh, 1))).mul_(0.3)
        # the touched blocks: from the start of the block that the first new row joins
        s["first"] = pos0 - pos0 % b
        s["count"] = pos0 % b + ntok
        s["span"] = max(p % b + m for p, m in lens)
        # where the window of touched blocks has rows, and blocks, that the call writes: (sequence, place in the window)
        wide = torch.arange(-(-s["span"] // b) * b, device="cuda") < s["count"].view(n, 1)
        s["rows"] = wide.nonzero(as_tuple=True)
        s["blocks"] = wide.view(n, -1, b).any(2).nonzero(as_tuple=True)
        s["k_out"] = torch.zeros(n, s["span"], kvh, DIM, device="cuda")
        s["v_out"] = torch.zeros_like(s["k_out"])
    else:
        s["q"] = rnd(n, t, case["q_heads"], DIM).mul_(0.9)
        s["out"] = torch.zeros(n, t, case["q_heads"], DIM, device="cuda")
        if case["op"] == "sparse":
            s["sel"] = torch.full((n, t, kvh, case["select"]), -1, dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        # the descriptor of the cache that a program keeps beside it
        s["cache"] = _library().Kv8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_sum"], nseq=case["nseq"],
                                         kv_heads=case["kv_heads"], max_context=_context(case), block=case["block"])
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        lib, s = _library(), state
        if op == "append":
            lib.kv8_append(s["cache"], s["tokens"], s["pos0"], s["new_k"], s["new_v"], n_tok=s["ntok"])
            lib.kv8_read(s["cache"], s["span"], s["first"], s["k_out"], s["v_out"], n_tok=s["count"])
            return {"k": s["k_out"], "v": s["v_out"], "k_scale": s["k_scale"], "v_scale": s["v_scale"],
                    "k_sum": s["k_sum"]}
        if op == "attn":
            lib.kv8_attn(s["cache"], s["case"]["q_heads"], s["tokens"], s["pos0"], s["q"], s["out"], n_tok=s["ntok"])
            return s["out"]
        lib.kv8_attn_sparse(s["cache"], s["case"]["q_heads"], s["tokens"], s["case"]["select"], s["pos0"], s["q"],
                            s["out"], s["sel"], n_tok=s["ntok"])
        return {"out": s["out"], "sel": s["sel"]}
    return {"append": _append, "attn": _attn, "sparse": _sparse}[op](state)


# ------------------------------------------------------------------ the plain forms


def _store(s, codes, scale, rows):
    """Quantises rows [n, t, kvh, 128] into codes / scale in place; what the touched blocks then stand for, and their codes."""
    n, kvh, ctx, _ = codes.shape
    b, span = s["block"], s["span"]
    nb = -(-span // b)
    dev = codes.device
    at = torch.arange(nb * b, device=dev)                                   # row of the window of touched blocks
    off = (s["pos0"] % b).view(n, 1)
    old = at < off                                                          # [n, nb * b]
    new = (at >= off) & (at < s["count"].view(n, 1))
    pos = s["first"].view(n, 1) + at
    inside = pos.clamp(max=ctx - 1).long()
    seq = torch.arange(n, device=dev).view(n, 1)
    x = rows[seq, (at - off).clamp(0, rows.shape[1] - 1)].masked_fill(~new.view(n, -1, 1, 1), 0.0)
    x = x.permute(0, 2, 1, 3).reshape(n, kvh, nb, b, DIM)                   # [n, kvh, nb, b, 128]
    c = codes[seq, :, inside].permute(0, 2, 1, 3).reshape(n, kvh, nb, b, DIM)
    blk = (s["first"].view(n, 1) // b + torch.arange(nb, device=dev)).clamp(max=scale.shape[2] - 1).long()
    was = scale[seq, :, blk].permute(0, 2, 1)                               # [n, kvh, nb]
    was = torch.where(old.view(n, 1, nb, b).any(3), was, torch.zeros_like(was))
    now = torch.maximum((x.abs().amax((3, 4)).double() / 127.0).float(), was)
    step = now.double().view(n, kvh, nb, 1, 1)
    step = torch.where(step > 0, step, torch.ones_like(step))
    fresh = (x.double() / step).round().clamp(-127, 127)
    kept = torch.where((now > was).view(n, kvh, nb, 1, 1), (c.double() * was.double().view(n, kvh, nb, 1, 1) / step).round(),
                       c.double())
    live = (old | new).view(n, 1, nb, b, 1)
    c = torch.where(new.view(n, 1, nb, b, 1), fresh, kept) * live
    c8 = c.to(torch.int8).view(n, kvh, nb * b, DIM)
    i, j = s["rows"]
    codes[i, :, pos[i, j].long()] = c8[i, :, j]
    i, j = s["blocks"]
    scale[i, :, blk[i, j]] = now[i, :, j]
    value = (c.float() * now.view(n, kvh, nb, 1, 1)).view(n, kvh, nb * b, DIM).permute(0, 2, 1, 3)
    return value[:, :span].contiguous(), c, blk


def _append(s):
    k, c, blk = _store(s, s["k"], s["k_scale"], s["new_k"])
    i, j = s["blocks"]
    s["k_sum"][i, :, blk[i, j]] = c.sum(3).to(torch.int16)[i, :, j]
    v, _, _ = _store(s, s["v"], s["v_scale"], s["new_v"])
    return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"], "k_sum": s["k_sum"]}


def _values(codes, scale, block, length):
    return codes[:, :, :length].float().mul_(scale.repeat_interleave(block, 2)[:, :, :length, None])


def _softmax_(x):
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    return x.div_(x.sum(-1, keepdim=True))


def _rows(s, out):
    """`out` where the sequence has that token, the buffer's own rows elsewhere."""
    n, t = out.shape[:2]
    there = torch.arange(t, device=out.device) < s["ntok"].view(n, 1)
    return torch.where(there.view(n, t, 1, 1), out, s["out"])


def _attn(s):
    q, b = s["q"], s["block"]
    n, t, qh, _ = q.shape
    kvh = s["k"].shape[1]
    length = max(p + m for p, m in s["lens"])
    k, v = _values(s["k"], s["k_scale"], b, length), _values(s["v"], s["v_scale"], b, length)
    rows = q.view(n, t, kvh, qh // kvh, DIM).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, DIM)
    score = torch.matmul(rows, k.transpose(2, 3)).mul_(1.0 / math.sqrt(DIM)).view(n, kvh, qh // kvh, t, length)
    at = s["pos0"].view(n, 1) + torch.arange(t, device=q.device)
    hidden = torch.arange(length, device=q.device) > at.view(n, 1, 1, t, 1)
    p = _softmax_(score.masked_fill_(hidden, -math.inf))
    out = torch.matmul(p.view(n, kvh, -1, length), v).view(n, qh, t, DIM).transpose(1, 2)
    return _rows(s, out.contiguous())


def _choose(s):
    """The blocks of each token and KV head, ascending, -1 behind them: its own block and the highest scores before it."""
    q, b, m = s["q"], s["block"], s["case"]["select"]
    n, t, qh, _ = q.shape
    kvh, nblk = s["k_scale"].shape[1:]
    pooled = q.double().view(n, t, kvh, qh // kvh, DIM).sum(3).transpose(1, 2)              # [n, kvh, t, 128]
    most = pooled.abs().amax(3, keepdim=True)
    code = (127.0 * pooled / torch.where(most > 0, most, torch.ones_like(most))).round()
    score = torch.matmul(code, s["k_sum"].double().transpose(2, 3)) * s["k_scale"].double().unsqueeze(2)
    mine = ((s["pos0"].view(n, 1) + torch.arange(t, device=q.device)) // b).view(n, 1, t, 1)
    before = torch.arange(nblk, device=q.device) < mine
    order = score.masked_fill_(~before, -math.inf).sort(dim=3, descending=True, stable=True).indices[..., : m - 1]
    far = 1 << 30
    order = torch.where(order < mine, order, far)
    sel = torch.cat([order, mine.expand(n, kvh, t, 1)], 3).sort(dim=3).values
    if sel.shape[3] < m:
        sel = torch.nn.functional.pad(sel, (0, m - sel.shape[3]), value=far)
    return torch.where(sel == far, -1, sel)


def _sparse(s):
    q, b, m = s["q"], s["block"], s["case"]["select"]
    n, t, qh, _ = q.shape
    kvh, ctx = s["k"].shape[1:3]
    sel = _choose(s)                                                                          # [n, kvh, t, m]
    at = (s["pos0"].view(n, 1) + torch.arange(t, device=q.device)).view(n, 1, t, 1)
    pos = (sel.unsqueeze(4) * b + torch.arange(b, device=q.device)).view(n, kvh, t, m * b)
    ok = (sel.unsqueeze(4) >= 0).expand(n, kvh, t, m, b).reshape(n, kvh, t, m * b) & (pos <= at)
    i, h = torch.arange(n, device=q.device).view(n, 1, 1, 1), torch.arange(kvh, device=q.device).view(1, kvh, 1, 1)
    row, blk = pos.clamp(0, ctx - 1), sel.clamp(min=0)
    k = s["k"][i, h, row].float().mul_(s["k_scale"][i, h, blk].repeat_interleave(b, 3).unsqueeze(4))
    v = s["v"][i, h, row].float().mul_(s["v_scale"][i, h, blk].repeat_interleave(b, 3).unsqueeze(4))
    rows = q.view(n, t, kvh, qh // kvh, DIM).transpose(1, 2)                                  # [n, kvh, t, group, 128]
    score = torch.matmul(rows, k.transpose(3, 4)).mul_(1.0 / math.sqrt(DIM)).masked_fill_(~ok.unsqueeze(3), -math.inf)
    out = torch.matmul(_softmax_(score), v).transpose(1, 2).reshape(n, t, qh, DIM)
    there = torch.arange(t, device=q.device).view(1, t, 1, 1) < s["ntok"].view(n, 1, 1, 1)
    sel = torch.where(there, sel.transpose(1, 2).to(torch.int32), s["sel"])
    return {"out": _rows(s, out), "sel": sel}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    lens, b, kvh, qh = _lengths(case), case["block"], case["kv_heads"], case["q_heads"]
    bytes_, flops = 0.0, 0.0
    for p, m in lens:
        if case["op"] == "append":
            rows, old = m * kvh * DIM * 2, (p % b) * kvh * DIM * 2
            touched = (p % b + m + b - 1) // b
            # new rows in, their codes out, the joined block's codes, scales and sums, and the values read back
            bytes_ += rows * 5 + old + touched * kvh * (2 * 4 + DIM * 2) + (rows + old) * 4
            flops += 2 * rows
        elif case["op"] == "attn":
            keys = m * p + m * (m + 1) // 2
            bytes_ += (p + m) * kvh * DIM * 2 + -(-(p + m) // b) * kvh * 8 + 2 * m * qh * DIM * 4
            flops += 4.0 * DIM * qh * keys
        else:
            cand, mine = (p + m - 1) // b, min(case["select"], (p + m - 1) // b + 1)
            read = min(p + m, m * mine * b)
            bytes_ += cand * kvh * (DIM * 2 + 4) + read * kvh * DIM * 2 + 2 * m * qh * DIM * 4 + m * kvh * mine * 4
            flops += 2.0 * DIM * m * kvh * cand + 4.0 * DIM * m * qh * mine * b
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------ the definitions, in 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "sparse": _exact_sparse}[case["op"]](case, s)


def _exact_append(case, s):
    b = case["block"]
    got = {}
    for name in ("k", "v"):
        out = torch.zeros(s["k_out"].shape, dtype=torch.float64, device="cuda")
        scales = s[name + "_scale"].double().clone()
        for i, (p, m) in enumerate(s["lens"]):
            first, done = p - p % b, 0
            while done < m:                                    # one block after the other
                at = p + done
                take = min(m - done, b - at % b)
                rows = s["new_" + name][i, done:done + take].double()                       # [take, kvh, 128]
                blk, kept = at // b, at % b
                scale = (rows.abs().amax((0, 2)) / 127.0).float().double()                   # a scale is held in 32 bits
                before = s[name][i, :, blk * b:blk * b + kept].double()                      # [kvh, kept, 128]
                if kept:
                    was = s[name + "_scale"][i, :, blk].double()
                    scale = torch.maximum(scale, was)
                    moved = torch.round(before * was.view(-1, 1, 1) / scale.view(-1, 1, 1))
                    before = torch.where((scale > was).view(-1, 1, 1), moved, before)
                    lo = blk * b - first
                    out[i, lo:lo + kept] = (before * scale.view(-1, 1, 1)).transpose(0, 1)
                lo = at - first
                out[i, lo:lo + take] = torch.round(rows / scale.view(1, -1, 1)) * scale.view(1, -1, 1)
                scales[i, :, blk] = scale
                done += take
        got[name], got[name + "_scale"] = out, scales
    got["k_sum"] = None
    return got


def _exact_head(q, codes, scale, at, b):
    """Attention of the rows q [t, group, 128] at positions `at` [t] over all of codes [length, 128], in 64 bits."""
    length = codes.shape[0]
    hidden = torch.arange(length, device=q.device).view(1, 1, -1) > at.view(-1, 1, 1)
    blk = torch.arange(length, device=q.device) // b
    k, v = codes.double() * scale[0].double()[blk, None], scale[1][:length].double() * scale[2].double()[blk, None]
    w = torch.einsum("tgd,ld->tgl", q.double(), k) / math.sqrt(DIM)
    return torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v


def _exact_attn(case, s):
    out = s["out"].double().clone()
    group = case["q_heads"] // case["kv_heads"]
    for i, (p, m) in enumerate(s["lens"]):
        for h in range(case["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            for t0 in range(0, m, 1024):
                t1 = min(m, t0 + 1024)
                at = torch.arange(p + t0, p + t1, device="cuda")
                out[i, t0:t1, heads] = _exact_head(s["q"][i, t0:t1, heads], s["k"][i, h, :p + t1],
                                                   (s["k_scale"][i, h], s["v"][i, h], s["v_scale"][i, h]), at,
                                                   case["block"])
    return out


def _exact_sparse(case, s):
    b, group = case["block"], case["q_heads"] // case["kv_heads"]
    out = s["out"].double().clone()
    for i, (p, m) in enumerate(s["lens"]):
        if m * case["kv_heads"] * len(s["lens"]) > 20000:
            return None
        for h in range(case["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            q = s["q"][i, :m, heads].double()
            pooled = q.sum(1)
            code = torch.round(127.0 * pooled / pooled.abs().amax(1, keepdim=True))
            score = (code @ s["k_sum"][i, h].double().T) * s["k_scale"][i, h].double()
            # a block is taken if fewer than select - 1 of those before the token's own stand higher
            mine = torch.arange(p, p + m, device="cuda") // b
            num = torch.arange(score.shape[1], device="cuda")
            score = score.masked_fill(num >= mine[:, None], -math.inf)
            rank = score.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
            taken = ((rank < case["select"] - 1) & (num < mine[:, None])) | (num == mine[:, None])
            where = torch.arange(p + m, device="cuda")
            seen = taken[:, where // b] & (where <= torch.arange(p, p + m, device="cuda")[:, None])
            k = s["k"][i, h, :p + m].double() * s["k_scale"][i, h].double()[where // b, None]
            v = s["v"][i, h, :p + m].double() * s["v_scale"][i, h].double()[where // b, None]
            w = torch.einsum("tgd,ld->tgl", q, k) / math.sqrt(DIM)
            out[i, :m, heads] = torch.softmax(w.masked_fill(~seen[:, None], -math.inf), -1) @ v
    return {"out": out, "sel": None}
