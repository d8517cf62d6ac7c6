"""GPU: the paged KV cache's calls at what their documentation allows and the other tests do not reach: values that are not finite
behind the chunk, weights that vanish, scores of -infinity, queries and outputs in one buffer, up to 4096 sequences."""
import pytest

import atlas_cuda
from paged_ref import DIM, TYPES, RefPaged, attend
from test_gpu_paged import Dev
from test_gpu_paged_attn import Setup, _i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("tokens,at", [(1, 400), (1, 399), (1, 40), (1, 0), (3, 40), (9, 130), (9, 402), (150, 0), (150, 300), (400, 40), (400, 399), (400, 400)])
def test_what_is_not_finite_in_the_cache(torch_cuda, kind, tokens, at):
    """A NaN or infinity among the values or the keys of a position behind the chunk, or of its first token: all rows from it on
    have it, and nothing else changes."""
    torch = torch_cuda
    x = Setup(torch, kind, 16, 2, [400 + tokens], 60, seed=tokens)
    q = x.rand(1, tokens, 10, DIM)
    clean = x.attn(q, [400])
    e, r = int(x.table[0, at // 16]), at % 16
    x.v[0, e, 0, r, 3] = float("inf")
    x.v[0, e, 0, r, 77] = float("nan")
    x.k[0, e, 1, r, 5] = float("nan")
    out = x.attn(q, [400])
    t = max(0, at - 400)
    assert torch.equal(out[0, :t], clean[0, :t])
    got, was = (y[0, t:].view(-1, 2, 5, DIM) for y in (out, clean))
    want = torch.ones_like(got, dtype=torch.bool)
    want[:, 0, :, 3] = want[:, 0, :, 77] = False
    want[:, 1] = False
    assert torch.equal(got.isfinite(), want)
    assert torch.equal(got[want], was[want])


def _halves(torch, x, high, strength=4.0):
    """Keys of the positions where `high` is true point along the queries, the others against them: weights there are 2^-1000."""
    n = high.numel()
    pos = torch.arange(n, device="cuda")
    e = x.table[0].long()[pos // x.page]
    x.k[0, e, :, pos % x.page] = torch.where(high, strength, -strength).view(n, 1, 1).to(x.kind).expand(n, x.k.shape[2], DIM)
    return e


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("tokens", [1, 3, 40, 300])
@pytest.mark.parametrize("pos,at", [(400, 3), (400, 200), (400, 300), (210, 3), (210, 200)])
def test_a_vanishing_weight_hides_nothing(torch_cuda, kind, tokens, pos, at):
    """Where a row's weight of a position is 0 in 32 bits, an infinite value there still shows: in a tile of keys of its own, next
    to such with all the weight, before and behind them."""
    torch = torch_cuda
    x = Setup(torch, kind, 16, 1, [pos + tokens], 60, seed=tokens)
    p = torch.arange(pos + tokens, device="cuda")
    e = _halves(torch, x, (p // 128 != at // 128) & (p // 16 != at // 16))
    q = (8.0 + x.rand(1, tokens, 5, DIM).float().abs()).to(x.kind)
    clean = x.attn(q, [pos])
    assert bool(clean.isfinite().all())
    x.v[0, e[at], 0, at % 16, 3] = float("inf")
    out = x.attn(q, [pos])
    assert not bool(out[..., 3].isfinite().any())
    keep = [d for d in range(DIM) if d != 3]
    assert torch.equal(out[..., keep], clean[..., keep])


@pytest.mark.parametrize("first", [True, False])
def test_a_vanishing_weight_in_a_long_piece(torch_cuda, first):
    """The same where a CTA's piece is so long that it is summed in several steps."""
    torch = torch_cuda
    nseq, kvh, pos, tokens = 16, 8, 40000, 20
    x = Setup(torch, "bf16", 128, kvh, [pos + tokens] * nseq, -(-(pos + tokens) // 128), seed=1, poison=False)
    at = 5 if first else 33000
    p = torch.arange(pos + tokens, device="cuda")
    e = _halves(torch, x, p // 32768 != at // 32768)
    q = (8.0 + x.rand(nseq, tokens, kvh, DIM).float().abs()).to(x.kind)
    clean = x.attn(q, [pos] * nseq)
    x.v[0, e[at], 0, at % 128, 3] = float("inf")
    out = x.attn(q, [pos] * nseq)
    assert not bool(out[0, :, 0, 3].isfinite().any())
    out[0, :, 0, 3] = clean[0, :, 0, 3]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("tokens", [1, 3, 40, 300])
def test_scores_of_minus_infinity(torch_cuda, kind, tokens):
    """A position whose score is -infinity has no weight; rows that have no other score are zeros."""
    torch = torch_cuda
    pos, at = 300, 150
    x = Setup(torch, kind, 32, 1, [pos + tokens], 40, seed=6)
    q = x.rand(1, tokens, 4, DIM).abs() + 0.125
    x.k[0, int(x.table[0, at // 32]), 0, at % 32, 7] = float("-inf")
    out = x.attn(q, [pos])
    one_term = atlas_cuda.paged_attn_form(x.c, 4, tokens) >= 128
    for t in {0, tokens // 2, tokens - 1}:
        p = torch.tensor([i for i in range(pos + t + 1) if i != at], device="cuda")
        e = x.table[0].long()[p // 32]
        k, v = (y[0, e, 0, p % 32].unsqueeze(1) for y in (x.k, x.v))
        want, bound = attend(q[0, t], k, v, torch.arange(p.numel(), device="cuda"), 1, p.numel() - 1, one_term)
        assert bool(((out[0, t].double() - want).abs() <= bound).all())
    x.k[0, x.table[0, :-(-(pos + tokens) // 32)].long(), 0, :, 7] = float("-inf")
    assert int(x.attn(q, [pos]).count_nonzero()) == 0


@pytest.mark.parametrize("tokens", [1, 3, 60, 300])
def test_queries_and_outputs_in_one_buffer(torch_cuda, tokens):
    """Side by side in a fused buffer; overlapping ones are refused and leave it as it was."""
    torch = torch_cuda
    heads = 6
    x = Setup(torch, "fp16", 32, 2, [90 + tokens, 200 + tokens], 20, seed=2)
    wide = x.rand(2, tokens, 2 * heads + 1, DIM)
    q, ld, pos = wide[:, :, :heads], (2 * heads + 1) * DIM, [90, 200]
    want = x.attn(q.contiguous(), pos)
    before = wide.clone()
    for first in (0, 1, heads - 1):
        with pytest.raises(atlas_cuda.AtlasError):
            x.attn(q, pos, out=wide[:, :, first:first + heads], ldq=ld, ldo=ld)
    torch.cuda.synchronize()
    assert torch.equal(wide, before)
    for first in (heads, heads + 1):
        x.attn(q, pos, out=wide[:, :, first:first + heads], ldq=ld, ldo=ld)
        assert torch.equal(wide[:, :, first:first + heads], want)
        wide[:, :, first:first + heads] = before[:, :, first:first + heads]
        assert torch.equal(wide, before)


@pytest.mark.parametrize("kind,nseq,kvh,grp,tokens,width", [("bf16", 4096, 1, 2, 1, 5), ("fp16", 4096, 2, 5, 3, 4), ("bf16", 1000, 2, 4, 2, 600), ("fp16", 300, 4, 7, 1, 12),
                                                           ("bf16", 129, 1, 8, 40, 8), ("fp16", 4095, 1, 1, 17, 5), ("bf16", 64, 4, 7, 1, 300)])
def test_many_sequences(torch_cuda, kind, nseq, kvh, grp, tokens, width):
    """Up to as many sequences as a cache may have, of all lengths, some without rows."""
    torch = torch_cuda
    page = 32
    room = min(width, 30) * page - tokens
    pos = [(s * 37) % room for s in range(nseq)]
    ntok = [(s * 7) % (tokens + 1) if s % 3 else tokens for s in range(nseq)]
    x = Setup(torch, kind, page, kvh, [p + n for p, n in zip(pos, ntok)], width, seed=nseq)
    q = x.rand(nseq, tokens, kvh * grp, DIM)
    out = x.attn(q, pos, ntok)
    assert torch.equal(out, x.attn(q, pos, ntok))
    here = torch.arange(tokens, device="cuda") < _i32(torch, ntok).view(nseq, 1)
    assert bool((out[~here] == 7.0).all()) and bool(out[here].isfinite().all())
    one_term = atlas_cuda.paged_attn_form(x.c, kvh * grp, tokens) >= 128
    for s in sorted({0, 1, 31, 32, 33, nseq // 2, nseq - 2, nseq - 1} | set(range(5, nseq, nseq // 23))):
        for t in {0, ntok[s] // 2, ntok[s] - 1} if ntok[s] else ():
            for h in range(kvh):
                want, bound = attend(q[s, t, h * grp:(h + 1) * grp], x.k[0, :, h], x.v[0, :, h], x.table[s], page, pos[s] + t, one_term)
                assert bool(((out[s, t, h * grp:(h + 1) * grp].double() - want).abs() <= bound).all()), (s, t, h)


@pytest.mark.parametrize("nseq", [4096, 1025])
def test_pages_of_many_sequences(torch_cuda, nseq):
    """Every call that changes the table, with as many sequences as a cache may have."""
    torch = torch_cuda
    ref = RefPaged("bf16", 1, 3 * nseq + 5, 1, 16, nseq, 3, seed=1)
    dev = Dev(torch, ref)
    pos, ntok = [0] * nseq, [(s * 5) % 33 for s in range(nseq)]
    short = torch.full((1,), 9, dtype=torch.int32, device="cuda")

    def reserve():
        want = ref.reserve(pos, ntok)
        atlas_cuda.paged_reserve(dev.c, max(ntok), _i32(torch, pos), short, n_tok=_i32(torch, ntok))
        assert int(short) == want == 0
        k = torch.randn(nseq, max(ntok), 1, DIM).to(TYPES["bf16"])
        ref.append(0, pos, ntok, k, k)
        atlas_cuda.paged_append(dev.c, 0, max(ntok), _i32(torch, pos), k.cuda(), k.cuda(), n_tok=_i32(torch, ntok))
        dev.equals(torch, ref)

    reserve()
    parent = [(s * 11) % nseq if s % 4 else s for s in range(nseq)]
    length = [ntok[p] for p in parent]
    ref.fork(parent, length)
    atlas_cuda.paged_fork(dev.c, _i32(torch, parent), _i32(torch, length))
    dev.equals(torch, ref)
    pos, ntok = length, [s % 3 for s in range(nseq)]
    reserve()
    assert ref.compact() == (atlas_cuda.paged_compact(dev.c, short), int(short))[1]
    dev.equals(torch, ref)
