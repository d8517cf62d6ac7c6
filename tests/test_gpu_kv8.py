"""GPU: the 8-bit KV cache (append, read, attention, attention over chosen blocks) against the definitions in 64 bits.

Codes, scales, sums and chosen blocks are equal; attention is within the bound that kv8_ref.attend derives."""
import numpy as np
import pytest

import atlas_cuda
from kv8_ref import DIM, RefCache, attend, choose

pytestmark = pytest.mark.gpu


class DevCache:
    """A RefCache's buffers on the device."""

    def __init__(self, torch, ref, sums=True):
        n, h, ctx, b, _ = ref.shape
        self.t = [torch.from_numpy(x.copy()).cuda() for x in (ref.k, ref.v, ref.ks, ref.vs, ref.ksum)]
        self.c = atlas_cuda.Kv8Cache(*self.t[:4], self.t[4] if sums else None, nseq=n, kv_heads=h, max_context=ctx,
                                     block=b)

    def equals(self, ref):
        for t, x in zip(self.t, (ref.k, ref.v, ref.ks, ref.vs, ref.ksum)):
            np.testing.assert_array_equal(t.cpu().numpy(), x)


def _i32(torch, x):
    return torch.tensor([int(np.uint32(i).view(np.int32)) for i in x], dtype=torch.int32, device="cuda")


def _f32(torch, x):
    return torch.from_numpy(np.array(x, dtype=np.float32, order="C")).cuda()


def filled(rng, nseq, heads, ctx, block, lens, v_spread=0.5, k_size=1.0):
    """A cache whose first lens[s] positions are stored, in blocks of different scales."""
    ref = RefCache(nseq, heads, ctx, block, rng)
    n = max(max(lens), 1)
    grow = lambda a: np.exp(a * rng.standard_normal((nseq, -(-n // block), heads)))[:, np.arange(n) // block]  # noqa: E731
    k = (k_size * rng.standard_normal((nseq, n, heads, DIM)) * grow(0.3)[..., None]).astype(np.float32)
    v = (rng.standard_normal((nseq, n, heads, DIM)) * grow(v_spread)[..., None]).astype(np.float32)
    ref.append([0] * nseq, lens, k, v)
    return ref


# ------------------------------------------------------------- append, read --


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("nseq,heads,ctx,pieces", [
    (1, 1, 40, [(0, 1), (1, 1), (2, 14), (16, 1), (17, 23)]),
    (1, 3, 300, [(0, 299), (299, 1)]),
    (2, 2, 260, [(0, 130), (130, 1), (131, 129)]),
    (1, 2, 200, [(0, 150), (37, 3), (40, 100)]),     # starts again earlier
])
def test_append_equals_the_definition(torch_cuda, block, nseq, heads, ctx, pieces):
    torch = torch_cuda
    rng = np.random.default_rng(block + ctx)
    ref = RefCache(nseq, heads, ctx, block, rng)
    dev = DevCache(torch, ref)
    for p, n in pieces:
        x, y = ((rng.standard_normal((nseq, n, heads, DIM)) * np.exp(rng.standard_normal((nseq, n, heads, 1)))
                 ).astype(np.float32) for _ in range(2))
        ref.append([p] * nseq, [n] * nseq, x, y)
        atlas_cuda.kv8_append(dev.c, n, _i32(torch, [p] * nseq), _f32(torch, x), _f32(torch, y))
        dev.equals(ref)


@pytest.mark.parametrize("block", [16, 128])
def test_append_ragged_strided(torch_cuda, block):
    """Sequences of different lengths (0 and one past the buffer among them), rows inside a wider buffer."""
    torch = torch_cuda
    rng = np.random.default_rng(7)
    nseq, heads, ctx, tokens, ld = 6, 2, 150, 70, 5 * DIM
    ref = RefCache(nseq, heads, ctx, block, rng)
    lens = [0, 3, 64, 100, 0, 17]
    x = rng.standard_normal((nseq, 128, heads, DIM)).astype(np.float32)
    ref.append([0] * nseq, lens, x, x[::-1])
    dev = DevCache(torch, ref)
    ntok = [70, 0, 1, 70, 33, 1000]              # 100 + 70 passes the cache's end, 1000 counts as 70
    wide = rng.standard_normal((nseq, tokens, 5, DIM)).astype(np.float32)
    ref.append(lens, ntok, wide[:, :, 1:3], wide[:, :, 3:5])
    w = _f32(torch, wide)
    atlas_cuda.kv8_append(dev.c, tokens, _i32(torch, lens), w[:, :, 1:], w[:, :, 3:], n_tok=_i32(torch, ntok), ld=ld)
    dev.equals(ref)
    # and back, into a buffer whose other rows stay
    back = torch.full((nseq, tokens, 5, DIM), 7.0, device="cuda")
    atlas_cuda.kv8_read(dev.c, tokens, _i32(torch, lens), back[:, :, 1:], back[:, :, 3:], n_tok=_i32(torch, ntok), ld=ld)
    got = back.cpu().numpy()
    want = np.full_like(got, 7.0)
    for s in range(nseq):
        for i in range(min(ntok[s], tokens)):
            p = lens[s] + i
            for j, (codes, scales) in enumerate(((ref.k, ref.ks), (ref.v, ref.vs))):
                want[s, i, 1 + 2 * j:3 + 2 * j] = (codes[s, :, p].astype(np.float32) * scales[s, :, p // block, None]
                                                   if p < ctx else np.nan)
    np.testing.assert_array_equal(got, want)


def test_append_rounds_ties_to_even_and_clamps(torch_cuda):
    torch = torch_cuda
    x = np.zeros((1, 4, 1, DIM), np.float32)
    x[0, 0, 0, :4] = [127.0, -127.0, 0.5, 1.5]          # scale 1: ties
    x[0, 1, 0, :6] = [2.5, -2.5, 126.5, -126.5, 125.5, np.nextafter(np.float32(2.5), np.float32(3))]
    x[0, 2, 0, :2] = [np.nextafter(np.float32(0.5), np.float32(0)), 1e-38]
    ref = RefCache(1, 1, 16, 16)
    dev = DevCache(torch, ref)
    ref.append([0], [4], x, -x)
    atlas_cuda.kv8_append(dev.c, 4, _i32(torch, [0]), _f32(torch, x), _f32(torch, -x))
    dev.equals(ref)
    assert ref.k[0, 0, 0, 2:4].tolist() == [0, 2] and ref.k[0, 0, 1, :6].tolist() == [2, -2, 126, -126, 126, 3]


@pytest.mark.parametrize("size", [0.0, 1e-45, 1.9e-43, 1e-40, 1.2e-36, 1e30, 3.4e38])
def test_append_extreme_sizes(torch_cuda, size):
    """All zeros, subnormal scales (rounded coarsely: codes are clamped), the largest values; then a larger row."""
    torch = torch_cuda
    rng = np.random.default_rng(5)
    x = np.clip(rng.uniform(-1, 1, (1, 9, 2, DIM)) * size, -3.4e38, 3.4e38).astype(np.float32)
    y = np.clip(np.float64(x[:, :1]) * 2.5, -3.4e38, 3.4e38).astype(np.float32)
    ref = RefCache(1, 2, 16, 16)
    dev = DevCache(torch, ref)
    for p, z in ((0, x), (9, y)):
        ref.append([p], [z.shape[1]], z, z[:, ::-1])
        atlas_cuda.kv8_append(dev.c, z.shape[1], _i32(torch, [p]), _f32(torch, z), _f32(torch, z[:, ::-1]))
        dev.equals(ref)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_non_finite(torch_cuda, bad):
    """A poisoned block stays poisoned until it is stored again from its start; the other blocks are untouched."""
    torch = torch_cuda
    rng = np.random.default_rng(6)
    ref = RefCache(1, 1, 64, 16)
    dev = DevCache(torch, ref)
    x = rng.standard_normal((1, 40, 1, DIM)).astype(np.float32)
    x[0, 20, 0, 77] = bad
    for p, n in ((0, 40), (24, 4), (16, 8)):            # the last call stores the block from its start, without the value
        z = x[:, :n] if p == 0 else rng.standard_normal((1, n, 1, DIM)).astype(np.float32)
        ref.append([p], [n], z, z)
        atlas_cuda.kv8_append(dev.c, n, _i32(torch, [p]), _f32(torch, z), _f32(torch, z))
        dev.equals(ref)
        assert np.isnan(ref.ks[0, 0, 1]) == (p != 16) and np.isfinite(ref.ks[0, 0, [0, 2]]).all()


def test_append_past_the_cache(torch_cuda):
    torch = torch_cuda
    ref = RefCache(2, 1, 30, 16)
    dev = DevCache(torch, ref)
    x = np.ones((2, 3, 1, DIM), np.float32)
    for pos in ([30, 31], [0xffffffff, 0x80000000]):    # nothing is stored
        atlas_cuda.kv8_append(dev.c, 3, _i32(torch, pos), _f32(torch, x), _f32(torch, x))
        dev.equals(ref)
    ref.append([29, 0], [3, 3], x, x)
    atlas_cuda.kv8_append(dev.c, 3, _i32(torch, [29, 0]), _f32(torch, x), _f32(torch, x))
    dev.equals(ref)


# ---------------------------------------------------------------- attention --


def check_attn(torch, rng, ref, q_heads, tokens, pos, ntok=None, n_sel=0, q=None, ldq=0, dev=None):
    """One call against the definition; rows that do not exist stay, positions past the cache give NaN."""
    nseq, heads, ctx, b, _ = ref.shape
    group = q_heads // heads
    dev = dev or DevCache(torch, ref)
    if q is None:
        q = rng.standard_normal((nseq, tokens, q_heads, DIM)).astype(np.float32)
    wide = max(ldq // DIM, q_heads)
    qw = np.full((nseq, tokens, wide, DIM), np.nan, np.float32)
    qw[:, :, :q_heads] = q
    out = torch.full((nseq, tokens, wide, DIM), 7.0, device="cuda")
    sel = torch.full((nseq, tokens, heads, max(n_sel, 1)), -5, dtype=torch.int32, device="cuda")
    n = None if ntok is None else _i32(torch, ntok)
    if n_sel:
        atlas_cuda.kv8_attn_sparse(dev.c, q_heads, tokens, n_sel, _i32(torch, pos), _f32(torch, qw), out, sel, n_tok=n,
                                   ldq=ldq, ldo=ldq)
    else:
        atlas_cuda.kv8_attn(dev.c, q_heads, tokens, _i32(torch, pos), _f32(torch, qw), out, n_tok=n, ldq=ldq, ldo=ldq)
    torch.cuda.synchronize()
    got, sel = out.cpu().numpy(), sel.cpu().numpy()
    assert (got[:, :, q_heads:] == 7.0).all()
    got = got[:, :, :q_heads]
    for s in range(nseq):
        m = tokens if ntok is None else min(ntok[s], tokens)
        assert (got[s, m:] == 7.0).all() and (sel[s, m:] == -5).all()
        for h in range(heads):
            at = pos[s] + np.arange(m)
            past = at >= ctx
            assert np.isnan(got[s, :m][past]).all()
            live = np.flatnonzero(~past)
            if not live.size:
                continue
            end = int(at[live].max()) + 1
            k, v = ref.values(s, h, end)
            seen = np.arange(end)[None] <= at[live, None]
            if n_sel:
                for j, i in enumerate(live):
                    blocks = choose(q[s, i, h * group:(h + 1) * group], ref, s, h, int(at[i]), n_sel)
                    want = np.full(n_sel, -1)
                    want[:len(blocks)] = blocks
                    np.testing.assert_array_equal(sel[s, i, h], want)
                    seen[j] &= np.isin(np.arange(end) // b, blocks)
            rows = q[s, live, h * group:(h + 1) * group].astype(np.float64).reshape(-1, DIM)
            want, bound = attend(rows, k, v, np.repeat(seen, group, 0))
            err = np.abs(got[s, live, h * group:(h + 1) * group].reshape(-1, DIM) - want)
            assert (err <= bound).all(), float((err / bound).max())
            if n_sel:
                assert (sel[s, :m, h][past] == -1).all()
    return got, sel


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("pos", [0, 1, 15, 16, 17, 63, 64, 127, 255, 1000])
def test_decode_lengths(torch_cuda, block, pos):
    rng = np.random.default_rng(pos * 7 + block)
    ref = filled(rng, 1, 2, pos + 1 + pos % 3, block, [pos + 1])
    check_attn(torch_cuda, rng, ref, 14, 1, [pos])


@pytest.mark.parametrize("q_heads,heads", [(1, 1), (2, 2), (6, 2), (5, 1), (7, 1), (8, 1), (9, 1), (24, 2), (16, 1), (33, 1)])
def test_decode_groups(torch_cuda, q_heads, heads):
    rng = np.random.default_rng(q_heads)
    ref = filled(rng, 2, heads, 401, 32, [401, 130])
    check_attn(torch_cuda, rng, ref, q_heads, 1, [400, 129])


@pytest.mark.parametrize("q_heads,heads", [(2, 2), (12, 2), (7, 1)])
@pytest.mark.parametrize("tokens,pos", [(2, 0), (3, 61), (5, 100), (16, 0), (17, 300), (33, 15), (64, 64), (129, 0),
                                        (130, 77), (300, 211)])
def test_prompt_pieces(torch_cuda, q_heads, heads, tokens, pos):
    rng = np.random.default_rng(tokens + pos)
    ref = filled(rng, 1, heads, pos + tokens, 64, [pos + tokens])
    check_attn(torch_cuda, rng, ref, q_heads, tokens, [pos])


@pytest.mark.parametrize("nseq,q_heads,heads,tokens,pos,ctx", [
    (1, 2, 1, 100, 1, 4000),        # one tile of rows, its positions over a cluster
    (1, 8, 1, 40, 1000, 5000),      # two tiles of rows, over a cluster
    (3, 14, 2, 150, 300, 480),      # one tile per CTA, none split
    (5, 40, 8, 60, 77, 140),        # two tiles per CTA, more units than fit at once
    (2, 28, 4, 99, 1500, 1700),     # odd row counts in the last tile
    (1, 130, 1, 3, 400, 500),       # a group larger than a tile of rows
])
def test_prompt_splits(torch_cuda, nseq, q_heads, heads, tokens, pos, ctx):
    rng = np.random.default_rng(ctx)
    at = [pos + 13 * s for s in range(nseq)]
    ref = filled(rng, nseq, heads, ctx, 32, [p + tokens for p in at])
    check_attn(torch_cuda, rng, ref, q_heads, tokens, at)


@pytest.mark.parametrize("block", [16, 32, 128])
def test_prompt_blocks(torch_cuda, block):
    rng = np.random.default_rng(block)
    ref = filled(rng, 1, 1, 400, block, [390])
    check_attn(torch_cuda, rng, ref, 5, 190, [200])


@pytest.mark.parametrize("tokens", [1, 4, 70, 150])
def test_attn_ragged_strided(torch_cuda, tokens):
    """Pieces of different lengths, an idle sequence, rows past the cache's end, rows inside wider buffers."""
    rng = np.random.default_rng(tokens)
    ctx, pos = 500, [0, 310, 499, 33, 128, 500 - tokens // 2]
    ntok = [tokens, max(1, tokens // 2), tokens, 0, tokens + 9, tokens]
    lens = [min(ctx, p + n) for p, n in zip(pos, ntok)]
    ref = filled(rng, 6, 2, ctx, 32, lens)
    check_attn(torch_cuda, rng, ref, 10, tokens, pos, ntok, ldq=13 * DIM)


@pytest.mark.parametrize("tokens", [1, 80])
def test_attn_positions_past_the_cache(torch_cuda, tokens):
    rng = np.random.default_rng(9)
    ref = filled(rng, 3, 1, 70, 16, [70, 70, 70])
    check_attn(torch_cuda, rng, ref, 3, tokens, [70, 0xffffffff, 0x7fffffff])


@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("q_size,k_size,v_spread", [(30.0, 3.0, 0.5), (1e-3, 1.0, 0.5), (1.0, 1.0, 4.0), (1e-30, 1e10, 0.1),
                                                    (1e8, 1e-8, 0.1)])
def test_attn_sizes(torch_cuda, tokens, q_size, k_size, v_spread):
    """Scores in the hundreds, flat ones, V blocks of very different scales, large and tiny queries."""
    rng = np.random.default_rng(11)
    ref = filled(rng, 1, 2, 300, 16, [300], v_spread=v_spread, k_size=k_size)
    q = (q_size * rng.standard_normal((1, tokens, 6, DIM))).astype(np.float32)
    check_attn(torch_cuda, rng, ref, 6, tokens, [300 - tokens], q=q)


@pytest.mark.parametrize("tokens", [1, 100])
def test_attn_zero_blocks_and_queries(torch_cuda, tokens):
    """Blocks of zeros (scale 0) at the start, in the middle and alone; a query of zeros weighs all positions alike."""
    rng = np.random.default_rng(12)
    ref = RefCache(1, 1, 160, 16, rng)
    x = rng.standard_normal((1, 160, 1, DIM)).astype(np.float32)
    x[:, :32] = 0
    x[:, 64:80] = 0
    ref.append([0], [160], x, x)
    q = rng.standard_normal((1, tokens, 4, DIM)).astype(np.float32)
    q[:, :, 1] = 0
    check_attn(torch_cuda, rng, ref, 4, tokens, [160 - tokens], q=q)
    z = RefCache(1, 1, 160, 16, rng)
    z.append([0], [160], 0 * x, 0 * x)
    got, _ = check_attn(torch_cuda, rng, z, 4, tokens, [160 - tokens], q=q)
    assert (got == 0).all()


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("tokens", [1, 100])
def test_attn_non_finite(torch_cuda, where, tokens):
    """A poisoned block shows in the rows that attend to it, and in no other; neither does what lies behind the end."""
    torch = torch_cuda
    rng = np.random.default_rng(13)
    ref = filled(rng, 1, 1, 256, 16, [256])
    (ref.ks if where == "k" else ref.vs)[0, 0, 12] = np.nan          # positions 192 .. 207
    for pos, hit in ((192 - tokens, False), (208, True), (150, tokens > 42)):
        q = rng.standard_normal((1, tokens, 2, DIM)).astype(np.float32)
        out = torch.zeros(1, tokens, 2, DIM, device="cuda")
        atlas_cuda.kv8_attn(DevCache(torch, ref).c, 2, tokens, _i32(torch, [pos]), _f32(torch, q), out)
        got = out.cpu().numpy()[0]
        at = pos + np.arange(tokens)
        inside = at < 256
        assert np.isnan(got[(at >= 192)]).all()
        assert np.isfinite(got[(at < 192) & inside]).all()
        if not hit:
            check_attn(torch, rng, ref, 2, tokens, [pos], q=q)


@pytest.mark.parametrize("tokens", [1, 100])
def test_attn_non_finite_query(torch_cuda, tokens):
    """A query row with a NaN or an infinity gives NaN, the others are as without it."""
    torch = torch_cuda
    rng = np.random.default_rng(14)
    ref = filled(rng, 1, 1, 256, 64, [256])
    q = rng.standard_normal((1, tokens, 4, DIM)).astype(np.float32)
    want, _ = check_attn(torch, rng, ref, 4, tokens, [256 - tokens], q=q)
    q[0, 0, 1, 5], q[0, -1, 2, 100] = np.nan, np.inf
    out = torch.zeros(1, tokens, 4, DIM, device="cuda")
    atlas_cuda.kv8_attn(DevCache(torch, ref).c, 4, tokens, _i32(torch, [256 - tokens]), _f32(torch, q), out)
    got = out.cpu().numpy()
    assert np.isnan(got[0, 0, 1]).all() and np.isnan(got[0, -1, 2]).all()
    ok = np.ones(got.shape[:3], bool)
    ok[0, 0, 1] = ok[0, -1, 2] = False
    np.testing.assert_array_equal(got[ok], want[ok])


def test_attn_many_positions(torch_cuda):
    """More positions than one round of the 32 scales that a warp holds, over all CTAs of a cluster."""
    rng = np.random.default_rng(15)
    ref = filled(rng, 1, 1, 40000, 16, [40000])
    check_attn(torch_cuda, rng, ref, 8, 1, [39999])


@pytest.mark.parametrize("q_heads,tokens,ctx", [
    (64, 300, 3300),      # two tiles of rows per CTA, all positions: three segments of 1024 in tensor memory
    (60, 150, 2500),      # one tile per CTA, the two groups of warps take turns at the keys
    (8, 7, 19000),        # over a cluster
    (1, 150, 20000),
    (64, 60, 12000),
])
@pytest.mark.parametrize("rising", [False, True])
def test_prompt_segments(torch_cuda, q_heads, tokens, ctx, rising):
    """Outputs of more positions than tensor memory sums up at once; scores and V scales that grow along the positions,
    so that maximum and V scale are raised in every segment, at its first tile as well as within."""
    rng = np.random.default_rng(ctx)
    q = rng.standard_normal((1, tokens, q_heads, DIM)).astype(np.float32)
    if not rising:
        ref = filled(rng, 1, 1, ctx, 64, [ctx])
    else:
        q[..., 0] = 4.0
        at = np.arange(ctx) / ctx
        k = 0.1 * rng.standard_normal((1, ctx, 1, DIM)).astype(np.float32)
        k[0, :, 0, 0] = 200.0 * at                # scores up to 70
        v = rng.standard_normal((1, ctx, 1, DIM)).astype(np.float32) * np.exp2(np.rint(12 * at)).astype(np.float32)[:, None, None]
        ref = RefCache(1, 1, ctx, 64, rng)
        ref.append([0], [ctx], k, v)
    check_attn(torch_cuda, rng, ref, q_heads, tokens, [ctx - tokens], q=q)


# Enough units of work for the prompt form also over few positions: 8 sequences, 2 KV heads, 600 rows each.


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_wide_prompts(torch_cuda, block):
    """Pieces of different lengths, an idle sequence, rows past the cache's end, rows inside wider buffers."""
    rng = np.random.default_rng(block)
    ctx, tokens, pos = 300, 150, [0, 150, 77, 33, 299, 128, 200, 0xfffffff0]
    ntok = [150, 150, 149, 0, 150, 1, 190, 150]
    ref = filled(rng, 8, 2, ctx, block, [min(ctx, p + n) for p, n in zip(pos, ntok)])
    check_attn(torch_cuda, rng, ref, 8, tokens, pos, ntok, ldq=11 * DIM)


@pytest.mark.parametrize("q_heads,tokens", [(2, 600), (14, 90), (130, 9)])
def test_wide_prompt_groups(torch_cuda, q_heads, tokens):
    rng = np.random.default_rng(q_heads)
    ref = filled(rng, 8, 2, 640, 32, [640] * 8)
    check_attn(torch_cuda, rng, ref, q_heads, tokens, [640 - tokens - 5 * s for s in range(8)])


@pytest.mark.parametrize("q_size,k_size,v_spread", [(30.0, 3.0, 0.5), (1e-3, 1.0, 0.5), (1.0, 1.0, 4.0), (1e-30, 1e10, 0.1),
                                                    (1e8, 1e-8, 0.1)])
def test_wide_prompt_sizes(torch_cuda, q_size, k_size, v_spread):
    rng = np.random.default_rng(31)
    ref = filled(rng, 8, 2, 300, 16, [300] * 8, v_spread=v_spread, k_size=k_size)
    q = (q_size * rng.standard_normal((8, 150, 8, DIM))).astype(np.float32)
    check_attn(torch_cuda, rng, ref, 8, 150, [150] * 8, q=q)


def test_wide_prompt_zeros_and_non_finite(torch_cuda):
    """Blocks of zeros, queries of zeros; a poisoned block of K or V shows in the rows that attend to it and in no other, a
    query row with a NaN or an infinity is NaN alone."""
    torch = torch_cuda
    rng = np.random.default_rng(32)
    ref = RefCache(8, 2, 300, 16, rng)
    x = rng.standard_normal((8, 300, 2, DIM)).astype(np.float32)
    x[:, :32] = 0
    x[:, 64:80] = 0
    ref.append([0] * 8, [300] * 8, x, x)
    q = rng.standard_normal((8, 150, 8, DIM)).astype(np.float32)
    q[:, :, 1] = 0
    want, _ = check_attn(torch, rng, ref, 8, 150, [100] * 8, q=q)
    ref.ks[2, 0, 12] = ref.vs[3, 1, 12] = np.nan      # positions 192 .. 207: tokens from 92 on
    q[5, 7, 3, 5], q[6, 149, 6, 100] = np.nan, np.inf
    out = torch.zeros(8, 150, 8, DIM, device="cuda")
    atlas_cuda.kv8_attn(DevCache(torch, ref).c, 8, 150, _i32(torch, [100] * 8), _f32(torch, q), out)
    got = out.cpu().numpy()
    bad = np.zeros(got.shape[:3], bool)
    bad[2, 92:, :4] = bad[3, 92:, 4:] = bad[5, 7, 3] = bad[6, 149, 6] = True
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], want[~bad])


@pytest.mark.parametrize("heads,q_heads,tokens", [(2, 2, 1), (1, 1, 200), (1, 64, 300)])
@pytest.mark.parametrize("at", [0, 100, 700, 2100])
def test_attn_of_one_position(torch_cuda, heads, q_heads, tokens, at):
    """One position takes all the weight, every other one rounds to none: the output is its value. With u = 2^-24, off by
    what a segment's sums are made up for though nothing was lost, 4.5e-6 = 75 u, and 24 u for the value's two terms, their
    scales and the states' merges."""
    torch, ctx = torch_cuda, 2500
    rng = np.random.default_rng(20)
    ref = RefCache(1, heads, ctx, 64, rng)
    k = np.zeros((1, ctx, heads, DIM), np.float32)
    k[..., 0] = -1.0
    k[:, at, :, 0] = 1.0
    ref.append([0], [ctx], k, rng.uniform(0.5, 1.0, k.shape).astype(np.float32))
    q = torch.zeros(1, tokens, q_heads, DIM, device="cuda")
    q[..., 0] = 2000.0
    out = torch.zeros_like(q)
    atlas_cuda.kv8_attn(DevCache(torch, ref).c, q_heads, tokens, _i32(torch, [ctx - tokens]), q, out)
    got = out.cpu().numpy().astype(np.float64)[0]
    for h in range(heads):
        want = ref.values(0, h, ctx)[1][at]
        rows = got[:, h * q_heads // heads:(h + 1) * q_heads // heads]
        assert (np.abs(rows / want - 1) <= 99 * 2.0 ** -24).all()


@pytest.mark.parametrize("heads,q_heads,tokens", [(8, 8, 1), (1, 1, 200), (1, 64, 300)])
def test_attn_sums_keep_their_precision(torch_cuda, heads, q_heads, tokens):
    """Equal weights over values of one sign. Relative to the output, with u = 2^-24: tensor cores truncate each of the 128
    sums of a segment (2 u of a sum that grows evenly: 128 u; the mean of that, at most 50 u, is made up for), the weights'
    terms 16 u, their sum and the segments' at most 64 u."""
    torch, ctx = torch_cuda, 8000
    rng = np.random.default_rng(17)
    ref = RefCache(1, heads, ctx, 128, rng)
    x = rng.uniform(0.5, 1.0, (1, ctx, heads, DIM)).astype(np.float32)
    ref.append([0], [ctx], x, x)
    out = torch.zeros(1, tokens, q_heads, DIM, device="cuda")
    atlas_cuda.kv8_attn(DevCache(torch, ref).c, q_heads, tokens, _i32(torch, [ctx - tokens]), torch.zeros_like(out), out)
    got = out.cpu().numpy().astype(np.float64)[0]
    for h in range(heads):
        v = ref.values(0, h, ctx)[1]
        want = (np.cumsum(v, 0) / np.arange(1, ctx + 1)[:, None])[ctx - tokens:]
        rows = got[:, h * q_heads // heads:(h + 1) * q_heads // heads]
        assert (np.abs(rows / want[:, None] - 1) <= 258 * 2.0 ** -24).all()


def test_attn_large_batch(torch_cuda):
    """More units of work than CTAs fit on the device (clusters of one)."""
    rng = np.random.default_rng(16)
    ref = filled(rng, 40, 16, 70, 32, list(range(30, 70)))
    check_attn(torch_cuda, rng, ref, 32, 1, list(range(29, 69)))


# ------------------------------------------------------------ chosen blocks --


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("n_sel", [1, 2, 5, 16, 100])
def test_sparse_decode(torch_cuda, block, n_sel):
    rng = np.random.default_rng(n_sel + block)
    ref = filled(rng, 2, 2, 1500, block, [1500, 700])
    check_attn(torch_cuda, rng, ref, 10, 1, [1499, 699], n_sel=n_sel)


@pytest.mark.parametrize("q_heads,heads", [(1, 1), (16, 2), (28, 4), (24, 2), (40, 1)])
@pytest.mark.parametrize("tokens,pos", [(1, 0), (5, 14), (37, 500)])
def test_sparse_tokens_and_groups(torch_cuda, q_heads, heads, tokens, pos):
    rng = np.random.default_rng(q_heads + tokens)
    ref = filled(rng, 1, heads, pos + tokens + 1, 16, [pos + tokens])
    check_attn(torch_cuda, rng, ref, q_heads, tokens, [pos], n_sel=7)


def test_sparse_many_tokens(torch_cuda):
    """Enough tokens that no clusters are formed."""
    rng = np.random.default_rng(21)
    ref = filled(rng, 2, 2, 900, 32, [900, 400])
    check_attn(torch_cuda, rng, ref, 4, 300, [600, 100], [300, 300], n_sel=4)


@pytest.mark.parametrize("nseq,q_heads,heads,tokens,pos,ctx,block,n_sel", [
    (2, 14, 2, 90, 700, 800, 16, 5),      # 360 units: chosen in one pass, attended in another
    (1, 24, 2, 90, 1000, 1100, 32, 8),    # two tiles of query rows per token
    (1, 4, 4, 100, 0, 100, 16, 3),        # the first tokens have no more blocks than they may choose
    (1, 4, 4, 100, 0, 100, 16, 100),      # nor has any
    (1, 8, 4, 80, 300, 380, 64, 1),       # the own block alone
    (1, 4, 4, 77, 9900, 10000, 16, 7),    # more blocks than a warp's registers hold the keys of
    (1, 8, 8, 43, 60000, 60050, 16, 4),   # more than the first pass takes
])
def test_sparse_many_units(torch_cuda, nseq, q_heads, heads, tokens, pos, ctx, block, n_sel):
    rng = np.random.default_rng(ctx + n_sel)
    at = [pos - 7 * s for s in range(nseq)]
    ref = filled(rng, nseq, heads, ctx, block, [p + tokens for p in at])
    check_attn(torch_cuda, rng, ref, q_heads, tokens, at, n_sel=n_sel)


def test_sparse_many_units_ragged_strided(torch_cuda):
    """Pieces of different lengths, an idle sequence, rows past the cache's end, rows inside wider buffers."""
    rng = np.random.default_rng(18)
    ctx, tokens, ntok, pos = 500, 61, [61, 8, 61, 0, 70], [400, 310, 460, 33, 0xffffffff]
    ref = filled(rng, 5, 2, ctx, 32, [461, 318, 500, 0, 500])
    check_attn(torch_cuda, rng, ref, 10, tokens, pos, ntok, n_sel=6, ldq=13 * DIM)


def test_sparse_many_units_ties_and_poison(torch_cuda):
    """Equal scores go to the lower block, a poisoned block is chosen, and scores of both signs and zero are in order."""
    torch = torch_cuda
    rng = np.random.default_rng(19)
    ref = RefCache(1, 4, 500, 16, rng)
    k = rng.standard_normal((1, 16, 4, DIM)).astype(np.float32)
    sign = np.array([1, -1, 0, 2, 1, 0, -1, 1])
    rows = np.concatenate([k * sign[i % 8] for i in range(32)], 1)[:, :500]
    ref.append([0], [500], rows, rng.standard_normal(rows.shape).astype(np.float32))
    q = rng.standard_normal((1, 90, 8, DIM)).astype(np.float32)
    q[0, 3] = 0                                   # every score 0: the lowest blocks
    check_attn(torch, rng, ref, 8, 90, [400], n_sel=9, q=q)
    ref.ks[0, 1, 17] = np.nan
    sel = torch.zeros(1, 90, 4, 9, dtype=torch.int32, device="cuda")
    out = torch.zeros(1, 90, 8, DIM, device="cuda")
    atlas_cuda.kv8_attn_sparse(DevCache(torch, ref).c, 8, 90, 9, _i32(torch, [400]), _f32(torch, q), out, sel)
    assert (sel[0, :, 1] == 17).any(-1).all() and torch.isnan(out[0, :, 2:4]).all()
    assert torch.isfinite(out[0, :, :2]).all() and torch.isfinite(out[0, :, 4:]).all()


def test_sparse_ragged_strided(torch_cuda):
    rng = np.random.default_rng(22)
    pos, ntok = [0, 310, 499, 33], [6, 2, 3, 0]
    ref = filled(rng, 4, 2, 500, 16, [6, 312, 500, 33])
    check_attn(torch_cuda, rng, ref, 10, 6, pos, ntok, n_sel=3, ldq=11 * DIM)


def test_sparse_ties_go_to_the_lower_block(torch_cuda):
    """A query of zeros (all scores equal), and blocks that repeat."""
    torch = torch_cuda
    rng = np.random.default_rng(23)
    x = np.tile(rng.standard_normal((1, 48, 1, DIM)).astype(np.float32), (1, 20, 1, 1))   # 20 times the same 3 blocks
    ref = RefCache(1, 1, 960, 16, rng)
    ref.append([0], [960], x, x)
    check_attn(torch, rng, ref, 4, 1, [959], n_sel=30)
    _, sel = check_attn(torch, rng, ref, 4, 1, [959], n_sel=9, q=np.zeros((1, 1, 4, DIM), np.float32))
    assert sel[0, 0, 0].tolist() == list(range(8)) + [59]


def test_sparse_scores_of_both_signs_and_zero(torch_cuda):
    """Scores below, at and above zero, and -0 beside 0: a block of zeros has scale 0."""
    rng = np.random.default_rng(24)
    x = rng.standard_normal((1, 640, 1, DIM)).astype(np.float32)
    for b in range(0, 40, 3):
        x[:, 16 * b:16 * b + 16] = 0
    ref = RefCache(1, 1, 640, 16, rng)
    ref.append([0], [640], x, x)
    ref.ksum[0, 0, [6, 12]] = [[-5], [5]]          # a scale of 0 with sums of either sign: equal scores
    for n in range(2, 41, 5):
        check_attn(torch_cuda, rng, ref, 3, 1, [639], n_sel=n)


def test_sparse_poisoned_block_is_chosen(torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(25)
    ref = filled(rng, 1, 1, 640, 16, [640])
    ref.ks[0, 0, 17] = np.nan
    out = torch.zeros(1, 1, 2, DIM, device="cuda")
    sel = torch.zeros(1, 1, 1, 4, dtype=torch.int32, device="cuda")
    q = rng.standard_normal((1, 1, 2, DIM)).astype(np.float32)
    atlas_cuda.kv8_attn_sparse(DevCache(torch, ref).c, 2, 1, 4, _i32(torch, [639]), _f32(torch, q), out, sel)
    assert 17 in sel.cpu().tolist()[0][0][0] and torch.isnan(out).all()
    assert sel.cpu().numpy()[0, 0, 0].tolist() == choose(q[0, 0], ref, 0, 0, 639, 4).tolist()


def test_sparse_past_the_cache(torch_cuda):
    rng = np.random.default_rng(26)
    ref = filled(rng, 2, 1, 100, 16, [100, 100])
    check_attn(torch_cuda, rng, ref, 2, 3, [98, 0xfffffff0], n_sel=3)


def test_sparse_of_all_blocks_is_dense(torch_cuda):
    """Choosing at least as many blocks as there are is the dense attention, to the bit where the split is the same."""
    rng = np.random.default_rng(27)
    ref = filled(rng, 1, 2, 777, 64, [777])
    q = rng.standard_normal((1, 1, 8, DIM)).astype(np.float32)
    a, _ = check_attn(torch_cuda, rng, ref, 8, 1, [776], q=q)
    b, sel = check_attn(torch_cuda, rng, ref, 8, 1, [776], q=q, n_sel=64)
    assert np.abs(a - b).max() <= 2e-6 and sel[0, 0, 0, :13].tolist() == list(range(13))


# ------------------------------------------------------ refusals, together --


def test_refusals_leave_outputs_alone(torch_cuda):
    torch = torch_cuda
    ref = RefCache(1, 2, 64, 16)
    dev = DevCache(torch, ref)
    pos, q = _i32(torch, [3]), torch.zeros(1, 1, 4, DIM, device="cuda")
    host, out = torch.zeros(1, 1, 4, DIM), torch.full((1, 1, 4, DIM), 7.0, device="cuda")
    sel = torch.full((1, 1, 2, 2), -5, dtype=torch.int32, device="cuda")
    C = dev.c
    bad = [lambda: atlas_cuda.kv8_attn(C, 3, 1, pos, q, out), lambda: atlas_cuda.kv8_attn(C, 0, 1, pos, q, out),
           lambda: atlas_cuda.kv8_attn(C, 4, 1, pos, q.view(-1)[1:], out), lambda: atlas_cuda.kv8_attn(C, 4, 1, pos, host, out),
           lambda: atlas_cuda.kv8_attn(C, 4, 1, pos.cpu(), q, out), lambda: atlas_cuda.kv8_attn(C, 4, 1, pos, q, host),
           lambda: atlas_cuda.kv8_attn(C, 4, 1, pos, q, out, ldq=508), lambda: atlas_cuda.kv8_attn(C, 4, 1, pos, q, out, ldo=514),
           lambda: atlas_cuda.kv8_attn(C, 4, 1 << 24, pos, q, out), lambda: atlas_cuda.kv8_attn(C, 4, 1, pos, q, out, n_tok=pos.cpu()),
           lambda: atlas_cuda.kv8_attn_sparse(C, 4, 1, 0, pos, q, out, sel),
           lambda: atlas_cuda.kv8_attn_sparse(C, 4, 1, 5000, pos, q, out, sel),
           lambda: atlas_cuda.kv8_attn_sparse(C, 4, 1, 2, pos, q, out, sel.cpu()),
           lambda: atlas_cuda.kv8_attn_sparse(DevCache(torch, ref, sums=False).c, 4, 1, 2, pos, q, out, sel),
           lambda: atlas_cuda.kv8_append(C, 1, pos, q, host), lambda: atlas_cuda.kv8_append(C, 1, pos, q, q, ld=128),
           lambda: atlas_cuda.kv8_read(C, 1, pos, out, host), lambda: atlas_cuda.kv8_read(C, 1, pos, out, out.view(-1)[2:])]
    for f in bad:
        with pytest.raises(atlas_cuda.AtlasError) as e:
            f()
        assert e.value.code == -1
    torch.cuda.synchronize()
    assert (out == 7.0).all() and (sel == -5).all()
    dev.equals(ref)
    # more blocks than fit beside the attention's buffers
    big = atlas_cuda.Kv8Desc(*(t.data_ptr() for t in dev.t), 1, 1, 1 << 20, 16)
    import ctypes
    assert atlas_cuda.lib().atlas_cuda_kv8_attn_sparse(ctypes.byref(big), 4, 1, 2, pos.data_ptr(), None, q.data_ptr(), 0,
                                                       out.data_ptr(), 0, sel.data_ptr(), None) == -1
    # no tokens: nothing to do
    atlas_cuda.kv8_attn(C, 4, 0, pos, q, out)
    atlas_cuda.kv8_append(C, 0, pos, q, q)
    torch.cuda.synchronize()
    assert (out == 7.0).all()


def test_a_prompt_and_steps_together_in_a_graph(torch_cuda):
    """As a decode loop uses them: a prompt is stored and attended, then one captured graph (append, attention, attention
    over chosen blocks, the positions advancing on the device) is replayed on a stream of its own, and every step is
    compared; at the end the cache is."""
    torch = torch_cuda
    rng = np.random.default_rng(31)
    nseq, heads, q_heads, ctx, block, steps = 2, 2, 10, 200, 16, 40
    lens = [70, 33]
    ref = RefCache(nseq, heads, ctx, block, rng)
    dev = DevCache(torch, ref)
    x, y = (rng.standard_normal((nseq, 70, heads, DIM)).astype(np.float32) for _ in range(2))
    ref.append([0, 0], lens, x, y)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        raw = stream.cuda_stream
        zero, n = _i32(torch, [0, 0]), _i32(torch, lens)
        q = rng.standard_normal((nseq, 70, q_heads, DIM)).astype(np.float32)
        dq, dk, dv, out = _f32(torch, q), _f32(torch, x), _f32(torch, y), torch.zeros(nseq, 70, q_heads, DIM, device="cuda")
        atlas_cuda.kv8_append(dev.c, 70, zero, dk, dv, n_tok=n, stream=raw)
        atlas_cuda.kv8_attn(dev.c, q_heads, 70, zero, dq, out, n_tok=n, stream=raw)
        stream.synchronize()
        dev.equals(ref)
        k_all, v_all = ((rng.standard_normal((steps, nseq, 1, heads, DIM)) * np.linspace(0.5, 2, steps)[:, None, None, None, None]
                         ).astype(np.float32) for _ in range(2))
        q_all = rng.standard_normal((steps, nseq, 1, q_heads, DIM)).astype(np.float32)
        dk, dv, dq = _f32(torch, k_all[0]), _f32(torch, v_all[0]), _f32(torch, q_all[0])
        pos = _i32(torch, lens)
        dense, sparse = torch.zeros(nseq, 1, q_heads, DIM, device="cuda"), torch.zeros(nseq, 1, q_heads, DIM, device="cuda")
        sel = torch.zeros(nseq, 1, heads, 3, dtype=torch.int32, device="cuda")
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            raw = torch.cuda.current_stream().cuda_stream
            atlas_cuda.kv8_append(dev.c, 1, pos, dk, dv, stream=raw)
            atlas_cuda.kv8_attn(dev.c, q_heads, 1, pos, dq, dense, stream=raw)
            atlas_cuda.kv8_attn_sparse(dev.c, q_heads, 1, 3, pos, dq, sparse, sel, stream=raw)
            pos += 1
        for i in range(steps):
            dk.copy_(_f32(torch, k_all[i]))
            dv.copy_(_f32(torch, v_all[i]))
            dq.copy_(_f32(torch, q_all[i]))
            graph.replay()
            stream.synchronize()
            at = [p + i for p in lens]
            ref.append(at, [1] * nseq, k_all[i], v_all[i])
            for s in range(nseq):
                for h in range(heads):
                    rows = slice(5 * h, 5 * h + 5)
                    k, v = ref.values(s, h, at[s] + 1)
                    qq = q_all[i, s, 0, rows].astype(np.float64)
                    blocks = choose(q_all[i, s, 0, rows], ref, s, h, at[s], 3)
                    assert sel[s, 0, h].tolist()[:len(blocks)] == blocks.tolist()
                    every = np.ones((5, at[s] + 1), bool)
                    some = every & np.isin(np.arange(at[s] + 1) // block, blocks)
                    for got, seen in ((dense, every), (sparse, some)):
                        want, bound = attend(qq, k, v, seen)
                        assert (np.abs(got[s, 0, rows].cpu().numpy() - want) <= bound).all()
    dev.equals(ref)
    assert pos.tolist() == [p + steps for p in lens]


def test_two_streams_at_once(torch_cuda):
    """Calls on different caches overlap freely: nothing is shared between them."""
    torch = torch_cuda
    rng = np.random.default_rng(32)
    work = []
    for i in range(4):
        ref = filled(rng, 1, 2, 3000, 64, [3000])
        q = rng.standard_normal((1, 1, 10, DIM)).astype(np.float32)
        want, _ = check_attn(torch, rng, ref, 10, 1, [2999], q=q)
        work.append((DevCache(torch, ref), _f32(torch, q), torch.zeros(1, 1, 10, DIM, device="cuda"), want, torch.cuda.Stream()))
    pos = _i32(torch, [2999])
    torch.cuda.synchronize()
    for _ in range(20):
        for dev, q, out, _, stream in work:
            atlas_cuda.kv8_attn(dev.c, 10, 1, pos, q, out, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for _, _, out, want, _ in work:
        np.testing.assert_array_equal(out.cpu().numpy(), want)
