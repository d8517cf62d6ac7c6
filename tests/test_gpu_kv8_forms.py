"""GPU: kv8_attn's forms, each at sizes that take it: rows that fill tiles and rows that do not, pieces of different lengths,
strides, poisoned blocks and extreme sizes, with one CTA per unit of rows and with clusters, some of whose CTAs have no keys.

Which form a call takes follows from an estimate on the host, so it is asked for and compared first."""
import numpy as np
import pytest

import atlas_cuda
from kv8_ref import DIM
from test_gpu_kv8 import DevCache, _f32, _i32, check_attn, filled

pytestmark = pytest.mark.gpu

# (sequences, query heads, KV heads, tokens, positions that there is room for): the form, as rows per CTA and CTAs per unit
FORMS = {
    "few rows": ((2, 10, 2, 1, 900), (8, 8)),
    "few rows, no cluster": ((20, 16, 8, 3, 200), (8, 1)),
    "tiles of 16": ((1, 8, 2, 9, 1500), (16, 12)),
    "tiles of 16, no cluster": ((5, 24, 8, 13, 120), (16, 1)),
    "one tile": ((8, 8, 2, 150, 300), (128, 1)),                                  # 600 rows: 88 in the last tile
    "one tile, 2 CTAs": ((8, 24, 8, 42, 2048), (128, 2)),
    "one tile, 8 CTAs": ((3, 12, 4, 40, 16384), (128, 8)),                        # 120 rows; most CTAs have no keys
    "two tiles, the last alone": ((4, 64, 16, 75, 640), (256, 1)),                # 300 rows: 256 and 44
    "two tiles, the last partly": ((4, 64, 16, 100, 640), (256, 1)),              # 256 and 144
    "two tiles, 2 CTAs": ((8, 32, 8, 34, 4096), (256, 2)),                        # 136 rows: 128 and 8
    "two tiles, 4 CTAs": ((4, 32, 8, 64, 8192), (256, 4)),                        # 256 rows
    "two tiles, 8 CTAs": ((3, 16, 4, 50, 16384), (256, 8)),                       # 200 rows
}


def _lengths(name):
    """Different first positions and token counts: an idle sequence, more tokens than there are, rows past the cache's end
    (where the cache is small), positions that end inside a tile."""
    nseq, _, _, tokens, ctx = FORMS[name][0]
    end = min(ctx, 420)
    pos = [max(0, end - tokens - 37 * s) for s in range(nseq)]
    ntok = [tokens] * nseq
    if nseq > 1:
        pos[0], ntok[1] = 0, max(1, tokens // 2)
    if nseq > 3:
        ntok[2], ntok[3] = 0, tokens + 9
    if ctx == end:
        pos[-1] = ctx - max(1, tokens // 2)
    return pos, ntok


def _form(name, c):
    (_, q_heads, _, tokens, _), want = FORMS[name]
    assert atlas_cuda.kv8_attn_form(c, q_heads, tokens) == want


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("block", [16, 128])
def test_ragged_strided(torch_cuda, name, block):
    nseq, q_heads, heads, tokens, ctx = FORMS[name][0]
    rng = np.random.default_rng(block)
    pos, ntok = _lengths(name)
    ref = filled(rng, nseq, heads, ctx, block, [min(ctx, p + n) for p, n in zip(pos, ntok)])
    dev = DevCache(torch_cuda, ref)
    _form(name, dev.c)
    check_attn(torch_cuda, rng, ref, q_heads, tokens, pos, ntok, ldq=(q_heads + 3) * DIM, dev=dev)


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("q_size,k_size,v_spread", [(30.0, 3.0, 0.5), (1e-3, 1.0, 0.5), (1.0, 1.0, 4.0), (1e-30, 1e10, 0.1),
                                                    (1e8, 1e-8, 0.1)])
def test_sizes(torch_cuda, name, q_size, k_size, v_spread):
    nseq, q_heads, heads, tokens, ctx = FORMS[name][0]
    rng = np.random.default_rng(41)
    end = min(ctx, 300)
    ref = filled(rng, nseq, heads, ctx, 16, [end] * nseq, v_spread=v_spread, k_size=k_size)
    q = (q_size * rng.standard_normal((nseq, tokens, q_heads, DIM))).astype(np.float32)
    check_attn(torch_cuda, rng, ref, q_heads, tokens, [max(0, end - tokens - s) for s in range(nseq)], q=q)


@pytest.mark.parametrize("name", FORMS)
def test_poison(torch_cuda, name):
    """A NaN scale of K or V shows in the rows that see its block and in no other, a query row with a NaN or an infinity is
    NaN alone, and every other row is, to the bit, as it was."""
    torch = torch_cuda
    nseq, q_heads, heads, tokens, ctx = FORMS[name][0]
    group = q_heads // heads
    rng = np.random.default_rng(42)
    end = min(ctx, 300)
    pos = [max(0, end - tokens)] * nseq
    ref = filled(rng, nseq, heads, ctx, 16, [pos[0] + tokens] * nseq)
    q = rng.standard_normal((nseq, tokens, q_heads, DIM)).astype(np.float32)
    want, _ = check_attn(torch, rng, ref, q_heads, tokens, pos, q=q)
    blk = (pos[0] + tokens // 2) // 16                       # the rows before it do not see it
    ref.ks[0, 0, blk] = ref.vs[nseq - 1, heads - 1, blk] = np.nan
    q[0, tokens - 1, q_heads - 1, 5], q[nseq - 1, 0, 0, 100] = np.nan, np.inf
    out = torch.zeros(nseq, tokens, q_heads, DIM, device="cuda")
    atlas_cuda.kv8_attn(DevCache(torch, ref).c, q_heads, tokens, _i32(torch, pos), _f32(torch, q), out)
    got = out.cpu().numpy()
    bad = np.zeros(got.shape[:3], bool)
    sees = pos[0] + np.arange(tokens) >= 16 * blk
    bad[0, sees, :group] = True
    bad[nseq - 1, sees, q_heads - group:] = True
    bad[0, tokens - 1, q_heads - 1] = bad[nseq - 1, 0, 0] = True
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], want[~bad])


def test_refusals(torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(1)
    c = DevCache(torch, filled(rng, 1, 2, 64, 16, [64])).c
    for q_heads, tokens in ((3, 1), (0, 1), (4, 0), (4, 1 << 24)):
        with pytest.raises(atlas_cuda.AtlasError) as e:
            atlas_cuda.kv8_attn_form(c, q_heads, tokens)
        assert e.value.code == -1


# The sizes at which both forms were measured: whichever took less time, in us (few rows, prompt)
MEASURED = [
    ((1, 28, 4, 16, 500), 6.7, 15.3), ((1, 28, 4, 6, 8000), 15.4, 28.0), ((1, 28, 4, 16, 8000), 27.1, 29.9),
    ((1, 40, 8, 4, 30000), 57.1, 81.4), ((1, 40, 8, 13, 30000), 107.4, 82.3), ((8, 40, 8, 4, 2000), 26.1, 32.1),
    ((8, 40, 8, 7, 2000), 50.7, 32.2), ((8, 40, 8, 4, 16000), 166.1, 196.8), ((8, 40, 8, 7, 16000), 324.6, 196.9),
]


def form_of(torch, nseq, q_heads, heads, tokens, ctx, block=64):
    """Only the sizes count: buffers of the right size without contents."""
    n = -(-ctx // block)
    k = torch.empty(nseq, heads, ctx, DIM, dtype=torch.int8, device="cuda")
    sc = torch.empty(nseq, heads, n, device="cuda")
    c = atlas_cuda.Kv8Cache(k, torch.empty_like(k), sc, torch.empty_like(sc), nseq=nseq, kv_heads=heads, max_context=ctx,
                            block=block)
    return atlas_cuda.kv8_attn_form(c, q_heads, tokens)


@pytest.mark.parametrize("sizes,few,prompt", MEASURED)
def test_the_faster_form_is_taken(torch_cuda, sizes, few, prompt):
    assert (form_of(torch_cuda, *sizes)[0] <= 16) == (few < prompt)


# (sequences, query heads, KV heads, tokens, positions), and us by (rows per CTA, CTAs per unit) where they differ by a fifth
# and more: clusters that do not all fit at once take a second wave
CUTS = [
    ((1, 28, 4, 256, 2048 + 13), {(128, 1): 43.8, (128, 2): 35.0, (256, 2): 43.8, (256, 3): 37.2, (256, 4): 33.4, (256, 5): 53.9}),
    ((4, 28, 4, 40, 6000 + 13), {(128, 1): 110, (128, 2): 81.5, (128, 3): 91.8, (256, 2): 94.7, (256, 3): 72.6, (256, 4): 59.8}),
    ((4, 16, 4, 64, 8000 + 13), {(128, 2): 82.5, (128, 3): 67.4, (128, 4): 57.0, (256, 4): 68.7, (256, 5): 64.9, (256, 6): 59.6,
                                 (256, 7): 97.6, (256, 8): 89.2}),
    ((1, 40, 8, 100, 6000 + 13), {(128, 2): 64.5, (128, 3): 54.2, (128, 4): 45.5, (256, 5): 53.5, (256, 6): 49.4, (256, 7): 82.9,
                                  (256, 8): 75.8}),
]


@pytest.mark.parametrize("sizes,took", CUTS)
def test_no_second_wave_of_clusters(torch_cuda, sizes, took):
    """The cut is one of those measured, and not a fifth slower than the best."""
    cut = form_of(torch_cuda, *sizes)
    assert took[cut] <= 1.2 * min(took.values())


@pytest.mark.parametrize("n_sel", [768, 769, 1000])
def test_many_chosen_blocks(torch_cuda, n_sel):
    """More blocks than a list beside which two CTAs fit an SM holds: clusters of another size."""
    rng = np.random.default_rng(n_sel)
    ref = filled(rng, 2, 2, 17100, 16, [17001, 9000])
    check_attn(torch_cuda, rng, ref, 10, 1, [17000, 8999], n_sel=n_sel)
