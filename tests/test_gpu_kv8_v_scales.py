"""GPU: attention over the 8-bit KV cache where V's block scales differ widely.

What a row's output may be off by goes by what its positions contribute, p |v|, whatever the scales of the blocks that have
no weight in it, or that it does not see. Every form of the attention is called: single tokens, few rows, prompts with one
and two tiles of rows per CTA, alone and in clusters, chosen blocks in one launch and in two."""
import numpy as np
import pytest

import atlas_cuda
from kv8_ref import DIM, RefCache, choose
from test_gpu_kv8 import DevCache, _f32, _i32

pytestmark = pytest.mark.gpu

U = 2.0 ** -24

# name: sequences, query heads, KV heads, tokens, first position, positions that the cache has room for, blocks to choose
SHAPES = {
    "single token": (2, 14, 2, 1, 9001, 9100, 0),       # long enough that every warp has several chunks of positions
    "few rows": (1, 8, 2, 5, 5005, 5200, 0),
    "one tile of rows": (8, 8, 2, 150, 0, 300, 0),
    "one tile of rows, clusters": (8, 24, 8, 42, 470, 2048, 0),
    "two tiles of rows": (4, 64, 16, 75, 130, 640, 0),
    "two tiles of rows, clusters": (4, 64, 8, 32, 480, 8192, 0),
    "chosen blocks": (1, 8, 2, 3, 5000, 5100, 320),     # all of them
    "chosen blocks, two launches": (2, 8, 4, 50, 2600, 2700, 170),
}


def attend_each(q, k, v, scale, seen):
    """Rows q [r, 128] over k, v [n, 128] (v's scales [n]) where seen [r, n]: the output and a bound of the error.

    With u = 2^-24, relative to what each position contributes: twice the error e of its score (q's terms, 4 u of the
    largest |q| per element; the score's own roundings, 8 u of the largest; the scale's logarithm as part of the exponent,
    4 u of its size), since the weight and the sum of weights have it; 32 u for exp's values and arguments, against a tile's
    maximum and the row's, the two binary16 terms and the merges of two levels of states; and the sums of n terms, of which
    one accumulator takes every 32nd, (n / 32 + 8) 2 u. Weights end at binary16's smallest number, so each position may be
    off by 2^-30 of what the row's largest contribution is worth."""
    s = np.where(seen, q @ k.T / np.sqrt(DIM), -np.inf)
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    size = np.abs(q).max(1) * np.where(seen, np.abs(k).sum(1)[None], 0).max(1) / np.sqrt(DIM)
    top = np.abs(np.where(seen, s, 0)).max(1)
    logs = np.where(seen, np.abs(np.log2(np.where(scale > 0, scale, 1.0)))[None] + 6, 0).max(1)
    e = 4 * U * size + 8 * U * top + 4 * U * logs
    n = k.shape[0]
    each = 2 * e + 32 * U + (n / 32 + 8) * 2 * U
    bound = (w @ np.abs(v)) * each[:, None] + (n * 2.0 ** -30 * (w * 127 * scale).max(1))[:, None]
    return w @ v, bound


def check(torch, ref, q, pos, q_heads, n_sel):
    nseq, heads, _, b, _ = ref.shape
    tokens, group = q.shape[1], q_heads // heads
    dev = DevCache(torch, ref)
    out = torch.full((nseq, tokens, q_heads, DIM), 7.0, device="cuda")
    if n_sel:
        sel = torch.zeros(nseq, tokens, heads, n_sel, dtype=torch.int32, device="cuda")
        atlas_cuda.kv8_attn_sparse(dev.c, q_heads, tokens, n_sel, _i32(torch, [pos] * nseq), _f32(torch, q), out, sel)
    else:
        atlas_cuda.kv8_attn(dev.c, q_heads, tokens, _i32(torch, [pos] * nseq), _f32(torch, q), out)
    got = out.cpu().numpy()
    at = pos + np.arange(tokens)
    n = pos + tokens
    for s in range(nseq):
        for h in range(heads):
            k, v = ref.values(s, h, n)
            rows = slice(h * group, (h + 1) * group)
            seen = np.arange(n)[None] <= at[:, None]
            if n_sel:
                for i in range(tokens):
                    seen[i] &= np.isin(np.arange(n) // b, choose(q[s, i, rows], ref, s, h, int(at[i]), n_sel))
            scale = ref.vs[s, h].astype(np.float64)[np.arange(n) // b]
            want, bound = attend_each(q[s, :, rows].astype(np.float64).reshape(-1, DIM), k, v, scale,
                                      np.repeat(seen, group, 0))
            err = np.abs(got[s, :, rows].reshape(-1, DIM) - want)
            assert (err <= bound).all(), float((err / np.maximum(bound, 1e-300)).max())


def cache_and_queries(shape, block, grown, apart, large):
    """Blocks where `grown` is true have values 2^large as large, and scores that are `apart` below the others' (in powers
    of e); the other dimensions of keys and queries are noise."""
    nseq, q_heads, heads, tokens, pos, ctx, n_sel = SHAPES[shape]
    rng = np.random.default_rng(int(max(large, -large, 0)) * 100 + block if np.isfinite(large) else block)
    n = pos + tokens
    ref = RefCache(nseq, heads, ctx, block, rng)
    k = 0.3 * rng.standard_normal((nseq, n, heads, DIM))
    v = rng.uniform(0.25, 1.0, k.shape) * rng.choice([-1, 1], k.shape)
    big = grown(np.arange(n) // block, n)
    k[..., 0] = np.where(big, -4.0, 4.0)[None, :, None]
    v[:, big] *= 2.0 ** large
    ref.append([0] * nseq, [n] * nseq, k.astype(np.float32), v.astype(np.float32))
    q = 0.3 * rng.standard_normal((nseq, tokens, q_heads, DIM))
    q[..., 0] = apart * np.sqrt(DIM) / 8.0
    return ref, q.astype(np.float32), pos, q_heads, n_sel


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("large", [10, 20, 30, 40])
def test_large_blocks_without_weight(torch_cuda, shape, large):
    """Every third block is 2^large as large, and has weights of e^-60."""
    args = cache_and_queries(shape, 16, lambda b, n: b % 3 == 1, 60.0, large)
    check(torch_cuda, *args)


@pytest.mark.parametrize("shape", [s for s in SHAPES if s != "single token"])
@pytest.mark.parametrize("large", [10, 20, 30, 40, 100])
def test_large_blocks_that_only_later_tokens_see(torch_cuda, shape, large):
    """The positions of the call's last tokens: earlier rows of the same tile do not see them."""
    tokens = SHAPES[shape][3]
    args = cache_and_queries(shape, 16, lambda b, n: b >= (n - 1 - tokens // 3) // 16, 0.0, large)
    check(torch_cuda, *args)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("large", [10, 20, 30, 40])
@pytest.mark.parametrize("more", [-4, 0, 6])
def test_large_blocks_of_little_weight(torch_cuda, shape, large, more):
    """Blocks 2^large as large with weights 2^(more - large): they make up the output, or as much of it as the others."""
    args = cache_and_queries(shape, 32, lambda b, n: b % 3 == 1, (large - more) * np.log(2.0), large)
    check(torch_cuda, *args)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [-60, 60, 126])
def test_values_of_any_size(torch_cuda, shape, size):
    """All values small, and so large that a sum of weighted ones passes fp32's range."""
    args = cache_and_queries(shape, 64, lambda b, n: b >= 0, 0.0, size)
    check(torch_cuda, *args)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("zero", ["first", "last", "every second"])
def test_zero_blocks_with_weight(torch_cuda, shape, zero):
    """Blocks of zeros (scale 0) that have most of the weight: whole parts of the positions, so that some warps and CTAs
    see nothing else, or every second block."""
    tokens = SHAPES[shape][3]
    grown = {"first": lambda b, n: b < (n - tokens) // 32, "last": lambda b, n: b >= (n - tokens) // 32,
             "every second": lambda b, n: b % 2 == 0}[zero]
    args = cache_and_queries(shape, 16, grown, -3.0, -np.inf)
    check(torch_cuda, *args)


@pytest.mark.parametrize("shape", [s for s in SHAPES if s != "single token"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_blocks_that_only_later_tokens_see_may_be_anything(torch_cuda, shape, bad, which):
    """A scale of NaN or infinity shows in the rows that see its block, and leaves the others as they were."""
    torch = torch_cuda
    ref, q, pos, q_heads, n_sel = cache_and_queries(shape, 16, lambda b, n: b >= 0, 0.0, 0)
    nseq, heads = ref.shape[:2]
    tokens = q.shape[1]
    blk = (pos + tokens - 1) // 16
    out = []
    for scale in (ref.vs[0, 0, blk], bad):
        (ref.ks if which == "k" else ref.vs)[:, :, blk] = scale
        dev = DevCache(torch, ref)
        out.append(torch.zeros(nseq, tokens, q_heads, DIM, device="cuda"))
        at = _i32(torch, [pos] * nseq)
        if n_sel:
            sel = torch.zeros(nseq, tokens, heads, n_sel, dtype=torch.int32, device="cuda")
            atlas_cuda.kv8_attn_sparse(dev.c, q_heads, tokens, n_sel, at, _f32(torch, q), out[-1], sel)
        else:
            atlas_cuda.kv8_attn(dev.c, q_heads, tokens, at, _f32(torch, q), out[-1])
    was, now = (x.cpu().numpy() for x in out)
    sees = pos + np.arange(tokens) >= 16 * blk
    if which == "v" or np.isnan(bad):   # an infinite K scale may make every score of the block -inf: no weight
        assert not np.isfinite(now[:, sees]).all(-1).any()
    np.testing.assert_array_equal(now[:, ~sees], was[:, ~sees])
