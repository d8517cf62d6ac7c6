"""GPU: attention over the 8-bit KV cache, rows whose weights come together in few positions.

Tensor cores truncate what they add up, so outputs of many like weights lose a little; a row whose weight lies in one place
must not gain or lose anything for that."""
import numpy as np
import pytest

import atlas_cuda
from kv8_ref import DIM, RefCache
from test_gpu_kv8 import DevCache, _i32

pytestmark = pytest.mark.gpu

U = 2.0 ** -24

# sequences, query heads, KV heads, tokens, over 2500 positions: a single token, few rows, two tiles of rows per CTA, one
SHAPES = [(1, 2, 2, 1), (1, 1, 1, 200), (1, 64, 1, 300), (8, 40, 8, 7)]


def run(torch, shape, ctx, score, v, block=64):
    """Attention of queries that see position i with the score score[i] (in powers of e, up to a constant), values v."""
    nseq, q_heads, heads, tokens = shape
    k = np.zeros((nseq, ctx, heads, DIM), np.float32)
    k[..., 0] = score[None, :, None]
    ref = RefCache(nseq, heads, ctx, block, np.random.default_rng(2))
    ref.append([0] * nseq, [ctx] * nseq, k, v)
    q = torch.zeros(nseq, tokens, q_heads, DIM, device="cuda")
    q[..., 0] = float(np.sqrt(DIM))
    out = torch.zeros_like(q)
    atlas_cuda.kv8_attn(DevCache(torch, ref).c, q_heads, tokens, _i32(torch, [ctx - tokens] * nseq), q, out)
    return ref, out.cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("at", [0, 127, 128, 511, 512, 700, 1023, 1024, 2100])
def test_one_position(torch_cuda, shape, at):
    """All weight on one position, the others' rounds to none: its value. With u = 2^-24, 4 u for the weight's two terms,
    2 u for the scale's reciprocal, 2 u each for the sum's and the output's additions, 4 u each for the powers of two of the
    states and of two levels of merges, 4 u for the last products: 24 u."""
    ctx = 2500
    rng = np.random.default_rng(at)
    score = np.full(ctx, -100.0)
    score[at] = 100.0
    ref, got = run(torch_cuda, shape, ctx, score, rng.uniform(0.5, 1.0, (shape[0], ctx, shape[2], DIM)).astype(np.float32))
    group = shape[1] // shape[2]
    for s, h in np.ndindex(shape[0], shape[2]):
        want = ref.values(s, h, ctx)[1][at]
        rows = got[s, :, h * group:(h + 1) * group]
        assert np.abs(rows / want - 1).max() <= 24 * U


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("at", [3, 1030, 2040])
def test_most_weight_on_one_position(torch_cuda, shape, at):
    """One position has 2^12 times the weight of each of the others, values of one sign: the others' sums, at most 8 of 13
    parts of the output, may be truncated by each of the additions that an accumulator takes (64 at most; 2 u, of a sum that
    grows evenly half), the one position's, once it is there, by as many additions that are less than its last bit: 64 u +
    24 u + what the scores' int8 steps and sums are off by, 16 u."""
    ctx = 2500
    rng = np.random.default_rng(at)
    score = np.full(ctx, -12 * np.log(2.0) / 2)
    score[at] = 12 * np.log(2.0) / 2
    ref, got = run(torch_cuda, shape, ctx, score, rng.uniform(0.5, 1.0, (shape[0], ctx, shape[2], DIM)).astype(np.float32))
    group = shape[1] // shape[2]
    for s, h in np.ndindex(shape[0], shape[2]):
        k, v = ref.values(s, h, ctx)
        w = np.exp(k[:, 0] - k[:, 0].max())
        want = (np.cumsum(w[:, None] * v, 0) / np.cumsum(w)[:, None])[ctx - shape[3]:]
        rows = got[s, :, h * group:(h + 1) * group]
        assert np.abs(rows / want[:, None] - 1).max() <= 104 * U
