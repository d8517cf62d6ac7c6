"""CPU: the 8-bit KV cache's entry points refuse bad arguments before they look for a device, and the definitions that
the GPU tests compare with hold by themselves."""
import ctypes

import numpy as np
import pytest

import atlas_cuda
from kv8_ref import RefCache

EINVAL, ENODEV = -1, -2


def _desc(**change):
    f = dict(k=0x1000, v=0x2000, k_scale=0x3000, v_scale=0x4000, k_sum=0x5000, nseq=1, kv_heads=2, max_context=64,
             block=16)
    f.update(change)
    return atlas_cuda.Kv8Desc(*(f[n] for n, _ in atlas_cuda.Kv8Desc._fields_))


def _calls(lib, d, q_heads=4, tokens=1, pos0=0x100, ntok=None, rows=0x200, ld=0, out=0x300, n_sel=2, sel=0x400):
    r = ctypes.byref(d) if d is not None else None
    return [lib.atlas_cuda_kv8_append(r, tokens, pos0, ntok, rows, out, ld, None),
            lib.atlas_cuda_kv8_read(r, tokens, pos0, ntok, rows, out, ld, None),
            lib.atlas_cuda_kv8_attn(r, q_heads, tokens, pos0, ntok, rows, ld, out, 0, None),
            lib.atlas_cuda_kv8_attn_sparse(r, q_heads, tokens, n_sel, pos0, ntok, rows, ld, out, 0, sel, None)]


@pytest.mark.parametrize("change", [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(block=0),
                                    dict(block=24), dict(block=256), dict(nseq=0), dict(nseq=70000), dict(kv_heads=0),
                                    dict(kv_heads=20000), dict(max_context=0), dict(max_context=0xffffffff),
                                    dict(k=0x1008), dict(v=0x2001), dict(k_sum=0x5008), dict(k_scale=0x3002),
                                    dict(v_scale=0x4001)])
def test_bad_cache_is_refused(lib, change):
    assert _calls(lib, _desc(**change)) == [EINVAL] * 4
    assert lib.atlas_cuda_last_error(None)


@pytest.mark.parametrize("change", [dict(pos0=None), dict(pos0=0x102), dict(ntok=0x101), dict(tokens=1 << 24)])
def test_bad_calls_are_refused(lib, change):
    assert _calls(lib, _desc(), **change) == [EINVAL] * 4


def test_attention_in_place_is_refused(lib):
    assert _calls(lib, _desc(), rows=0x300)[2:] == [EINVAL] * 2


def test_null_cache_is_refused(lib):
    assert _calls(lib, None) == [EINVAL] * 4


def test_no_device_is_reported(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert _calls(lib, _desc()) == [ENODEV] * 4


def test_python_cache_checks_its_buffers():
    import torch
    ok = dict(nseq=1, kv_heads=2, max_context=20, block=16)
    k, sc, sums = torch.zeros(1, 2, 20, 128, dtype=torch.int8), torch.zeros(1, 2, 2), torch.zeros(1, 2, 2, 128,
                                                                                                 dtype=torch.int16)
    c = atlas_cuda.Kv8Cache(k, k, sc, sc, sums, **ok)
    assert c.desc.k == k.data_ptr() and c.desc.k_sum == sums.data_ptr() and c.desc.block == 16
    assert atlas_cuda.Kv8Cache(k, k, sc, sc, None, **ok).desc.k_sum is None
    for bad in ((k[:, :, :19], k, sc, sc, sums), (k, k.float(), sc, sc, sums), (k, k, sc[:, :, :1], sc, sums),
                (k, k, sc, sc, sums.int()), (k.transpose(1, 2), k, sc, sc, sums), (k, k, sc, sc.double(), sums)):
        with pytest.raises(ValueError):
            atlas_cuda.Kv8Cache(*bad, **ok)


def test_definition_append_in_pieces_and_at_once():
    """A block filled at once is off by half a step; filled in pieces, by at most half a step for each rounding again."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((1, 40, 1, 128)).astype(np.float32) * np.linspace(0.1, 3, 40)[None, :, None, None].astype(
        np.float32)
    once, steps = RefCache(1, 1, 64, 16), RefCache(1, 1, 64, 16)
    once.append([0], [40], x, x)
    for p in range(40):
        steps.append([p], [1], x[:, p:p + 1], x[:, p:p + 1])
    np.testing.assert_array_equal(once.ks[0, 0, :3], steps.ks[0, 0, :3])
    for c, rounds in ((once, 1), (steps, 16)):
        k, _ = c.values(0, 0, 40)
        step = c.ks[0, 0].astype(np.float64)[np.arange(40) // 16, None]
        # half a step each, and 2^-24 of the value for the scale's own rounding
        assert (np.abs(k - x[0, :, 0]) <= rounds * 0.5 * step * (1 + 2.0 ** -20)).all()
        np.testing.assert_array_equal(c.ksum[0, 0, 2], c.k[0, 0, 32:40].astype(int).sum(0))
