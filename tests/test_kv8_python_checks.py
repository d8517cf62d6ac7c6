"""CPU: the Python calls of the 8-bit KV cache refuse tensors of another type, layout or size before the library sees their
addresses. (Tensors that pass get the library's own answer: no device, or memory of another one.)"""
import ctypes

import pytest

import atlas_cuda

torch = pytest.importorskip("torch")

N, H, QH, CTX, B, TOKENS = 2, 2, 6, 40, 16, 3
EINVAL = -1


def _cache():
    blocks = -(-CTX // B)
    z = torch.zeros
    return atlas_cuda.Kv8Cache(z(N, H, CTX, 128, dtype=torch.int8), z(N, H, CTX, 128, dtype=torch.int8), z(N, H, blocks),
                               z(N, H, blocks), z(N, H, blocks, 128, dtype=torch.int16), nseq=N, kv_heads=H, max_context=CTX,
                               block=B)


def _args(**change):
    a = dict(pos0=torch.zeros(N, dtype=torch.int32), n_tok=torch.zeros(N, dtype=torch.int32),
             k=torch.zeros(N, TOKENS, H, 128), v=torch.zeros(N, TOKENS, H, 128), q=torch.zeros(N, TOKENS, QH, 128),
             out=torch.zeros(N, TOKENS, QH, 128), sel=torch.zeros(N, TOKENS, H, 4, dtype=torch.int32), ld=0, ldq=0, ldo=0)
    return {**a, **change}


def _calls(a):
    c, t = _cache(), TOKENS
    return [lambda: atlas_cuda.kv8_append(c, t, a["pos0"], a["k"], a["v"], n_tok=a["n_tok"], ld=a["ld"]),
            lambda: atlas_cuda.kv8_read(c, t, a["pos0"], a["k"], a["v"], n_tok=a["n_tok"], ld=a["ld"]),
            lambda: atlas_cuda.kv8_attn(c, QH, t, a["pos0"], a["q"], a["out"], n_tok=a["n_tok"], ldq=a["ldq"], ldo=a["ldo"]),
            lambda: atlas_cuda.kv8_attn_sparse(c, QH, t, 4, a["pos0"], a["q"], a["out"], a["sel"], n_tok=a["n_tok"],
                                               ldq=a["ldq"], ldo=a["ldo"])]


@pytest.fixture
def seen(monkeypatch):
    """The library's calls, counted instead of made."""
    n = []
    real = atlas_cuda.lib()

    class Fake:
        def __getattr__(self, name):
            if name.startswith("atlas_cuda_kv8_"):
                return lambda *a: n.append(name) or 0
            return getattr(real, name)

    monkeypatch.setattr(atlas_cuda, "lib", lambda: Fake())
    return n


def _refused(a, which, seen):
    for i, f in enumerate(_calls(a)):
        seen.clear()
        if i in which:
            with pytest.raises(atlas_cuda.AtlasError) as e:
                f()
            assert e.value.code == EINVAL and not seen
        else:
            f()
            assert len(seen) == 1


def test_right_tensors_pass(seen):
    wide, rows = torch.zeros(N, TOKENS, 9, 128), torch.zeros(N * TOKENS * QH * 128)
    for a in (_args(), _args(n_tok=None), _args(pos0=torch.zeros(N, dtype=torch.uint32)), _args(pos0=torch.zeros(5, dtype=torch.int32)),
              _args(k=wide[:, :, 1:3], v=wide[:, :, 7:], ld=9 * 128), _args(q=wide, out=wide[:, :, 3:], ldq=9 * 128, ldo=9 * 128),
              _args(q=rows, out=rows.clone()), _args(sel=torch.zeros(N * TOKENS * H * 4 + 1, dtype=torch.int32))):
        _refused(a, (), seen)


@pytest.mark.parametrize("name", ["pos0", "n_tok"])
@pytest.mark.parametrize("bad", [torch.zeros(N, dtype=torch.int64), torch.zeros(N), torch.zeros(N, dtype=torch.int16),
                                 torch.zeros(N - 1, dtype=torch.int32), torch.zeros(2 * N, dtype=torch.int32)[::2]])
def test_positions_and_counts(seen, name, bad):
    _refused(_args(**{name: bad}), (0, 1, 2, 3), seen)


@pytest.mark.parametrize("name,heads,which", [("k", H, (0, 1)), ("v", H, (0, 1)), ("q", QH, (2, 3)), ("out", QH, (2, 3))])
def test_rows(seen, name, heads, which):
    good = torch.zeros(N, TOKENS, heads, 128)
    for bad in (good.half(), good.double(), good.int(), good[:, :, : heads - 1], good[:, : TOKENS - 1].contiguous(), good[:1],
                torch.zeros(N, heads, TOKENS, 128).transpose(1, 2), torch.zeros(N, TOKENS, heads, 256)[..., ::2],
                torch.zeros(N, TOKENS + 1, heads, 128)[:, :TOKENS], good.view(-1)[4:], good.view(-1)[::2]):
        _refused(_args(**{name: bad}), which, seen)


def test_rows_apart(seen):
    """Rows inside a wider buffer: the stride that is named has to be the tensor's, and the last row has to end in it."""
    wide = torch.zeros(N, TOKENS, 9, 128)
    _refused(_args(q=wide, ldq=8 * 128), (2, 3), seen)
    _refused(_args(out=wide[:, :, 4:], ldo=9 * 128), (2, 3), seen)       # 4 + 6 heads of 9
    _refused(_args(k=wide[:, :, 8:], ld=9 * 128, v=wide[:, :, 1:]), (0, 1), seen)
    _refused(_args(k=wide.view(-1)[128:], v=wide, ld=9 * 128), (), seen)


@pytest.mark.parametrize("bad", [torch.zeros(N, TOKENS, H, 3, dtype=torch.int32), torch.zeros(N, TOKENS, H, 4),
                                 torch.zeros(N, TOKENS, H, 4, dtype=torch.int64),
                                 torch.zeros(N, H, TOKENS, 4, dtype=torch.int32).transpose(1, 2)])
def test_selection(seen, bad):
    _refused(_args(sel=bad), (3,), seen)


def test_no_tokens_need_no_rows(seen):
    c, p, none = _cache(), torch.zeros(N, dtype=torch.int32), torch.zeros(0)
    atlas_cuda.kv8_append(c, 0, p, none, none)
    atlas_cuda.kv8_attn(c, QH, 0, p, none, none)
    assert len(seen) == 2


def test_cache_types():
    ok = dict(nseq=1, kv_heads=2, max_context=20, block=16)
    k, sc, sums = torch.zeros(1, 2, 20, 128, dtype=torch.int8), torch.zeros(1, 2, 2), torch.zeros(1, 2, 2, 128, dtype=torch.int16)
    for bad in ((k.view(torch.uint8), k, sc, sc, sums), (k, k.bool(), sc, sc, sums), (k, k, sc.view(torch.int32), sc, sums),
                (k, k, sc, sc, sums.view(torch.float16)), (k, k, sc, sc, sums.view(torch.bfloat16))):
        with pytest.raises(ValueError):
            atlas_cuda.Kv8Cache(*bad, **ok)


def test_form_needs_a_cache_and_a_device(lib):
    rows, ctas = ctypes.c_uint32(7), ctypes.c_uint32(7)
    args = ctypes.byref(rows), ctypes.byref(ctas)
    assert lib.atlas_cuda_kv8_attn_form(None, 4, 1, *args) == EINVAL
    assert lib.atlas_cuda_kv8_attn_form(_cache()._ref, 4, 1, None, args[1]) == EINVAL
    if not torch.cuda.is_available():
        with pytest.raises(atlas_cuda.AtlasError) as e:
            atlas_cuda.kv8_attn_form(_cache(), 4, 1)
        assert e.value.code == -2
    assert rows.value == ctas.value == 7
