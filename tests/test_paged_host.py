"""CPU: the paged KV cache's calls refuse what they cannot take: cache shapes and workspaces by the library, tensors of another
type, layout or size by the Python calls before the library sees their addresses."""
import ctypes

import pytest

import atlas_cuda

torch = pytest.importorskip("torch")

N, H, QH, PAGE, PAGES, MAXP, TOKENS, LAYERS = 2, 2, 6, 16, 7, 3, 5, 2
EINVAL, ENODEV = -1, -2


def _buffers(kind=torch.bfloat16, **change):
    b = dict(k=torch.zeros(LAYERS, PAGES, H, PAGE, 128, dtype=kind), v=torch.zeros(LAYERS, PAGES, H, PAGE, 128, dtype=kind),
             table=torch.full((N, MAXP), -1, dtype=torch.int32), refs=torch.zeros(PAGES, dtype=torch.int32))
    return {**b, **change}


def _desc(**change):
    """A descriptor of made-up addresses: what the library checks before it looks at them."""
    d = dict(k=1 << 20, v=2 << 20, table=3 << 20, refs=4 << 20, work=5 << 20, work_bytes=1 << 40, type=0, layers=LAYERS, pages=PAGES,
             kv_heads=H, page=PAGE, nseq=N, max_pages=MAXP)
    return atlas_cuda.PagedDesc(*{**d, **change}.values())


def _message():
    f = atlas_cuda.lib().atlas_cuda_last_error
    f.restype = ctypes.c_char_p
    return f(None).decode()


BAD = [(dict(type=2), "type"), (dict(page=48), "pages of"), (dict(page=8), "pages of"), (dict(page=256), "pages of"), (dict(layers=0), "pool"),
       (dict(pages=0), "pool"), (dict(kv_heads=0), "pool"), (dict(pages=1 << 27, layers=1 << 10), "pool"), (dict(nseq=0), "table"),
       (dict(nseq=4097), "table"), (dict(max_pages=0), "table"), (dict(max_pages=1 << 28), "table"), (dict(k=0), "null"), (dict(v=0), "null"),
       (dict(table=0), "null"), (dict(refs=0), "null"), (dict(work=0), "null"), (dict(k=(1 << 20) + 8), "aligned"),
       (dict(refs=(4 << 20) + 4), "aligned"), (dict(table=(3 << 20) + 2), "aligned"), (dict(work=(5 << 20) + 128), "aligned"),
       (dict(work_bytes=1 << 10), "workspace")]


@pytest.mark.parametrize("change,word", BAD)
def test_caches_that_the_library_refuses(lib, change, word):
    ref, some = ctypes.byref(_desc(**change)), ctypes.c_void_p(6 << 20)
    for call in (lambda: lib.atlas_cuda_paged_fork(ref, some, some, None, None),
                 lambda: lib.atlas_cuda_paged_reserve(ref, 1, some, None, some, None),
                 lambda: lib.atlas_cuda_paged_compact(ref, some, None),
                 lambda: lib.atlas_cuda_paged_append(ref, 0, 1, some, None, some, some, 0, None),
                 lambda: lib.atlas_cuda_paged_attn(ref, 0, QH, 1, some, None, some, 0, ctypes.c_void_p(7 << 20), 0, None)):
        assert call() == EINVAL
        assert word in _message(), _message()


def test_workspace(lib):
    n = ctypes.c_uint64()
    assert lib.atlas_cuda_paged_work(ctypes.byref(_desc()), ctypes.byref(n)) == 0 and n.value > 0
    small = n.value
    assert lib.atlas_cuda_paged_work(ctypes.byref(_desc(pages=PAGES + 100000)), ctypes.byref(n)) == 0
    assert n.value >= small + 4 * 100000
    assert lib.atlas_cuda_paged_work(ctypes.byref(_desc(page=0)), ctypes.byref(n)) == EINVAL
    assert lib.atlas_cuda_paged_work(None, ctypes.byref(n)) == EINVAL
    assert lib.atlas_cuda_paged_work(ctypes.byref(_desc()), None) == EINVAL


def test_output_is_not_the_query(lib):
    ref, some = ctypes.byref(_desc()), ctypes.c_void_p(6 << 20)
    assert lib.atlas_cuda_paged_attn(ref, 0, QH, 1, some, None, some, 0, some, 0, None) == EINVAL


def test_no_device_is_an_error(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert lib.atlas_cuda_paged_compact(ctypes.byref(_desc()), ctypes.c_void_p(6 << 20), None) == ENODEV


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(LAYERS, PAGES, H, PAGE, 128)), dict(v=torch.zeros(LAYERS, PAGES, H, PAGE, 128, dtype=torch.float16)),
    dict(v=torch.zeros(LAYERS, PAGES, H, PAGE + 16, 128, dtype=torch.bfloat16)),
    dict(k=torch.zeros(LAYERS, PAGES, PAGE, H, 128, dtype=torch.bfloat16).transpose(2, 3)),
    dict(k=torch.zeros(LAYERS, PAGES, H, PAGE, 64, dtype=torch.bfloat16), v=torch.zeros(LAYERS, PAGES, H, PAGE, 64, dtype=torch.bfloat16)),
    dict(k=torch.zeros(PAGES, H, PAGE, 128, dtype=torch.bfloat16)), dict(table=torch.zeros(N, MAXP, dtype=torch.int64)),
    dict(table=torch.zeros(N * MAXP, dtype=torch.int32)), dict(table=torch.zeros(N, 2 * MAXP, dtype=torch.int32)[:, ::2]),
    dict(refs=torch.zeros(PAGES - 1, dtype=torch.int32)), dict(refs=torch.zeros(PAGES)), dict(refs=torch.zeros(PAGES, 1, dtype=torch.int32)),
    dict(work=torch.zeros(64, dtype=torch.uint8))])
def test_buffers_that_the_cache_refuses(change):
    with pytest.raises(ValueError):
        atlas_cuda.PagedCache(**_buffers(**change))


def test_page_sizes_that_the_cache_refuses():
    z = torch.zeros(LAYERS, PAGES, H, 24, 128, dtype=torch.bfloat16)
    with pytest.raises(atlas_cuda.AtlasError):
        atlas_cuda.PagedCache(**_buffers(k=z, v=z.clone()))


@pytest.fixture
def seen(monkeypatch):
    """The library's calls, counted instead of made."""
    n = []
    real = atlas_cuda.lib()

    class Fake:
        def __getattr__(self, name):
            if name.startswith("atlas_cuda_paged_") and name != "atlas_cuda_paged_work":
                return lambda *a: n.append(name) or 0
            return getattr(real, name)

    monkeypatch.setattr(atlas_cuda, "lib", lambda: Fake())
    return n


def _args(**change):
    i = lambda n=N: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    a = dict(pos0=i(), n_tok=i(), short=i(1), used=i(1), parent=i(), length=i(), first=i(), ld=0, ldq=0, ldo=0,
             k=torch.zeros(N, TOKENS, H, 128, dtype=torch.bfloat16), v=torch.zeros(N, TOKENS, H, 128, dtype=torch.bfloat16),
             q=torch.zeros(N, TOKENS, QH, 128, dtype=torch.bfloat16), out=torch.zeros(N, TOKENS, QH, 128, dtype=torch.bfloat16))
    return {**a, **change}


def _calls(a):
    c = atlas_cuda.PagedCache(**_buffers())
    return dict(
        fork=lambda: atlas_cuda.paged_fork(c, a["parent"], a["length"], first=a["first"]),
        reserve=lambda: atlas_cuda.paged_reserve(c, TOKENS, a["pos0"], a["short"], n_tok=a["n_tok"]),
        compact=lambda: atlas_cuda.paged_compact(c, a["used"]),
        append=lambda: atlas_cuda.paged_append(c, 1, TOKENS, a["pos0"], a["k"], a["v"], n_tok=a["n_tok"], ld=a["ld"]),
        attn=lambda: atlas_cuda.paged_attn(c, 1, QH, TOKENS, a["pos0"], a["q"], a["out"], n_tok=a["n_tok"], ldq=a["ldq"], ldo=a["ldo"]))


def _wide(heads, extra=2):
    return torch.zeros(N, TOKENS, heads + extra, 128, dtype=torch.bfloat16)[:, :, :heads]


REFUSED = [(dict(pos0=torch.zeros(N, dtype=torch.int64)), "reserve append attn"), (dict(pos0=torch.zeros(N - 1, dtype=torch.int32)), "reserve append attn"),
           (dict(n_tok=torch.zeros(N)), "reserve append attn"), (dict(n_tok=torch.zeros(2 * N, dtype=torch.int32)[::2]), "reserve append attn"),
           (dict(short=torch.zeros(1)), "reserve"), (dict(used=torch.zeros(0, dtype=torch.int32)), "compact"),
           (dict(parent=torch.zeros(N - 1, dtype=torch.int32)), "fork"), (dict(length=torch.zeros(N)), "fork"),
           (dict(first=torch.zeros(N, dtype=torch.int64)), "fork"),
           (dict(k=torch.zeros(N, TOKENS, H, 128)), "append"), (dict(v=torch.zeros(N, TOKENS, H, 128, dtype=torch.float16)), "append"),
           (dict(k=torch.zeros(N, TOKENS - 1, H, 128, dtype=torch.bfloat16)), "append"), (dict(k=_wide(H)), "append"),
           (dict(q=_wide(QH)), "attn"), (dict(q=torch.zeros(N, TOKENS, QH, 128)), "attn"),
           (dict(out=torch.zeros(N - 1, TOKENS, QH, 128, dtype=torch.bfloat16)), "attn"),
           (dict(out=torch.zeros(N, TOKENS, QH, 128, dtype=torch.bfloat16).transpose(1, 2)), "attn"),
           (dict(ldq=QH * 128 + 8), "attn"), (dict(ld=H * 128 + 8), "append")]


@pytest.mark.parametrize("change,which", REFUSED)
def test_tensors_that_the_calls_refuse(seen, change, which):
    for name, f in _calls(_args(**change)).items():
        seen.clear()
        if name in which.split():
            with pytest.raises(atlas_cuda.AtlasError) as e:
                f()
            assert e.value.args and name in str(e.value) and not seen
        else:
            f()
            assert seen == ["atlas_cuda_paged_" + name]


def test_strided_rows_pass(seen):
    wide = 128 * (QH + 2)
    a = _args(q=_wide(QH), out=_wide(QH), ldq=wide, ldo=wide, k=_wide(H), v=_wide(H), ld=128 * (H + 2))
    for name in ("append", "attn"):
        _calls(a)[name]()
    assert seen == ["atlas_cuda_paged_append", "atlas_cuda_paged_attn"]
