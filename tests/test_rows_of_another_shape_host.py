"""CPU: the Python calls of both KV caches refuse dense token rows of the right size in another order, as [nseq, heads, tokens,
128], and take those whose dimensions only group the same rows differently."""
import pytest

import atlas_cuda

torch = pytest.importorskip("torch")

N, H, QH, PAGE, CTX, B = 2, 2, 6, 16, 40, 16


@pytest.fixture
def seen(monkeypatch):
    """The library's calls, counted instead of made."""
    n = []
    real = atlas_cuda.lib()

    class Fake:
        def __getattr__(self, name):
            if name.startswith(("atlas_cuda_paged_", "atlas_cuda_kv8_")) and name != "atlas_cuda_paged_work":
                return lambda *a: n.append(name) or 0
            return getattr(real, name)

    monkeypatch.setattr(atlas_cuda, "lib", lambda: Fake())
    return n


def _calls(which, tokens):
    """(a call with two row tensors, their heads, their type) of each operator."""
    z, pos = torch.zeros, torch.zeros(N, dtype=torch.int32)
    if which == "paged":
        bf = torch.bfloat16
        c = atlas_cuda.PagedCache(z(1, 7, H, PAGE, 128, dtype=bf), z(1, 7, H, PAGE, 128, dtype=bf),
                                  torch.full((N, 3), -1, dtype=torch.int32), z(7, dtype=torch.int32))
        return [(lambda a, b: atlas_cuda.paged_append(c, 0, tokens, pos, a, b), H, bf),
                (lambda a, b: atlas_cuda.paged_attn(c, 0, QH, tokens, pos, a, b), QH, bf)]
    blocks = -(-CTX // B)
    c = atlas_cuda.Kv8Cache(z(N, H, CTX, 128, dtype=torch.int8), z(N, H, CTX, 128, dtype=torch.int8), z(N, H, blocks), z(N, H, blocks),
                            z(N, H, blocks, 128, dtype=torch.int16), nseq=N, kv_heads=H, max_context=CTX, block=B)
    sel = z(N, tokens, H, 4, dtype=torch.int32)
    f32 = torch.float32
    return [(lambda a, b: atlas_cuda.kv8_append(c, tokens, pos, a, b), H, f32), (lambda a, b: atlas_cuda.kv8_read(c, tokens, pos, a, b), H, f32),
            (lambda a, b: atlas_cuda.kv8_attn(c, QH, tokens, pos, a, b), QH, f32),
            (lambda a, b: atlas_cuda.kv8_attn_sparse(c, QH, tokens, 4, pos, a, b, sel), QH, f32)]


@pytest.mark.parametrize("which", ["paged", "kv8"])
@pytest.mark.parametrize("tokens", [3, 1])
def test_the_order_of_dimensions(seen, which, tokens):
    for call, heads, kind in _calls(which, tokens):
        right = torch.zeros(N, tokens, heads, 128, dtype=kind)
        takes = [(N, tokens, heads, 128), (1, N * tokens, heads, 128), (N * tokens, heads, 128), (N, tokens, 1, heads * 128), (N * tokens * heads * 128,),
                 (N, tokens * heads, 1, 128), (N, tokens, heads * 128, 1)]
        refuses = [(N, tokens, 128, heads), (128, N, tokens, heads)] + [(3, N, heads, 128)] * (tokens == 3) + [(heads, N, 1, 128)] * (tokens == 1 and heads != N)
        (takes if tokens == 1 else refuses).append((N, heads, tokens, 128))
        for shape in takes:
            for pair in ((torch.zeros(shape, dtype=kind), right), (right, torch.zeros(shape, dtype=kind))):
                seen.clear()
                call(*pair)
                assert len(seen) == 1, shape
        for shape in refuses:
            for pair in ((torch.zeros(shape, dtype=kind), right), (right, torch.zeros(shape, dtype=kind))):
                seen.clear()
                with pytest.raises(atlas_cuda.AtlasError):
                    call(*pair)
                assert not seen, shape
