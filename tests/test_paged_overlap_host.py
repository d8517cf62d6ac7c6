"""CPU: paged_attn refuses queries and outputs whose rows share memory, before it looks for a device; rows that lie beside one
another pass this check."""
import ctypes

import pytest

import atlas_cuda

torch = pytest.importorskip("torch")

N, H, QH, TOKENS = 2, 2, 6, 5
EINVAL, ROW = -1, 2 * 128          # bytes of a head's row


def _message():
    f = atlas_cuda.lib().atlas_cuda_last_error
    f.restype = ctypes.c_char_p
    return f(None).decode()


def _refused(lib, q, ldq, out, ldo, tokens=TOKENS, nseq=N):
    """Whether the call is refused for its rows' place (made-up addresses, which come to be looked at later)."""
    d = atlas_cuda.PagedDesc(1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, 1 << 40, 1, 2, 7, H, 16, nseq, 3)
    some = ctypes.c_void_p(6 << 20)
    rc = lib.atlas_cuda_paged_attn(ctypes.byref(d), 0, QH, tokens, some, None, ctypes.c_void_p(q), ldq, ctypes.c_void_p(out), ldo, None)
    assert rc != 0
    return rc == EINVAL and "overlap" in _message()


def _share(q, ldq, out, ldo, tokens, nseq):
    """The same, row by row."""
    n = nseq * tokens
    rows = [(q + 2 * i * (ldq or QH * 128), out + 2 * i * (ldo or QH * 128)) for i in range(n)]
    return any(abs(a - b) < QH * ROW for a, _ in rows for _, b in rows)


BASE = 1 << 30
WIDE = (2 * QH + 1) * 128          # values from token to token in a buffer that holds both


@pytest.mark.parametrize("nseq,tokens", [(1, 1), (2, 1), (1, 4), (2, 5)])
@pytest.mark.parametrize("ld", [0, QH * 128 + 8, 2 * QH * 128, WIDE])
def test_rows_the_same_distance_apart(lib, nseq, tokens, ld):
    step, width = 2 * (ld or QH * 128), QH * ROW
    at = set()
    for k in (0, 1, 2, nseq * tokens - 1, nseq * tokens, nseq * tokens + 1):
        for d in (-16, 0, 16, ROW, width - 16, width, width + 16, step - width - 16, step - width, step - width + 16):
            at |= {k * step + d, -(k * step + d)}
    for d in sorted(at):
        got, want = (f(BASE, ld, BASE + d, ld, tokens, nseq) for f in (lambda *a: _refused(lib, *a), _share))
        assert got == want, (d, got, want)


@pytest.mark.parametrize("ldq,ldo", [(0, WIDE), (WIDE, 0), (WIDE, WIDE + 8)])
def test_rows_of_different_distances(lib, ldq, ldo):
    """Nothing that overlaps passes, and ranges that do not meet are not refused."""
    n, width = N * TOKENS, QH * ROW
    lo = -((n - 1) * 2 * (ldo or QH * 128) + width)
    hi = (n - 1) * 2 * (ldq or QH * 128) + width
    for d in (lo - 16, lo, lo + 16, lo // 2 // 16 * 16, -16, 0, 16, hi // 2 // 16 * 16, hi - 16, hi, hi + 16):
        got = _refused(lib, BASE, ldq, BASE + d, ldo)
        assert got or not _share(BASE, ldq, BASE + d, ldo, TOKENS, N), d
        assert not got or lo < d < hi, d


def test_sizes_past_the_limits_are_still_refused(lib):
    big = 0xffffffff
    for tokens, nseq, ld in ((big, 4096, 0), (0xffffff, 4096, 0), (5, 2, 1 << 63), (5, 2, 8)):
        d = atlas_cuda.PagedDesc(1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, 1 << 40, 1, 2, 7, H, 16, nseq, 3)
        p = [ctypes.c_void_p(x << 20) for x in (6, 7, 1 << 30)]
        assert lib.atlas_cuda_paged_attn(ctypes.byref(d), 0, QH, tokens, p[0], None, p[1], ld, p[2], ld, None) != 0


def test_views_of_one_tensor():
    """Through the Python call: a fused buffer's overlapping views are refused, its separate ones get the library's next answer
    (no device, or memory of another one)."""
    c = atlas_cuda.PagedCache(*(torch.zeros(1, 7, H, 16, 128, dtype=torch.bfloat16) for _ in range(2)),
                              torch.full((N, 3), -1, dtype=torch.int32), torch.zeros(7, dtype=torch.int32))
    pos = torch.zeros(N, dtype=torch.int32)
    wide = torch.zeros(N, TOKENS, 2 * QH, 128, dtype=torch.bfloat16)
    ld = 2 * QH * 128
    for first, overlaps in ((0, True), (1, True), (QH - 1, True), (QH, False)):
        with pytest.raises(atlas_cuda.AtlasError) as e:
            atlas_cuda.paged_attn(c, 0, QH, TOKENS, pos, wide[:, :, :QH], wide[:, :, first:first + QH], ldq=ld, ldo=ld)
        assert ("overlap" in str(e.value)) == overlaps
