"""GPU: the paged KV cache's calls that store and move rows (append, fork, reserve, compact) against the definitions entry by
entry: pools, tables and counts are equal."""
import pytest

import atlas_cuda
from paged_ref import DIM, TYPES, RefPaged

pytestmark = pytest.mark.gpu


def _i32(torch, x):
    return torch.tensor([int(i) - (1 << 32) if int(i) > 0x7fffffff else int(i) for i in x], dtype=torch.int32, device="cuda")


class Dev:
    """A RefPaged's buffers on the device."""

    def __init__(self, torch, ref):
        self.k, self.v, self.table, self.refs = (x.cuda() for x in (ref.k, ref.v, ref.table, ref.refs))
        self.c = atlas_cuda.PagedCache(self.k, self.v, self.table, self.refs)
        self.c.buffers[4].fill_(float("nan"))        # what is in the workspace means nothing
        self.out = torch.full((1,), 77, dtype=torch.int32, device="cuda")

    def equals(self, torch, ref):
        assert torch.equal(self.table.cpu(), ref.table)
        assert torch.equal(self.refs.cpu(), ref.refs)
        for x, y in ((self.k, ref.k), (self.v, ref.v)):
            assert torch.equal(x.cpu().view(torch.int16), y.view(torch.int16))


def _both(torch, *shape, **more):
    ref = RefPaged(*shape, **more)
    return ref, Dev(torch, ref)


def _fork(torch, ref, dev, parent, length, first=None):
    ref.fork(parent, length, first)
    atlas_cuda.paged_fork(dev.c, _i32(torch, parent), _i32(torch, length), first=None if first is None else _i32(torch, first))


def _reserve(torch, ref, dev, pos0, ntok):
    want = ref.reserve(pos0, ntok)
    atlas_cuda.paged_reserve(dev.c, max(max(ntok), 1), _i32(torch, pos0), dev.out, n_tok=_i32(torch, ntok))
    assert int(dev.out) == want
    return want


def _compact(torch, ref, dev):
    want = ref.compact()
    atlas_cuda.paged_compact(dev.c, dev.out)
    assert int(dev.out) == want


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_sequences_come_fork_and_go(torch_cuda, kind, page):
    """The calls as a server makes them, compared after each."""
    torch = torch_cuda
    g = torch.Generator().manual_seed(page)
    layers, heads, nseq = 3, 2, 5
    ref, dev = _both(torch, kind, layers, 40, heads, page, nseq, 6, seed=1)
    pos = [0] * nseq

    def store(ntok):
        assert _reserve(torch, ref, dev, pos, ntok) == 0
        dev.equals(torch, ref)
        for layer in range(layers):
            k, v = (torch.randn(nseq, max(ntok), heads, DIM, generator=g).to(TYPES[kind]) for _ in range(2))
            ref.append(layer, pos, ntok, k, v)
            atlas_cuda.paged_append(dev.c, layer, max(ntok), _i32(torch, pos), k.cuda(), v.cuda(), n_tok=_i32(torch, ntok))
        dev.equals(torch, ref)
        for s in range(nseq):
            pos[s] += ntok[s]

    store([page, 3, 0, 2 * page + 5, 0])
    _fork(torch, ref, dev, [0, 1, 3, 3, 0], [pos[0], pos[1], pos[3], pos[3], page // 2])       # two forks, one of a part
    pos[2], pos[4] = pos[3], page // 2
    dev.equals(torch, ref)
    store([1, 1, 1, 1, 1])                                                                       # copies of shared ends
    _fork(torch, ref, dev, [3, 2, 1, 0, -1], [pos[3], pos[2], pos[1], pos[0], 9])                # exchanged, one freed
    pos[:] = [pos[3], pos[2], pos[1], pos[0], 0]
    dev.equals(torch, ref)
    _compact(torch, ref, dev)
    dev.equals(torch, ref)
    store([page - 1, 2, 0, 1, 3 * page])
    _fork(torch, ref, dev, range(nseq), pos, first=[max(0, p - page) for p in pos])              # a window
    dev.equals(torch, ref)
    _compact(torch, ref, dev)
    dev.equals(torch, ref)
    store([1, 0, 2, 1, 0])


@pytest.mark.parametrize("nseq,pages,max_pages,layers,heads,page", [(1, 1, 1, 1, 1, 16), (3, 5, 2, 1, 1, 128), (8, 61, 9, 2, 3, 16), (33, 1030, 37, 1, 1, 16),
                                                                    (300, 35000, 5, 1, 1, 16)])
def test_random_tables(torch_cuda, nseq, pages, max_pages, layers, heads, page):
    """Calls in a random order, short pools among them."""
    torch = torch_cuda
    import random
    r = random.Random(nseq * 1000 + pages)
    ref, dev = _both(torch, "bf16", layers, pages, heads, page, nseq, max_pages, seed=pages)
    pos = [0] * nseq
    end = max_pages * page
    for step in range(8 if nseq > 100 else 16):
        do = r.choice(["fork", "reserve", "reserve", "compact"]) if step else "reserve"
        if do == "fork":
            parent = [r.choice([s, r.randrange(nseq), r.randrange(-2, nseq + 2)]) for s in range(nseq)]
            length = [r.randint(0, pos[p]) if 0 <= p < nseq else r.randint(0, end) for p in parent]
            first = r.choice([None, [r.randint(0, n) if r.random() < 0.3 else 0 for n in length]])
            pos = [n if 0 <= p < nseq else 0 for n, p in zip(length, parent)]
            _fork(torch, ref, dev, parent, length, first)
        elif do == "reserve":
            most = max(1, 2 * pages * page // nseq)
            ntok = [r.choice([0, 1, r.randint(0, most)]) for _ in range(nseq)]
            if _reserve(torch, ref, dev, pos, ntok) == 0:
                pos = [min(p + n, end) for p, n in zip(pos, ntok)]
        else:
            _compact(torch, ref, dev)
        dev.equals(torch, ref)


def test_a_pool_that_is_too_small_changes_nothing(torch_cuda):
    torch = torch_cuda
    ref, dev = _both(torch, "fp16", 1, 4, 1, 16, 3, 4)
    assert _reserve(torch, ref, dev, [0, 0, 0], [16, 17, 0]) == 0
    _fork(torch, ref, dev, [0, 1, 1], [16, 17, 17])
    before = ref.table.clone()
    # the shared end's last writer keeps it: two pages are wanted, one is free
    assert _reserve(torch, ref, dev, [16, 17, 17], [1, 1, 1]) == 1
    assert torch.equal(before, ref.table)
    dev.equals(torch, ref)
    assert _reserve(torch, ref, dev, [16, 17, 17], [0, 1, 1]) == 0
    dev.equals(torch, ref)
    assert _reserve(torch, ref, dev, [16, 0, 0], [48, 0, 0]) == 3
    dev.equals(torch, ref)


def test_entries_that_name_no_page(torch_cuda):
    """Numbers out of the pool's range are no pages: never followed, dropped by forks, replaced by reservations."""
    torch = torch_cuda
    ref, dev = _both(torch, "bf16", 2, 6, 1, 16, 2, 4)
    wild = torch.tensor([[-5, 2 ** 31 - 1, 6, -2 ** 31], [1, 7, -1, 6]], dtype=torch.int32)
    for x in (ref, dev):
        x.table.copy_(wild)
        x.refs.copy_(torch.tensor([0, 1, 0, 0, 0, 0], dtype=torch.int32))
    k = torch.randn(2, 64, 1, DIM).to(torch.bfloat16)
    ref.append(1, [0, 0], [64, 64], k, k)
    atlas_cuda.paged_append(dev.c, 1, 64, _i32(torch, [0, 0]), k.cuda(), k.cuda())
    dev.equals(torch, ref)
    assert _reserve(torch, ref, dev, [20, 3], [1, 20]) == 0
    dev.equals(torch, ref)
    _compact(torch, ref, dev)
    dev.equals(torch, ref)
    _fork(torch, ref, dev, [1, 0], [64, 64])
    dev.equals(torch, ref)


def test_append_leaves_shared_pages_and_lost_positions(torch_cuda):
    """Strided rows inside wider buffers, positions behind the table and past 2^31, a larger n_tok, sequences left out."""
    torch = torch_cuda
    nseq, heads, page, tokens = 6, 3, 32, 50
    ref, dev = _both(torch, "fp16", 2, 24, heads, page, nseq, 4)
    assert _reserve(torch, ref, dev, [0] * nseq, [40, 40, 70, 128, 0, 128]) == 0
    _fork(torch, ref, dev, [0, 0, 2, 3, 4, 5], [40, 33, 70, 128, 0, 128])     # sequences 0 and 1 share both pages
    wide = torch.randn(nseq, tokens, heads + 2, DIM).to(torch.float16)
    k, v = wide[:, :, :heads], wide[:, :, 2:]
    pos, ntok = [0, 10, 60, 100, 0, 0xffffffff], [1, 50, 10 ** 9, 28, 7, 50]
    ref.append(1, pos, ntok, k, v)
    dk, dv = wide.cuda(), wide.cuda()
    atlas_cuda.paged_append(dev.c, 1, tokens, _i32(torch, pos), dk[:, :, :heads], dv[:, :, 2:], n_tok=_i32(torch, ntok), ld=(heads + 2) * DIM)
    dev.equals(torch, ref)
    atlas_cuda.paged_append(dev.c, 0, 0, _i32(torch, pos), dk[:, :0], dv[:, :0])
    dev.equals(torch, ref)


def test_a_large_pool(torch_cuda):
    """Rows whose offsets pass 32 bits, in elements too."""
    torch = torch_cuda
    pages, heads, page = 5000, 2, 128
    layers = 2
    # 2 x 5000 x 2 x 128 x 128 values: 5.2 GB a pool; row offsets in bytes pass 2^32 in the second layer
    k = torch.zeros(layers, pages, heads, page, DIM, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[[4997, 4998, 4999]] = 0
    c = atlas_cuda.PagedCache(k, v, table, refs)
    short = torch.zeros(1, dtype=torch.int32, device="cuda")
    atlas_cuda.paged_reserve(c, 130, _i32(torch, [0, 0]), short, n_tok=_i32(torch, [130, 0]))
    assert table.tolist() == [[4997, 4998, -1], [-1, -1, -1]] and int(short) == 0
    rows = torch.randn(2, 130, heads, DIM, device="cuda").to(torch.bfloat16)
    atlas_cuda.paged_append(c, 1, 130, _i32(torch, [0, 0]), rows, rows, n_tok=_i32(torch, [130, 0]))
    assert torch.equal(k[1, 4997], rows[0, :128].transpose(0, 1)) and torch.equal(v[1, 4998, :, :2], rows[0, 128:].transpose(0, 1))
    assert int(k.count_nonzero()) == int(rows[0].count_nonzero())
    atlas_cuda.paged_fork(c, _i32(torch, [0, 0]), _i32(torch, [130, 130]))
    atlas_cuda.paged_reserve(c, 1, _i32(torch, [130, 130]), short)
    # sequence 0 leaves the shared end, which stays sequence 1's
    assert table.tolist() == [[4997, 4999, -1], [4997, 4998, -1]] and refs[4997:].tolist() == [2, 1, 1]
    assert torch.equal(k[1, 4999, :, :2], k[1, 4998, :, :2]) and int(k[1, 4999, :, 2:].count_nonzero()) == 0
    refs[:4990] = 0
    atlas_cuda.paged_compact(c, short)
    assert int(short) == 10
    assert table.tolist() == [[7, 9, -1], [7, 8, -1]] and refs[:11].tolist() == [1] * 7 + [2, 1, 1, 0] and int(refs[10:].sum()) == 0
    assert torch.equal(k[1, 7], rows[0, :128].transpose(0, 1)) and torch.equal(v[1, 9, :, :2], rows[0, 128:].transpose(0, 1))


def test_captured_step_replays(torch_cuda):
    """Fork, reserve, append and compact captured once on a stream of their own, replayed while positions advance on the device."""
    torch = torch_cuda
    page, nseq, heads = 16, 4, 1
    ref, dev = _both(torch, "bf16", 1, 40, heads, page, nseq, 6)
    pos, parent = _i32(torch, [0, 0, 0, 0]), _i32(torch, [0, 1, 1, 0])
    k = torch.zeros(nseq, 3, heads, DIM, dtype=torch.bfloat16, device="cuda")
    short = torch.zeros(1, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()

    def step():
        s = torch.cuda.current_stream().cuda_stream
        atlas_cuda.paged_fork(dev.c, parent, pos, stream=s)
        atlas_cuda.paged_reserve(dev.c, 3, pos, short, stream=s)
        atlas_cuda.paged_append(dev.c, 0, 3, pos, k, k, stream=s)
        atlas_cuda.paged_compact(dev.c, dev.out, stream=s)
        pos.add_(3)

    start = [x.clone() for x in (dev.k, dev.v, dev.table, dev.refs)]
    with torch.cuda.stream(side):
        step()                                   # warm
    torch.cuda.synchronize()
    for x, y in zip((dev.k, dev.v, dev.table, dev.refs), start):
        x.copy_(y)
    pos.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(9):
        k.copy_(torch.full_like(k, i + 1))
        graph.replay()
        torch.cuda.synchronize()
        p = [3 * i] * nseq
        ref.fork([0, 1, 1, 0], p)
        assert ref.reserve(p, [3] * nseq) == 0
        ref.append(0, p, [3] * nseq, k.cpu(), k.cpu())
        assert ref.compact() == int(dev.out)
        dev.equals(torch, ref)


def test_many_copies(torch_cuda):
    """More to copy than one cluster is given: forks of one sequence that each go on inside its last page, in several layers."""
    torch = torch_cuda
    nseq, layers, heads, page = 60, 4, 3, 64
    ref, dev = _both(torch, "fp16", layers, 200, heads, page, nseq, 4, seed=3)
    assert _reserve(torch, ref, dev, [0] * nseq, [150] + [0] * (nseq - 1)) == 0
    _fork(torch, ref, dev, [0] * nseq, [150 - s for s in range(nseq)])
    assert _reserve(torch, ref, dev, [150 - s for s in range(nseq)], [1 + s % 3 for s in range(nseq)]) == 0
    dev.equals(torch, ref)
    _compact(torch, ref, dev)
    dev.equals(torch, ref)


@pytest.mark.parametrize("nseq,tokens,pages", [(3, 400, 90), (1024, 16, 1100), (40, 700, 2000)])
def test_more_entries_than_threads_or_as_many(torch_cuda, nseq, tokens, pages):
    """Reservations of about a thousand entries and more, of pages that sequences share."""
    torch = torch_cuda
    width = -(-tokens // 16) + 2
    ref, dev = _both(torch, "bf16", 1, pages, 1, 16, nseq, width, seed=nseq)
    _reserve(torch, ref, dev, [0] * nseq, [min(tokens, 16 * (pages // (2 * nseq)) + 5)] * nseq)
    dev.equals(torch, ref)
    _fork(torch, ref, dev, [s // 3 for s in range(nseq)], [tokens] * nseq)
    dev.equals(torch, ref)
    _reserve(torch, ref, dev, [7 * (s % 2) for s in range(nseq)], [tokens if s % 4 else 0 for s in range(nseq)])
    dev.equals(torch, ref)


def test_first_calls_inside_a_capture(torch_cuda):
    """A program whose first calls of all are captured: nothing they set up at first use spoils the capture. In a process of its
    own, with both forms of attention."""
    import os
    import subprocess
    import sys
    code = """
import sys, torch
sys.path[:0] = %r
import atlas_cuda
pool = lambda: torch.zeros(2, 40, 2, 32, 128, dtype=torch.bfloat16, device="cuda")
table = torch.full((2, 16), -1, dtype=torch.int32, device="cuda")
c = atlas_cuda.PagedCache(pool(), pool(), table, torch.zeros(40, dtype=torch.int32, device="cuda"))
i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
pos, zero, parent, length, short = i(0, 0), i(0, 0), i(0, 1), i(0, 0), i(5)
q = torch.ones(2, 300, 4, 128, dtype=torch.bfloat16, device="cuda")
out, one = torch.zeros_like(q), torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16, device="cuda")
k = torch.ones(2, 300, 2, 128, dtype=torch.bfloat16, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    atlas_cuda.paged_fork(c, parent, length, stream=s)
    atlas_cuda.paged_reserve(c, 300, pos, short, stream=s)
    atlas_cuda.paged_compact(c, short, stream=s)
    atlas_cuda.paged_reserve(c, 300, pos, short, stream=s)
    atlas_cuda.paged_append(c, 1, 300, pos, k, k, stream=s)
    atlas_cuda.paged_attn(c, 1, 4, 300, pos, q, out, stream=s)
    atlas_cuda.paged_attn(c, 1, 4, 1, pos, q[:, :1].contiguous(), one, stream=s)
for _ in range(2):
    g.replay()
torch.cuda.synchronize()
assert int(short) == 0 and bool((out == 1).all()) and bool((one == 1).all())
""" % ([os.path.dirname(atlas_cuda.__file__)],)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
