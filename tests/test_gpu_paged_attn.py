"""GPU: attention over the paged KV cache against the definition in 64 bits, within the bound that paged_ref.attend derives."""
import pytest

import atlas_cuda
from paged_ref import DIM, TYPES, attend

pytestmark = pytest.mark.gpu


def _i32(torch, x):
    return torch.tensor([int(i) - (1 << 32) if int(i) > 0x7fffffff else int(i) for i in x], dtype=torch.int32, device="cuda")


class Setup:
    """Sequences whose first lens[s] positions have pages, in a random order; everything else in the pool is not finite."""

    def __init__(self, torch, kind, page, kv_heads, lens, width, layers=1, layer=0, seed=0, spare=3, poison=True, spread=1.0):
        self.torch, self.page, self.layer, self.kind = torch, page, layer, TYPES[kind]
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g = g
        per = [-(-n // page) for n in lens]
        pages = sum(per) + spare
        order = torch.randperm(pages, generator=g, device="cuda").tolist()
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(per):
            table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.table = table.cuda()
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.refs[order[:at]] = 1
        shape = (layers, pages, kv_heads, page, DIM)
        self.k = (spread * torch.randn(shape, generator=g, device="cuda")).to(self.kind)
        self.v = torch.randn(shape, generator=g, device="cuda").to(self.kind)
        if poison:
            here = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
            for s, n in enumerate(lens):
                p = torch.arange(n, device="cuda")
                here[self.table[s].long()[p // page], p % page] = True
            bad = torch.tensor([float("nan"), float("inf"), float("-inf")], dtype=self.kind, device="cuda")
            hide = ~here.view(1, pages, 1, page, 1).expand(shape)
            for pool in (self.k, self.v):
                pool[hide] = bad[torch.arange(int(hide.sum()), device="cuda") % 3]
                for other in range(layers):
                    if other != layer:
                        pool[other] = float("nan")
        self.c = atlas_cuda.PagedCache(self.k, self.v, self.table, self.refs)
        self.c.buffers[4].fill_(float("nan"))

    def rand(self, *shape, size=1.0):
        return (size * self.torch.randn(shape, generator=self.g, device="cuda")).to(self.kind)

    def attn(self, q, pos, ntok=None, out=None, ldq=0, ldo=0):
        out = self.torch.full_like(q, 7.0) if out is None else out
        atlas_cuda.paged_attn(self.c, self.layer, q.shape[2], q.shape[1], _i32(self.torch, pos), q, out,
                              n_tok=None if ntok is None else _i32(self.torch, ntok), ldq=ldq, ldo=ldo)
        return out

    def check(self, out, q, pos, ntok=None, sample=None):
        """Every row that the call has (or `sample` tokens of each sequence, ends among them), and that the others are as they were."""
        torch = self.torch
        n, tokens, heads, _ = q.shape
        kvh = self.k.shape[2]
        grp = heads // kvh
        one_term = atlas_cuda.paged_attn_form(self.c, heads, tokens) >= 128
        for s in range(n):
            m = tokens if ntok is None else min(int(ntok[s]), tokens)
            assert torch.equal(out[s, m:], torch.full_like(out[s, m:], 7.0))
            at = range(m)
            if sample and m > sample:
                at = sorted(set([0, 1, m - 1] + torch.randint(0, m, (sample,), generator=self.g, device="cuda").tolist()))
            for t in at:
                p = int(pos[s]) + t
                for h in range(kvh):
                    want, bound = attend(q[s, t, h * grp:(h + 1) * grp], self.k[self.layer, :, h], self.v[self.layer, :, h], self.table[s], self.page, p,
                                         one_term)
                    got = out[s, t, h * grp:(h + 1) * grp].double()
                    err = (got - want).abs()
                    assert bool((err <= bound).all()), (s, t, h, p, float((err / bound).nan_to_num(1e9).max()))


# (KV heads, query heads per KV head, first positions, tokens, tokens of each sequence or None)
SHAPES = [
    (1, 1, [0], 1, None), (4, 7, [0], 1, None), (2, 8, [15], 1, None), (2, 6, [16], 1, None), (4, 7, [640], 1, None),
    (8, 5, [126, 127, 128, 129], 1, None), (1, 16, [300, 5000], 1, None), (1, 20, [77], 1, None), (1, 40, [2000], 1, None),
    (8, 5, [2303, 1500, 0, 700, 31, 2000, 16, 1], 1, [1, 1, 1, 1, 1, 1, 0, 1]),
    (2, 4, [100], 2, None), (1, 3, [0], 5, None), (2, 8, [1000, 30], 4, [4, 3]), (8, 5, [801] * 4, 7, None), (2, 1, [50], 16, None),
    (1, 1, [0], 17, None), (1, 1, [0], 130, None), (4, 7, [0], 40, None), (2, 8, [0, 513], 33, [33, 20]), (1, 5, [63], 100, None),
    (4, 7, [0], 300, None), (2, 8, [700, 0, 40], 260, [260, 1, 255]), (1, 12, [129], 129, None), (1, 40, [10], 70, None), (1, 64, [3], 9, None),
    (1, 100, [9], 30, None), (1, 130, [9], 5, None), (1, 7, [13 * i for i in range(40)], 1, None), (2, 2, [300 - 5 * i for i in range(37)], 5, [i % 7 for i in range(37)]),
    (1, 4, [11 * i for i in range(45)], 50, [(7 * i) % 60 for i in range(45)]), (1, 8, [0] * 33, 70, None),
]


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%d-%d-%s-%d" % (s[0], s[1], s[2][0], s[3]))
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_against_the_definition(torch_cuda, kind, shape, page):
    kvh, grp, pos, tokens, ntok = shape
    lens = [p + (tokens if ntok is None else min(ntok[s], tokens)) for s, p in enumerate(pos)]
    x = Setup(torch_cuda, kind, page, kvh, lens, -(-max(lens) // page) + 2, seed=page + tokens)
    q = x.rand(len(pos), tokens, kvh * grp, DIM)
    x.check(x.attn(q, pos, ntok), q, pos, ntok, sample=12 if len(pos) < 10 else 2)


@pytest.mark.parametrize("kind,page,kvh,grp,pos,tokens", [
    ("bf16", 64, 8, 5, [32767, 20000], 1), ("fp16", 128, 2, 8, [30000], 5), ("bf16", 16, 1, 7, [70000], 1), ("fp16", 32, 4, 7, [0], 2048),
    ("bf16", 64, 8, 5, [6000], 513), ("fp16", 128, 1, 8, [40000], 300), ("bf16", 128, 1, 1, [0, 9000], 4000)])
def test_long_ones(torch_cuda, kind, page, kvh, grp, pos, tokens):
    lens = [p + tokens for p in pos]
    x = Setup(torch_cuda, kind, page, kvh, lens, -(-max(lens) // page), seed=5)
    q = x.rand(len(pos), tokens, kvh * grp, DIM)
    x.check(x.attn(q, pos), q, pos, sample=8)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("size", [0.0, 4.0, 30.0])
@pytest.mark.parametrize("tokens", [1, 3, 60, 400])
def test_flat_and_peaked_rows(torch_cuda, kind, size, tokens):
    """Scores that are all equal, and such that one position has nearly all the weight."""
    pos = [500, 37]
    x = Setup(torch_cuda, kind, 32, 2, [p + tokens for p in pos], 40, seed=3, spread=3.0)
    q = x.rand(2, tokens, 14, DIM, size=size)
    x.check(x.attn(q, pos), q, pos, sample=8)


@pytest.mark.parametrize("tokens", [1, 4, 20, 90, 300])
def test_values_of_one_sign_and_great_size(torch_cuda, tokens):
    """Sums that are truncated lose most where all values have one sign; binary16's largest values stay finite."""
    for kind, big in (("fp16", 65000.0), ("bf16", 2.0 ** 120)):
        x = Setup(torch_cuda, kind, 64, 1, [3000 + tokens], 60, seed=4)
        x.v.copy_(torch_cuda.where(x.v.isfinite(), (0.5 + 0.5 * torch_cuda.rand(x.v.shape, device="cuda")) * big, x.v.float()).to(x.kind))
        q = x.rand(1, tokens, 5, DIM)
        out = x.attn(q, [3000])
        x.check(out, q, [3000], sample=6)


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("tokens", [1, 5, 37, 200])
@pytest.mark.parametrize("gone", ["first", "middle", "last", "own", "all", "many"])
def test_positions_without_a_page(torch_cuda, page, tokens, gone):
    torch = torch_cuda
    pos = [900, 300]
    x = Setup(torch, "bf16", page, 2, [p + tokens for p in pos], 80, seed=page)
    used = -(-(pos[0] + tokens) // page)
    cut = {"first": range(0, used // 2), "middle": [used // 3, used // 2], "last": [used - 1], "own": range(pos[0] // page, used), "all": range(used),
           "many": range(0, used, 2)}[gone]
    x.table[0, list(cut)] = torch.tensor([(-1, 1 << 20, -7, x.refs.numel())[i % 4] for i in range(len(cut))], dtype=torch.int32, device="cuda")
    q = x.rand(2, tokens, 10, DIM)
    out = x.attn(q, pos)
    x.check(out, q, pos, sample=10)
    if gone == "all":
        assert int(out[0].count_nonzero()) == 0


@pytest.mark.parametrize("tokens", [1, 6, 50, 260])
def test_positions_behind_the_table(torch_cuda, tokens):
    """Rows there see what the table holds; positions up to 2^32 - 1."""
    x = Setup(torch_cuda, "fp16", 32, 1, [96, 64, 96], 3, seed=9)
    q = x.rand(3, tokens, 8, DIM)
    pos = [90, 60, 0xffffffff]
    x.table[1, 2] = -1
    x.check(x.attn(q, pos), q, pos, sample=8)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("tokens,at", [(1, 100), (9, 104), (9, 100), (150, 130), (150, 240), (400, 401)])
def test_what_is_not_finite_stays_with_who_sees_it(torch_cuda, kind, tokens, at):
    """A NaN or infinity among the values of one position of the chunk, or among its keys: only rows from it on have it."""
    torch = torch_cuda
    pos = [96]
    x = Setup(torch, kind, 16, 2, [96 + tokens], 40, seed=tokens)
    q = x.rand(1, tokens, 10, DIM)
    clean = x.attn(q, pos)
    e, r = int(x.table[0, at // 16]), at % 16
    if at >= 96 + tokens:
        pytest.skip("not a position of the chunk")
    x.v[0, e, 0, r, 3] = float("inf")
    x.v[0, e, 0, r, 77] = float("nan")
    x.k[0, e, 1, r, 5] = float("nan")
    out = x.attn(q, pos)
    t = max(0, at - 96)
    assert torch.equal(out[0, :t], clean[0, :t])
    seen = out[0, t:].view(-1, 2, 5, DIM).isfinite()
    want = torch.ones_like(seen)
    want[:, 0, :, 3] = want[:, 0, :, 77] = False
    want[:, 1] = False
    assert torch.equal(seen, want)
    assert torch.equal(out[0, t:].view(-1, 2, 5, DIM)[:, 0][seen[:, 0]], clean[0, t:].view(-1, 2, 5, DIM)[:, 0][seen[:, 0]])


def test_a_query_that_is_not_finite_is_its_rows_own(torch_cuda):
    torch = torch_cuda
    for tokens in (3, 40, 300):
        x = Setup(torch, "bf16", 64, 1, [200 + tokens], 10, seed=2)
        q = x.rand(1, tokens, 7, DIM)
        clean = x.attn(q, [200])
        q[0, tokens // 2, 3, 9] = float("nan")
        out = x.attn(q, [200])
        assert bool(out[0, tokens // 2, 3].isnan().all())
        out[0, tokens // 2, 3] = clean[0, tokens // 2, 3]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("tokens", [1, 3, 70, 300])
def test_strides_layers_and_shared_pages(torch_cuda, tokens):
    """Rows inside wider buffers, what lies between them left alone; a layer in the middle; a common prefix; a table wider than used."""
    torch = torch_cuda
    x = Setup(torch, "fp16", 32, 2, [200 + tokens, 90 + tokens], 64, layers=3, layer=1, seed=11)
    x.table[1, :2] = x.table[0, :2]                    # the second sequence's first 64 positions
    x.refs[x.table[0, :2].long()] = 2
    wide = x.rand(2, tokens, 16, DIM)
    q = wide[:, :, 2:14]
    canvas = torch.full((2, tokens, 14, DIM), 7.0, dtype=x.kind, device="cuda")
    x.attn(q, [200, 90], [tokens, 1], out=canvas[:, :, 1:13], ldq=16 * DIM, ldo=14 * DIM)
    assert bool((canvas[:, :, [0, 13]] == 7.0).all())
    x.check(canvas[:, :, 1:13], q, [200, 90], [tokens, 1], sample=10)


def test_no_rows_and_no_tokens(torch_cuda):
    torch = torch_cuda
    x = Setup(torch, "bf16", 16, 2, [50, 60], 8)
    for tokens in (1, 100):
        q = x.rand(2, tokens, 4, DIM)
        out = x.attn(q, [40, 50], [0, 0])
        assert bool((out == 7.0).all())
    q = x.rand(2, 0, 4, DIM)
    x.attn(q, [40, 50])


def test_a_chunk_at_a_time_is_the_whole(torch_cuda):
    """A prompt in pieces of many sizes, through every form, stored and attended as a server does: each within the bound."""
    torch = torch_cuda
    page, kvh, grp, total = 16, 2, 6, 700
    x = Setup(torch, "bf16", page, kvh, [0, 0], 50, spare=100, seed=21)
    g = x.g
    k, v, q = (torch.randn(2, total, n, DIM, generator=g, device="cuda").to(torch.bfloat16) for n in (kvh, kvh, kvh * grp))
    short = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = 0
    for n in (1, 2, 13, 200, 1, 5, 50, 400, 28):
        pos = [p, p]
        atlas_cuda.paged_reserve(x.c, n, _i32(torch, pos), short)
        part = [t[:, p:p + n].contiguous() for t in (k, v, q)]
        atlas_cuda.paged_append(x.c, 0, n, _i32(torch, pos), part[0], part[1])
        assert int(short) == 0
        out = x.attn(part[2], pos)
        x.check(out, part[2], pos, sample=4)
        p += n
    assert p == total


def test_replays_and_streams(torch_cuda):
    """A captured decode step on a stream of its own replays at advancing positions, beside another cache's on another stream;
    the same call gives the same bits."""
    torch = torch_cuda
    caches = [Setup(torch, "fp16", 32, 2, [700, 500], 24, seed=s, poison=False) for s in (1, 2)]
    state = []
    for x in caches:
        q, out, pos = x.rand(2, 1, 14, DIM), torch.zeros(2, 1, 14, DIM, dtype=x.kind, device="cuda"), _i32(torch, [600, 400])
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            atlas_cuda.paged_attn(x.c, 0, 14, 1, pos, q, out, stream=side.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            atlas_cuda.paged_attn(x.c, 0, 14, 1, pos, q, out, stream=torch.cuda.current_stream().cuda_stream)
            pos.add_(1)
        state.append((x, q, out, pos, side, graph))
    for i in range(40):
        torch.cuda.synchronize()
        for x, q, out, pos, side, graph in state:
            out.fill_(7.0)
        torch.cuda.synchronize()
        for x, q, out, pos, side, graph in state:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for x, q, out, pos, side, graph in state:
            at = [600 + i, 400 + i]
            assert pos.tolist() == [a + 1 for a in at]
            if i % 13 == 0:
                x.check(out, q, at)
            again = x.attn(q, at)
            assert torch.equal(out, again) and torch.equal(again, x.attn(q, at))


def test_refusals_on_the_device(torch_cuda):
    torch = torch_cuda
    x = Setup(torch, "bf16", 16, 2, [50], 8)
    q, out, pos = x.rand(1, 2, 4, DIM), x.rand(1, 2, 4, DIM), _i32(torch, [40])
    before = out.clone()
    bad = [lambda: atlas_cuda.paged_attn(x.c, 1, 4, 2, pos, q, out), lambda: atlas_cuda.paged_attn(x.c, 0, 3, 2, pos, q[:, :, :3].contiguous(), out[:, :, :3].contiguous()),
           lambda: atlas_cuda.paged_attn(x.c, 0, 4, 2, pos, q, q), lambda: atlas_cuda.paged_attn(x.c, 0, 4, 2, pos.cpu(), q, out),
           lambda: atlas_cuda.paged_attn(x.c, 0, 4, 2, pos, q.cpu(), out), lambda: atlas_cuda.paged_attn(x.c, 0, 4, 2, pos, q, out.cpu()),
           lambda: atlas_cuda.paged_append(x.c, 1, 2, pos, q[:, :, :2].contiguous(), q[:, :, 2:].contiguous()),
           lambda: atlas_cuda.paged_append(x.c, 0, 2, pos, q[:, :, :2].contiguous().cpu(), q[:, :, 2:].contiguous()),
           lambda: atlas_cuda.paged_fork(x.c, pos.cpu(), pos), lambda: atlas_cuda.paged_fork(x.c, pos, pos, first=pos.cpu()),
           lambda: atlas_cuda.paged_reserve(x.c, 2, pos, pos.cpu()), lambda: atlas_cuda.paged_compact(x.c, pos.cpu())]
    for f in bad:
        with pytest.raises(atlas_cuda.AtlasError):
            f()
    torch.cuda.synchronize()
    assert torch.equal(out, before)


def test_two_graphs_of_one_cache(torch_cuda):
    """A prompt's graph and a decode step's, captured over one cache and its workspace, replayed in turn on one stream."""
    torch = torch_cuda
    x = Setup(torch, "bf16", 32, 2, [1500, 1300], 60, seed=31)
    long_q, step_q = x.rand(2, 200, 10, DIM), x.rand(2, 1, 10, DIM)
    long_out, step_out = torch.zeros_like(long_q), torch.zeros_like(step_q)
    long_pos, step_pos = _i32(torch, [1300, 1100]), _i32(torch, [1499, 1299])
    want = x.attn(long_q, [1300, 1100]), x.attn(step_q, [1499, 1299])
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for g, args in zip(graphs, ((200, long_pos, long_q, long_out), (1, step_pos, step_q, step_out))):
        with torch.cuda.graph(g):
            atlas_cuda.paged_attn(x.c, 0, 10, *args, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(10):
        for g in graphs + graphs[::-1]:
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(long_out, want[0]) and torch.equal(step_out, want[1])


@pytest.mark.parametrize("kvh,grp,lens,tokens", [(1, 7, [5000], 1), (2, 8, [9000], 1), (8, 5, [8447], 1), (4, 7, [640] * 5, 1), (4, 7, [3000, 10, 700], 1), (8, 5, [2000] * 9, 1),
                                                 (1, 5, [20, 9000, 300, 40], 2), (6, 5, [4000, 3900, 3800], 3), (16, 1, [1000] * 9, 1), (3, 4, [100, 20000], 4)])
def test_units_shared_by_clusters_and_not(torch_cuda, kvh, grp, lens, tokens):
    """Few sequences (a cluster has a unit), many or uneven ones (a line of all), with room for much more than they have."""
    torch = torch_cuda
    x = Setup(torch, "fp16", 64, kvh, lens, 600, seed=sum(lens))
    pos = [n - tokens for n in lens]
    q = x.rand(len(lens), tokens, kvh * grp, DIM)
    out = x.attn(q, pos)
    x.check(out, q, pos)
    assert torch.equal(out, x.attn(q, pos))


def test_a_row_goes_by_what_it_sees(torch_cuda):
    """Other rows' queries, and keys and values behind it, change no bit of a row."""
    torch = torch_cuda
    for tokens in (3, 60, 500):
        x = Setup(torch, "bf16", 16, 2, [300 + tokens], 60, seed=8)
        q = x.rand(1, tokens, 10, DIM)
        out = x.attn(q, [300])
        t = tokens // 2
        other = q.clone()
        other[:, :t] = x.rand(1, t, 10, DIM, size=5.0)
        other[:, t + 1:] = x.rand(1, tokens - t - 1, 10, DIM, size=5.0)
        e = x.table[0].long()[torch.arange(300 + t + 1, 300 + tokens, device="cuda") // 16]
        at = torch.arange(300 + t + 1, 300 + tokens, device="cuda") % 16
        x.k[0, e, :, at] = x.rand(tokens - t - 1, 2, DIM, size=5.0)
        x.v[0, e, :, at] = x.rand(tokens - t - 1, 2, DIM, size=5.0)
        assert torch.equal(x.attn(other, [300])[0, t], out[0, t])


@pytest.mark.parametrize("kvh,grp,pos,tokens,ntok", [
    (1, 1, [5 * i for i in range(32)], 200, [37 * i % 201 for i in range(32)]), (1, 1, [0], 4300, None), (1, 1, [0], 4096, None), (2, 1, [0] * 31 + [900], 40, None),
    (1, 4, list(range(33)), 100, [0] * 32 + [100]), (1, 4, list(range(32)), 100, [0] * 31 + [100]), (3, 2, [100] * 16, 140, [0] * 7 + [140] + [0] * 8),
    (1, 2, [300] * 32, 8, [8, 0] * 16), (1, 2, [300] * 33, 8, [0, 0, 8] * 11), (2, 8, [50] * 32, 6, [0] * 32), (2, 8, [50] * 33, 6, [0] * 33), (1, 1, [0], 18000, None)])
def test_sequences_and_units_at_the_edges(torch_cuda, kvh, grp, pos, tokens, ntok):
    """As many sequences and tiles of rows as a warp has lanes, one more, and sequences without rows around those that have some."""
    torch = torch_cuda
    lens = [p + (tokens if ntok is None else ntok[s]) for s, p in enumerate(pos)]
    for width in (-(-max(lens) // 32), 700):   # with room for what they have, and for much more
        x = Setup(torch, "fp16", 32, kvh, lens, width, seed=len(pos) + tokens)
        q = x.rand(len(pos), tokens, kvh * grp, DIM)
        out = x.attn(q, pos, ntok)
        x.check(out, q, pos, ntok, sample=2)
        assert torch.equal(out, x.attn(q, pos, ntok))
