"""GPU: the KV caches' calls from host threads other than the one that set CUDA up: as a thread's first call of all, and several
threads at the same time."""
import threading

import pytest

import atlas_cuda
from paged_ref import DIM
from test_gpu_paged_attn import Setup, _i32

pytestmark = pytest.mark.gpu


def _in_threads(works):
    wrong = []

    def guarded(work):
        try:
            work()
        except Exception as e:   # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=guarded, args=(w,)) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def _paged(torch, tokens):
    x = Setup(torch, "fp16", 32, 2, [300 + tokens, 100 + tokens], 30, seed=tokens, poison=False)
    pos, q, k = _i32(torch, [300, 100]), x.rand(2, tokens, 10, DIM), x.rand(2, tokens, 2, DIM)
    out, one = torch.full_like(q, 7.0), torch.zeros(1, dtype=torch.int32, device="cuda")
    same = torch.arange(2, dtype=torch.int32, device="cuda")
    return {"append": lambda: atlas_cuda.paged_append(x.c, 0, tokens, pos, k, k), "fork": lambda: atlas_cuda.paged_fork(x.c, same, pos + tokens),
            "reserve": lambda: atlas_cuda.paged_reserve(x.c, tokens, pos, one), "compact": lambda: atlas_cuda.paged_compact(x.c, one),
            "attn": lambda: atlas_cuda.paged_attn(x.c, 0, 10, tokens, pos, q, out)}, (out, x.k, x.v, x.table, x.refs, one)


def _kv8(torch, tokens):
    nseq, heads, ctx, block = 2, 2, 600, 16
    g = torch.Generator(device="cuda").manual_seed(tokens)
    blocks = -(-ctx // block)
    z = lambda *s, kind: torch.zeros(*s, dtype=kind, device="cuda")  # noqa: E731
    c = atlas_cuda.Kv8Cache(z(nseq, heads, ctx, DIM, kind=torch.int8), z(nseq, heads, ctx, DIM, kind=torch.int8), z(nseq, heads, blocks, kind=torch.float32),
                            z(nseq, heads, blocks, kind=torch.float32), z(nseq, heads, blocks, DIM, kind=torch.int16), nseq=nseq, kv_heads=heads, max_context=ctx,
                            block=block)
    rand = lambda n, h: torch.randn(nseq, n, h, DIM, generator=g, device="cuda")  # noqa: E731
    k, v, q, pos = rand(200, heads), rand(200, heads), rand(tokens, 10), _i32(torch, [200 - tokens] * 2)
    atlas_cuda.kv8_append(c, 200, _i32(torch, [0, 0]), k, v)
    out, sel, back = torch.zeros_like(q), z(nseq, tokens, heads, 4, kind=torch.int32), torch.zeros_like(k)
    start = _i32(torch, [0, 0])
    return {"append": lambda: atlas_cuda.kv8_append(c, 200, start, k, v), "read": lambda: atlas_cuda.kv8_read(c, 200, start, back, back.clone()),
            "attn": lambda: atlas_cuda.kv8_attn(c, 10, tokens, pos, q, out),
            "attn_sparse": lambda: atlas_cuda.kv8_attn_sparse(c, 10, tokens, 4, pos, q, out, sel)}, (out, sel, *c.buffers)


@pytest.mark.parametrize("cache", [_paged, _kv8])
@pytest.mark.parametrize("tokens", [1, 3, 40, 150])
def test_first_call_of_a_thread(torch_cuda, cache, tokens):
    """Each call, made by a thread that has made no other, gives what it gives in this one."""
    torch = torch_cuda
    for name in cache(torch, tokens)[0]:
        calls, want = cache(torch, tokens)
        calls[name]()
        torch.cuda.synchronize()
        calls, got = cache(torch, tokens)
        torch.cuda.synchronize()
        _in_threads([calls[name]])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name


def test_threads_with_caches_of_their_own(torch_cuda):
    """Threads that call at the same time, each on its own cache and stream."""
    torch = torch_cuda
    jobs = []
    for i, tokens in enumerate((1, 3, 40, 300)):
        x = Setup(torch, "fp16", 32, 2, [300 + tokens, 100 + tokens], 30, seed=i, poison=False)
        q, pos = x.rand(2, tokens, 10, DIM), _i32(torch, [300, 100])
        jobs.append((x, q, pos, x.attn(q, [300, 100]), torch.full_like(q, 7.0), torch.cuda.Stream()))
    torch.cuda.synchronize()

    def work(x, q, pos, want, out, side):
        for _ in range(50):
            atlas_cuda.paged_attn(x.c, 0, 10, q.shape[1], pos, q, out, stream=side.cuda_stream)
        side.synchronize()
        assert torch.equal(out, want)

    _in_threads([lambda j=j: work(*j) for j in jobs])
