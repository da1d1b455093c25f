"""The paged cache's calls in captured graphs, beside other calls: what a graph names stays its own."""

import gc
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def pages(pkg, lib):
    return importlib.import_module(pkg.__name__ + ".pages")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool_of(pages, lens, dtype=BF, h=2, d=64, page=32, seed=0):
    pool = pages.PagePool.empty(1, sum(-(-n // page) for n in lens) + 2, page, h, d, len(lens), max(lens) // page + 2, dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool.k.normal_(generator=g)
    pool.v.normal_(generator=g)
    pool.extend(ints(list(range(len(lens)))), ints(lens))
    return pool


def settled(pkg, lib):
    torch.cuda.synchronize()
    lib.attn_set_stream(None)
    assert lib.attn_sync() == 0, pkg.last_error(lib)


@pytest.mark.parametrize("dtype", [BF, F])
def test_a_larger_call_leaves_a_graph_its_workspace(pkg, lib, pages, dtype):
    """Capture a small call; make a far larger one on the same stream; fill what memory it may have given back;
    replay: the same bits."""
    lens = [700 + 13 * i for i in range(200)]
    pool = pool_of(pages, lens, dtype, 4, 128, 64)
    few, all_of = ints([3, 1, 2]), ints(list(range(200)))
    q = torch.randn((600, 8, 128), device="cuda").to(dtype)
    starts = ints([0, 100, 200, 300])
    out = [torch.empty((n, 8, 128), device="cuda", dtype=dtype) for n in (3, 3, 300)]

    def small():
        pool.attend_window(q[:3], 0, few, None, 1, 3400, 0, 0, 0.1, out=out[0])
        pool.attend_prefix(q[:3], 0, few, 0, 3400, 0.1, out=out[1])
        pool.attend_window(q[:300], 0, few, starts, 100, 3400, 300, 4, 0.1, out=out[2])

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        small()
    side.synchronize()
    want = [x.clone() for x in out]
    with torch.cuda.graph(graph, stream=side):
        small()
    with torch.cuda.stream(side):
        pool.attend_window(q[:200], 0, all_of, None, 1, 3400, 0, 0, 0.1)
        pool.attend_prefix(q[:200], 0, all_of, 640, 3400, 0.1)
        pool.attend_window(q, 0, all_of, ints([3 * i for i in range(201)]), 3, 3400, 0, 0, 0.1)
    side.synchronize()
    filled = [torch.full((1 << 20,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(256)]  # whoever gets that memory next
    for _ in range(3):
        for x in out:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for x, w in zip(out, want):
            assert torch.equal(x, w)
    assert all(bool((x == 0xFF).all()) for x in filled)
    settled(pkg, lib)


def test_two_pools_captured_on_one_stream_replay_on_two(pkg, lib, pages):
    pools = [pool_of(pages, [3000 + 100 * i + 7 * p for i in range(6)], BF, 8, 128, 64, seed=p) for p in range(2)]
    seqs = ints(list(range(6)))
    q = [torch.randn((6, 16, 128), device="cuda").to(BF) for _ in pools]
    out = [torch.empty_like(x) for x in q]
    call = lambda i: pools[i].attend_window(q[i], 0, seqs, None, 1, 3600, 0, 0, 0.1, out=out[i])  # noqa: E731
    for i in range(2):
        call(i)
    torch.cuda.synchronize()
    want = [x.clone() for x in out]
    side, graphs = torch.cuda.Stream(), [torch.cuda.CUDAGraph() for _ in pools]
    for i in range(2):
        with torch.cuda.graph(graphs[i], stream=side):  # not the stream of the calls before
            for _ in range(8):
                call(i)
    streams = [torch.cuda.Stream() for _ in pools]
    for _ in range(10):
        for x in out:
            x.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for x, w in zip(out, want):
            assert torch.equal(x, w)
    settled(pkg, lib)


def test_a_capture_that_would_need_more_is_refused(pkg, lib, pages):
    pool = pool_of(pages, [500] * 300, F, 4, 64, 16)
    q = torch.randn((300, 8, 64), device="cuda")
    out, one = torch.empty_like(q), torch.empty_like(q[:1])
    pool.attend_window(q[:1], 0, ints([0]), None, 1, 500, 0, 0, 0.1, out=one)
    torch.cuda.synchronize()
    want, graph, seqs, first = one.clone(), torch.cuda.CUDAGraph(), ints(list(range(300))), ints([0])
    big = lambda: pool.attend_prefix(q, 0, seqs, 480, 500, 0.1, out=out)  # noqa: E731
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="while the stream is captured"):
            big()
        pool.attend_window(q[:1], 0, first, None, 1, 500, 0, 0, 0.1, out=one)
    one.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(one, want)
    big()
    settled(pkg, lib)


def test_a_dropped_pool_gives_its_handle_back(pkg, lib, pages):
    pages._dropped.clear()
    pool = pool_of(pages, [100])
    keep = pool.k, pool.v, pool.table, pool.len, pool.ref
    handle = pool._handle
    del pool
    gc.collect()
    assert [x[1] for x in pages._dropped] == [handle]
    again = pages.PagePool(*keep)
    assert not pages._dropped
    again.close()
    del again
    gc.collect()
    assert not pages._dropped
    settled(pkg, lib)
