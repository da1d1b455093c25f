"""Attention over the paged cache (a shared prefix, a window with sinks) against 64-bit attention from
its definition; the tolerances are derived in pages_model.tolerance."""

import importlib

import pytest
import torch

from pages_model import attention, rows_of, tolerance

pytestmark = pytest.mark.gpu

BF, F = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def pages(pkg, lib):
    return importlib.import_module(pkg.__name__ + ".pages")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def synced(pkg, lib):
    lib.attn_sync()
    msg = pkg.last_error(lib)
    lib.attn_clear_error()
    return msg


def filled(pages, lens, page, h, d, dtype, seed, layers=1, layer=0, spare=5):
    """A pool of random rows in scattered pages; everything else in it is NaN."""
    need = [-(-n // page) for n in lens]
    n = sum(need) + spare
    pool = pages.PagePool.empty(layers, n, page, h, d, len(lens) + 2, max(need + [1]) + 1, dtype)
    pool.k.fill_(float("nan"))
    pool.v.fill_(float("nan"))
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(n, generator=g).tolist()
    for s, c in enumerate(lens):
        mine = [order.pop() for _ in range(need[s])]
        pool.table[s, :need[s]] = ints(mine)
        pool.len[s] = c
        for e, p in enumerate(mine):
            m = min(page, c - e * page)
            pool.k[layer, p, :, :m] = torch.randn((h, m, d), generator=g).to("cuda", dtype)
            pool.v[layer, p, :, :m] = torch.randn((h, m, d), generator=g).to("cuda", dtype)
            pool.ref[p] = 1
    return pool


def close(got, want, pool, io):
    out, mean_abs, size = want
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    off = (got - out).abs() - tolerance(out, mean_abs, size, pool.k.dtype == BF, io == BF)
    assert (off <= 0).all(), f"over by {off.max().item():.3g} (values about {out.abs().mean().item():.3g})"


def queries(n, hq, d, io, pool, seed):
    q = torch.randn((n, hq, d), generator=torch.Generator().manual_seed(seed)).to("cuda", io)
    return q, (q.to(BF) if pool.k.dtype == BF else q).double().cpu()  # a BF16 pool multiplies BF16 operands


SHAPES = [(16, 8, 128), (8, 8, 64), (12, 4, 64), (10, 2, 128), (16, 1, 128), (7, 7, 128), (32, 2, 64), (9, 3, 64)]


@pytest.mark.parametrize("dtype,io", [(BF, BF), (F, F), (BF, F), (F, BF)])
@pytest.mark.parametrize("hq,h,d", SHAPES[:4])
@pytest.mark.parametrize("page,batch,prefix,own", [(16, 2, 16, 1), (64, 5, 100, 30), (32, 37, 333, 70), (128, 3, 1000, 300),
                                                  (64, 70, 0, 40), (16, 9, 15, 3)])
def test_prefix(pkg, lib, pages, dtype, io, hq, h, d, page, batch, prefix, own):
    # Sequence 0 holds the prefix; the others branch off it, then each grows by its own rows.
    pool = filled(pages, [prefix], page, h, d, dtype, batch + prefix, spare=batch * (own // page + 3))
    big = pages.PagePool(pool.k, pool.v, torch.full((batch + 1, prefix // page + own // page + 3), -1, dtype=torch.int32, device="cuda"),
                         torch.zeros(batch + 1, dtype=torch.int32, device="cuda"), pool.ref)
    w = pool.table.shape[1]
    big.table[0, :min(w, big.table.shape[1])] = pool.table[0, :big.table.shape[1]]
    big.len[0] = prefix
    big.fork(ints([0] * batch), ints(list(range(1, batch + 1))))
    counts = [1 + (7 * i) % own for i in range(batch)]
    seqs = ints([batch - i for i in range(batch)])
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn((starts[-1], h, d), generator=g).to("cuda", dtype) for _ in range(2))
    big.extend(seqs, ints(counts))
    big.write(0, seqs, ints(starts), k, v)
    q, q64 = queries(batch, hq, d, io, pool, 4)
    scale = d**-0.5
    got = big.attend_prefix(q, 0, seqs, prefix, prefix + own, scale)
    assert synced(pkg, lib) == ""
    for b in range(0, batch, 1 + batch // 12):
        kk, vv, there = rows_of(big, 0, batch - b)
        close(got[b:b + 1], attention(q64[b:b + 1], kk, vv, there[None], scale), big, io)


def see_window(pos, n, there, window, sinks):
    j = torch.arange(n)[None]
    p = torch.tensor(pos)[:, None]
    see = (j <= p) & there[None]
    if window:
        see &= (j > p - window) | (j < sinks)
    return see


@pytest.mark.parametrize("dtype,io", [(BF, BF), (F, F), (BF, F)])
@pytest.mark.parametrize("hq,h,d", SHAPES)
@pytest.mark.parametrize("page,window,sinks", [(16, 5, 0), (64, 100, 4), (32, 1, 1), (128, 0, 0), (64, 10000, 70), (16, 64, 300)])
def test_window_tokens(pkg, lib, pages, dtype, io, hq, h, d, page, window, sinks):
    lens = [1, 2, 15, 16, 17, 64, 200, 333, 1030, 0]
    pool = filled(pages, lens, page, h, d, dtype, 7, layers=2, layer=1)
    q, q64 = queries(len(lens), hq, d, io, pool, 8)
    scale = 1.7 * d**-0.5
    order = [3, 8, 0, 9, 5, 1, 7, 2, 6, 4]
    got = pool.attend_window(q, 1, ints(order), None, 1, max(lens), window, sinks, scale)
    assert synced(pkg, lib) == ""
    for b, s in enumerate(order):
        if lens[s] == 0:  # nothing to see
            assert (got[b] == 0).all()
            continue
        k, v, there = rows_of(pool, 1, s)
        close(got[b:b + 1], attention(q64[b:b + 1], k, v, see_window([lens[s] - 1], lens[s], there, window, sinks), scale), pool, io)


@pytest.mark.parametrize("dtype,io", [(BF, BF), (F, F), (BF, F)])
@pytest.mark.parametrize("hq,h,d", SHAPES)
@pytest.mark.parametrize("page,window,sinks", [(16, 5, 0), (64, 100, 4), (32, 1, 1), (128, 0, 0), (64, 300, 140)])
def test_window_chunks(pkg, lib, pages, dtype, io, hq, h, d, page, window, sinks):
    new = [1, 0, 130, 64, 3, 257]
    past = [0, 50, 0, 333, 128, 700]
    lens = [a + b for a, b in zip(new, past)]
    pool = filled(pages, lens, page, h, d, dtype, 9)
    starts = [0]
    for c in new:
        starts.append(starts[-1] + c)
    q, q64 = queries(starts[-1], hq, d, io, pool, 10)
    scale = d**-0.5
    got = pool.attend_window(q, 0, ints(list(range(6))), ints(starts), max(new), max(lens), window, sinks, scale)
    assert synced(pkg, lib) == ""
    for s in range(6):
        if not new[s]:
            continue
        k, v, there = rows_of(pool, 0, s)
        see = see_window(list(range(past[s], lens[s])), lens[s], there, window, sinks)
        close(got[starts[s]:starts[s + 1]], attention(q64[starts[s]:starts[s + 1]], k, v, see, scale), pool, io)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("n", [1, 70])
def test_pages_given_back_are_not_seen(pkg, lib, pages, dtype, n):
    """After a trim the window form is unchanged; rows whose pages are all gone see nothing and give zeros."""
    pool = filled(pages, [700, 700], 32, 2, 64, dtype, 11)
    q, q64 = queries(2 * n, 4, 64, F, pool, 12)
    args = (0, ints([0, 1]), ints([0, n, 2 * n]), n, 700, 100, 40, 0.125)
    before = pool.attend_window(q, *args)
    pool.trim(ints([0, 1]), 100 + n, 40)
    gone = int((pool.table[:2, :700 // 32 + 1] < 0).sum())
    assert gone == 2 * ((700 - 100 - n) // 32 - 2)
    for t in (pool.k, pool.v):
        t[:, pool.ref == 0] = float("nan")
    assert torch.equal(pool.attend_window(q, *args), before)
    pool.free(ints([0]))
    pool.len[0] = 700  # a table of nothing
    got = pool.attend_window(q, *args)
    assert (got[:n] == 0).all() and torch.equal(got[n:], before[n:])
    # the first pages gone: early queries without sinks see less, the first none
    pool.table[1, :3] = -1
    got = pool.attend_window(q[n:], 0, ints([1]), ints([0, n]), n, 700, 0, 0, 0.125)
    assert synced(pkg, lib) == ""
    k, v, there = rows_of(pool, 0, 1)
    close(got, attention(q64[n:], k, v, see_window(list(range(700 - n, 700)), 700, there, 0, 0), 0.125), pool, F)


@pytest.mark.parametrize("dtype", [BF, F])
def test_a_long_prompt_from_the_first_token(pkg, lib, pages, dtype):
    pool = filled(pages, [1500], 64, 8, 128, dtype, 13)
    q, q64 = queries(1500, 16, 128, dtype, pool, 14)
    got = pool.attend_window(q, 0, ints([0]), ints([0, 1500]), 1500, 1500, 256, 4, 128**-0.5)
    assert synced(pkg, lib) == ""
    k, v, there = rows_of(pool, 0, 0)
    close(got, attention(q64, k, v, see_window(list(range(1500)), 1500, there, 256, 4), 128**-0.5), pool, dtype)


@pytest.mark.parametrize("dtype", [BF, F])
def test_large_scores(pkg, lib, pages, dtype):
    """Scores in the hundreds, rising and falling along the sequence: the running maximum has to move."""
    pool = filled(pages, [900], 64, 2, 128, dtype, 15)
    pool.k *= 12
    q, q64 = queries(300, 4, 128, dtype, pool, 16)
    for window in (0, 200):
        got = pool.attend_window(q, 0, ints([0]), ints([0, 300]), 300, 900, window, 2, 1.0)
        k, v, there = rows_of(pool, 0, 0)
        close(got, attention(q64, k, v, see_window(list(range(600, 900)), 900, there, window, 2), 1.0), pool, dtype)
        got = pool.attend_window(q[:1], 0, ints([0]), None, 1, 900, window, 2, 1.0)
        close(got, attention(q64[:1], k, v, see_window([899], 900, there, window, 2), 1.0), pool, dtype)
    assert synced(pkg, lib) == ""


def test_a_strided_query_and_an_own_output(pkg, lib, pages):
    pool = filled(pages, [300, 200], 32, 2, 128, BF, 17)
    fused = torch.randn((50, 8 * 128), device="cuda").to(BF)
    q = fused[:, 256:768].view(50, 4, 128)
    out = torch.full((50, 4, 128), float("nan"), device="cuda", dtype=BF)
    args = (0, ints([1, 0]), ints([0, 20, 50]), 30, 300, 64, 2, 0.1)
    assert pool.attend_window(q, *args, out=out) is out
    assert torch.equal(out, pool.attend_window(q.contiguous(), *args))
    a = pool.attend_prefix(q[:2], 0, ints([0, 1]), 0, 300, 0.1)
    assert torch.equal(a, pool.attend_prefix(q[:2].contiguous(), 0, ints([0, 1]), 0, 300, 0.1))
    assert synced(pkg, lib) == ""


def test_bad_numbers_on_the_device(pkg, lib, pages):
    """Sequences, lengths, pages and query ranges outside their bounds: a status, and nothing out of bounds."""
    pool = filled(pages, [300, 200], 32, 2, 64, BF, 18)
    q = torch.randn((2, 4, 64), device="cuda").to(BF)
    qs = torch.randn((80, 4, 64), device="cuda").to(BF)

    def bad(fn):
        fn()
        assert "index check failed" in synced(pkg, lib)

    bad(lambda: pool.attend_window(q, 0, ints([0, 4]), None, 1, 300, 10, 0, 1.0))
    bad(lambda: pool.attend_window(q, 0, ints([-1, 1]), None, 1, 300, 10, 0, 1.0))
    bad(lambda: pool.attend_prefix(q, 0, ints([9, 1]), 64, 300, 1.0))
    bad(lambda: pool.attend_window(qs, 0, ints([0, 7]), ints([0, 40, 80]), 40, 300, 10, 0, 1.0))
    bad(lambda: pool.attend_window(qs, 0, ints([0, 1]), ints([0, 40, 90]), 50, 300, 10, 0, 1.0))
    pool.len[1] = 10  # more queries than tokens
    bad(lambda: pool.attend_window(qs, 0, ints([0, 1]), ints([0, 40, 80]), 40, 300, 10, 0, 1.0))
    pool.len[1] = 32 * pool.table.shape[1] + 1
    bad(lambda: pool.attend_window(q, 0, ints([0, 1]), None, 1, 300, 10, 0, 1.0))
    pool.len[1] = 200
    pool.table[1, 5] = pool.ref.numel()
    bad(lambda: pool.attend_window(q, 0, ints([0, 1]), None, 1, 300, 0, 0, 1.0))
    bad(lambda: pool.attend_window(qs, 0, ints([0, 1]), ints([0, 40, 80]), 40, 300, 0, 0, 1.0))


def test_repeatable_and_on_another_stream(pkg, lib, pages):
    pool = filled(pages, [900, 800, 700], 64, 8, 128, BF, 19)
    q = torch.randn((300, 16, 128), device="cuda").to(BF)
    calls = [lambda: pool.attend_window(q, 0, ints([0, 1, 2]), ints([0, 100, 200, 300]), 100, 900, 300, 4, 0.09),
             lambda: pool.attend_window(q[:3], 0, ints([0, 1, 2]), None, 1, 900, 300, 4, 0.09),
             lambda: pool.attend_prefix(q[:3], 0, ints([0, 1, 2]), 0, 900, 0.09)]
    first = [c() for c in calls]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = [c() for c in calls]
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    lib.attn_set_stream(None)
    assert synced(pkg, lib) == ""


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("hq,h,d", [(16, 8, 128), (8, 8, 64), (12, 4, 64), (32, 2, 64)])
@pytest.mark.parametrize("batch", [3, 8, 20])
def test_a_shared_prefix_repeats_exactly(pkg, lib, pages, dtype, hq, h, d, batch):
    # Which sequences a run joins together is a matter of timing; the sums are not.
    prefix, page = 1500, 64
    pool = filled(pages, [prefix], page, h, d, dtype, 30, spare=batch)
    big = pages.PagePool(pool.k, pool.v, torch.full((batch + 1, pool.table.shape[1] + 1), -1, dtype=torch.int32, device="cuda"),
                         torch.zeros(batch + 1, dtype=torch.int32, device="cuda"), pool.ref)
    big.table[0, :pool.table.shape[1]] = pool.table[0]
    big.len[0] = prefix
    big.fork(ints([0] * batch), ints(list(range(1, batch + 1))))
    seqs = ints(list(range(1, batch + 1)))
    q, _ = queries(batch, hq, d, dtype, pool, 31)
    want = big.attend_prefix(q, 0, seqs, 1472, prefix, d**-0.5)
    for _ in range(20):
        assert torch.equal(big.attend_prefix(q, 0, seqs, 1472, prefix, d**-0.5), want)
    assert synced(pkg, lib) == ""


@pytest.mark.parametrize("hq,h,d,batch,prefix,own", [(4, 2, 64, 1100, 700, 20), (16, 8, 128, 70, 2000, 300), (9, 3, 64, 200, 3000, 30),
                                                     (14, 7, 128, 33, 1000, 90)])
def test_a_large_batch_in_a_graph(pkg, lib, pages, hq, h, d, batch, prefix, own):
    # Shared rows on the tensor cores with the own rows beside them: more sequences than one launch has, odd numbers of
    # KV heads, and replays back to back, each of which overwrites what the one before left.
    page = 16
    pool = filled(pages, [prefix], page, h, d, BF, 40, spare=batch * (own // page + 3))
    big = pages.PagePool(pool.k, pool.v, torch.full((batch + 1, prefix // page + own // page + 3), -1, dtype=torch.int32, device="cuda"),
                         torch.zeros(batch + 1, dtype=torch.int32, device="cuda"), pool.ref)
    w = min(pool.table.shape[1], big.table.shape[1])
    big.table[0, :w] = pool.table[0, :w]
    big.len[0] = prefix
    seqs = ints(list(range(1, batch + 1)))
    big.fork(ints([0] * batch), seqs)
    counts = [1 + 7 * i % own for i in range(batch)]
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    g = torch.Generator().manual_seed(41)
    k, v = (torch.randn((starts[-1], h, d), generator=g).to("cuda", BF) for _ in range(2))
    big.extend(seqs, ints(counts))
    big.write(0, seqs, ints(starts), k, v)
    q, q64 = queries(batch, hq, d, BF, pool, 42)
    other = torch.randn_like(q)
    scale = d**-0.5
    want = big.attend_prefix(q, 0, seqs, prefix, prefix + own, scale)
    want_other = big.attend_prefix(other, 0, seqs, prefix, prefix + own, scale)
    assert synced(pkg, lib) == ""
    for b in (0, 1, batch // 2, batch - 1):
        kk, vv, there = rows_of(big, 0, b + 1)
        close(want[b:b + 1], attention(q64[b:b + 1], kk, vv, there[None], scale), big, BF)
    side, graph, out, out_other = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.empty_like(q), torch.empty_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big.attend_prefix(q, 0, seqs, prefix, prefix + own, scale, out=out)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        big.attend_prefix(q, 0, seqs, prefix, prefix + own, scale, out=out)
        big.attend_prefix(other, 0, seqs, prefix, prefix + own, scale, out=out_other)
    for _ in range(5):
        out.zero_()
        out_other.zero_()
        for _ in range(4):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out_other, want_other)
    lib.attn_set_stream(None)
    assert synced(pkg, lib) == ""
