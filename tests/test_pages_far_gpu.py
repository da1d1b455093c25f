"""The paged cache where offsets pass 32 bits and sequences are long: pages at the end of slabs of more than 2^31
elements, positions past a million, and every row of a hundred thousand."""

import importlib

import pytest
import torch

from pages_model import attention, rows_of, tolerance

pytestmark = pytest.mark.gpu

BF, F = torch.bfloat16, torch.float32
H, D, PAGE, HQ = 8, 128, 64, 16


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


def normal(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to("cuda", dtype)


def close(got, want, bf16_pool, bf16_io, rows):
    # Beside the tolerance of one step's arithmetic: a running FP32 sum rounds once per 32 rows at least, each time by
    # at most 2^-24 of the magnitudes so far.
    out, mean_abs, size = want
    off = (got.double().cpu() - out).abs() - tolerance(out, mean_abs, size, bf16_pool, bf16_io) - mean_abs * (rows / 32 + 1) * 2.0**-24
    assert (off <= 0).all(), f"over by {off.max().item():.3g}"


def seen(n, m, window, sinks):
    """The last n of m rows as queries."""
    p, j = torch.arange(m - n, m)[:, None], torch.arange(m)[None]
    return (j <= p) & ((j > p - window) | (j < sinks)) if window else j <= p


@pytest.fixture(params=[BF, F], ids=["bf16", "f32"])
def far(request, pages):
    """Two layers whose slabs have more than 2^31 elements each; sequence 0 has all pages but the last 60."""
    n = 17000
    pool = pages.PagePool.empty(2, n, PAGE, H, D, 8, n, request.param)
    assert pool.k.numel() > 2**31
    pool.k.fill_(float("nan"))
    pool.v.fill_(float("nan"))
    pool.extend(ints([0]), ints([(n - 60) * PAGE]))
    yield pool
    pool.close()
    del pool
    torch.cuda.empty_cache()


def test_the_last_pages_of_a_large_slab(pkg, lib, far):
    pool, dtype, n = far, far.k.dtype, [700, 130, 1]
    seqs = ints([1, 2, 3])
    pool.extend(seqs, ints(n))
    assert pool.table[1, 0] == far.k.shape[1] - 60
    k, v = (normal((sum(n), H, D), s, dtype) for s in (1, 2))
    for layer in (0, 1):
        pool.write(layer, seqs, ints([0, 700, 830, 831]), k + layer, v - layer)
    # two branches of the 700, one a copy; each grows by its own rows
    pool.fork(ints([1]), ints([4]))
    pool.copy(ints([1]), ints([5]))
    more = ints([4, 5])
    pool.extend(more, ints([30, 30]))
    k2, v2 = (normal((60, H, D), s, dtype) for s in (3, 4))
    pool.write(1, more, ints([0, 30, 60]), k2, v2)
    assert synced(pkg, lib) == ""
    rows = {s: rows_of(pool, 1, s) for s in (1, 2, 3, 4, 5)}
    assert torch.equal(rows[1][0], (k[:700] + 1).double().cpu()) and torch.equal(rows[2][1], (v[700:830] - 1).double().cpu())
    assert torch.equal(rows[4][0], torch.cat([k[:700] + 1, k2[:30]]).double().cpu())
    assert torch.equal(rows[5][1], torch.cat([v[:700] - 1, v2[30:]]).double().cpu())

    def attend():
        q = normal((5, HQ, D), 5, dtype)
        one = pool.attend_window(q, 1, ints([1, 2, 3, 4, 5]), None, 1, 730, 200, 3, 0.1)
        shared = pool.attend_prefix(q[:3], 1, ints([4, 1, 4]), 640, 730, 0.1)
        wide = pool.attend_prefix(q[:1].repeat(40, 1, 1), 1, ints([4] * 40), 700, 730, 0.1)
        chunk = pool.attend_window(normal((160, HQ, D), 6, dtype), 1, ints([4, 2]), ints([0, 30, 160]), 130, 730, 200, 3, 0.1)
        assert synced(pkg, lib) == ""
        return one, shared, wide, chunk

    before = attend()
    q = normal((5, HQ, D), 5, dtype).double().cpu()
    bf = dtype == BF
    for i, s in enumerate((1, 2, 3, 4, 5)):
        kk, vv, _ = rows[s]
        close(before[0][i:i + 1], attention(q[i:i + 1], kk, vv, seen(1, len(kk), 200, 3), 0.1), bf, bf, len(kk))
    kk, vv, _ = rows[4]
    close(before[1][:1], attention(q[:1], kk, vv, seen(1, 730, 0, 0), 0.1), bf, bf, 730)
    close(before[2][39:], attention(q[:1], kk, vv, seen(1, 730, 0, 0), 0.1), bf, bf, 730)
    close(before[3][:30], attention(normal((160, HQ, D), 6, dtype)[:30].double().cpu(), kk, vv, seen(30, 730, 200, 3), 0.1), bf, bf, 730)

    # The large sequence goes; what is left moves to the slab's start and reads the same.
    pool.free(ints([0]))
    live = ints([0])
    pool.compact(live)
    assert synced(pkg, lib) == "" and int(live) == int((pool.ref > 0).sum()) and int(pool.table.max()) == int(live) - 1
    for a, b in zip(before, attend()):
        assert torch.equal(a, b)


def test_positions_past_a_million(pkg, lib, far):
    pool, dtype, n = far, far.k.dtype, 1500
    first = int(pool.len[0])
    assert first > 2**20
    pool.extend(ints([0]), ints([n]))
    k, v = (normal((n, H, D), s, dtype) for s in (7, 8))
    pool.write(1, ints([0]), ints([0, n]), k, v)
    for i, x in ((0, pool.k), (1, pool.v)):
        x[1, int(pool.table[0, 0])] = normal((H, PAGE, D), 9 + i, dtype)
    sinks, window, c = 5, 1000, 200
    q = normal((c, HQ, D), 11, dtype)
    got = pool.attend_window(q, 1, ints([0]), ints([0, c]), c, first + n, window, sinks, 0.09)
    one = pool.attend_window(q[-1:], 1, ints([0]), None, 1, first + n, window, sinks, 0.09)
    assert synced(pkg, lib) == ""
    head = [x[1, int(pool.table[0, 0]), :, :sinks].transpose(0, 1) for x in (pool.k, pool.v)]
    kk, vv = (torch.cat([a, b]).double().cpu() for a, b in zip(head, (k, v)))
    want = attention(q.double().cpu(), kk, vv, seen(c, n + sinks, window, sinks), 0.09)
    bf = dtype == BF
    close(got, want, bf, bf, window)
    close(one, [w[-1:] for w in want], bf, bf, window)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("batch", [3, 50])
def test_every_row_of_a_hundred_thousand(pkg, lib, pages, dtype, batch):
    n, h, d, hq = 100_003, 2, 64, 6
    pool = pages.PagePool.empty(1, n // 16 + 2 * batch + 2, 16, h, d, batch + 1, n // 16 + 3, dtype)
    k, v = (normal((n, h, d), s, dtype) for s in (12, 13))
    pool.extend(ints([0]), ints([n]))
    pool.write(0, ints([0]), ints([0, n]), k, v)
    pool.fork(ints([0] * batch), ints(list(range(1, batch + 1))))
    q = normal((batch, hq, d), 14, dtype)
    seqs = ints(list(range(1, batch + 1)))
    alone = pool.attend_window(q, 0, seqs, None, 1, n, 0, 0, 0.2)
    behind = pool.attend_prefix(q, 0, seqs, n - 50, n, 0.2)
    assert synced(pkg, lib) == ""
    want = attention(q.double().cpu()[-2:], k.double().cpu(), v.double().cpu(), seen(1, n, 0, 0).expand(2, n), 0.2)
    close(alone[-2:], want, dtype == BF, dtype == BF, n)
    close(behind[-2:], want, dtype == BF, dtype == BF, n)
