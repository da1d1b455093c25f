"""Windows and sinks at the ends of their range."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32
MOST = 2**31 - 1


@pytest.fixture(scope="module")
def pages(pkg, lib):
    return importlib.import_module(pkg.__name__ + ".pages")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool_of(pages, lens, dtype, h, d, page, seed=0):
    pool = pages.PagePool.empty(1, sum(-(-n // page) for n in lens) + 2, page, h, d, len(lens), max(lens) // page + 2, dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool.k.normal_(generator=g)
    pool.v.normal_(generator=g)
    pool.extend(ints(list(range(len(lens)))), ints(lens))
    return pool


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("window,sinks", [(1, MOST), (1, MOST - 15), (1, MOST - 126), (MOST, 0), (MOST, MOST), (MOST - 1, 3), (400, 1000), (1, 1000)])
def test_a_trim_that_keeps_everything(pkg, lib, pages, page, window, sinks):
    pool = pool_of(pages, [1000, 1, 400], BF, 2, 64, page)
    books = [x.clone() for x in (pool.table, pool.len, pool.ref)]
    pool.trim(ints([0, 1, 2]), window, sinks)
    assert lib.attn_sync() == 0, pkg.last_error(lib)
    for x, y in zip(books, (pool.table, pool.len, pool.ref)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("window,sinks", [(MOST, 0), (MOST, MOST), (1, MOST), (MOST - 1, 7), (10, MOST - 3)])
def test_attention_that_sees_everything(pkg, lib, pages, dtype, window, sinks):
    """The same rows in sight as without a window, so the same sums."""
    pool = pool_of(pages, [700, 33], dtype, 2, 64, 32)
    q = torch.randn((130, 4, 64), device="cuda").to(dtype)
    for args in ((q[:2], 0, ints([0, 1]), None, 1, 700), (q, 0, ints([0, 1]), ints([0, 100, 130]), 100, 700)):
        assert torch.equal(pool.attend_window(*args, window, sinks, 0.125), pool.attend_window(*args, 0, 0, 0.125))
    assert lib.attn_sync() == 0, pkg.last_error(lib)
