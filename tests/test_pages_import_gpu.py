"""A BF16 static cache becomes a sequence of a BF16 pool: every row of every layer, bit for bit."""

import importlib

import numpy as np
import pytest
import torch

from gpu_helpers import check, new_cache, vp

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pages(pkg, lib):
    return importlib.import_module(pkg.__name__ + ".pages")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page,rows,capacity", [(16, 75, 100), (64, 128, 128), (128, 1, 300), (32, 301, 333)])
def test_a_bf16_cache(pkg, lib, pages, page, rows, capacity):
    rng = np.random.default_rng(rows)
    h = new_cache(pkg, lib, capacity, pkg.ATTN_KV_BF16)
    try:
        k, v = (rng.standard_normal((28, rows, 8, 128), dtype=np.float32) for _ in range(2))
        for layer in range(28):
            lib.kv_cache_append_prefill(h, layer, vp(k[layer]), vp(v[layer]), rows)
        lib.kv_cache_advance(h, rows)
        check(pkg, lib, "append")
        need = -(-rows // page)
        pool = pages.PagePool.empty(28, need + 3, page, 8, 128, 3, need + 1, torch.bfloat16)
        for t in (pool.k, pool.v):
            t.fill_(7)
        pool.extend(ints([0]), ints([page + 1]))  # pages 0 and 1 are taken
        pool.import_cache(2, h)
        assert lib.attn_sync() == 0, pkg.last_error(lib)
        assert pool.len.tolist() == [page + 1, 0, rows]
        assert pool.table[2].tolist() == list(range(2, 2 + need)) + [-1]
        for got, want in ((pool.k, k), (pool.v, v)):
            mine = got[:, 2:2 + need].transpose(2, 3).reshape(28, need * page, 8, 128)
            # the cache rounds to nearest, ties to even, as torch does
            assert torch.equal(mine[:, :rows], torch.from_numpy(want).cuda().to(torch.bfloat16))
            assert bool((mine[:, rows:] == 7).all())
            assert bool((got[:, :2] == 7).all()) and bool((got[:, 2 + need:] == 7).all())
    finally:
        lib.kv_cache_free(h)
