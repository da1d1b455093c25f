"""What the paged KV cache refuses, and what it does when a wait runs out or memory does."""

import importlib
import os

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


def refused(fn, word, kind=RuntimeError):
    with pytest.raises(kind, match=word):
        fn()


def test_attention_refusals(pkg, lib, pages):
    pool = pool_of(pages, [100, 70])
    q = torch.randn((2, 4, 64), device="cuda").to(BF)
    s = ints([0, 1])
    window = lambda q=q, layer=0, seqs=s, starts=None, new=1, most=100, w=10, sinks=0, scale=1.0, out=None: pool.attend_window(  # noqa: E731
        q, layer, seqs, starts, new, most, w, sinks, scale, out)
    refused(lambda: window(layer=1), "layer")
    refused(lambda: window(layer=-1), "layer")
    refused(lambda: window(w=-1), "window")
    refused(lambda: window(sinks=-1), "sinks")
    refused(lambda: window(new=-1, starts=ints([0, 1, 2])), "max_new")
    refused(lambda: window(most=-1), "max_len")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(lambda: window(scale=scale), "scale")
    refused(lambda: window(q=q[:, :3].contiguous()), "q_heads")
    refused(lambda: window(q=torch.randn((2, 2 * 17, 64), device="cuda")), "q_heads")
    refused(lambda: window(q=q.half()), "bfloat16 or float32", ValueError)
    refused(lambda: window(q=q[:, :, :32]), "wanted", ValueError)
    refused(lambda: window(q=torch.randn((2, 8, 64), device="cuda")[:, ::2]), "one after another", ValueError)
    refused(lambda: window(seqs=s.long()), "int32", ValueError)
    refused(lambda: window(starts=ints([0, 1]), new=2), "list of 3", ValueError)
    refused(lambda: window(new=2), "starts")
    refused(lambda: window(out=torch.empty((2, 4, 64), device="cuda")), "q's shape", ValueError)
    refused(lambda: window(q=q.cpu()), "not device memory")
    refused(lambda: window(seqs=s.cpu()), "not device memory")
    refused(lambda: window(out=q.cpu()), "not device memory")
    off = torch.empty(2 * 4 * 64 + 8, device="cuda", dtype=BF)[4:4 + 512].view(2, 4, 64)
    refused(lambda: window(q=off), "aligned")
    refused(lambda: window(out=off), "aligned")
    odd = torch.empty((2, 4 * 64 + 4), device="cuda", dtype=BF)[:, :256].view(2, 4, 64)
    refused(lambda: window(q=odd), "apart")
    refused(lambda: pool.attend_prefix(q, 0, s, 101, 100, 1.0), "prefix_len")
    refused(lambda: pool.attend_prefix(q, 0, s, -1, 100, 1.0), "prefix_len")
    # nothing to do is done
    none = torch.empty((0, 4, 64), device="cuda", dtype=BF)
    assert pool.attend_prefix(none, 0, ints([]), 0, 0, 1.0).numel() == 0
    assert pool.attend_window(none, 0, s, ints([0, 0, 0]), 0, 100, 0, 0, 1.0).numel() == 0
    assert lib.attn_sync() == 0


def test_a_length_beyond_max_len_is_reported(pkg, lib, pages):
    pool = pool_of(pages, [100, 70])
    q = torch.randn((2, 4, 64), device="cuda").to(BF)
    pool.attend_window(q, 0, ints([0, 1]), None, 1, 99, 10, 0, 1.0)
    assert lib.attn_sync() != 0
    assert "index check failed" in pkg.last_error(lib)
    lib.attn_clear_error()


def test_maintenance_refusals(pkg, lib, pages):
    pool = pool_of(pages, [100, 70])
    k = torch.randn((5, 2, 64), device="cuda").to(BF)
    refused(lambda: pool.trim(ints([0]), 0), "window")
    refused(lambda: pool.trim(ints([0]), 1, -1), "sinks")
    refused(lambda: pool.extend(ints([0]), ints([1, 2])), "list of 1", ValueError)
    refused(lambda: pool.extend(ints([0]).cpu(), ints([1])), "not device memory")
    refused(lambda: pool.write(1, ints([0]), ints([0, 5]), k, k), "layer")
    refused(lambda: pool.write(0, ints([0]), ints([0, 5]), k, k[:4]), "like k_new", ValueError)
    refused(lambda: pool.write(0, ints([0]), ints([0, 5]), k.half(), k.half()), "bfloat16 or float32", ValueError)
    refused(lambda: pool.compact(torch.zeros(1, dtype=torch.int32)), "not device memory")
    refused(lambda: pool.import_cache(0, None), "KVCache is NULL")
    h = lib.kv_cache_alloc_ex(8, pkg.ATTN_KV_BF16)
    try:
        refused(lambda: pool.import_cache(0, h), "have to be the cache's")
    finally:
        lib.kv_cache_free(h)
    with pytest.raises(ValueError):
        pages.PagePool(pool.k.half(), pool.v.half(), pool.table, pool.len, pool.ref)
    with pytest.raises(ValueError):
        pages.PagePool(pool.k, pool.v, pool.table.long(), pool.len, pool.ref)
    with pytest.raises(ValueError):
        pages.PagePool(pool.k, pool.v, pool.table, pool.len, pool.ref[:-1].contiguous())
    refused(lambda: pages.PagePool(pool.k.cpu(), pool.v.cpu(), pool.table.cpu(), pool.len.cpu(), pool.ref.cpu()), "device", (RuntimeError, ValueError))
    lib.attn_clear_error()
    pool.close()
    refused(lambda: pool.compact(), "closed")
    assert lib.attn_sync() == 0


def test_waits_that_run_out_leave_the_next_call_right(pkg, lib, pages):
    """With every wait limited to a microsecond, calls may give up (and say so); with the limit back, the same
    calls give what they gave before."""
    lens = [3000, 2500, 2000, 1500]
    pools = [pool_of(pages, lens, BF, 8, 128, 64), pool_of(pages, lens, F, 2, 64, 16)]
    calls = []
    for pool in pools:
        h, d = pool.kv_heads, pool.head_dim
        q = torch.randn((400, 2 * h, d), device="cuda").to(pool.k.dtype)
        s = ints([0, 1, 2, 3])
        calls += [lambda p=pool, q=q, s=s: p.attend_window(q[:4], 0, s, None, 1, 3000, 0, 0, 0.1),
                  lambda p=pool, q=q, s=s: p.attend_window(q, 0, s, ints([0, 100, 200, 300, 400]), 100, 3000, 700, 4, 0.1),
                  lambda p=pool, q=q, s=s: p.attend_prefix(q[:4], 0, s, 0, 3000, 0.1)]
    want = [c() for c in calls]
    assert lib.attn_sync() == 0, pkg.last_error(lib)
    gave_up = 0
    assert lib.attn_set_wait_limit_ns(1000) == 0
    try:
        for c in calls:
            c()
            if lib.attn_sync() != 0:
                assert "wait timed out" in pkg.last_error(lib)
                gave_up += 1
                lib.attn_clear_error()
    finally:
        assert lib.attn_set_wait_limit_ns(2_000_000_000) == 0
    for c, w in zip(calls, want):
        assert torch.equal(c(), w)
    assert lib.attn_sync() == 0, pkg.last_error(lib)


def test_pool_allocation_failures(pkg, lib):
    """Injected on the host: NULL, a message, and everything freed."""
    torch.cuda.synchronize()
    try:
        for n in (1, 2, 3):
            os.environ["TYB_FAULT_ALLOC"] = f"{n} pages"
            free = torch.cuda.mem_get_info()[0]
            lib.attn_clear_error()
            assert not lib.kv_pages_alloc(1, 4096, 64, 8, 128, 4, 1024, pkg.ATTN_KV_BF16)
            assert "injected" in pkg.last_error(lib)
            assert torch.cuda.mem_get_info()[0] == free
    finally:
        os.environ.pop("TYB_FAULT_ALLOC", None)
        lib.attn_clear_error()
    h = lib.kv_pages_alloc(1, 8, 64, 8, 128, 4, 8, pkg.ATTN_KV_BF16)
    assert h, pkg.last_error(lib)
    lib.kv_pages_release(h)
