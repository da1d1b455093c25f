"""Host threads that share a stream: each call's launches stay together, whatever the other threads queue."""

import importlib
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def pages(pkg, lib):
    return importlib.import_module(pkg.__name__ + ".pages")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool_of(pages, lens, dtype, h, d, page, seqs, spare, seed):
    pool = pages.PagePool.empty(2, sum(-(-n // page) for n in lens) + spare, page, h, d, seqs, max(lens) // page + 2, dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool.k.normal_(generator=g)
    pool.v.normal_(generator=g)
    pool.extend(ints(list(range(len(lens)))), ints(lens))
    return pool


@pytest.mark.parametrize("shared", [False, True])
def test_two_threads_on_one_stream(pkg, lib, pages, shared):
    """Each thread copies and forks a parent of its own, decodes the branches behind the parent's rows and frees them,
    over and over; the branches answer as their parent does.  In one pool, and in one each."""
    lens, threads, batch, rounds = [1100, 830], 2, 40, 30
    make = lambda seed: pool_of(pages, lens, BF, 4, 64, 32, 2 + threads * batch, 4000, seed)  # noqa: E731
    pools = [make(1)] * 2 if shared else [make(1), make(2)]
    q = [torch.randn((1, 8, 64), device="cuda").to(BF).expand(batch, -1, -1).contiguous() for _ in range(threads)]
    want, got, errors = [], [[] for _ in range(threads)], []
    for i in range(threads):
        want.append(pools[i].attend_window(q[i][:1], 1, ints([i]), None, 1, 1100, 0, 0, 0.125))
    lists = [(ints([i] * batch), ints(list(range(2 + i * batch, 2 + (i + 1) * batch)))) for i in range(threads)]
    torch.cuda.synchronize()

    def go(i):
        try:
            src, dst = lists[i]
            for r in range(rounds):
                (pools[i].copy if r % 2 else pools[i].fork)(src, dst)
                # a fork's shared rows at once, a copy's each by themselves
                out = (pools[i].attend_window(q[i], 1, dst, None, 1, 1100, 0, 0, 0.125) if r % 2 else
                       pools[i].attend_prefix(q[i], 1, dst, lens[i], 1100, 0.125))
                pools[i].free(dst)
                got[i].append(out)
        except Exception as e:  # noqa: BLE001 (raised below)
            errors.append(e)

    ts = [threading.Thread(target=go, args=(i,)) for i in range(threads)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert lib.attn_sync() == 0, pkg.last_error(lib)
    for i in range(threads):
        for r, out in enumerate(got[i]):
            # The same rows in other groups of sums: FP32 sums, weights rounded to BF16 or not (at most 2^-8 of the mean
            # |v|, which is below 1 here), and the output's own rounding.
            assert float((out.float() - want[i].float()).abs().max()) < 2.0**-7, (i, r)
    for pool in set(pools):
        mine = [i for i in range(2)]
        assert pool.len.tolist() == [lens[i] for i in mine] + [0] * (threads * batch)
        assert int((pool.ref > 0).sum()) == sum(-(-n // 32) for n in lens)
        assert int((pool.table >= 0).sum()) == int(pool.ref.sum())
