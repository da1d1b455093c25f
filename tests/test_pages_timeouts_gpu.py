"""Waits of the paged attention that run out, and what follows: the limit is set to its least, a microsecond, so that
calls of some hundred megabytes, whose copies take longer to come, give up; nothing hangs and nothing faults."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32
LEAST, USUAL = 1000, 2_000_000_000


@pytest.fixture(scope="module")
def pages(pkg, lib):
    return importlib.import_module(pkg.__name__ + ".pages")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def outcome(pkg, lib):
    """attn_sync: "" or its message."""
    rc = lib.attn_sync()
    msg = pkg.last_error(lib) if rc else ""
    lib.attn_clear_error()
    return msg


class Setup:
    """Some long sequences whose decode is cut into many runs."""

    def __init__(self, pages, dtype):
        self.lens = [5003 + 97 * i for i in range(40)]
        self.pool = pages.PagePool.empty(1, sum(-(-n // 64) for n in self.lens) + 2, 64, 8, 128, 40, 150, dtype)
        self.pool.k.normal_()
        self.pool.v.normal_()
        self.all = ints(list(range(40)))
        self.pool.extend(self.all, ints(self.lens))
        self.q = torch.randn((40, 16, 128), device="cuda").to(dtype)
        self.few = ints([0, 20, 39])

        self.busy = torch.empty((2, 1 << 28), dtype=torch.uint8, device="cuda")
        self.side = torch.cuda.Stream()

    def large(self, out=None):
        return self.pool.attend_window(self.q, 0, self.all, None, 1, 9000, 0, 0, 0.1, out=out)

    def small(self, out=None):
        return self.pool.attend_window(self.q[:3], 0, self.few, None, 1, 9000, 3000, 4, 0.1, out=out)


def give_up(lib, s, limit):
    """A large call at a small limit, beside copies that keep the memory busy."""
    with torch.cuda.stream(s.side):
        for _ in range(2):
            s.busy[1].copy_(s.busy[0])
    assert lib.attn_set_wait_limit_ns(limit) == 0
    try:
        s.large()
        torch.cuda.synchronize()
    finally:
        assert lib.attn_set_wait_limit_ns(USUAL) == 0


@pytest.mark.parametrize("dtype", [BF, F])
def test_graphs_after_a_wait_that_ran_out(pkg, lib, pages, dtype):
    """Once attn_sync has reported it, replays and calls give the bits they gave before, however far the call had
    counted when it gave up."""
    s = Setup(pages, dtype)
    out, out_large = torch.empty_like(s.q[:3]), torch.empty_like(s.q)
    want, want_large = s.small().clone(), s.large().clone()
    small, large = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(small):
        s.small(out)
    with torch.cuda.graph(large):
        s.large(out_large)
    lib.attn_set_stream(None)
    assert outcome(pkg, lib) == ""
    gave_up = 0
    for limit in (LEAST, 2000, 3000, 4000, 6000, 8000):
        for _ in range(6):
            give_up(lib, s, limit)
            msg = outcome(pkg, lib)
            assert msg == "" or "wait timed out" in msg
            gave_up += msg != ""
            for _ in range(2):  # no call of the host's between the report and the replays
                out.fill_(float("nan"))
                out_large.fill_(float("nan"))
                small.replay()
                large.replay()
                torch.cuda.synchronize()
                assert outcome(pkg, lib) == ""
                assert torch.equal(out, want) and torch.equal(out_large, want_large)
    assert gave_up > 0
    assert torch.equal(s.large(), want_large)
    assert outcome(pkg, lib) == ""


def test_another_pool_goes_on(pkg, lib, pages):
    s, other = Setup(pages, BF), Setup(pages, BF)
    want = other.small().clone()
    assert outcome(pkg, lib) == ""
    gave_up = 0
    for _ in range(10):
        give_up(lib, s, LEAST)
        assert torch.equal(other.small(), want)
        gave_up += outcome(pkg, lib) != ""
        assert torch.equal(other.small(), want)
        s.small()
        assert outcome(pkg, lib) == ""
    assert gave_up > 0
