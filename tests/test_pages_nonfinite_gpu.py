"""Rows of the paged cache that are not finite: whoever sees one has outputs that are not finite, on every form of the
attention and however little the row weighs; who does not see it (behind a sequence's end, before its window, another
sequence, another head) has the outputs it would have without."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def pages(pkg, lib):
    return importlib.import_module(pkg.__name__ + ".pages")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


PAGE, H, D = 16, 3, 64


class Batch:
    """`seqs` sequences behind `prefix` shared tokens, each with `own` more.  Queries are +-1 in every component; a key is
    noise, or -5 times the query: a score of -320 at a scale of 1, whose weight is 0 in FP32."""

    def __init__(self, pages, dtype, group, seqs, prefix, own):
        g = torch.Generator(device="cuda").manual_seed(seqs + prefix)
        self.group, self.seqs, self.prefix, self.total = group, seqs, prefix, prefix + own
        entries = -(-self.total // PAGE) + 1
        self.pool = pages.PagePool.empty(1, prefix // PAGE + seqs * (-(-own // PAGE) + 2) + 3, PAGE, H, D, seqs + 1, entries, dtype)
        self.pool.k.normal_(0, 0.05, generator=g)
        self.pool.v.normal_(generator=g)
        self.list = ints(list(range(1, seqs + 1)))
        self.pool.extend(ints([0]), ints([prefix]))
        self.pool.fork(ints([0] * seqs), self.list)
        self.pool.extend(self.list, ints([own] * seqs))
        self.u = torch.randint(0, 2, (H, D), generator=g, device="cuda") * 2.0 - 1.0

    def q(self, rows, io):
        return self.u.repeat_interleave(self.group, 0)[None].expand(rows, -1, -1).to(io).contiguous()

    def place(self, seq, at):
        return int(self.pool.table[seq, at // PAGE]), at % PAGE

    def low(self, seq, lo, hi):
        for at in range(lo, hi):
            p, r = self.place(seq, at)
            self.pool.k[0, p, :, r] = (-5 * self.u).to(self.pool.k.dtype)

    def bad(self, x, seq, at, head, value):
        p, r = self.place(seq, at)
        x[0, p, head, r] = value


def lost(out, head, group):
    """Whether each row of out is not finite throughout in a KV head, and finite throughout in the others."""
    mine = out[:, head * group:(head + 1) * group].float().flatten(1)
    others = torch.cat([out[:, :head * group], out[:, (head + 1) * group:]], 1).float().flatten(1)
    return (~torch.isfinite(mine)).all(1), torch.isfinite(others).all(1)


# seqs, prefix, own: few rows (the prefix streams) and many (on the tensor cores for BF16, with the own rows after it or beside)
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("group,seqs,prefix,own", [(1, 3, 2048, 40), (4, 3, 4000, 3), (2, 70, 2048, 90), (4, 130, 1024, 500), (1, 40, 4096, 1)])
@pytest.mark.parametrize("what", ["v nan", "v inf", "k nan"])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_a_shared_row(pkg, lib, pages, dtype, group, seqs, prefix, own, what, where):
    b = Batch(pages, dtype, group, seqs, prefix, own)
    b.low(0, 0, prefix // PAGE * PAGE)  # all shared rows: their records weigh nothing
    q = b.q(seqs, dtype)
    call = lambda: b.pool.attend_prefix(q, 0, b.list, prefix, b.total, 1.0)  # noqa: E731
    plain = call()
    at = {"first": 0, "middle": prefix // 2 + 5, "last": prefix // PAGE * PAGE - 1}[where]
    b.bad(b.pool.v if what[0] == "v" else b.pool.k, 0, at, 1, INF if what[2:] == "inf" else NAN)
    mine, others = lost(call(), 1, group)
    assert bool(mine.all()) and bool(others.all())
    assert lib.attn_sync() == 0, pkg.last_error(lib)
    assert bool(torch.isfinite(plain.float()).all())


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("group,seqs,prefix,own", [(2, 70, 2048, 90), (1, 3, 512, 3000), (4, 1, 0, 5000)])
@pytest.mark.parametrize("what", ["v nan", "v inf", "k nan"])
@pytest.mark.parametrize("window", [False, True])
def test_an_own_row(pkg, lib, pages, dtype, group, seqs, prefix, own, what, window):
    """Of one sequence of a decode batch, among rows that weigh nothing."""
    b = Batch(pages, dtype, group, seqs, prefix, own)
    one = seqs // 2 + 1
    b.low(one, b.total - own, b.total - 2)
    q = b.q(seqs, dtype)
    if window:
        call = lambda: b.pool.attend_window(q, 0, b.list, None, 1, b.total, own, 0, 1.0)  # noqa: E731
    else:
        call = lambda: b.pool.attend_prefix(q, 0, b.list, prefix, b.total, 1.0)  # noqa: E731
    plain = call()
    b.bad(b.pool.v if what[0] == "v" else b.pool.k, one, b.total - own // 2 - 3, 1, INF if what[2:] == "inf" else NAN)
    out = call()
    mine, others = lost(out, 1, group)
    assert mine.tolist() == [i + 1 == one for i in range(seqs)] and bool(others.all())
    rest = [i for i in range(seqs) if i + 1 != one]
    assert torch.equal(out[rest], plain[rest])
    assert lib.attn_sync() == 0, pkg.last_error(lib)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("new", [5, 30, 300])  # both tile heights, with splits and without
@pytest.mark.parametrize("what", ["v nan", "v inf", "k nan"])
def test_a_row_that_a_chunk_sees(pkg, lib, pages, dtype, group, new, what):
    """Long before two chunks of two sequences, among rows that weigh nothing: every query of its own sequence."""
    b = Batch(pages, dtype, group, 2, 0, 2000)
    b.low(1, 0, 1500)
    q = b.q(2 * new, dtype)
    call = lambda: b.pool.attend_window(q, 0, b.list, ints([0, new, 2 * new]), new, b.total, 0, 0, 1.0)  # noqa: E731
    plain = call()
    b.bad(b.pool.v if what[0] == "v" else b.pool.k, 1, 700, 1, INF if what[2:] == "inf" else NAN)
    out = call()
    mine, others = lost(out, 1, group)
    assert mine.tolist() == [True] * new + [False] * new and bool(others.all())
    assert torch.equal(out[new:], plain[new:])
    assert lib.attn_sync() == 0, pkg.last_error(lib)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("new", [1, 7, 300])
def test_rows_out_of_sight(pkg, lib, pages, dtype, value, new):
    """Before the window of all queries, past the sinks, and behind the sequence's end in its last page."""
    b = Batch(pages, dtype, 2, 2, 0, 1001)
    q, window, sinks = b.q(2 * new, dtype), 300, 5
    call = lambda: b.pool.attend_window(q, 0, b.list, ints([0, new, 2 * new]), new, b.total, window, sinks, 1.0)  # noqa: E731
    plain = call()
    for seq in (1, 2):
        for at in [sinks, 100, b.total - new - window] + list(range(b.total, -(-b.total // PAGE) * PAGE)):
            for x in (b.pool.k, b.pool.v):
                for head in range(H):
                    b.bad(x, seq, at, head, value)
    assert torch.equal(call(), plain)
    assert lib.attn_sync() == 0, pkg.last_error(lib)
