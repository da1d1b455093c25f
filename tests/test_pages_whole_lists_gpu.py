"""A maintenance call that a single entry of its list makes wrong changes nothing, wherever that entry stands; a write
places row by row."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def pages(pkg, lib):
    return importlib.import_module(pkg.__name__ + ".pages")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def outcome(pkg, lib):
    rc = lib.attn_sync()
    msg = pkg.last_error(lib) if rc else ""
    lib.attn_clear_error()
    return msg


PAGE = 16


def pool_of(pages, seqs, entries=20):
    """`seqs` sequences of 3 .. 300 tokens, and two that are not in use."""
    lens = [3 + 31 * i % 298 for i in range(seqs)]
    pool = pages.PagePool.empty(1, sum(-(-n // PAGE) for n in lens) + 50, PAGE, 1, 64, seqs + 2, entries, BF)
    pool.extend(ints(list(range(seqs))), ints(lens))
    return pool


def books(pool):
    return [x.clone() for x in (pool.table, pool.len, pool.ref)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


CALLS = {"free": lambda pool, s: pool.free(s), "trim": lambda pool, s: pool.trim(s, 20, 17)}


@pytest.mark.parametrize("call", list(CALLS))
@pytest.mark.parametrize("seqs", [2, 7, 255, 256, 257, 700])
@pytest.mark.parametrize("bad", [-1, 10**6, -(2**31), 2**31 - 1])
def test_a_number_that_is_no_sequence(pkg, lib, pages, call, seqs, bad):
    pool = pool_of(pages, seqs)
    before = books(pool)
    for at in {0, 1, seqs // 2, seqs - 1}:
        wrong = list(range(seqs))
        wrong[at] = bad
        CALLS[call](pool, ints(wrong))
        assert "index check failed" in outcome(pkg, lib)
        assert same(books(pool), before), at
    CALLS[call](pool, ints(list(range(seqs))))
    assert outcome(pkg, lib) == ""
    assert same(books(pool), before) == (call == "trim" and seqs == 2)  # (3 and 34 tokens: nothing to trim)


@pytest.mark.parametrize("call", list(CALLS))
@pytest.mark.parametrize("seqs", [1, 7, 256, 700])
def test_a_table_that_names_no_page(pkg, lib, pages, call, seqs):
    pool = pool_of(pages, seqs)
    last = seqs - 1
    pool.len[last] = 20 * PAGE
    for entry in (2, 9, 17):  # of those that either call would take
        keep = int(pool.table[last, entry])
        for bad in (pool.ref.numel(), 2**31 - 1):
            pool.table[last, entry] = bad
            before = books(pool)
            CALLS[call](pool, ints(list(range(seqs))))
            assert "index check failed" in outcome(pkg, lib)
            assert same(books(pool), before)
        pool.table[last, entry] = keep
    CALLS[call](pool, ints(list(range(seqs))))
    assert outcome(pkg, lib) == ""


@pytest.mark.parametrize("seqs", [3, 300])
@pytest.mark.parametrize("bad", [-1, 20 * PAGE + 1, -(2**31), 2**31 - 1])
def test_a_length_that_is_none(pkg, lib, pages, seqs, bad):
    """Trim goes by it and refuses; free does not, and puts it right."""
    pool = pool_of(pages, seqs)
    pool.len[1] = bad
    before, all_of = books(pool), ints(list(range(seqs)))
    pool.trim(all_of, 20, 17)
    assert "index check failed" in outcome(pkg, lib)
    assert same(books(pool), before)
    pool.free(all_of)
    assert outcome(pkg, lib) == ""
    assert int(pool.ref.abs().sum()) == 0 and int(pool.len.abs().sum()) == 0 and bool((pool.table == -1).all())


@pytest.mark.parametrize("seqs", [1, 3, 100, 256, 300])
def test_a_sequence_named_often_is_freed_once(pkg, lib, pages, seqs):
    pool = pool_of(pages, 3)
    pool.fork(ints([0]), ints([3]))
    pool.free(ints([0] * seqs))
    assert outcome(pkg, lib) == ""
    assert pool.len.tolist()[0] == 0
    named = pool.table[pool.table >= 0].long()
    assert torch.equal(torch.bincount(named, minlength=pool.ref.numel()).to(torch.int32), pool.ref)


@pytest.mark.parametrize("deep", [False, True])
@pytest.mark.parametrize("children,at", [(1, 0), (5, 4), (40, 33), (70, 69)])
@pytest.mark.parametrize("entry", [0, 1, 37, 61, 62])
def test_a_branch_of_a_table_that_names_no_page(pkg, lib, pages, deep, children, at, entry):
    """Among the entries that the branch would share, or copy, of one source of the list."""
    pool = pages.PagePool.empty(1, 70 * 63 + 200, PAGE, 1, 64, 80, 70, BF)
    pool.extend(ints([0, 1]), ints([62 * PAGE + 5, 62 * PAGE + 3]))
    src = [0] * children
    src[at] = 1
    src, dst = ints(src), ints(list(range(2, 2 + children)))
    keep = int(pool.table[1, entry])
    for bad in (pool.ref.numel(), 2**31 - 1):
        pool.table[1, entry] = bad
        before = books(pool)
        (pool.copy if deep else pool.fork)(src, dst)
        assert "index check failed" in outcome(pkg, lib)
        assert same(books(pool), before)
    pool.table[1, entry] = keep
    (pool.copy if deep else pool.fork)(src, dst)
    assert outcome(pkg, lib) == ""
    named = pool.table[pool.table >= 0].long()
    assert torch.equal(torch.bincount(named, minlength=pool.ref.numel()).to(torch.int32), pool.ref)


@pytest.mark.parametrize("wrong", ["sequence", "length", "page given back", "page beyond the pool", "first start"])
def test_a_write_places_what_has_a_place(pkg, lib, pages, wrong):
    pool = pages.PagePool.empty(1, 12, PAGE, 2, 64, 4, 5, BF)
    pool.extend(ints([0, 1, 2]), ints([40, 20, 33]))
    for t in (pool.k, pool.v):
        t.fill_(7)
    k, v = (torch.randn((15, 2, 64), device="cuda").to(BF) for _ in range(2))
    seqs, starts, placed = [0, 1, 2], [0, 5, 10, 15], [0, 2]  # items whose rows have places
    if wrong == "sequence":
        seqs[1] = 4
    elif wrong == "length":
        pool.len[1] = 4
        placed = [0, (1, 1), 2]  # all but the first of its five rows
    elif wrong == "page given back":
        pool.table[1, 0] = -1  # rows 15 .. 19: row 15 lies in it
        placed = [0, (1, 1), 2]
    elif wrong == "page beyond the pool":
        pool.table[1, 1] = 12  # and rows 16 .. 19 in this one
        placed = [0, (1, 0, 1), 2]
    else:
        starts[0] = 2
        placed = [(0, 2), 1, 2]
    before, want = books(pool), [pool.k.clone(), pool.v.clone()]
    pool.write(0, ints(seqs), ints(starts), k, v)
    assert "index check failed" in outcome(pkg, lib)
    for x in placed:
        i, lo, hi = x if isinstance(x, tuple) and len(x) == 3 else (*x, 5) if isinstance(x, tuple) else (x, 0, 5)
        for r in range(lo, hi):
            at = int(before[1][seqs[i]]) - 5 + r
            page = int(before[0][seqs[i], at // PAGE])
            for t, new in zip(want, (k, v)):
                t[0, page, :, at % PAGE] = new[5 * i + r]
    assert torch.equal(pool.k, want[0]) and torch.equal(pool.v, want[1])
    assert same(books(pool), before)
