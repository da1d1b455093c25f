"""Batches behind a shared prefix in which a sequence does not have all of it."""

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


def outcome(pkg, lib):
    rc = lib.attn_sync()
    msg = pkg.last_error(lib) if rc else ""
    lib.attn_clear_error()
    return msg


def branches(pages, dtype, seqs, prefix):
    """`seqs` branches of one sequence, some rows further each; one more that is not in use."""
    pool = pages.PagePool.empty(1, prefix // 32 + 4 * seqs + 5, 32, 2, 64, seqs + 2, prefix // 32 + 5, dtype)
    g = torch.Generator(device="cuda").manual_seed(seqs)
    pool.k.normal_(generator=g)
    pool.v.normal_(generator=g)
    all_of = ints(list(range(1, seqs + 1)))
    pool.extend(ints([0]), ints([prefix]))
    pool.fork(ints([0] * seqs), all_of)
    pool.extend(all_of, ints([1 + i % 50 for i in range(seqs)]))
    q = torch.randn((seqs, 4, 64), generator=g, device="cuda").to(dtype)
    return pool, all_of, q


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("seqs,prefix", [(3, 1000), (60, 2000), (1030, 70)])  # streamed, on the tensor cores, in two launches
def test_a_sequence_without_all_of_the_prefix_is_reported(pkg, lib, pages, dtype, seqs, prefix):
    pool, all_of, q = branches(pages, dtype, seqs, prefix)
    call = lambda: pool.attend_prefix(q, 0, all_of, prefix, prefix + 50, 0.125)  # noqa: E731
    want = call()
    assert outcome(pkg, lib) == ""
    shared = prefix // 32 * 32
    for at in {0, 1, seqs - 1}:
        keep = int(pool.len[1 + at])
        for short in (1, shared - 1):
            pool.len[1 + at] = short
            call()
            assert "index check failed" in outcome(pkg, lib), (at, short)
        pool.len[1 + at] = shared  # the shared pages and nothing besides
        out = call()
        assert outcome(pkg, lib) == ""
        assert bool(torch.isfinite(out.float()).all())
        pool.len[1 + at] = keep
    assert torch.equal(call(), want)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("seqs,prefix", [(3, 1000), (60, 2000)])
def test_a_sequence_not_in_use(pkg, lib, pages, dtype, seqs, prefix):
    """It fills up a batch, the others answering as ever; but the shared rows are found by the first."""
    pool, all_of, q = branches(pages, dtype, seqs, prefix)
    filled = all_of.clone()
    filled[1::2] = seqs + 1
    call = lambda s: pool.attend_prefix(q, 0, s, prefix, prefix + 50, 0.125)  # noqa: E731
    want = call(all_of)
    out = call(filled)
    assert outcome(pkg, lib) == ""
    # other runs of the same sums: FP32 sums, the output's rounding; values are below 4 here
    assert float((out[::2].float() - want[::2].float()).abs().max()) <= (2.0**-6 if dtype == BF else 2.0**-16)
    filled[0] = seqs + 1
    call(filled)
    assert "index check failed" in outcome(pkg, lib)
