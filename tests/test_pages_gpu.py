"""Maintenance of the paged KV cache against a plain model: tables, counts and rows have to be equal."""

import importlib
import random

import pytest
import torch

from gpu_helpers import check
from pages_model import Model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pages(pkg, lib):
    return importlib.import_module(pkg.__name__ + ".pages")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def sync(pkg, lib):
    """attn_sync; "" or the message of a status bit."""
    lib.attn_sync()
    msg = pkg.last_error(lib)
    lib.attn_clear_error()
    return msg


class Mirror:
    """A pool, its model, and the rows that each sequence should hold."""

    def __init__(self, pages, layers, n, page, h, d, seqs, entries, dtype, seed):
        self.pool = pages.PagePool.empty(layers, n, page, h, d, seqs, entries, dtype)
        self.pool.k.fill_(float("nan"))
        self.pool.v.fill_(float("nan"))
        self.model = Model(n, page, seqs)
        self.rows = {}  # sequence -> (k, v) [layers][len][h][d]
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.shape = (layers, h, d)

    def extend(self, seqs, counts, io=None):
        self.model.extend(seqs, counts)
        self.pool.extend(ints(seqs), ints(counts))
        layers, h, d = self.shape
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        new = torch.randn((2, layers, starts[-1], h, d), generator=self.gen, device="cuda").to(io or self.pool.k.dtype)
        for layer in range(layers):
            self.pool.write(layer, ints(seqs), ints(starts), new[0, layer], new[1, layer])
        for i, s in enumerate(seqs):
            mine = new[:, :, starts[i]:starts[i + 1]].to(self.pool.k.dtype)
            self.rows[s] = torch.cat([self.rows[s], mine], 2) if s in self.rows else mine

    def fork(self, src, dst, deep=False):
        self.model.fork(src, dst, deep)
        (self.pool.copy if deep else self.pool.fork)(ints(src), ints(dst))
        for s, d in zip(src, dst):
            if s in self.rows:
                self.rows[d] = self.rows[s]

    def free(self, seqs):
        self.model.free(seqs)
        self.pool.free(ints(seqs))
        for s in seqs:
            self.rows.pop(s, None)

    def check(self):
        self.model.check(self.pool)
        page = self.model.page
        for s, want in self.rows.items():
            for e, p in enumerate(self.model.table[s]):
                if p < 0:
                    continue
                m = min(page, self.model.len[s] - e * page)
                got = torch.stack([self.pool.k[:, p, :, :m], self.pool.v[:, p, :, :m]]).transpose(2, 3)
                assert torch.equal(got, want[:, :, e * page:e * page + m]), (s, e, p)


@pytest.mark.parametrize("page,dtype,h,d,layers", [(16, torch.bfloat16, 8, 128, 2), (32, torch.float32, 3, 64, 1),
                                                  (64, torch.bfloat16, 2, 64, 3), (128, torch.float32, 8, 128, 1)])
def test_a_long_history_matches_the_model(pkg, lib, pages, page, dtype, h, d, layers):
    m = Mirror(pages, layers, 96, page, h, d, 12, 20, dtype, page)
    r = random.Random(page)
    for _ in range(60):
        free = [s for s in range(12) if m.model.len[s] == 0]
        used = [s for s in range(12) if m.model.len[s] > 0]
        room = m.model.ref.count(0)
        op = r.choice(["extend", "extend", "fork", "copy", "free", "trim", "compact"])
        if op == "extend":
            seqs = r.sample(range(12), r.randint(1, 4))
            counts = [r.choice([0, 1, 2, page - 1, page, 2 * page + 3]) for _ in seqs]
            if all(m.model.len[s] + c <= 20 * page for s, c in zip(seqs, counts)) and room >= 12:
                m.extend(seqs, counts, r.choice([torch.float32, torch.bfloat16]))
        elif op in ("fork", "copy") and free and used:
            n = r.randint(1, min(3, len(free)))
            src = [r.choice(used) for _ in range(n)]
            if sum(len(m.model.table[s]) for s in src) <= room:
                m.fork(src, free[:n], op == "copy")
        elif op == "free" and used:
            m.free(r.sample(range(12), 2))
        elif op == "trim" and used:
            window, sinks = r.choice([1, page, 3 * page + 1]), r.choice([0, 1, page, page + 1])
            m.model.trim(used, window, sinks)
            m.pool.trim(ints(used), window, sinks)
        elif op == "compact":
            live = torch.zeros(1, dtype=torch.int32, device="cuda")
            want = m.model.compact()
            m.pool.compact(live)
            assert live.item() == want
        m.check()
    assert sync(pkg, lib) == ""


def test_many_sequences_and_pages(pkg, lib, pages):
    """More list items than the planning CTA has threads, more pages than one of its turns."""
    m = Mirror(pages, 1, 5000, 16, 1, 64, 2600, 4, torch.bfloat16, 1)
    seqs = list(range(1300))
    random.Random(0).shuffle(seqs)
    m.extend(seqs, [1 + s % 40 for s in seqs])
    m.check()
    m.free(seqs[::3])
    m.fork([s for s in seqs if m.model.len[s]], list(range(1300, 1300 + sum(x > 0 for x in m.model.len[:1300]))))
    m.check()
    m.free(seqs[:700])
    m.model.compact()
    m.pool.compact()
    m.check()
    assert sync(pkg, lib) == ""


def test_rows_from_a_strided_projection(pkg, lib, pages):
    m = Mirror(pages, 1, 16, 16, 4, 64, 2, 8, torch.bfloat16, 2)
    fused = torch.randn((37, 4 * 64 * 3), device="cuda", dtype=torch.bfloat16)
    k, v = fused[:, 256:512].view(37, 4, 64), fused[:, 512:].view(37, 4, 64)
    m.pool.extend(ints([1]), ints([37]))
    m.pool.write(0, ints([1]), ints([0, 37]), k, v)
    m.model.extend([1], [37])
    m.rows[1] = torch.stack([k, v])[:, None]
    m.check()


def test_refused_requests_change_nothing(pkg, lib, pages):
    m = Mirror(pages, 1, 10, 16, 2, 64, 6, 6, torch.bfloat16, 3)
    m.extend([0, 1], [40, 16])
    m.check()
    for fn, args in ((m.pool.extend, ([0, 0], [1, 1])), (m.pool.extend, ([6], [1])), (m.pool.extend, ([-1], [1])),
                     (m.pool.extend, ([0], [-1])), (m.pool.extend, ([0], [57])), (m.pool.fork, ([0], [1])),
                     (m.pool.fork, ([0, 1], [2, 2])), (m.pool.fork, ([0, 2], [2, 3])), (m.pool.fork, ([6], [2])),
                     (m.pool.copy, ([0], [9])), (m.pool.extend, ([2, 2**31 - 1], [1, 1]))):
        fn(*[ints(a) for a in args])
        assert "index check failed" in sync(pkg, lib), (fn, args)
        m.check()
    for fn, args in ((m.pool.extend, ([2, 3], [80, 17])), (m.pool.copy, ([0, 0], [2, 3])), (m.pool.copy, ([0, 0, 0], [2, 3, 4]))):
        fn(*[ints(a) for a in args])
        if fn == m.pool.copy and len(args[0]) == 2:  # six pages of the six that are free
            m.model.fork(*args, deep=True)
            m.rows[2] = m.rows[3] = m.rows[0]
            assert sync(pkg, lib) == ""
            m.free([2, 3])
        else:
            assert "out of pages" in sync(pkg, lib), (fn, args)
        m.check()
    # freeing is harmless twice, and for a sequence that is not in use
    m.pool.free(ints([0, 0, 5]))
    m.model.free([0])
    m.rows.pop(0)
    m.check()
    assert sync(pkg, lib) == ""
    m.pool.free(ints([6]))
    assert "index check failed" in sync(pkg, lib)
    m.check()


def test_empty_lists_and_empty_sequences(pkg, lib, pages):
    m = Mirror(pages, 1, 4, 16, 1, 64, 3, 2, torch.float32, 4)
    none = ints([])
    m.pool.extend(none, none)
    m.pool.fork(none, none)
    m.pool.free(none)
    m.pool.trim(none, 1)
    m.pool.compact()
    m.extend([0], [0])
    m.fork([0], [1])
    m.check()
    assert sync(pkg, lib) == ""


def test_a_static_cache_becomes_a_sequence(pkg, lib, pages):
    from gpu_helpers import new_cache, vp
    import numpy as np
    rng = np.random.default_rng(5)
    h = new_cache(pkg, lib, 100, pkg.ATTN_KV_F32)
    try:
        k = [rng.standard_normal((75, 8, 128), dtype=np.float32) for _ in range(28)]
        v = [rng.standard_normal((75, 8, 128), dtype=np.float32) for _ in range(28)]
        one = rng.standard_normal((2, 8, 128), dtype=np.float32)
        for layer in range(28):
            lib.kv_cache_append_prefill(h, layer, vp(k[layer]), vp(v[layer]), 75)
        lib.kv_cache_advance(h, 75)
        lib.kv_cache_append(h, 3, vp(one[0]), vp(one[1]))  # from host memory: written by the next use of the layer
        pkg.cache_struct(h).seq_len = 76
        check(pkg, lib, "append")
        pool = pages.PagePool.empty(28, 9, 16, 8, 128, 3, 6, torch.float32)
        pool.extend(ints([0]), ints([17]))
        pool.import_cache(2, h)
        assert sync(pkg, lib) == ""
        assert pool.len.tolist() == [17, 0, 76]
        assert pool.table[2].tolist() == [2, 3, 4, 5, 6, -1]
        for layer in (0, 3, 27):
            got = pool.k[layer, 2:7].transpose(1, 2).reshape(80, 8, 128)[:76].cpu().numpy()
            assert np.array_equal(got[:75], k[layer])
            if layer == 3:
                assert np.array_equal(got[75], one[0])
            got = pool.v[layer, 2:7].transpose(1, 2).reshape(80, 8, 128)[:75].cpu().numpy()
            assert np.array_equal(got, v[layer])
        pool.import_cache(2, h)  # in use by now
        assert "index check failed" in sync(pkg, lib)
        pool.import_cache(1, h)
        assert "out of pages" in sync(pkg, lib)
        assert pool.len.tolist() == [17, 0, 76]
    finally:
        lib.kv_cache_free(h)


def test_library_pool(pkg, lib):
    """kv_pages_alloc: an empty pool of the library's own memory."""
    lib.attn_set_stream(None)
    h = lib.kv_pages_alloc(2, 8, 32, 4, 64, 3, 4, pkg.ATTN_KV_BF16)
    assert h, pkg.last_error(lib)
    from gpu_helpers import d2h
    import numpy as np
    s = pkg.pages_struct(h)
    assert lib.kv_pages_extend(h, ints([1]).data_ptr(), ints([40]).data_ptr(), 1) == 0
    assert sync(pkg, lib) == ""
    assert d2h(s.len, 3, np.int32).tolist() == [0, 40, 0]
    assert d2h(s.table, 12, np.int32).tolist() == [-1] * 4 + [0, 1, -1, -1] + [-1] * 4
    assert d2h(s.ref, 8, np.int32).tolist() == [1, 1] + [0] * 6
    lib.kv_pages_release(h)
    check(pkg, lib, "release")


def test_other_streams(pkg, lib, pages):
    """Two pools driven on two streams at once, and a captured call."""
    a, b = (Mirror(pages, 1, 400, 16, 2, 64, 9, 64, torch.bfloat16, i) for i in (6, 7))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for step in range(8):
        for m, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                m.extend([step], [100 + step])
                m.pool.compact()
    torch.cuda.synchronize()
    a.model.compact()
    a.check()
    b.check()
    graph = torch.cuda.CUDAGraph()
    seqs, counts = ints([8]), ints([5])
    with torch.cuda.stream(streams[0]):
        a.pool.extend(seqs, ints([1]))  # sizes this stream's workspace
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=streams[0]):
        a.pool.extend(seqs, counts)
    a.model.extend([8], [1])
    for _ in range(3):
        graph.replay()
        a.model.extend([8], [5])
    torch.cuda.synchronize()
    a.model.check(a.pool)
    lib.attn_set_stream(None)
    assert sync(pkg, lib) == ""
