"""The host side of the paged cache (csrc/pages.c) over a CUDA runtime that only keeps books
(pages_host_fake.c): what becomes of a pool's workspace, and what reaches a launch."""

import ctypes
import shutil
import subprocess
import threading
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
VP = ctypes.c_void_p


def cuda_headers():
    for at in ("/usr/local/cuda/include",):
        if (Path(at) / "cuda_runtime_api.h").exists():
            return at
    pytest.skip("no CUDA headers")


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    cc = shutil.which("gcc", path="/usr/bin") or shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    out = tmp_path_factory.mktemp("host") / "pages_host.so"
    subprocess.run([cc, "-shared", "-fPIC", "-std=gnu11", "-w", "-g", "-I", str(ROOT / "include"), "-I", str(ROOT / "typhoon-ocr-server_b200" / "csrc"),
                    "-I", cuda_headers(), str(ROOT / "typhoon-ocr-server_b200" / "csrc" / "pages.c"), str(ROOT / "tests" / "pages_host_fake.c"),
                    "-o", str(out), "-Wl,-Bsymbolic", "-lpthread"], check=True)
    return ctypes.CDLL(str(out))


class Host:
    def __init__(self, lib):
        self.lib = lib
        self.buf = (ctypes.c_char * 4096)()
        self.at = (ctypes.addressof(self.buf) + 63) & ~63
        lib.kv_pages_attach.restype = VP
        lib.fake_error.restype = ctypes.c_char_p

    def get(self, name, kind=ctypes.c_int):
        return kind.in_dll(self.lib, name).value

    def set(self, name, value):
        ctypes.c_int.in_dll(self.lib, name).value = value

    def pool(self, pages=8, entries=4):
        a = VP(self.at)
        h = self.lib.kv_pages_attach(a, a, a, a, a, 1, pages, 16, 2, 64, 3, entries, 1)
        assert h, self.lib.fake_error()
        return VP(h)

    def attend(self, h, batch, window=0, sinks=0):
        a = VP(self.at)
        return self.lib.attention_pages_window_gqa(a, ctypes.c_longlong(128), h, 0, a, None, batch, batch, 2, 1, 64, window, sinks, a, 1,
                                                   ctypes.c_float(1.0))

    def ws(self):
        return self.get("fake_ws", VP)

    def tickets(self):
        return self.get("fake_tickets", VP)

    def live(self, p):
        return bool(self.lib.fake_is_live(VP(p)))


@pytest.fixture
def host(built):
    h = Host(built)
    h.set("fake_capturing", 0)
    h.lib.fake_stream(VP(0))
    return h


def test_what_a_captured_call_was_given_stays(host):
    """A graph keeps the addresses of its calls: no later call, larger or on another stream, frees them."""
    pool = host.pool()
    assert host.attend(pool, 4) == 0
    host.set("fake_capturing", 1)
    assert host.attend(pool, 4) == 0
    ws, tickets = host.ws(), host.tickets()
    host.set("fake_capturing", 0)
    assert host.attend(pool, 256) == 0
    assert host.ws() != ws
    assert host.live(ws) and host.live(tickets)
    for s in range(1, 70):  # more streams than anything is kept for
        host.lib.fake_stream(VP(64 * s))
        assert host.attend(pool, 4) == 0
        assert host.live(ws) and host.live(tickets)
    assert host.lib.kv_pages_compact(pool, None) == 0
    host.lib.kv_pages_release(pool)
    assert host.live(ws) and host.live(tickets)


def test_a_pools_workspace_is_its_own(host):
    """Two pools driven on two streams, through graphs captured on one: no scratch, no tickets in common."""
    a, b = host.pool(), host.pool()
    given = []
    for p in (a, b):
        assert host.attend(p, 4) == 0
        given += [host.ws(), host.tickets()]
    assert len(set(given)) == 4
    host.lib.kv_pages_release(a)
    host.lib.kv_pages_release(b)


def test_what_pools_give_back_serves_the_next(host):
    """Outgrown and released buffers: some are kept for pools to come, after all work has ended, and no more than that."""
    pool = host.pool()
    assert host.attend(pool, 4) == 0
    mallocs, syncs = host.get("fake_mallocs"), host.get("fake_syncs")
    host.lib.kv_pages_release(pool)
    assert host.get("fake_syncs") > syncs
    for _ in range(100):
        pool, memsets = host.pool(), host.get("fake_memsets")
        assert host.attend(pool, 4) == 0
        assert host.get("fake_mallocs") == mallocs
        assert host.get("fake_memsets") == memsets + 1  # the tickets
        host.lib.kv_pages_release(pool)
    pools = [host.pool() for _ in range(100)]  # all at once
    for i, p in enumerate(pools):
        assert host.attend(p, 1 + 5 * i) == 0
    assert len({p.value for p in pools}) == 100 and host.lib.fake_live() >= 200
    for p in pools:
        host.lib.kv_pages_release(p)
    left = host.lib.fake_live()
    assert left < 40  # (what earlier tests captured is kept too)
    for n in (1, 30, 300, 3000, 2, 9000):  # one that grows: its former buffers do not pile up
        pool = host.pool()
        assert host.attend(pool, n) == 0 and host.attend(pool, 2 * n) == 0
        host.lib.kv_pages_release(pool)
    assert host.lib.fake_live() <= left


def test_a_spare_buffer_is_not_in_use_twice(host):
    pools = [host.pool() for _ in range(6)]
    for _ in range(3):
        given = []
        for p in pools:
            assert host.attend(p, 4) == 0
            given += [host.ws(), host.tickets()]
        assert len(set(given)) == 12
        host.lib.kv_pages_release(pools.pop())
        pools.append(host.pool())
    for p in pools:
        host.lib.kv_pages_release(p)


def test_a_capture_is_refused_what_it_would_have_to_allocate(host):
    pool = host.pool()
    assert host.attend(pool, 4) == 0
    host.set("fake_capturing", 1)
    mallocs, syncs, memsets, launches = (host.get("fake_" + x) for x in ("mallocs", "syncs", "memsets", "launches"))
    assert host.attend(pool, 400) != 0
    assert b"captured" in host.lib.fake_error()
    assert [host.get("fake_" + x) for x in ("mallocs", "syncs", "memsets", "launches")] == [mallocs, syncs, memsets, launches]
    assert host.attend(pool, 4) == 0  # what fits goes on
    host.set("fake_capturing", 0)
    assert host.attend(pool, 400) == 0
    host.lib.kv_pages_release(pool)


def test_threads_that_share_a_pool_queue_whole_calls(host):
    """A call may be several launches with one workspace: another thread's call on the pool comes before or after."""
    pool = host.pool()
    for x in ("overlaps", "lost"):
        host.set("fake_" + x, 0)
    host.set("fake_launch_us", 300)
    a, n = VP(host.at), [0]
    calls = [lambda i: host.lib.kv_pages_fork(pool, a, a, 1 + 100000 * i), lambda i: host.lib.kv_pages_compact(pool, None),
             lambda i: host.attend(pool, 1 + 10 * i), lambda i: host.lib.kv_pages_free(pool, a, 1)]

    def go(call):
        for i in range(40):
            n[0] += call(i) != 0

    threads = [threading.Thread(target=go, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    host.set("fake_launch_us", 0)
    assert (n[0], host.get("fake_overlaps"), host.get("fake_lost")) == (0, 0, 0)
    host.lib.kv_pages_release(pool)


def test_tickets_after_a_wait_that_ran_out(host):
    """Those of the pool whose kernel gave up are cleared, its mark too; another pool's, perhaps in use, are left."""
    a, b = host.pool(), host.pool()
    words = []
    for p in (a, b):
        assert host.attend(p, 4) == 0
        words.append(ctypes.cast(host.tickets(), ctypes.POINTER(ctypes.c_uint32)))
    for w in words:
        w[16], w[40] = 3, 1
    words[0][0] = 1
    host.lib.tyb_pages_after_timeout()
    assert [words[0][i] for i in (0, 16, 40)] == [0, 0, 0]
    assert [words[1][i] for i in (0, 16, 40)] == [0, 3, 1]
    words[1][0] = 1
    host.lib.kv_pages_release(a)
    host.lib.tyb_pages_after_timeout()
    assert [words[1][i] for i in (0, 16, 40)] == [0, 0, 0]
    host.lib.kv_pages_release(b)


@pytest.mark.parametrize("sinks", [2**31 - 1, 2**31 - 16, 65, 64])
def test_sinks_beyond_a_table_reach_no_kernel(host, sinks):
    """A kernel rounds the sinks up to pages in 32 bits: past 2^31 - page_size that would be a row far before the table."""
    pool = host.pool(entries=4)
    a = VP(host.at)
    assert host.lib.kv_pages_trim(pool, a, 1, 1, sinks) == 0
    assert host.get("fake_sinks") == 4 * 16
    assert host.lib.kv_pages_trim(pool, a, 1, 2**31 - 1, 5) == 0
    assert (host.get("fake_window"), host.get("fake_sinks")) == (2**31 - 1, 5)
    host.lib.kv_pages_release(pool)


def test_memory_of_another_device_is_refused(host):
    """Every pointer of every call, before anything is launched."""
    lib, a = host.lib, VP(host.at)
    foreign = VP((ctypes.addressof((ctypes.c_char * 64).in_dll(lib, "fake_foreign")) + 15) & ~15)
    pool, launches = host.pool(), host.get("fake_launches")
    one, scale = ctypes.c_longlong(128), ctypes.c_float(1.0)

    def each(call, *names):
        """call(*pointers) with each pointer in turn on the other device."""
        for i, name in enumerate(names):
            args = [a] * len(names)
            args[i] = foreign
            assert call(*args), name
            assert f"{name} is on device 1".encode() in lib.fake_error()
        assert host.get("fake_launches") == launches
        assert not call(*[a] * len(names))
        host.set("fake_launches", launches)

    each(lambda s, c: lib.kv_pages_extend(pool, s, c, 1), "seqs", "counts")
    each(lambda s, d: lib.kv_pages_fork(pool, s, d, 1), "src", "dst")
    each(lambda s, d: lib.kv_pages_copy(pool, s, d, 1), "src", "dst")
    each(lambda s: lib.kv_pages_free(pool, s, 1), "seqs")
    each(lambda s: lib.kv_pages_trim(pool, s, 1, 1, 0), "seqs")
    each(lambda s: lib.kv_pages_compact(pool, s), "live_out")
    each(lambda s, t, k, v: lib.kv_pages_write(pool, 0, s, t, 1, 1, k, v, 1, one), "seqs", "starts", "k_new", "v_new")
    each(lambda q, s, o: lib.attention_pages_prefix_gqa(q, one, pool, 0, s, 2, 2, 0, 64, o, 1, scale), "q", "seqs", "output")
    each(lambda q, s, t, o: lib.attention_pages_window_gqa(q, one, pool, 0, s, t, 1, 2, 2, 2, 64, 0, 0, o, 1, scale), "q", "seqs", "starts",
         "output")
    for i, name in enumerate(("k", "v", "table", "len", "ref")):
        args = [a] * 5
        args[i] = foreign
        assert not lib.kv_pages_attach(*args, 1, 8, 16, 2, 64, 3, 4, 1)
        assert f"{name} is on device 1".encode() in lib.fake_error()
    lib.kv_pages_release(pool)
