"""The paged KV cache over torch tensors (include/kv_pages.h has the rules).

A ``PagePool`` names tensors that the caller holds; every call queues work on torch's current
stream (which becomes the calling thread's library stream, and stays it: static calls that belong on
another set that again) and returns.  ``attn_sync`` reports what only the device can see, a pool
without enough free pages among it.
"""

from __future__ import annotations

import torch

_lib = None


def _package():
    return __import__(__name__.rsplit(".", 1)[0])


def _library():
    global _lib
    if _lib is None:
        _lib = _package().load_attention_lib()
    return _lib


def _ints(x, what):
    if x.dtype is not torch.int32 or not x.is_contiguous():
        raise ValueError(f"{what}: a contiguous int32 tensor is wanted")
    return x


_raw_stream = torch._C._cuda_getCurrentRawStream  # what torch.cuda.current_stream().cuda_stream is, without the objects

_dropped = []  # (library, handle, device) of pools that nobody closed


class PagePool:
    """k, v [layers][pages][kv_heads][page_size][head_dim] (bfloat16 or float32); table [seqs][entries],
    length [seqs] and ref [pages] int32; all contiguous CUDA tensors of one device."""

    def __init__(self, k, v, table, length, ref, lib=None):
        pkg = _package()
        self._handle = None
        self.lib = lib or _library()
        self.k, self.v, self.table, self.len, self.ref = k, v, _ints(table, "table"), _ints(length, "length"), _ints(ref, "ref")
        if k.dtype not in (torch.bfloat16, torch.float32) or v.dtype != k.dtype or v.shape != k.shape or k.dim() != 5:
            raise ValueError("k and v: [layers][pages][kv_heads][page_size][head_dim] of one type, bfloat16 or float32")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("k and v have to be contiguous")
        if table.dim() != 2 or length.shape != table.shape[:1] or ref.shape != k.shape[1:2]:
            raise ValueError("table [seqs][entries], length [seqs], ref [pages] are wanted")
        self.device, self._index = k.device, k.device.index
        self._codes = {torch.float32: pkg.ATTN_DT_F32, torch.bfloat16: pkg.ATTN_DT_BF16}
        layers, pages, self.kv_heads, page, self.head_dim = k.shape
        dtype = pkg.ATTN_KV_BF16 if k.dtype == torch.bfloat16 else pkg.ATTN_KV_F32
        while _dropped and not torch.cuda.is_current_stream_capturing():
            old, handle, device = _dropped.pop()
            with torch.cuda.device(device):
                old.kv_pages_release(handle)
        with torch.cuda.device(self.device):
            self._handle = self.lib.kv_pages_attach(k.data_ptr(), v.data_ptr(), table.data_ptr(), length.data_ptr(),
                                                    ref.data_ptr(), layers, pages, page, self.kv_heads, self.head_dim,
                                                    table.shape[0], table.shape[1], dtype)
        if not self._handle:
            raise RuntimeError(pkg.last_error(self.lib))

    @classmethod
    def empty(cls, layers, pages, page_size, kv_heads, head_dim, seqs, entries, dtype=torch.bfloat16, device="cuda", lib=None):
        """A pool of tensors of its own, with nothing in it."""
        shape = (layers, pages, kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                   torch.full((seqs, entries), -1, dtype=torch.int32, device=device),
                   torch.zeros(seqs, dtype=torch.int32, device=device), torch.zeros(pages, dtype=torch.int32, device=device), lib)

    def close(self):
        """Gives the handle back (after waiting for the stream); the tensors stay the caller's."""
        if self._handle:
            handle, self._handle = self._handle, None
            with torch.cuda.device(self.device):
                self.lib.attn_set_stream(_raw_stream(self._index))
                self.lib.kv_pages_release(handle)

    def __del__(self, dropped=_dropped):
        # The collector may run anywhere, in a capture too, so this calls no CUDA: the next pool made gives the handle back.
        if getattr(self, "_handle", None):
            dropped.append((self.lib, self._handle, self.device))

    def _call(self, fn, *args):
        if not self._handle:
            raise RuntimeError("the pool is closed")
        self.lib.attn_set_stream(_raw_stream(self._index))
        if fn(*args):
            msg = _package().last_error(self.lib)
            self.lib.attn_clear_error()
            raise RuntimeError(msg)

    def _dtype(self, x):
        code = self._codes.get(x.dtype)
        if code is None:
            raise ValueError(f"bfloat16 or float32 is wanted, not {x.dtype}")
        return code

    def _tokens(self, x, heads, what):
        """Row stride, in elements, of [rows][heads][head_dim] (any row stride, as in a slice of a fused projection)."""
        shape, d = x.shape, self.head_dim
        if len(shape) != 3 or shape[1] != heads or shape[2] != d:
            raise ValueError(f"{what}: [rows][{heads}][{d}] is wanted, not {tuple(shape)}")
        stride = x.stride()
        if stride[2] != 1 or (stride[1] != d and heads > 1):
            raise ValueError(f"{what}: the heads of a row have to lie one after another")
        return stride[0] if shape[0] > 1 else heads * d

    # ---- maintenance ----------------------------------------------------------------------------

    def _list(self, x, what, n=None):
        if x.dtype is not torch.int32 or x.dim() != 1 or not x.is_contiguous() or (n is not None and x.shape[0] != n):
            raise ValueError(f"{what}: a contiguous int32 list{'' if n is None else f' of {n}'} is wanted")
        return x.data_ptr()

    def extend(self, seqs, counts):
        """Sequence seqs[i] grows by counts[i] tokens, whose rows are written next."""
        self._call(self.lib.kv_pages_extend, self._handle, self._list(seqs, "seqs"), self._list(counts, "counts", seqs.numel()),
                   seqs.numel())

    def write(self, layer, seqs, starts, k_new, v_new):
        """The last starts[i + 1] - starts[i] rows of sequence seqs[i], from [rows][kv_heads][head_dim]; a row without a
        place is reported by ``attn_sync`` and the others are written."""
        stride = self._tokens(k_new, self.kv_heads, "k_new")
        if v_new.shape != k_new.shape or v_new.dtype != k_new.dtype or self._tokens(v_new, self.kv_heads, "v_new") != stride:
            raise ValueError("v_new has to be like k_new")
        self._call(self.lib.kv_pages_write, self._handle, layer, self._list(seqs, "seqs"),
                   self._list(starts, "starts", seqs.numel() + 1), seqs.numel(), k_new.shape[0], k_new.data_ptr(),
                   v_new.data_ptr(), self._dtype(k_new), stride)

    def import_cache(self, seq, cache):
        """The rows of a static cache (a KVCache handle of the library) become sequence `seq`."""
        self._call(self.lib.kv_pages_import, self._handle, seq, cache)

    def fork(self, src, dst):
        """Sequence dst[i] becomes a branch of src[i], sharing its full pages."""
        self._call(self.lib.kv_pages_fork, self._handle, self._list(src, "src"), self._list(dst, "dst", src.numel()), src.numel())

    def copy(self, src, dst):
        """Sequence dst[i] becomes a copy of src[i] in pages of its own."""
        self._call(self.lib.kv_pages_copy, self._handle, self._list(src, "src"), self._list(dst, "dst", src.numel()), src.numel())

    def free(self, seqs):
        """The sequences are no longer in use."""
        self._call(self.lib.kv_pages_free, self._handle, self._list(seqs, "seqs"), seqs.numel())

    def trim(self, seqs, window, sinks=0):
        """Gives back the pages that a window with sinks no longer reaches."""
        self._call(self.lib.kv_pages_trim, self._handle, self._list(seqs, "seqs"), seqs.numel(), window, sinks)

    def compact(self, live=None):
        """Moves the pages in use to the front; live: an int32 tensor of one element that receives their number."""
        self._call(self.lib.kv_pages_compact, self._handle, None if live is None else self._list(live, "live", 1))

    # ---- attention ------------------------------------------------------------------------------

    def _output(self, q, out):
        if out is None:
            return torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if out.shape != q.shape or out.dtype is not q.dtype or not out.is_contiguous():
            raise ValueError("out: contiguous, of q's shape and type, is wanted")
        return out

    def attend_prefix(self, q, layer, seqs, prefix_len, max_len, scale, out=None):
        """One token for each sequence, q [batch][q_heads][head_dim], their first prefix_len tokens shared."""
        rows, heads = q.shape[0], q.shape[1]
        stride = self._tokens(q, heads, "q")
        out = self._output(q, out)
        self._call(self.lib.attention_pages_prefix_gqa, q.data_ptr(), stride, self._handle, layer,
                   self._list(seqs, "seqs", rows), rows, heads, prefix_len, max_len, out.data_ptr(), self._dtype(q), scale)
        return out

    def attend_window(self, q, layer, seqs, starts, max_new, max_len, window, sinks, scale, out=None):
        """Causal attention of each sequence's last tokens, q [rows][q_heads][head_dim], through a window (0: none) with
        sinks; starts None: one token for each sequence."""
        rows, heads = q.shape[0], q.shape[1]
        stride = self._tokens(q, heads, "q")
        out = self._output(q, out)
        batch = seqs.shape[0]
        self._call(self.lib.attention_pages_window_gqa, q.data_ptr(), stride, self._handle, layer, self._list(seqs, "seqs"),
                   None if starts is None else self._list(starts, "starts", batch + 1), batch, rows, heads, max_new, max_len,
                   window, sinks, out.data_ptr(), self._dtype(q), scale)
        return out
