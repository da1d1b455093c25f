"""A plain model of the paged cache for the tests: tables as lists, rows as 64-bit arrays, and
attention in 64 bits from its definition."""

import numpy as np
import torch


class Model:
    """Sequences as lists of pages; new pages are the lowest free ones in the order of the call."""

    def __init__(self, pages, page, seqs):
        self.page = page
        self.ref = [0] * pages
        self.table = [[] for _ in range(seqs)]
        self.len = [0] * seqs

    def take(self):
        p = self.ref.index(0)
        self.ref[p] = 1
        return p

    def extend(self, seqs, counts):
        for s, c in zip(seqs, counts):
            self.len[s] += c
            while len(self.table[s]) < -(-self.len[s] // self.page):
                self.table[s].append(self.take())

    def fork(self, src, dst, deep=False):
        copies = []
        for s, d in zip(src, dst):
            self.table[d] = list(self.table[s])
            self.len[d] = self.len[s]
        for d in dst:
            for e, p in enumerate(self.table[d]):
                rows = min(self.page, self.len[d] - e * self.page)
                if p < 0:
                    continue
                if deep or rows < self.page:
                    self.table[d][e] = self.take()
                    copies.append((p, self.table[d][e], rows))
                else:
                    self.ref[p] += 1
        return copies

    def drop(self, s, e):
        p = self.table[s][e]
        if p >= 0:
            self.ref[p] -= 1
        self.table[s][e] = -1

    def free(self, seqs):
        for s in seqs:
            for e in range(len(self.table[s])):
                self.drop(s, e)
            self.table[s], self.len[s] = [], 0

    def trim(self, seqs, window, sinks):
        for s in seqs:
            for e in range(len(self.table[s])):
                if e * self.page >= sinks and (e + 1) * self.page <= self.len[s] - window:
                    self.drop(s, e)

    def compact(self):
        live = sum(r > 0 for r in self.ref)
        moved = [p for p in range(live, len(self.ref)) if self.ref[p] > 0]
        holes = [p for p in range(live) if self.ref[p] == 0]
        to = dict(zip(moved, holes))
        for t in self.table:
            t[:] = [to.get(p, p) for p in t]
        for a, b in to.items():
            self.ref[b], self.ref[a] = self.ref[a], 0
        return live

    def check(self, pool):
        entries = pool.table.shape[1]
        want = [t + [-1] * (entries - len(t)) for t in self.table]
        assert pool.table.tolist() == want
        assert pool.len.tolist() == self.len
        assert pool.ref.tolist() == self.ref


def attention(q, k, v, see, scale):
    """q [n][H][d], k and v [m][h][d], see [n][m] (what each query sees), float64: the output, and for the
    tolerances the weighted mean of |v| and the largest scale * sum |q_i k_i| of a visible key."""
    n, hq, d = q.shape
    g = hq // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    see = see[:, None, :]
    s = torch.einsum("nhd,mhd->nhm", q, k) * scale
    s = torch.where(see, s, torch.full_like(s, -torch.inf))
    top = s.amax(-1, keepdim=True)
    w = torch.where(see, torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top)), torch.zeros_like(s))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, torch.ones_like(total), total)
    size = torch.where(see, torch.einsum("nhd,mhd->nhm", q.abs(), k.abs()) * scale, torch.zeros_like(s)).amax(-1, keepdim=True)
    return torch.einsum("nhm,mhd->nhd", w, v), torch.einsum("nhm,mhd->nhd", w, v.abs()), size


def tolerance(out, mean_abs, size, pool_bf16, io_bf16):
    """Elementwise bound of |kernel - out|.

    FP32 sums of n products err by at most a few 2^-24 of the sum of magnitudes per step; with the
    operands' split (2^-21 per product) and the base-2 exponential (2^-22), 2^-19 of `size` per score
    covers it, which enters numerator and denominator of the softmax; 2^-18 covers the value products
    and the joins.  BF16 pools: products of BF16 operands are exact in FP32, and each weight is rounded
    to BF16 at most once (8 significant bits: half an ulp is up to 2^-8 of the value).  A BF16 output adds
    its own rounding, 2^-8 of the value.
    """
    tol = mean_abs * (2 * size * 2.0**-19 + 2.0**-18)
    if pool_bf16:
        tol = tol + mean_abs * 2.0**-8
    if io_bf16:
        tol = tol + out.abs() * 2.0**-8 + 1e-30
    return tol * 1.01 + 1e-30


def rows_of(pool, layer, seq, cpu=True):
    """K and V rows of a sequence, [len][h][d] float64; rows of pages given back as zeros, and which rows are there."""
    table, n = pool.table[seq].tolist(), int(pool.len[seq])
    page, h, d = pool.k.shape[3], pool.k.shape[2], pool.k.shape[4]
    k, v = torch.zeros((n, h, d), dtype=torch.float64), torch.zeros((n, h, d), dtype=torch.float64)
    there = np.zeros(n, dtype=bool)
    for e in range(-(-n // page)):
        p = table[e]
        if p < 0:
            continue
        m = min(page, n - e * page)
        k[e * page:e * page + m] = pool.k[layer, p, :, :m].transpose(0, 1).double().cpu()
        v[e * page:e * page + m] = pool.v[layer, p, :, :m].transpose(0, 1).double().cpu()
        there[e * page:e * page + m] = True
    return k, v, torch.from_numpy(there)
