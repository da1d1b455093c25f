"""The paged-cache operators as they are measured: page maintenance (fork, compact, trim + extend +
write), decode attention of a batch over a shared prefix, and sliding-window attention with sinks
(single tokens and prompt chunks).

``own`` false: plain torch forms (elementary operations, 32-bit sums, one rounding at the end);
``own`` true: the library's entry points through the package's ``pages.PagePool``.

A pool holds K and V as [layers][pages][kv_heads][page_size][head_dim]; ``table[s][i]`` is the page
of rows [i * page_size, (i + 1) * page_size) of sequence s (-1: none), ``len[s]`` its tokens,
``ref[p]`` the number of table entries that name page p (0: free).
"""

import importlib
import importlib.util
import random
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _package():
    name = "typhoon_ocr_server_b200"
    if name not in sys.modules:
        at = ROOT / "typhoon-ocr-server_b200"
        spec = importlib.util.spec_from_file_location(name, at / "__init__.py", submodule_search_locations=[str(at)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ---- cases ------------------------------------------------------------------------------------

# The decoder's own heads (16 query, 8 KV, 128 wide), and generic layouts.
OWN_HEADS = {"q_heads": 16, "kv_heads": 8, "d": 128}


def listed():
    return [
        # Four answers sampled about one small page (1,024 tokens): a decode step's latency.
        {"name": "prefix, 4 answers", "op": "prefix", "batch": 4, "prefix": 1024, "lo": 1, "hi": 40, "page": 64,
         "dtype": "bf16", "lens": 1, **OWN_HEADS},
        # 23 requests behind one long instruction, full precision, narrow heads in groups of three, ragged ends.
        {"name": "prefix, 23 in f32", "op": "prefix", "batch": 23, "prefix": 1537, "lo": 1, "hi": 300, "page": 16,
         "dtype": "f32", "lens": 2, "q_heads": 12, "kv_heads": 4, "d": 64},
        # A full server: 256 questions about one 4,096-token page, each with its own turn behind it.
        {"name": "prefix, 256 questions", "op": "prefix", "batch": 256, "prefix": 4096, "lo": 1, "hi": 512, "page": 64,
         "dtype": "bf16", "lens": 3, **OWN_HEADS},
        # One request at the end of a 32K-token document, reading its last 1,024 tokens: latency again.
        {"name": "window, 1 token", "op": "window", "batch": 1, "past_lo": 32767, "past_hi": 32767, "new_lo": 1, "new_hi": 1,
         "window": 1024, "sinks": 4, "page": 64, "dtype": "bf16", "lens": 4, **OWN_HEADS},
        # The batched decode of 512 requests with 1,024 to 8,192 tokens each, the last 2,048 in view.
        {"name": "window, 512 requests", "op": "window", "batch": 512, "past_lo": 1023, "past_hi": 8191, "new_lo": 1,
         "new_hi": 1, "window": 2048, "sinks": 16, "page": 64, "dtype": "bf16", "lens": 5, **OWN_HEADS},
        # Prompt chunks of three requests at different depths, full precision, odd everything.
        {"name": "window, chunks in f32", "op": "window", "batch": 3, "past_lo": 0, "past_hi": 901, "new_lo": 37,
         "new_hi": 733, "window": 301, "sinks": 5, "page": 32, "dtype": "f32", "lens": 6, "q_heads": 8, "kv_heads": 2, "d": 64},
        # A 4,096-token page as one prompt.
        {"name": "window, page prompt", "op": "window", "batch": 1, "past_lo": 0, "past_hi": 0, "new_lo": 4096, "new_hi": 4096,
         "window": 1024, "sinks": 4, "page": 64, "dtype": "bf16", "lens": 7, **OWN_HEADS},
        # A long document as one prompt.
        {"name": "window, long prompt", "op": "window", "batch": 1, "past_lo": 0, "past_hi": 0, "new_lo": 16384,
         "new_hi": 16384, "window": 4096, "sinks": 4, "page": 64, "dtype": "bf16", "lens": 8, **OWN_HEADS},
        # One page's cache branches into four answers.
        {"name": "fork, 1 into 4", "op": "fork", "parents": 1, "children": 4, "lo": 1000, "hi": 1000, "layers": 28,
         "page": 64, "dtype": "bf16", "lens": 9, **OWN_HEADS},
        # Eight pages branch into 16 questions each.
        {"name": "fork, 8 into 128", "op": "fork", "parents": 8, "children": 128, "lo": 1024, "hi": 4096, "layers": 28,
         "page": 64, "dtype": "bf16", "lens": 10, **OWN_HEADS},
        # Requests have ended here and there: the live half of the pool moves to its front, the rest goes back.
        {"name": "compact, 512 pages", "op": "compact", "seqs": 40, "pages": 512, "live": 250, "layers": 28, "page": 64,
         "dtype": "bf16", "lens": 11, **OWN_HEADS},
        # A decode step's bookkeeping for 256 requests: what left the window goes, one token each comes, its rows are written.
        {"name": "step, 256 requests", "op": "step", "batch": 256, "lo": 100, "hi": 4000, "window": 1024, "sinks": 4,
         "new": 1, "page": 64, "dtype": "bf16", "lens": 12, **OWN_HEADS},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    heads = rng.choice([OWN_HEADS, OWN_HEADS, {"q_heads": 12, "kv_heads": 4, "d": 64}, {"q_heads": 8, "kv_heads": 8, "d": 128},
                        {"q_heads": 32, "kv_heads": 4, "d": 128}, {"q_heads": 10, "kv_heads": 2, "d": 64}])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    c = {"page": rng.choice([16, 32, 64, 128]), "dtype": dtype, "lens": rng.randrange(1 << 20), **heads}
    half = 1 if dtype == "bf16" else 2  # full precision: half the tokens
    op = rng.choice(["prefix", "prefix", "decode", "chunk", "chunk", "fork", "compact", "step"])
    if op == "prefix":
        return {"op": "prefix", "batch": _log(rng, 2, 200 // half), "prefix": _log(rng, 64, 4000 // half), "lo": 1,
                "hi": _log(rng, 1, 400 // half), **c}
    if op == "decode":
        lo = _log(rng, 1, 4000 // half)
        return {"op": "window", "batch": _log(rng, 1, 300 // half), "past_lo": lo, "past_hi": lo + _log(rng, 1, 4000 // half),
                "new_lo": 1, "new_hi": 1, "window": _log(rng, 16, 2000), "sinks": rng.choice([0, 1, 4, 16, 70]), **c}
    if op == "chunk":
        new = _log(rng, 16, 4000 // half)
        past = _log(rng, 1, 4000 // half) - 1
        return {"op": "window", "batch": 1 if new > 1000 else rng.randint(1, 4), "past_lo": past // 2, "past_hi": past,
                "new_lo": (new + 1) // 2, "new_hi": new, "window": _log(rng, 16, 2000), "sinks": rng.choice([0, 1, 4, 16, 70]), **c}
    if op == "fork":
        n = _log(rng, 2, 100 // half)
        lo = _log(rng, 1, 2000 // half)
        return {"op": "fork", "parents": rng.randint(1, min(8, n)), "children": n, "lo": lo, "hi": 2 * lo,
                "layers": _log(rng, 1, 28), **c}
    if op == "compact":
        pages = _log(rng, 16, 400 // half)
        return {"op": "compact", "seqs": rng.randint(1, 16), "pages": pages, "live": max(16, int(pages * rng.uniform(0.2, 0.9))),
                "layers": _log(rng, 1, 28), **c}
    lo = _log(rng, 1, 2000 // half)
    return {"op": "step", "batch": _log(rng, 1, 200 // half), "lo": lo, "hi": 2 * lo, "window": _log(rng, 16, 1500),
            "sinks": rng.choice([0, 1, 4, 70]), "new": rng.choice([1, 1, 5, 70]), **c}


# ---- lengths and tables: from the case alone, so that work() knows them ---------------------------


def _lens(c, n, lo, hi):
    r = random.Random(c["lens"] * 7919 + lo)
    return [r.randint(lo, hi) for _ in range(n)]


def _ceil(a, b):
    return -(-a // b)


def _chunks(c):
    """(tokens before the chunk, tokens of the chunk) of each sequence of a window case."""
    return list(zip(_lens(c, c["batch"], c["past_lo"], c["past_hi"]), _lens({**c, "lens": c["lens"] + 1}, c["batch"], c["new_lo"],
                                                                        c["new_hi"])))


def _sequences(c):
    """Tokens of each sequence at the start, the shared tokens at their front, and the sequences and pages besides."""
    if c["op"] == "prefix":
        return [c["prefix"] + n for n in _lens(c, c["batch"], c["lo"], c["hi"])], c["prefix"], 0, 4
    if c["op"] == "window":
        return [a + b for a, b in _chunks(c)], 0, 0, 4
    if c["op"] == "fork":
        return _lens(c, c["parents"], c["lo"], c["hi"]), 0, c["children"], c["children"] + 2
    if c["op"] == "compact":
        n = c["seqs"]
        entries = [c["live"] // n + (i < c["live"] % n) for i in range(n)]
        r = random.Random(c["lens"])
        return [max(0, e * c["page"] - r.randrange(c["page"])) for e in entries], 0, 0, c["pages"] - c["live"]
    lens = _lens(c, c["batch"], c["lo"], c["hi"])
    return lens, 0, 0, c["batch"] * (_ceil(c["new"], c["page"]) + 1)


def prepare(case, seed):
    c = case
    dt, ps, h, d = DTYPES[c["dtype"]], c["page"], c["kv_heads"], c["d"]
    lens, shared, more_seqs, spare = _sequences(c)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    layers = c.get("layers", 1)
    n = len(lens) + more_seqs
    common = shared // ps
    own_pages = [max(0, _ceil(x, ps) - common) for x in lens]
    used = common + sum(own_pages)
    num_pages = used + spare
    most = max(_ceil(x + c.get("new", 0), ps) for x in lens) + 1
    order = torch.randperm(num_pages, generator=cpu).to(torch.int32)  # pages in the order of a pool long in use
    table = torch.full((n, most), -1, dtype=torch.int32)
    ref = torch.zeros(num_pages, dtype=torch.int32)
    at = common
    for s, k in enumerate(own_pages):
        table[s, :common] = order[:common]
        table[s, common:common + k] = order[at:at + k]
        at += k
    ref[order[:used].long()] = 1
    ref[order[:common].long()] = len(lens)
    length = torch.tensor(lens + [0] * more_seqs, dtype=torch.int32)
    # One buffer for the bookkeeping, so that it is put back to where it was with one copy.
    books = torch.cat([table.flatten(), length, ref]).cuda()
    s = {"case": c, "books0": books.clone(), "books": books, "scale": d ** -0.5, "shared": shared, "max_len": max(lens)}
    s["table"] = books[:n * most].view(n, most)
    s["len"] = books[n * most:n * most + n]
    s["ref"] = books[n * most + n:]
    # Keys as QK normalisation leaves them (unit root mean square), values about half as large.
    s["k"] = torch.empty((layers, num_pages, h, ps, d), dtype=dt, device="cuda").normal_(generator=gen)
    s["v"] = torch.empty((layers, num_pages, h, ps, d), dtype=dt, device="cuda").normal_(0.0, 0.5, generator=gen)
    if shared % ps:  # the shared rows of a partly filled page: every sequence has its copy, as a fork leaves them
        at = table[:len(lens), common].long().cuda()
        for x in ("k", "v"):
            s[x][:, at, :, :shared % ps] = s[x][:, at[:1], :, :shared % ps]
    if c["op"] in ("prefix", "window"):
        rows = c["batch"]
        if c["op"] == "window":
            new = [b for _, b in _chunks(c)]
            s["max_new"] = max(new)
            s["starts"] = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
            rows = sum(new)
        s["seqs"] = torch.arange(c["batch"], dtype=torch.int32).cuda()
        s["q"] = torch.empty((rows, c["q_heads"], d), dtype=dt, device="cuda").normal_(generator=gen)
        s["out"] = torch.empty_like(s["q"])
    elif c["op"] == "fork":
        s["src"] = (torch.arange(c["children"]) % c["parents"]).to(torch.int32).cuda()
        s["dst"] = (torch.arange(c["children"]) + c["parents"]).to(torch.int32).cuda()
    elif c["op"] == "step":
        s["seqs"] = torch.randperm(c["batch"], generator=cpu).to(torch.int32).cuda()
        s["counts"] = torch.full((c["batch"],), c["new"], dtype=torch.int32).cuda()
        s["starts"] = (torch.arange(c["batch"] + 1) * c["new"]).to(torch.int32).cuda()
        for x in ("k_new", "v_new"):
            s[x] = torch.empty((c["batch"] * c["new"], h, d), dtype=dt, device="cuda").normal_(generator=gen)
    return s


# ---- the passes ----------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"prefix": _plain_prefix, "window": _plain_window, "fork": _plain_fork, "compact": _plain_compact,
            "step": _plain_step}[op](state)


def _own(s, op):
    c = s["case"]
    pool = s.get("pool")
    if pool is None:  # the handle that a program keeps beside its pool
        pkg = _package()
        pool = s["pool"] = importlib.import_module(pkg.__name__ + ".pages").PagePool(s["k"], s["v"], s["table"], s["len"], s["ref"])
    if op == "prefix":
        return pool.attend_prefix(s["q"], 0, s["seqs"], s["shared"], s["max_len"], s["scale"], out=s["out"])
    if op == "window":
        return pool.attend_window(s["q"], 0, s["seqs"], s["starts"], s["max_new"], s["max_len"], c["window"], c["sinks"],
                                  s["scale"], out=s["out"])
    # The bookkeeping goes back to its snapshot, as when a step is thrown away; page contents need no such thing.
    s["books"].copy_(s["books0"])
    if op == "fork":
        pool.fork(s["src"], s["dst"])
    elif op == "compact":
        pool.compact()
    else:
        pool.trim(s["seqs"], c["window"], c["sinks"])
        pool.extend(s["seqs"], s["counts"])
        pool.write(0, s["seqs"], s["starts"], s["k_new"], s["v_new"])
    return {x: s[x] for x in ("table", "len", "ref", "k", "v")}


def _rows(s, x, seqs, at):
    """Rows at[b, j] of sequences seqs[b] as [b][j][kv_heads][d] in 32 bits; at is clamped to what the table holds."""
    ps = x.shape[3]
    at = at.clamp(min=0)
    page = s["table"][seqs.long()].gather(1, at // ps).clamp(min=0).long()
    return x[0][page, :, at % ps].float()


def _softmax(x, seen):
    x = x.masked_fill(~seen, float("-inf"))
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prefix(s):
    c, q, p = s["case"], s["q"], s["shared"]
    b, h, g, d = c["batch"], c["kv_heads"], c["q_heads"] // c["kv_heads"], c["d"]
    qf = q.float().view(b, h, g, d)
    first = torch.arange(p, device="cuda")[None]
    kp, vp = (_rows(s, s[x], s["seqs"][:1], first)[0] for x in ("k", "v"))  # [p][h][d]
    own_at = torch.arange(p, s["max_len"], device="cuda")[None].expand(b, -1)
    seen = own_at < s["len"][s["seqs"].long()][:, None]
    at = torch.where(seen, own_at, torch.full_like(own_at, p))
    ks, vs = (_rows(s, s[x], s["seqs"], at) for x in ("k", "v"))  # [b][j][h][d]
    x = torch.cat([torch.einsum("bhgd,jhd->bhgj", qf, kp), torch.einsum("bhgd,bjhd->bhgj", qf, ks)], -1) * s["scale"]
    seen = torch.cat([torch.ones((b, p), dtype=torch.bool, device="cuda"), seen], 1)[:, None, None]
    w = _softmax(x, seen)
    o = torch.einsum("bhgj,jhd->bhgd", w[..., :p], vp) + torch.einsum("bhgj,bjhd->bhgd", w[..., p:], vs)
    return o.reshape(q.shape).to(q.dtype)


def _plain_window(s):
    c, q, seqs = s["case"], s["q"], s["seqs"]
    b, h, g, d = c["batch"], c["kv_heads"], c["q_heads"] // c["kv_heads"], c["d"]
    n = s["max_new"]
    starts = s["starts"].long()
    new = starts[1:] - starts[:-1]
    total = s["len"][seqs.long()].long()
    t = torch.arange(n, device="cuda")[None].expand(b, -1)
    live = t < new[:, None]  # queries of a padded batch
    pos = (total - new)[:, None] + t
    qf = q.float()[(starts[:-1, None] + t).clamp(max=q.shape[0] - 1)].view(b, n, h, g, d)
    if n == 1:  # single tokens: the rows in view alone
        first = torch.arange(c["sinks"], device="cuda")[None].expand(b, -1)
        last = pos - c["window"] + 1 + torch.arange(c["window"], device="cuda")[None]
        at = torch.cat([first, last], 1)
        seen = torch.cat([first <= pos, (last >= c["sinks"]) & (last >= 0)], 1)
        at = torch.where(seen, at, torch.zeros_like(at))
        seen = seen[:, None]
    else:
        at = torch.arange(s["max_len"], device="cuda")[None].expand(b, -1)
        seen = (at[:, None] <= pos[..., None]) & ((at[:, None] < c["sinks"]) | (at[:, None] > pos[..., None] - c["window"]))
        at = torch.where(at < total[:, None], at, torch.zeros_like(at))
    kf, vf = (_rows(s, s[x], seqs, at) for x in ("k", "v"))
    w = _softmax(torch.einsum("bnhgd,bjhd->bhgnj", qf, kf) * s["scale"], seen[:, None, None])
    o = torch.einsum("bhgnj,bjhd->bnhgd", w, vf)
    return o[live].reshape(q.shape).to(q.dtype)


def _free_pages(ref):
    """Page numbers, the free ones first, each group in rising order."""
    return torch.argsort((ref != 0).to(torch.int32), stable=True)


def _plain_fork(s):
    s["books"].copy_(s["books0"])
    table, length, ref, src, dst = s["table"], s["len"], s["ref"], s["src"].long(), s["dst"].long()
    ps = s["case"]["page"]
    n = length[src].long()
    rows = table[src]
    end = (n // ps).clamp(max=table.shape[1] - 1)[:, None]
    cut = torch.nonzero(n % ps).squeeze(1)  # children whose last page is partly filled: it becomes their own
    old = rows.gather(1, end)[cut, 0].long()
    new = _free_pages(ref)[:cut.numel()]
    rows[cut, end[cut, 0]] = new.to(torch.int32)
    table[dst] = rows
    length[dst] = n.to(torch.int32)
    named = rows >= 0
    ref.scatter_add_(0, rows[named].long(), torch.ones_like(rows[named]))
    held = (torch.arange(ps, device="cuda") < (n % ps)[cut, None])[None, :, None, :, None]
    for x in (s["k"], s["v"]):
        x[:, new] = torch.where(held, x[:, old], x[:, new])
    return {x: s[x] for x in ("table", "len", "ref", "k", "v")}


def _plain_compact(s):
    s["books"].copy_(s["books0"])
    table, ref = s["table"], s["ref"]
    live = int((ref > 0).sum())
    pages = torch.arange(ref.numel(), device="cuda")
    moved = torch.nonzero((ref > 0) & (pages >= live)).squeeze(1)
    holes = torch.nonzero((ref == 0) & (pages < live)).squeeze(1)
    to = pages.clone()
    to[moved] = holes
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table))
    ref[holes] = ref[moved]
    ref[moved] = 0
    for x in (s["k"], s["v"]):
        x[:, holes] = x[:, moved]
    return {x: s[x] for x in ("table", "len", "ref", "k", "v")}


def _plain_step(s):
    s["books"].copy_(s["books0"])
    c = s["case"]
    ps, table, length, ref, seqs = c["page"], s["table"], s["len"], s["ref"], s["seqs"].long()
    entry = torch.arange(table.shape[1], device="cuda")[None]
    # trim: pages wholly behind the window and past the sinks
    n = length[seqs].long()[:, None]
    rows = table[seqs]
    gone = (rows >= 0) & (entry * ps >= c["sinks"]) & ((entry + 1) * ps <= n - c["window"])
    ref.scatter_add_(0, rows[gone].long(), -torch.ones_like(rows[gone]))
    rows = torch.where(gone, -torch.ones_like(rows), rows)
    # extend: new pages, the lowest free ones, in the order of the list
    add = s["counts"].long()[:, None]
    wanted = (entry >= (n + ps - 1) // ps) & (entry < (n + add + ps - 1) // ps)
    fresh = _free_pages(ref)[:int(wanted.sum())]
    rows[wanted] = fresh.to(torch.int32)
    ref[fresh] = 1
    table[seqs] = rows
    length[seqs] += s["counts"]
    # write: each sequence's last rows
    t = torch.arange(s["k_new"].shape[0], device="cuda")
    b = torch.bucketize(t, s["starts"].long(), right=True) - 1
    at = n[b, 0] + t - s["starts"].long()[b]
    page = rows[b, at // ps].long()
    s["k"][0][page, :, at % ps] = s["k_new"]
    s["v"][0][page, :, at % ps] = s["v_new"]
    return {x: s[x] for x in ("table", "len", "ref", "k", "v")}


# ---- what a pass cannot do without ---------------------------------------------------------------


def _seen_pairs(past, new, window, sinks):
    """Visible (query, key) pairs of a chunk, and the distinct keys among them."""
    pairs = 0
    for p in range(past, past + new):
        first = max(0, p - window + 1)
        pairs += p + 1 - first + min(sinks, first)
    first = max(0, past - window + 1)
    return pairs, past + new - first + min(sinks, first)


def work(case):
    c = case
    e = 2 if c["dtype"] == "bf16" else 4
    row = 2 * c["kv_heads"] * c["d"] * e  # one token's K and V rows of a layer
    qo = 2 * c["q_heads"] * c["d"] * e  # one token's query and output
    lens, shared, _, _ = _sequences(c)
    if c["op"] == "prefix":
        return {"bytes": row * (shared + sum(x - shared for x in lens)) + qo * c["batch"],
                "flops": 4 * c["d"] * c["q_heads"] * sum(lens)}
    if c["op"] == "window":
        seen = [_seen_pairs(a, b, c["window"], c["sinks"]) for a, b in _chunks(c)]
        return {"bytes": row * sum(k for _, k in seen) + qo * sum(b for _, b in _chunks(c)),
                "flops": 4 * c["d"] * c["q_heads"] * sum(p for p, _ in seen)}
    ps = c["page"]
    if c["op"] == "fork":
        src = [i % c["parents"] for i in range(c["children"])]
        read = sum(lens[i] % ps for i in set(src))
        return {"bytes": c["layers"] * row * (read + sum(lens[i] % ps for i in src)) + 8 * sum(_ceil(lens[i], ps) for i in src),
                "flops": 0}
    if c["op"] == "compact":
        live, pages = sum(_ceil(x, ps) for x in lens), c["pages"]
        moved = live * (pages - live) / pages  # of pages spread evenly
        return {"bytes": 2 * c["layers"] * row * ps * moved + 8 * live + 8 * pages, "flops": 0}
    return {"bytes": 2 * row * c["batch"] * c["new"] + 8 * sum(_ceil(x, ps) for x in lens), "flops": 0}


# ---- the definition in 64 bits ---------------------------------------------------------------------


def exact(case, seed):
    """Each query by itself against the keys that it sees; None for page maintenance, which computes no numbers."""
    if case["op"] not in ("prefix", "window"):
        return None
    s = prepare(case, seed)
    c, ps, h = case, case["page"], case["kv_heads"]
    g = c["q_heads"] // h
    if c["op"] == "prefix":
        starts, window = list(range(c["batch"] + 1)), 0
    else:
        starts, window = s["starts"].tolist(), c["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        total = int(s["len"][b])
        pages = s["table"][b, :_ceil(total, ps)].long()
        k, v = (s[x][0][pages].permute(1, 0, 2, 3).reshape(h, -1, c["d"])[:, :total].double() for x in ("k", "v"))
        new = starts[b + 1] - starts[b]
        for lo in range(0, new, 512):
            hi = min(new, lo + 512)
            q = s["q"][starts[b] + lo:starts[b] + hi].double().view(hi - lo, h, g, c["d"])
            pos = torch.arange(total - new + lo, total - new + hi, device="cuda")[:, None]
            key = torch.arange(total, device="cuda")[None]
            see = key <= pos
            if window:
                see &= (pos - key < window) | (key < c["sinks"])
            first = int(torch.nonzero(see.any(0))[0])
            a = torch.einsum("thgd,hjd->hgtj", q, k[:, first:]) * s["scale"]
            a = torch.where(see[:, first:], a, torch.full_like(a, -torch.inf)).softmax(-1)
            out[starts[b] + lo:starts[b] + hi] = torch.einsum("hgtj,hjd->thgd", a, v[:, first:]).reshape(hi - lo, h * g, c["d"])
    return out
