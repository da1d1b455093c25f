"""One page, many answers: a prompt is prefilled once into a static cache, becomes a sequence of a page
pool, branches into several answers that share its pages, and the answers are decoded together; long
answers go on through a sliding window, and what ends is given back.

    python examples/one_page_many_answers.py [--answers 16] [--steps 32]

Weights are not needed: queries, keys and values are synthetic, of the decoder's shapes (16 query heads,
8 KV heads, 128 wide, 28 layers).  Everything runs on the library's kernels:

    attention_prefill_fused_gqa        the prompt, layer by layer, into the static cache
    kv_pages_import                    the static cache's rows become a sequence
    kv_pages_fork                      a branch for every answer
    kv_pages_extend / kv_pages_write   a step's new rows
    attention_pages_prefix_gqa         a step's attention, the prompt read once for all answers
    attention_pages_window_gqa         the same through a window with sinks
    kv_pages_trim / _free / _compact   what left the window, what ended, and the pool's free end
"""

import argparse
import ctypes
import importlib
import importlib.util
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]


def package():
    name = "typhoon_ocr_server_b200"
    if name not in sys.modules:
        at = ROOT / "typhoon-ocr-server_b200"
        spec = importlib.util.spec_from_file_location(name, at / "__init__.py", submodule_search_locations=[str(at)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def run(answers=16, steps=32, prompt=1024, window=512, sinks=4, page=64, seed=0):
    """Decodes `answers` answers for `steps` steps each way; returns the figures that main() prints."""
    pkg = package()
    pages = importlib.import_module(pkg.__name__ + ".pages")
    lib = pkg.load_attention_lib()
    layers, heads, kv_heads, d = pkg.NUM_LAYERS, pkg.NUM_Q_HEADS, pkg.NUM_KV_HEADS, pkg.HEAD_DIM
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32)  # noqa: E731
    at = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    lib.attn_set_stream(torch.cuda.current_stream().cuda_stream)

    def ok(rc, what):
        if rc:
            raise RuntimeError(f"{what}: {pkg.last_error(lib)}")

    # The prompt, into a static cache.
    cache = lib.kv_cache_alloc_ex(prompt, pkg.ATTN_KV_BF16)
    if not cache:
        raise RuntimeError(pkg.last_error(lib))
    try:
        norm = torch.ones(d, device="cuda")
        angle = torch.arange(prompt, device="cuda")[:, None] * pkg.MROPE_THETA ** (-torch.arange(d // 2, device="cuda") / (d // 2))[None]
        cos, sin = angle.cos().contiguous(), angle.sin().contiguous()
        out = torch.empty((prompt, heads, d), device="cuda")
        for layer in range(layers):
            q, k, v = rand(prompt, heads, d), rand(prompt, kv_heads, d), rand(prompt, kv_heads, d)
            ok(lib.attention_prefill_fused_gqa(at(q), at(k), at(v), pkg.ATTN_DT_F32, at(norm), at(norm), at(cos), at(sin), cache, layer,
                                               at(out), pkg.ATTN_DT_F32, prompt, pkg.SCALE, pkg.RMS_EPS), "prefill")
        lib.kv_cache_advance(cache, prompt)
        # A pool with room for the prompt and, per answer, its copy of the prompt's last page and its own rows.
        own = -(-(2 * steps) // page) + 2
        pool = pages.PagePool.empty(layers, -(-prompt // page) + answers * own, page, kv_heads, d, answers + 1, -(-prompt // page) + own, lib=lib)
        pool.import_cache(0, cache)
        ok(lib.attn_sync(), "import")
    finally:
        lib.kv_cache_free(cache)

    seqs = ints(list(range(1, answers + 1)))
    pool.fork(ints([0] * answers), seqs)
    ones, starts = ints([1] * answers), ints(list(range(answers + 1)))
    figures = {"pages for the prompt and its branches": int((pool.ref > 0).sum()),
               "pages of as many copies": (answers + 1) * -(-prompt // page)}

    def step(length, attend):
        """One token for every answer: its rows in every layer, then that layer's attention."""
        pool.extend(seqs, ones)
        outs = []
        for layer in range(layers):
            q, k, v = (rand(answers, n, d).bfloat16() for n in (heads, kv_heads, kv_heads))
            pool.write(layer, seqs, starts, k, v)
            outs.append((q, attend(q, layer, length)))
        return outs

    # Decoding with the prompt shared; the last step once more with every answer reading it for itself.
    length = prompt
    for _ in range(steps):
        length += 1
        outs = step(length, lambda q, layer, n: pool.attend_prefix(q, layer, seqs, prompt, n, pkg.SCALE))
    apart = [pool.attend_window(q, layer, seqs, None, 1, length, 0, 0, pkg.SCALE) for layer, (q, _) in enumerate(outs)]
    figures["largest difference, shared prompt against each for itself"] = max(
        float((o.float() - a.float()).abs().max()) for (_, o), a in zip(outs, apart))

    # On through a window: the pages that it leaves behind go back as it moves.
    for _ in range(steps):
        length += 1
        pool.trim(seqs, window, sinks)
        outs = step(length, lambda q, layer, n: pool.attend_window(q, layer, seqs, None, 1, n, window, sinks, pkg.SCALE))
    figures["pages through the window"] = int((pool.ref > 0).sum())

    # Every second answer ends, the prompt itself is no longer needed, and the rest moves to the pool's front.
    pool.free(ints([0] + list(range(2, answers + 1, 2))))
    kept, q = seqs[::2].contiguous(), outs[0][0][::2].contiguous()
    before = pool.attend_window(q, 0, kept, None, 1, length, window, sinks, pkg.SCALE)
    live = torch.zeros(1, dtype=torch.int32, device="cuda")
    pool.compact(live)
    after = pool.attend_window(q, 0, kept, None, 1, length, window, sinks, pkg.SCALE)
    ok(lib.attn_sync(), "decoding")
    figures["pages of the answers that go on"] = int(live)
    figures["their outputs unchanged by the move"] = torch.equal(before, after)
    pool.close()
    return figures


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--answers", type=int, default=16)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    for name, value in run(a.answers, a.steps).items():
        print(f"{name}: {value}")


if __name__ == "__main__":
    main()
