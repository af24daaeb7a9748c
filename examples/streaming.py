"""Streaming attention end to end: a prompt prefix, video frame by frame over a paged cache,
then several continuations decoded token by token from the same pages.

    python examples/streaming.py [--frames 6] [--tokens 720] [--e4m3]

One attention layer of random weights stands for a model: what counts is the order of the
calls.  The frames' outputs are compared with window_attention over the whole sequence.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-minimaxh3_b200"))

from h3b import PagedKVCache, decode_attention, device_status  # noqa: E402
from h3b import context as C  # noqa: E402
from h3b.streaming import WindowAttentionB200  # noqa: E402


def ints(values) -> torch.Tensor:
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def stream(frames: int = 6, tokens: int = 720, prefix: int = 77, heads: int = 8, kv_heads: int = 4, seen: int = 3,
           continuations: int = 3, steps: int = 20, e4m3: bool = False, seed: int = 0) -> dict:
    """Runs the whole course; returns the frames' outputs, the whole-sequence ones and the decoded rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = prefix + frames * tokens
    q, k, v = (torch.randn(total, h, 128, device="cuda", generator=g).to(torch.bfloat16) for h in (heads, kv_heads, kv_heads))
    page = 64
    cache = PagedKVCache.create(layers=1, pages=-(-total // page) + continuations * 2 + 2, page_tokens=page,
                                kv_heads=kv_heads, slots=1 + continuations, max_tokens=total + steps)
    backend = WindowAttentionB200(frames=seen)
    out = torch.empty_like(q)
    slot = ints([0])
    with C.attention_protected_prefix(prefix), C.attention_video_layout(frames, tokens):
        at = 0
        for n in [prefix] + [tokens] * frames:  # the prefix, then a frame at a time
            rows = slice(at, at + n)
            cache.append(slot, k[rows], v[rows], starts=ints([0, n]))
            out[rows] = backend.cached(q[rows], cache, slot)
            at += n
        whole = backend(q, k, v)

    # continuations share the pages of slot 0 until their first own token
    children = ints(range(1, 1 + continuations))
    cache.fork(ints([0] * continuations), children)
    decoder = cache
    if e4m3:  # the same sequence again, in 8 bits
        scale = torch.full((1, kv_heads), 0.02, device="cuda")
        decoder = PagedKVCache.create(1, cache.k.shape[1], page, kv_heads, 1 + continuations, total + steps,
                                      torch.float8_e4m3fn, k_scale=scale, v_scale=scale)
        decoder.append(slot, k, v, starts=ints([0, total]))
        decoder.fork(ints([0] * continuations), children)
    decoded = []
    for _ in range(steps):
        nq, nk, nv = (torch.randn(continuations, h, 128, device="cuda", generator=g).to(torch.bfloat16)
                      for h in (heads, kv_heads, kv_heads))
        decoder.append(children, nk, nv)
        decoded.append(decode_attention(nq, decoder, children, window=4 * tokens, sinks=prefix))
    decoder.truncate(children, ints([total + steps // 2] * continuations))  # drop the last half again
    decoder.free(ints([0]))
    decoder.compact()
    decoder.check()
    cache.check()
    assert device_status(0) == 0
    return dict(frames=out, whole=whole, decoded=torch.stack(decoded), cache=decoder, total=total)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--frames", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=720)
    ap.add_argument("--e4m3", action="store_true")
    args = ap.parse_args()
    r = stream(args.frames, args.tokens, e4m3=args.e4m3)
    off = (r["frames"].float() - r["whole"].float()).norm() / r["whole"].float().norm()
    used = int((r["cache"].refs > 0).sum())
    print(f"{r['total']} tokens frame by frame against the whole sequence: relative difference {float(off):.1e}")
    print(f"decoded {tuple(r['decoded'].shape)}; {used} pages in use after the continuations were cut back")


if __name__ == "__main__":
    main()
