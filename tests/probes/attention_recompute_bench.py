"""The engines' attention gradient from stored and from recomputed probabilities (tuning aid, not a test):  python tests/probes/attention_recompute_bench.py
At the UNets' attention levels, from an fp16 tape: ops.attention(probs_only) + ops.attention_bwd as the engines call them, against ops.attention_recompute_bwd
(DIFFPURE_ATTN_RECOMPUTE=1).  Prints microseconds a call, both sides in turn, and how far the two results are apart."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
from diffpure_amd import ops  # noqa: E402

DEV = "cuda:0"
#        name, batch, tokens, heads, head dimension, layout
LEVELS = [("guided 32 x 32", 32, 1024, 8, 64, "legacy"), ("guided 16 x 16", 32, 256, 16, 64, "legacy"), ("guided 8 x 8", 32, 64, 16, 64, "legacy"),
          ("NCSN++ 16 x 16", 128, 256, 1, 256, "split")]


def timeit(fn, iters=20):
    for _ in range(3):
        fn()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(iters):
        fn()
    e1.record()
    torch.cuda.synchronize()
    return e0.elapsed_time(e1) / iters * 1e3


def main():
    for name, b, t, h, d, layout in LEVELS:
        qkv, dout = torch.randn(b, t, 3 * h * d, device=DEV).half(), torch.randn(b, t, h * d, device=DEV)

        def stored():
            x = qkv if ops.attention_h16_serves(t, d) else qkv.float()
            _, probs = ops.attention(x, h, layout, probs_only=True, h16=True)
            return ops.attention_bwd(x, probs, dout, h, layout, h16=True)

        def recomputed():
            return ops.attention_recompute_bwd(qkv, dout, h, layout)

        a, r = stored(), recomputed()
        apart = ((a - r).abs().max() / a.abs().max()).item()
        del a, r
        times = [[timeit(f) for f in (stored, recomputed)] for _ in range(3)]
        print(f"{name:16s} B={b:4d} | stored {min(x[0] for x in times):8.1f} us | recomputed {min(x[1] for x in times):8.1f} us | apart by {apart:.1e} of the largest element", flush=True)


if __name__ == "__main__":
    main()
