"""Frames arriving one by one through a global-attention layer with a bounded cache.

    python examples/stream_frames.py [--frames 40] [--budget-frames 31]

Each frame has 5 special tokens and a 37 x 37 patch grid (1,374 tokens, 16
heads of 64, as the layers of the 32-frame configuration).  The layer turns
queries and keys by their grid positions, writes keys and values into the paged
cache, attends from the frame to everything cached, adds up what each cached
token received and evicts the tokens of least weight once the cache is over its
budget.  Prints the time of each step's operators and what the cache holds.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "sparse-attention-vggt_b200"))
import vggt_sparse  # noqa: E402


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--frames", type=int, default=40)
    ap.add_argument("--budget-frames", type=int, default=31)
    ap.add_argument("--heads", type=int, default=16)
    args = ap.parse_args()
    dev, side, special = torch.device("cuda"), 37, 5
    tokens = special + side * side
    layer = vggt_sparse.StreamingGlobalLayer(args.heads, 64, tokens, args.budget_frames * tokens,
                                             special=special, device=dev)
    yy, xx = torch.meshgrid(torch.arange(side), torch.arange(side), indexing="ij")
    pos = torch.cat((torch.zeros(special, 2), torch.stack((yy.flatten() + 1, xx.flatten() + 1), -1)))
    pos = pos.to(torch.int32).to(dev)
    gen = torch.Generator(device=dev).manual_seed(0)
    scene = torch.randn(side * side + special, args.heads, 64, generator=gen, device=dev)
    ms = []
    for f in range(args.frames):
        # neighbouring frames look alike
        noise = lambda: torch.randn(scene.shape, generator=gen, device=dev)  # noqa: E731
        scene = 0.9 * scene + 0.44 * noise()
        q, k, v = ((scene + 0.5 * noise()).to(torch.bfloat16) for _ in range(3))
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        layer(q, k, v, pos)
        end.record()
        end.synchronize()
        ms.append(begin.elapsed_time(end))
    layer.cache.check()
    held = layer.cache.ids[0, 0, :layer.cache.lengths[0]]
    frames = torch.bincount(held // tokens, minlength=args.frames)
    print("ms per frame: " + " ".join("%.2f" % t for t in ms))
    print("cached %d of %d tokens; head 0 holds of each frame: %s"
          % (layer.cache.lengths[0], args.frames * tokens, frames.tolist()))


if __name__ == "__main__":
    main()
