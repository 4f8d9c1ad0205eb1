"""Trains a feed-forward sublayer on a synthetic target, then serves it in 8 bits.

    python examples/feed_forward.py [--width 1024] [--inner 4096] [--rows 4096] [--steps 20]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from maloq_amd.feed_forward import FeedForward  # noqa: E402


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("width", 1024), ("inner", 4096), ("rows", 4096), ("steps", 20)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args(argv)
    dev, dt = torch.device("cuda:0"), torch.bfloat16
    torch.manual_seed(0)
    layer, teacher = (FeedForward(a.width, a.inner, device=dev, dtype=dt) for _ in range(2))
    opt = torch.optim.SGD(layer.parameters(), lr=0.2, momentum=0.9)
    losses = []
    for step in range(a.steps):
        x, r = (torch.randn(a.rows, a.width, device=dev, dtype=dt) for _ in range(2))
        with torch.no_grad():
            target = teacher(x, r)
        opt.zero_grad()
        loss = (layer(x, r) - target).float().square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {a.steps} steps", flush=True)

    served = layer.quantized()
    off = []
    with torch.no_grad():
        for rows in (1, 24, a.rows):
            x, r = (torch.randn(rows, a.width, device=dev, dtype=dt) for _ in range(2))
            y, q = layer(x, r).float(), served(x, r).float()
            off.append(((q - y).norm() / (y - x.float() - r.float()).norm()).item())
            times = []
            for f in (layer, served):
                for _ in range(3):
                    f(x, r)
                torch.cuda.synchronize()
                start = time.perf_counter()
                for _ in range(20):
                    f(x, r)
                torch.cuda.synchronize()
                times.append((time.perf_counter() - start) / 20 * 1e6)
            print(f"{rows} rows: bf16 {times[0]:.0f} us, e4m3 {times[1]:.0f} us; the sublayer's output is off by {off[-1]:.3f}", flush=True)
    return losses, off


if __name__ == "__main__":
    main()
