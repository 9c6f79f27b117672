"""Train the embedding heads of a few maps and score detections against 4- and 8-bit memory banks.

Each map's camera turns the embeddings it sees by a rotation of its own; the head learns to undo it.  Prints the
share of detections whose best-scoring object is the right one, before and after, per bank format.

    python examples/map_heads.py [--maps 8] [--objects 512] [--dim 256] [--steps 200]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "robot-agent_b200"))
from scenemap_b200 import products  # noqa: E402
from scenemap_b200.heads import MapHeads  # noqa: E402


def unit(v):
    return v / v.norm(dim=-1, keepdim=True)


def run(maps=8, objects=512, dim=256, steps=200, lr=None, seed=0, say=print):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    vectors = unit(rand(maps, objects, dim))                               # what the maps remember
    turn = torch.linalg.qr(rand(maps, dim, dim)).Q
    lr = 0.2 * dim if lr is None else lr                                   # unit rows: a curvature of about 1 / dim

    def detections():
        """Ragged numbers of detections per map: (rows, off, map of each row, object of each row)."""
        n = torch.randint(0, 2 * objects, (maps,), generator=g, device="cuda")
        off = torch.cat((n.new_zeros(1), n.cumsum(0))).to(torch.int32)
        m = torch.repeat_interleave(torch.arange(maps, device="cuda"), n)
        o = torch.randint(0, objects, m.shape, generator=g, device="cuda")
        seen = torch.bmm(vectors, turn)[m, o]
        return unit(seen + 0.02 * rand(*seen.shape)).to(torch.bfloat16), off, m, o

    heads = MapHeads(maps, dim)
    banks = {bits: heads.bank(vectors, bits) for bits in (4, 8)}
    z, off, _, o = detections()

    def right(bits):
        return float((heads.scores(z, off, banks[bits]).argmax(1) == o).float().mean())

    out = {"before": {b: right(b) for b in banks}}
    losses = []
    for _ in range(steps):
        zt, offt, mt, ot = detections()
        losses.append(heads.train_step(zt, vectors[mt, ot], offt, lr))
    out["after"] = {b: right(b) for b in banks}
    out["loss"] = [float(losses[0]), float(losses[-1])]
    assert products.error() == 0
    for when in ("before", "after"):
        say(f"{when}: " + ", ".join(f"{b}-bit bank {100 * v:.1f}% right" for b, v in out[when].items()))
    say(f"loss {out['loss'][0]:.4f} -> {out['loss'][1]:.4f} in {steps} steps")
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    for name, v in (("maps", 8), ("objects", 512), ("dim", 256), ("steps", 200)):
        ap.add_argument("--" + name, type=int, default=v)
    run(**vars(ap.parse_args()))
