"""A small point network on this library: attention between neighbouring patches.

The cloud is put in the curve order of its BVH and cut into patches of 64 points,
which are the tree's own nodes.  Every patch attends to the patches nearest to it,
with a learned bias of the relative position; a group norm with SiLU goes before.
The network learns a smooth field at the points, and is then asked for it at
single places that are no points of the cloud.

    python examples/point_attention.py [--points 20000] [--steps 60] [--float32]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import torchbvh_amd as tb  # noqa: E402

HEADS, CHANNELS, PATCH, NEAREST, REACH, SIZES = 4, 16, 64, 8, 24, 12


class PatchAttention(torch.nn.Module):
    """x + project(attention(norm(x))) over chosen patches."""

    def __init__(self, width: int):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(width))
        self.bias = torch.nn.Parameter(torch.zeros(width))
        self.qkv = torch.nn.Linear(width, 3 * HEADS * CHANNELS)
        self.project = torch.nn.Linear(HEADS * CHANNELS, width)
        self.table = torch.nn.Parameter(torch.zeros(3, 2 * SIZES - 1, HEADS))

    def forward(self, x, where, layout, selected, buckets):
        y = tb.group_norm_act(x, 8, self.weight, self.bias, layout)
        q, k, v = self.qkv(y).reshape(-1, 3, HEADS, CHANNELS).unbind(1)  # read in place
        bias = tb.RelativeBias(self.table, buckets, where, where)
        out = tb.block_attention(q, k, v, selected, layout, layout, bias=bias)
        return x + self.project(out.reshape(x.size(0), -1))


def field(points: torch.Tensor) -> torch.Tensor:
    return torch.sin(6.0 * points[:, 0]) * torch.cos(5.0 * points[:, 1]) + points[:, 2] ** 2


def main(points: int = 20_000, steps: int = 60, kind: torch.dtype = torch.bfloat16, seed: int = 0) -> list[float]:
    """The loss of every step; prints some of them."""
    torch.manual_seed(seed)
    device = torch.device("cuda")
    cloud = torch.rand((points, 3), device=device)
    bvh = tb.build_bvh(cloud)
    cloud = cloud[bvh["sorted_indices"]]                      # curve order, as the layout has it
    layout, boxes = tb.block_layout(bvh, PATCH), tb.block_boxes(bvh, PATCH)
    selected = tb.select_blocks(cloud, boxes, NEAREST, layout, layout)
    where = (cloud * points ** (1 / 3)).int()                 # cells of about one point
    buckets = tb.relative_buckets(SIZES, REACH)

    width = 32
    embed = torch.nn.Linear(3, width).to(device, kind)
    layers = torch.nn.ModuleList(PatchAttention(width) for _ in range(2)).to(device, kind)
    head = torch.nn.Linear(width, 1).to(device, kind)
    # Half the field is given; the network fills in the other half.
    target = field(cloud)
    given = torch.rand(points, device=device) < 0.5
    features = torch.stack([torch.where(given, target, torch.zeros_like(target)), given.float(), cloud[:, 0]], 1).to(kind)
    wanted = [*embed.parameters(), *layers.parameters(), *head.parameters()]
    optimizer = torch.optim.Adam(wanted, lr=4e-3)
    losses = []
    for step in range(steps):
        x = embed(features)
        for layer in layers:
            x = layer(x, where, layout, selected, buckets)
        loss = (head(x).float().squeeze(1) - target)[~given].square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if step % 20 == 0 or step == steps - 1:
            print(f"step {step}: loss {losses[-1]:.4f}", flush=True)

    # Single places: each chooses its own patches and attends to the cloud's features.
    with torch.no_grad():
        places = torch.rand((16, 3), device=device)
        one = tb.block_layout((1, places.size(0)), 1)
        chosen = tb.select_blocks(places, boxes, NEAREST, one, layout)
        keys = x.reshape(points, 1, width)
        asked = keys[torch.randint(points, (places.size(0),), device=device)]
        answer = tb.block_attention(asked.contiguous(), keys, keys, chosen, one, layout)
    assert answer.shape == (16, 1, width) and bool(torch.isfinite(answer).all())
    tb.destroy_bvh(bvh)
    return losses


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--points", type=int, default=20_000)
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--float32", action="store_true")
    a = p.parse_args()
    main(a.points, a.steps, torch.float32 if a.float32 else torch.bfloat16)
