"""Regions of a 3-D head that look at the whole map: RoIAlign, a linear layer, two decoder layers.

    python examples/region_decoder.py [--steps N]

Trains on random maps and boxes to tell which of four quarters of the map a box lies in (bfloat16), then runs the same
layers for inference with their linear layers in 8 bits and prints how often the two agree."""
import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from medvision_amd.ops import BlockScaledLinear, RegionDecoderLayer, RoIAlign, map_tokens  # noqa: E402


class Head(nn.Module):
    def __init__(self, channels=64, heads=4, layers=2, cells=4, classes=4):
        super().__init__()
        self.pool = RoIAlign((cells,) * 3, 1.0, 2)
        self.first = nn.Linear(channels * cells ** 3, channels)
        self.layers = nn.ModuleList(RegionDecoderLayer(channels, heads, key_heads=heads // 2) for _ in range(layers))
        self.classes = nn.Linear(channels, classes)

    def forward(self, features, rois, key_lengths):
        batch = features.size(0)
        pooled = self.pool(features, rois).flatten(1)
        regions, residual = self.first(pooled).unflatten(0, (batch, -1)), None   # as many rois for each sample
        tokens = map_tokens(features)
        for layer in self.layers:
            regions, residual = layer(regions, tokens, residual, key_lengths=key_lengths)
        return self.classes(regions + residual)

    def for_inference(self, dtype):
        head = Head.__new__(Head)
        nn.Module.__init__(head)
        head.pool, head.classes = self.pool, self.classes
        head.first = BlockScaledLinear.from_linear(self.first, dtype)
        head.layers = nn.ModuleList(layer.for_inference(dtype) for layer in self.layers)
        return head.eval()


def batch_of(generator, batch, regions, shape, dtype):
    """Maps with a different pattern in each quarter, boxes, and the quarter that each box's middle lies in."""
    depth, height, width = shape
    features = torch.randn(batch, 64, *shape, generator=generator, device="cuda")
    for i in range(4):
        y, x = i // 2 * (height // 2), i % 2 * (width // 2)
        features[:, 8 * i:8 * i + 8, :, y:y + height // 2, x:x + width // 2] += 1.0
    size = torch.tensor([width, height, depth], device="cuda", dtype=torch.float32)
    middle = torch.rand(batch * regions, 3, generator=generator, device="cuda") * (size - 6) + 3
    index = torch.arange(batch, device="cuda").repeat_interleave(regions)[:, None]
    rois = torch.cat((index.float(), middle - 3, middle + 3), 1)
    quarter = (middle[:, 1] >= height / 2) * 2 + (middle[:, 0] >= width / 2)
    lengths = torch.full((batch,), depth * height * width, device="cuda", dtype=torch.int32)
    return features.to(dtype), rois, quarter.long().view(batch, regions), lengths


def main(steps=30):
    torch.manual_seed(0)
    generator = torch.Generator(device="cuda").manual_seed(0)
    dtype = torch.bfloat16
    head = Head().cuda().to(dtype)
    optimizer = torch.optim.AdamW(head.parameters(), lr=2e-3)
    losses = []
    for step in range(steps):
        features, rois, quarter, lengths = batch_of(generator, 2, 100, (8, 24, 24), dtype)
        loss = nn.functional.cross_entropy(head(features, rois, lengths).float().flatten(0, 1), quarter.flatten())
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    with torch.no_grad():
        features, rois, quarter, lengths = batch_of(generator, 2, 100, (8, 24, 24), dtype)
        full = head(features, rois, lengths).argmax(-1)
        small = head.for_inference(dtype)(features, rois, lengths).argmax(-1)
    right, agree = (full == quarter).float().mean().item(), (full == small).float().mean().item()
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f}, right {right:.3f}, the same class in 8 bits {agree:.3f}")
    return losses, right, agree


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=30)
    main(parser.parse_args().steps)
