"""A new head trained on a detector that stays as it is: the detector's neck maps come from the whole-network
HIP forward, the head is convolutions with ``kadconv.GroupNormAct`` (statistics of a group, so that a batch of
one or two large images trains as a batch of many does), and ``kadconv.AdamW`` steps all of its tensors in one
launch, with states in 8 bits if asked to.

    python -m kadcnet.finetune --steps 50 --batch 8 --size 640 --dtype bf16 --state-bits 8

runs it on synthetic images: a cell's class is the largest of fixed random projections of its neck map.
"""
import argparse
import time

import torch
import torch.nn as nn
import torch.nn.functional as F

import kadconv

from .fast import enable_fast_inference

DTYPES = {'fp32': torch.float32, 'fp16': torch.float16, 'bf16': torch.bfloat16}


class GroupNormHead(nn.Module):
    """Class logits of each cell from each neck map: two 3 x 3 convolutions with group norm and SiLU, and a
    1 x 1 convolution."""

    def __init__(self, channels, classes, width=64, groups=8):
        super().__init__()
        self.scales = nn.ModuleList(nn.Sequential(
            nn.Conv2d(c, width, 3, padding=1, bias=False), kadconv.GroupNormAct(groups, width),
            nn.Conv2d(width, width, 3, padding=1, bias=False), kadconv.GroupNormAct(groups, width),
            nn.Conv2d(width, classes, 1)) for c in channels)

    def forward(self, maps):
        return [scale(m) for scale, m in zip(self.scales, maps)]


def neck_maps(model, images):
    """The maps that the detector's own head reads, [N, C, H, W] in channels-last memory (slices of wider maps
    among them), from a model with ``enable_fast_inference``."""
    with torch.no_grad():
        _, layers = model._kad_plan.forward(images, keep_layers=True)
    return [layers[i].permute(0, 3, 1, 2) for i in model.model[-1].f]


def synthetic_images(n, size, device, dtype, generator):
    """Images of smooth colours with noise."""
    coarse = torch.rand(n, 3, 7, 7, generator=generator).to(device)
    colours = F.interpolate(coarse, size=(size, size), mode='bicubic', align_corners=False)
    return (colours + 0.1 * torch.randn(n, 3, size, size, generator=generator).to(device)).clamp(0, 1).to(dtype)


def projected_classes(maps, projections):
    """Each cell's class: which of the projections [classes, C] of its values is largest, its map's mean and
    spread of each channel taken out."""
    out = []
    for m, p in zip(maps, projections):
        v = m.float()
        v = (v - v.mean(dim=(2, 3), keepdim=True)) / (v.std(dim=(2, 3), keepdim=True) + 1e-3)
        out.append(F.conv2d(v, p[:, :, None, None]).argmax(1))
    return out


def train_head(head, batches, lr=2e-3, weight_decay=1e-2, state_bits=8, seed=0):
    """One step a batch of (neck maps, targets); the losses as a GPU tensor."""
    masters = next(head.parameters()).dtype != torch.float32
    optimizer = kadconv.AdamW(head.parameters(), lr=lr, weight_decay=weight_decay, state_bits=state_bits,
                              master_weights=masters, seed=seed)
    losses = []
    for maps, targets in batches:
        logits = head(maps)
        loss = sum(F.cross_entropy(z.float(), t) for z, t in zip(logits, targets)) / len(targets)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split('\n\n')[0])
    ap.add_argument('--steps', type=int, default=50)
    ap.add_argument('--batch', type=int, default=8)
    ap.add_argument('--size', type=int, default=640)
    ap.add_argument('--classes', type=int, default=8)
    ap.add_argument('--dtype', choices=sorted(DTYPES), default='bf16')
    ap.add_argument('--state-bits', type=int, choices=(8, 32), default=8)
    ap.add_argument('--lr', type=float, default=2e-3)
    ap.add_argument('--seed', type=int, default=0)
    a = ap.parse_args(argv)
    if a.steps < 1 or a.batch < 1 or a.size < 128 or a.size % 32:
        ap.error('steps and batch must be positive, size a multiple of 32 from 128 on')
    from .synthetic import build_kadcnet_s
    device, dtype = torch.device('cuda'), DTYPES[a.dtype]
    model = build_kadcnet_s(seed=a.seed).fuse().to(device, dtype)
    enable_fast_inference(model)
    generator = torch.Generator().manual_seed(a.seed)

    def maps():
        return neck_maps(model, synthetic_images(a.batch, a.size, device, dtype, generator))

    channels = [m.shape[1] for m in maps()]
    projections = [torch.randn(a.classes, c, generator=generator).to(device) for c in channels]

    def batches():
        for _ in range(a.steps):
            m = maps()
            yield m, projected_classes(m, projections)

    torch.manual_seed(a.seed)
    head = GroupNormHead(channels, a.classes).to(device, dtype).to(memory_format=torch.channels_last)
    torch.cuda.synchronize()
    start = time.perf_counter()
    losses = train_head(head, batches(), lr=a.lr, state_bits=a.state_bits, seed=a.seed).tolist()
    ms = (time.perf_counter() - start) * 1e3 / a.steps
    tenth = max(1, a.steps // 10)
    print(f'{a.steps} steps of {a.batch} x 3 x {a.size} x {a.size} {a.dtype}, {a.state_bits}-bit states: {ms:.1f} ms a step, '
          f'loss {sum(losses[:tenth]) / tenth:.4f} -> {sum(losses[-tenth:]) / tenth:.4f}')
    return losses


if __name__ == '__main__':
    main()
