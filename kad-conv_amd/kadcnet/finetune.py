"""A new head trained on a detector that stays as it is: the detector's neck maps come from the whole-network
HIP forward, the head is convolutions with ``kadconv.GroupNormAct`` (statistics of a group, so that a batch of
one or two large images trains as a batch of many does), and ``kadconv.AdamW`` steps all of its tensors in one
launch, with states in 8 bits if asked to.

    python -m kadcnet.finetune --steps 50 --batch 8 --size 640 --dtype bf16 --state-bits 8

runs it on synthetic images: a cell's class is the largest of fixed random projections of its neck map.

    python -m kadcnet.finetune --distill 4

goes on with a smaller head that learns from the first one's 4 best logits of each cell alone (``kadconv.distill_loss``):
1 x 1 convolutions whose products are in 8 bits (``kadconv.Linear8``), with ``kadconv.LayerNorm`` over each cell's channels.
``StudentHead.serve`` keeps its weights in 8 bits.
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


class StudentHead(nn.Module):
    """Class logits of each cell from each neck map, cell by cell: two 1 x 1 convolutions in 8 bits with layer norm over the
    channels and SiLU, and a third."""

    def __init__(self, channels, classes, width=64):
        super().__init__()
        self.scales = nn.ModuleList(nn.Sequential(
            kadconv.Linear8(c, width, dim=1), kadconv.LayerNorm(width, dim=1), nn.SiLU(),
            kadconv.Linear8(width, width, dim=1), kadconv.LayerNorm(width, dim=1), nn.SiLU(),
            kadconv.Linear8(width, classes, dim=1)) for c in channels)

    def forward(self, maps):
        return [scale(m) for scale, m in zip(self.scales, maps)]

    def serve(self):
        """In eval mode, the weights kept in 8 bits; until ``train()``."""
        self.eval()
        for m in self.modules():
            if isinstance(m, kadconv.Linear8):
                m.keep()
        return self


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


def top_logits(head, maps, entries):
    """(logits, classes) of each cell's best ``entries`` classes, a pair of maps [N, entries, H, W] for each neck map: what a
    student needs of its teacher."""
    with torch.no_grad():
        return [tuple(torch.topk(z, min(entries, z.shape[1]), dim=1)) for z in head(maps)]


def distill_head(student, batches, temperature=2.0, lr=2e-3, weight_decay=1e-2, state_bits=8, seed=0):
    """One step a batch of (neck maps, a teacher's top logits on them); the losses as a GPU tensor."""
    masters = next(student.parameters()).dtype != torch.float32
    optimizer = kadconv.AdamW(student.parameters(), lr=lr, weight_decay=weight_decay, state_bits=state_bits,
                              master_weights=masters, seed=seed)
    losses = []
    for maps, top in batches:
        loss = sum(kadconv.distill_loss(z, t, i, temperature, dim=1) for z, (t, i) in zip(student(maps), top)) / len(top)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses)


def agreement(student, teacher, maps):
    """The share of cells whose best class both heads agree on."""
    with torch.no_grad():
        same = [(a.argmax(1) == b.argmax(1)).float().flatten() for a, b in zip(student(maps), teacher(maps))]
    return torch.cat(same).mean().item()


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
    ap.add_argument('--distill', type=int, default=0, metavar='ENTRIES',
                    help="then train a head of 8-bit 1 x 1 convolutions by the first one's best ENTRIES logits of each cell")
    ap.add_argument('--temperature', type=float, default=2.0)
    a = ap.parse_args(argv)
    if a.steps < 1 or a.batch < 1 or a.size < 128 or a.size % 32:
        ap.error('steps and batch must be positive, size a multiple of 32 from 128 on')
    if a.distill < 0 or not 1e-6 <= a.temperature <= 1e6:
        ap.error('distill must not be negative, and temperature lie in 1e-6 to 1e6')
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
    if a.distill:
        losses = losses, distill(a, head, channels, maps)
    return losses


def distill(a, teacher, channels, maps):
    """The student's part of the program: its losses."""
    teacher.eval()

    def batches():
        for _ in range(a.steps):
            m = maps()
            yield m, top_logits(teacher, m, a.distill)

    device, dtype = torch.device('cuda'), DTYPES[a.dtype]
    student = StudentHead(channels, a.classes).to(device, dtype)
    torch.cuda.synchronize()
    start = time.perf_counter()
    losses = distill_head(student, batches(), a.temperature, lr=a.lr, state_bits=a.state_bits, seed=a.seed).tolist()
    ms = (time.perf_counter() - start) * 1e3 / a.steps
    tenth = max(1, a.steps // 10)
    print(f'student: {a.steps} steps by {a.distill} entries a cell: {ms:.1f} ms a step, loss {sum(losses[:tenth]) / tenth:.4f} -> '
          f'{sum(losses[-tenth:]) / tenth:.4f}, served in 8 bits it agrees on {agreement(student.serve(), teacher, maps()):.3f} of the cells')
    return losses


if __name__ == '__main__':
    main()
