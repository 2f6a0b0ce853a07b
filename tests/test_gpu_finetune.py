"""The head trained on a frozen detector: the path that runs group norm and AdamW together."""
import pytest
import torch

from kadcnet import finetune

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype,bits', [('fp32', 32), ('bf16', 8), ('fp16', 8)])
def test_loss_falls(dtype, bits, capsys):
    """Eight classes: from ln 8 = 2.1 at least a quarter of the way down in 40 steps."""
    losses = finetune.main(['--steps', '40', '--batch', '2', '--size', '256', '--dtype', dtype, '--state-bits', str(bits)])
    assert len(losses) == 40 and all(x == x for x in losses)
    assert sum(losses[-4:]) / 4 < 0.75 * sum(losses[:4]) / 4
    assert f'{bits}-bit states' in capsys.readouterr().out


def test_the_detector_stays_as_it_is():
    from kadcnet import build_kadcnet_s, enable_fast_inference
    model = build_kadcnet_s(seed=3).fuse().cuda()
    enable_fast_inference(model)
    before = [p.clone() for p in model.parameters()]
    gen = torch.Generator().manual_seed(0)
    maps = finetune.neck_maps(model, finetune.synthetic_images(1, 256, 'cuda', torch.float32, gen))
    targets = finetune.projected_classes(maps, [torch.randn(4, m.shape[1], generator=gen).cuda() for m in maps])
    head = finetune.GroupNormHead([m.shape[1] for m in maps], 4).cuda()
    held = [p.clone() for p in head.parameters()]
    finetune.train_head(head, [(maps, targets)] * 2, state_bits=32)
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), before))
    assert not any(torch.equal(p, q) for p, q in zip(head.parameters(), held))
