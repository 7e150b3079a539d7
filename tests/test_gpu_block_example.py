"""The operators together, as a network uses them: the example that learns from a bundle adjustment."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


def _example():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples'))
    import depth_correction
    return depth_correction


def test_the_example_learns():
    losses = _example().main(n_imgs=12, n_tracks=800, train_steps=30, verbose=False)
    assert losses[-1] < 0.8 * losses[0]


def test_packed_images_do_not_see_each_other():
    """Another image's tokens change nothing but its own outputs and gradients."""
    ex = _example()
    torch.manual_seed(0)
    model = ex.Correction(8)
    table = ex.rotary_table(64, 16, base=100.0)
    cu = torch.tensor([0, 70, 70, 230, 301], dtype=torch.int32, device='cuda')
    tokens = torch.randn(301, 8, device='cuda').bfloat16()
    patches = torch.randint(0, 32, (301, 2), device='cuda', dtype=torch.int32)
    outs = []
    for scale in (1.0, 3.0):
        t = tokens.clone()
        t[70:230] *= scale
        t.requires_grad_()
        y = model(t, patches, cu, 160, table)
        (g,) = torch.autograd.grad(y[230:].square().sum(), t)
        outs.append((y.detach(), g))
    keep = torch.ones(301, dtype=torch.bool, device='cuda')
    keep[70:230] = False
    assert torch.equal(outs[0][0][keep], outs[1][0][keep]) and torch.equal(outs[0][1], outs[1][1])
    assert float(outs[0][1][:230].abs().max()) == 0 and float(outs[0][1][230:].abs().max()) > 0
