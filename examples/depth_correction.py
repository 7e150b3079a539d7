"""Learns a correction of a network's log-depths from a bundle adjustment's result.

One bundle adjustment refines cameras and points from what a depth network answered with; the depth of
every observed point then says how far the network's first log-depth channel is off.  This example
runs a few Levenberg-Marquardt steps on a synthetic scene and trains a small transformer on that
difference: an image's observations are one sequence (the observations of all images lie packed
one after the other, as the bundle adjustment has them), their patches give the rotary positions, and
the blocks use this package's operators: ``rotary``, ``attention`` and ``residual_norm``, forward and
backward.

    python examples/depth_correction.py
"""
import math
import os
import sys

import numpy as np
import torch

if __name__ == '__main__':
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from blast3r_b200.attention import attention, check_attention   # noqa: E402
from blast3r_b200.engine import lm_step                          # noqa: E402
from blast3r_b200.norm import check_norm, residual_norm                      # noqa: E402
from blast3r_b200.rotary import rotary, rotary_table             # noqa: E402
from blast3r_b200.synthetic import make_scene                    # noqa: E402

PATCH = 16


class Correction(torch.nn.Module):
    """Blocks of attention and a two-layer perceptron between norms with a scale for each channel."""

    def __init__(self, n_in, dim=128, heads=4, blocks=2, dtype=torch.bfloat16, device='cuda'):
        super().__init__()
        kw = dict(device=device, dtype=dtype)
        self.heads, self.n_blocks = heads, blocks
        self.embed = torch.nn.Linear(n_in, dim, **kw)
        self.qkv = torch.nn.ModuleList(torch.nn.Linear(dim, 3 * dim, **kw) for _ in range(blocks))
        self.out = torch.nn.ModuleList(torch.nn.Linear(dim, dim, **kw) for _ in range(blocks))
        self.up = torch.nn.ModuleList(torch.nn.Linear(dim, 2 * dim, **kw) for _ in range(blocks))
        self.down = torch.nn.ModuleList(torch.nn.Linear(2 * dim, dim, **kw) for _ in range(blocks))
        self.head = torch.nn.Linear(dim, 1, **kw)
        ones = lambda n, v: torch.nn.ParameterList(torch.full((dim,), v, device=device) for _ in range(n))   # noqa: E731
        self.weight, self.bias, self.scale = ones(2 * blocks + 1, 1.0), ones(2 * blocks + 1, 0.0), ones(2 * blocks, 0.3)

    def forward(self, tokens, patches, cu, longest, table):
        """tokens (n, n_in); patches (n, 2) integer positions; cu (images + 1,): where each image begins."""
        pre = lambda i: (self.weight[i], self.bias[i])                                                          # noqa: E731
        x = torch.zeros(tokens.shape[0], self.embed.out_features, device=tokens.device)   # float32 residual stream
        x, h = residual_norm(self.embed(tokens), x, pre=pre(0))
        for b in range(self.n_blocks):
            q, k, v = self.qkv[b](h).unflatten(-1, (3, self.heads, -1)).unbind(1)
            q, k = (t[0] for t in rotary((q[None], k[None]), table, patches))
            y = attention(q, k, v, cu_q=cu, cu_k=cu, max_q=longest, max_k=longest)
            x, h = residual_norm(self.out[b](y.flatten(1)), x, gate=self.scale[2 * b], pre=pre(2 * b + 1))
            y = self.down[b](torch.nn.functional.gelu(self.up[b](h)))
            x, h = residual_norm(y, x, gate=self.scale[2 * b + 1], pre=pre(2 * b + 2))
        return self.head(h).squeeze(-1).float()


def observed_log_depth(p):
    """log of every observation's depth in its camera, from the parameters of a bundle adjustment."""
    n = torch.diff(p['rigs'][0].long(), prepend=p['rigs'].new_zeros(1).long())
    img = torch.repeat_interleave(torch.arange(len(n), device=n.device), n)
    P = p['P_rig2cam'][p['rigs'][2].long()] @ p['P_w2rig'][p['rigs'][1].long()]
    X = p['pts3d'][p['pids'].long()]
    return (P[img, 2, :3] * X).sum(-1).add(P[img, 2, 3]).clamp(min=1e-3).log()


def main(n_imgs=24, n_tracks=3000, lm_steps=3, train_steps=60, seed=0, verbose=True):
    """Returns the training losses."""
    torch.manual_seed(seed)
    sc = make_scene(0, n_imgs=n_imgs, n_tracks=n_tracks, seed=seed + 1)
    p = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in sc.lm_inputs().items()}
    scale = torch.tensor([2 / 512, 2 / 384], device='cuda')
    at = p['pix2d'] * scale - 1                                # -1..1 over the image
    p['pix2d_dep'][:, 0] += 0.3 * at.square().sum(-1)          # this network sees the image's borders too far away
    for _ in range(lm_steps):
        p.update(lm_step(**p, weight_z=1e-3, pnorm=1, huber_delta=1.0)[0])

    dep = p['pix2d_dep']
    target = observed_log_depth(p) - dep[:, 0]                 # what the network's log-depth lacks
    target = (target - target.mean()) / target.std().clamp(min=1e-6)
    tokens = torch.cat([dep, at, at.square()], dim=1).bfloat16()
    patches = (p['pix2d'] / PATCH).floor().clamp(0, 63).int()
    cu = torch.cat([p['rigs'].new_zeros(1), p['rigs'][0]]).int()
    longest = int(torch.diff(cu).max())
    model = Correction(tokens.shape[1])
    table = rotary_table(64, 16, base=100.0)                   # two axes of 16 of the head's 32 elements
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3)
    losses = []
    for step in range(train_steps):
        loss = (model(tokens, patches, cu, longest, table) - target).square().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if verbose and step % 10 == 0:
            print(f'step {step:3d}  loss {losses[-1]:.4f}')
    check_attention()
    check_norm()
    if verbose:
        print(f'{sc.n_obs} observations of {n_imgs} images: loss {losses[0]:.4f} -> {losses[-1]:.4f}')
    assert all(math.isfinite(v) for v in losses)
    return losses


if __name__ == '__main__':
    main()
