"""Distils a teacher's class logits into a scene's feature field.

A few thousand Gaussians carry feature channels next to their geometry.  Each
step renders one view's features, decodes every pixel with a gated feed-forward
block and compares the logits with the few largest that a teacher kept for that
pixel; the gradient trains the features and the block together.  The teacher
here is synthetic: every Gaussian belongs to a class by where it lies, and the
teacher sees the classes' composited weights.

    python examples/distil_feature_field.py [steps]
"""

from __future__ import annotations

import math
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from mlx3d_amd.cameras import Camera  # noqa: E402
from mlx3d_amd.losses import distillation_value_and_grad  # noqa: E402
from mlx3d_amd.nn import GatedFeedForward  # noqa: E402
from mlx3d_amd.optim import Adam, adam_step  # noqa: E402
from mlx3d_amd.splatting import render_gaussian_features  # noqa: E402

CLASSES, TOP, CHANNELS = 12, 4, 16


def scene(n: int, seed: int = 0, device="cuda"):
    """Geometry of n Gaussians in a ball, and the class of each (by direction)."""
    g = torch.Generator().manual_seed(seed)
    means = torch.randn((n, 3), generator=g) * 0.6
    quats = torch.randn((n, 4), generator=g)
    scales = torch.exp(torch.randn((n, 3), generator=g) * 0.3 - 2.6)
    opacities = torch.sigmoid(torch.randn((n,), generator=g) + 1.0)
    angle = torch.atan2(means[:, 1], means[:, 0]) / (2 * math.pi) + 0.5
    label = (angle * CLASSES).long().clamp(0, CLASSES - 1)
    return [t.to(device) for t in (means, quats, scales, opacities, label)]


def cameras(count: int, size: int):
    return [Camera.look_at(eye=(3.5 * math.sin(a), 0.4, -3.5 * math.cos(a)), width=size,
                           height=size * 3 // 4, fov=45.0)
            for a in (2 * math.pi * k / count for k in range(count))]


@torch.no_grad()
def teacher(camera, means, quats, scales, opacities, label):
    """The teacher's largest logits of each pixel and their classes; pixels that
    no Gaussian covers have none."""
    weights = torch.nn.functional.one_hot(label, CLASSES).float()
    out = render_gaussian_features(camera, means, quats, scales, opacities, weights)
    values, indices = torch.topk(torch.log(out["features"] + 1e-3) * 2.0, TOP, dim=-1)
    return values, torch.where(out["alpha"][..., None] > 0.05, indices, -1)


def train(steps: int = 60, n: int = 4000, size: int = 160, views: int = 4, verbose: bool = True):
    """Trains from zero; returns the loss of every step."""
    means, quats, scales, opacities, label = scene(n)
    views_ = cameras(views, size)
    told = [teacher(c, means, quats, scales, opacities, label) for c in views_]
    g = torch.Generator().manual_seed(1)
    field = {"features": (torch.randn((n, CHANNELS), generator=g) * 0.1).cuda()
             .requires_grad_(True)}
    block = GatedFeedForward(CHANNELS, 64, CLASSES, seed=2)
    updates = [(Adam(2e-2, eps=1e-15), field), (Adam(2e-3, eps=1e-15), block.params)]
    losses = []
    for step in range(steps):
        values, indices = told[step % views]
        out = render_gaussian_features(views_[step % views], means, quats, scales, opacities,
                                       field["features"])
        logits = block(out["features"])
        loss, grad = distillation_value_and_grad(logits, values, indices, temperature=2.0)
        logits.backward(grad)
        with torch.no_grad():
            adam_step([(opt, {k: p.grad for k, p in params.items()}, params)
                       for opt, params in updates])
            for _, params in updates:
                for p in params.values():
                    p.grad = None
        losses.append(loss)
        if verbose and (step + 1) % 20 == 0:
            print(f"step {step + 1}: loss {float(loss):.4f}", flush=True)
    with torch.no_grad():  # how many covered pixels the decoded view names as the teacher does
        out = render_gaussian_features(views_[0], means, quats, scales, opacities,
                                       field["features"])
        named = block(out["features"]).argmax(dim=-1)
        covered = told[0][1][..., 0] >= 0
        same = float((named == told[0][1][..., 0])[covered].float().mean())
    if verbose:
        print(f"the first view's labels agree in {100 * same:.1f} % of its pixels")
    return [float(v) for v in losses], same


if __name__ == "__main__":
    train(int(sys.argv[1]) if len(sys.argv) > 1 else 60)
