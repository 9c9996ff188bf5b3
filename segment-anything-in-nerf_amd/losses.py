"""Losses with the reference's names (nerfstudio/model_components/losses.py:46-143)."""
from __future__ import annotations

import torch

from . import ops


def ray_samples_to_sdist(ray_samples) -> torch.Tensor:
    return ray_samples.spacing_bins


def interlevel_loss(weights_list, ray_samples_list) -> torch.Tensor:
    c = ray_samples_to_sdist(ray_samples_list[-1]).detach()
    w = weights_list[-1][..., 0].detach()
    loss = 0.0
    for ray_samples, weights in zip(ray_samples_list[:-1], weights_list[:-1]):
        loss = loss + ops.interlevel_loss(weights[..., 0], ray_samples_to_sdist(ray_samples), c, w)
    return loss


def distortion_loss(weights_list, ray_samples_list) -> torch.Tensor:
    return ops.distortion_loss(weights_list[-1][..., 0], ray_samples_to_sdist(ray_samples_list[-1]))


class MSELoss(torch.nn.Module):
    """nn.MSELoss() (nerfacto.py:226: `self.rgb_loss = MSELoss()`), one HIP launch per direction on the GPU."""

    def forward(self, target: torch.Tensor, pred: torch.Tensor) -> torch.Tensor:
        # the reference calls rgb_loss(image, outputs["rgb"]); MSE is symmetric, the gradient goes to whichever needs it
        if pred.requires_grad or not target.requires_grad:
            return ops.mse_loss(pred, target)
        return ops.mse_loss(target, pred)


class TopLogitsDistillLoss(torch.nn.Module):
    """weight * T^2 KL(teacher || student) from the teacher's top logits (`ops.top_logits`), mean over the rows that have a target.
    with_rest: the mass of the logits that the teacher's list leaves out is one class of its own; otherwise the teacher's
    probabilities are those of its list alone.  The teacher's temperature must be this one where `with_rest` is on."""

    def __init__(self, temperature: float = 1.0, weight: float = 1.0, with_rest: bool = True):
        super().__init__()
        self.temperature, self.weight, self.with_rest = temperature, weight, with_rest

    def forward(self, student: torch.Tensor, teacher) -> torch.Tensor:
        ids, logits, rest = teacher
        return ops.top_logits_distill_loss(student, ids, logits, rest=rest if self.with_rest else None, temperature=self.temperature,
                                           weight=self.weight)
