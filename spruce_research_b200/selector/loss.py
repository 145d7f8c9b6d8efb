"""The gate's training loss: distillation of a teacher's top entries into rows of scores, on the GPU.

The reference trains its gate against the teacher's attention weight of key blocks (selector/loss.py:15 `kl_loss`).  Here the
teacher is ``native.block_mass`` cut to its heaviest blocks, and the loss with its gradient are the kernels of
csrc/distill.cu.  The same loss serves a vocabulary's rows.
"""
from __future__ import annotations

import torch

from .. import native


class _TopkDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, ids, teacher, visible, temperature, status):
        loss, stats = native.topk_distill_forward(scores, ids, teacher, visible=visible, temperature=temperature,
                                                  status=status)
        ctx.save_for_backward(scores, ids, teacher, stats, visible)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        scores, ids, teacher, stats, visible = ctx.saved_tensors
        grad = native.topk_distill_backward(scores, ids, teacher, stats, grad_loss.float(), visible=visible,
                                            temperature=ctx.temperature)
        return grad, None, None, None, None, None


def topk_distill_loss(scores: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, *,
                      visible: torch.Tensor | None = None, temperature: float = 1.0,
                      status: torch.Tensor | None = None) -> torch.Tensor:
    """Losses float32 [...] of rows of scores [..., n] (see :func:`native.topk_distill`), recorded by autograd for the scores.

    The teacher gets no gradient.  A second backward through the gradient is refused.
    """
    return _TopkDistill.apply(scores, ids, teacher.detach(), visible, float(temperature), status)


def teacher_top_blocks(mass: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The heaviest ``k`` blocks of each row of ``native.block_mass`` [..., qb, qb]: ``(ids, logits)`` [..., qb, k].

    ids are int32, -1 where a row has fewer blocks with any weight; logits are the weights' logs, so that their softmax at
    temperature 1 is the weight within the top k.
    """
    if k < 1:
        raise ValueError(f"k must be positive, got {k}")
    best, ids = mass.topk(min(k, mass.shape[-1]), dim=-1)
    gone = ~(best > 0)
    return ids.masked_fill(gone, -1).int(), best.log().masked_fill(gone, 0.0)
