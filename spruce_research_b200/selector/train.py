"""Teaching a gate on the GPU: a layer's own attention weight of key blocks, distilled into the gate's scores.

The reference trains its gate on stored teacher weights (selector/train.py:274 `train_document`, selector/loss.py:15 `kl_loss`).
Here the teacher is formed from the layer's post-RoPE Q and K (``native.block_mass``), cut to each row's heaviest blocks, and the
loss and its gradient by the scores are one kernel each; the projections' gradients are plain matrix products.

    python -m spruce_research_b200.selector.train     # a gate taught on one synthetic layer
"""
from __future__ import annotations

import torch

from .. import native
from .gate import FlatGate
from .loss import teacher_top_blocks, topk_distill_loss


def layer_teacher(query: torch.Tensor, key: torch.Tensor, top: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The teacher of one layer from its post-RoPE Q [B, Hq, T, D] and K [B, Hkv, T, D]: ids and logits [B, Hkv, qb, top]."""
    return teacher_top_blocks(native.block_mass(query, key), top)


def gate_training_scores(gate: FlatGate, q_feat: torch.Tensor, k_feat: torch.Tensor) -> torch.Tensor:
    """``FlatGate.forward``'s scores [L, G, qb, kb], recorded by autograd for ``Wq`` and ``Wk``."""
    gate._check_prototypes(q_feat, single=False)
    gate._check_prototypes(k_feat, single=False)
    if q_feat.shape[3] != k_feat.shape[3]:
        raise ValueError("query and key features must have the same number of prototypes")
    L, G, qb, P, _ = q_feat.shape
    kb = k_feat.shape[2]
    q = torch.einsum("lgqpd,lde->lgqpe", q_feat.float(), gate.Wq).reshape(L, G, qb * P, -1)
    k = torch.einsum("lgkpd,lde->lgkpe", k_feat.float(), gate.Wk).reshape(L, G, kb * P, -1)
    s = (q @ k.transpose(-1, -2)) * gate.proj_dim ** -0.5
    return s if P == 1 else s.view(L, G, qb, P, kb, P).amax((3, 5))


def gate_loss(gate: FlatGate, q_feat: torch.Tensor, k_feat: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, *,
              temperature: float = 1.0) -> torch.Tensor:
    """Mean distillation loss of the gate's rows: q_feat [L, G, qb, P, d], k_feat [L, G, qb, P, d], ids and teacher [L, G, qb, K].

    Row i scores the key blocks up to its own.  The teacher gets no gradient.
    """
    L, G, qb = q_feat.shape[:3]
    if k_feat.shape[2] != qb:
        raise ValueError(f"a causal gate scores as many key blocks as query blocks, got {k_feat.shape[2]} and {qb}")
    scores = gate_training_scores(gate, q_feat, k_feat)
    visible = torch.arange(1, qb + 1, device=scores.device, dtype=torch.int32).expand(L, G, qb)
    return topk_distill_loss(scores, ids, teacher, visible=visible, temperature=temperature).mean()


def main(tokens: int = 8192, steps: int = 50, top: int = 16) -> list:
    """Teach a random gate one synthetic layer (28 query / 4 KV heads); prints and returns the losses."""
    from ..synthetic import LayerShape, make_layer_inputs
    from ..teacher.chunked_extract import pool_selector_features

    q, k, _ = make_layer_inputs(LayerShape(1, 28, 4, tokens, 128), torch.bfloat16, seed=3)
    q, k = q.cuda(), k.cuda()
    ids, teacher = layer_teacher(q, k, top)
    q_feat, k_feat = pool_selector_features(q, k, 1)
    gate = FlatGate(1, 128).cuda()
    opt = torch.optim.Adam(gate.parameters(), lr=1e-3)
    losses = []
    for i in range(steps):
        loss = gate_loss(gate, q_feat, k_feat, ids, teacher)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if i % 10 == 0 or i + 1 == steps:
            print(f"step {i}: loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    main()
