"""The inference-only mark that every operator's output carries."""
from __future__ import annotations

import torch


class _NoBackward(torch.autograd.Function):
    """Marks the output as produced by an inference-only op: backward raises."""

    @staticmethod
    def forward(ctx, out, *inputs):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("mtlflashattn_b200: backward is not supported (inference-only)")


def _guard_grad(out, *inputs):
    if torch.is_grad_enabled():
        for t in inputs:
            if torch.is_tensor(t) and t.requires_grad:
                return _NoBackward.apply(out, *[x for x in inputs if torch.is_tensor(x)])
    return out
