"""Dropout whose mask is regenerated in backward from a seed instead of being
stored (reference: operators/efficient_dropout.py).  The reference's drivers
always build it with ``p = 0`` (train_gsm8k.py:540-541), where it is the
identity; for ``p > 0`` the mask comes from a seeded device generator.

``EfficientMemoryCounterDropout`` draws its mask inside the kernel from a counter-based generator instead: no random tensor in
either direction, an optional residual in the same launch, and a state on the device that a recorded graph moves on."""
import torch

from .. import rowops


class EfficientMemoryDropoutFunc(torch.autograd.Function):
    @staticmethod
    def _mask(x, p, seed):
        gen = torch.Generator(device=x.device)
        gen.manual_seed(int(seed))
        return torch.rand(x.shape, device=x.device, generator=gen) > p

    @staticmethod
    def forward(ctx, x, p, seed):
        ctx.p, ctx.seed = p, seed
        if p == 0.0:
            return x.clone()
        return torch.where(EfficientMemoryDropoutFunc._mask(x, p, seed), x / (1 - p), torch.zeros_like(x))

    @staticmethod
    def backward(ctx, grad_output):
        if ctx.p == 0.0:
            return grad_output, None, None
        keep = EfficientMemoryDropoutFunc._mask(grad_output, ctx.p, ctx.seed)
        return torch.where(keep, grad_output / (1 - ctx.p), torch.zeros_like(grad_output)), None, None


class EfficientMemoryDropout(torch.nn.Module):
    def __init__(self, p: float = 0.5):
        super().__init__()
        self.p = p
        self.seed = 0

    def forward(self, x):
        if not self.training or self.p == 0.0:
            return x
        self.seed += 1
        return EfficientMemoryDropoutFunc.apply(x, self.p, self.seed)


def new_rng_state(seed=None, device=None) -> torch.Tensor:
    """int64 [2] = (seed, next call number), the state a counter-based module draws its calls from.  Without a seed one is
    taken from torch's default CPU generator, so ``torch.manual_seed`` makes a run repeatable."""
    if seed is None:
        seed = int(torch.randint(0, 2 ** 62, (1,)).item())
    return torch.tensor([int(seed), 0], dtype=torch.int64, device=device)


class CounterDropoutFunc(torch.autograd.Function):
    """``residual + dropout(x)`` with the mask of ``rng`` (seed, call); the mask is drawn again in backward, nothing but
    ``rng`` is kept.  The residual's gradient is the arriving one."""

    @staticmethod
    def forward(ctx, x, residual, p, rng):
        ctx.p = p
        ctx.save_for_backward(rng)
        return rowops.dropout(x, p, rng, residual=residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        rng, = ctx.saved_tensors
        dx = rowops.dropout(grad_output, ctx.p, rng) if ctx.needs_input_grad[0] else None
        return dx, grad_output if ctx.needs_input_grad[1] else None, None, None


class EfficientMemoryCounterDropout(torch.nn.Module):
    """Dropout from a counter-based generator, with an optional residual added in the same kernel.

    ``forward(x, residual=None, rng=None)``; the residual has x's shape and dtype, in training and in evaluation.  The state
    (seed and call number) is a buffer on the device: it moves with the module, is saved with it, and a step recorded into a
    CUDA graph draws a new mask at every replay.  Copies of a module draw the same masks as the original; give ranks that
    should differ seeds of their own.  (Under torch's DistributedDataParallel that takes ``broadcast_buffers=False``: by
    default it copies rank 0's buffers, this state among them, to all ranks in front of every forward pass.
    ``hyc_lora_b200.ddp`` exchanges gradients only.)  A forward pass that is run again by activation checkpointing has to see
    its first mask: take ``rng = module.take()`` outside the checkpointed function and hand it to ``forward``."""

    def __init__(self, p: float = 0.5, seed=None, device=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability has to be between 0 and 1, got {p}")
        self.p = p
        self.register_buffer("rng_state", new_rng_state(seed, device))

    def take(self) -> torch.Tensor:
        return rowops.rng_take(self.rng_state)

    def forward(self, x, residual=None, rng=None):
        if not self.training or self.p == 0.0:
            if residual is None:
                return x
            rowops.check_like("residual", residual, x)         # the same calls as with dropout
            return residual + x
        return CounterDropoutFunc.apply(x, residual, self.p, self.take() if rng is None else rng)

    def extra_repr(self):
        return f"p={self.p}"
