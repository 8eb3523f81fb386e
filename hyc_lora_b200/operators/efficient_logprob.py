"""Token log probabilities with entropy and alternatives, and the language-model loss made of them.

The host models take their loss by eager ops from an fp32 copy of the shifted logits (reference: models/modeling_llama.py);
here the logits are read in their own dtype, two floats per row are kept, and the gradient is written once in the logits'
dtype."""
import torch

from .. import rowops


class TokenLogprobFunc(torch.autograd.Function):
    """``(logprob, entropy, top_logprob, top_index)`` of :func:`rowops.token_logprobs`, None for what was not asked for."""

    @staticmethod
    def forward(ctx, logits, targets, ignore_index, entropy, top):
        out = rowops.token_logprobs(logits, targets, ignore_index=ignore_index, entropy=entropy, top=top)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        if out.top_index is not None:
            ctx.mark_non_differentiable(out.top_index)
        ctx.save_for_backward(logits, targets, out.stats, out.entropy, out.top_index)
        return out.logprob, out.entropy, out.top_logprob, out.top_index

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_logprob, d_entropy, d_top, _d_index):
        logits, targets, stats, entropy, top_index = ctx.saved_tensors
        if d_logprob is None and d_entropy is None and d_top is None:
            return (None,) * 5
        grad = rowops.token_logprobs_bwd(logits, stats, targets, d_logprob, ignore_index=ctx.ignore_index, entropy=entropy,
                                         d_entropy=d_entropy, top_index=top_index, d_top=d_top)
        return (grad,) + (None,) * 4


class EfficientMemoryTokenLogprob(torch.nn.Module):
    """``forward(logits, targets)`` -> :class:`rowops.TokenLogprobs`-like tuple ``(logprob, entropy, top_logprob, top_index)``,
    differentiable in the first three; ``entropy`` and ``top`` say what is made."""

    def __init__(self, ignore_index: int = -100, entropy: bool = False, top: int = 0):
        super().__init__()
        self.ignore_index, self.entropy, self.top = ignore_index, entropy, top

    def forward(self, logits, targets=None):
        return TokenLogprobFunc.apply(logits, targets, self.ignore_index, self.entropy, self.top)

    def extra_repr(self):
        return f"ignore_index={self.ignore_index}, entropy={self.entropy}, top={self.top}"


def token_cross_entropy(logits, targets, ignore_index: int = -100, reduction: str = "mean"):
    """``F.cross_entropy(logits.float(), targets)`` over the last dimension without the fp32 copy.  ``reduction`` is "mean" (over
    the rows that have a target; NaN where none has, as there), "sum" or "none"."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"unknown reduction {reduction!r}")
    nll = -TokenLogprobFunc.apply(logits, targets, ignore_index, False, 0)[0]
    if reduction == "none":
        return nll
    return nll.sum() if reduction == "sum" else nll.sum() / (targets != ignore_index).sum()
