"""LayerNorm with a compressed saved input (reference: operators/efficient_layernorm.py:203-405), and the layer norm of a
residual sum with dropout on the joining branch, uncompressed."""
import torch

from .. import rowops
from ._norm_common import make_norm
from .efficient_dropout import new_rng_state

EfficientMemoryLayerNormFunc, EfficientMemoryLayerNorm = make_norm(
    "ln", "EfficientMemoryLayerNormFunc", "EfficientMemoryLayerNorm",
    "LayerNorm whose saved input is compressed (reference: operators/efficient_layernorm.py:203-405).")


class DropoutAddLayerNormFunc(torch.autograd.Function):
    """``z = residual + dropout(x)`` and its layer norm; returns ``(y, z)``, z being None where it would be x itself.  Kept for
    backward: z (or x), two floats per row, and the two words that name the mask."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, p, rng):
        out = rowops.layer_norm(x, weight, bias, eps, residual=residual, p=p, rng=rng)
        ctx.p, ctx.param_dtype = p, bias.dtype if bias is not None else None
        ctx.set_materialize_grads(False)
        own_sum = residual is not None or p > 0.0
        ctx.save_for_backward(out.z if own_sum else x, weight, out.mean, out.rstd, rng if p > 0.0 else None)
        return out.y, out.z if own_sum else None

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dz):
        z, weight, mean, rstd, rng = ctx.saved_tensors
        need_x, need_residual, need_w, need_b = ctx.needs_input_grad[:4]
        if dy is None:                                    # only the sum went on
            if dz is None:
                return (None,) * 7
            dx = rowops.dropout(dz, ctx.p, rng) if need_x and ctx.p > 0.0 else dz
            return dx if need_x else None, dz if need_residual else None, None, None, None, None, None
        dx, dresidual, dw, db = rowops.layer_norm_bwd(dy, z, weight, mean, rstd, p=ctx.p, rng=rng, dz=dz, need_dweight=need_w,
                                                      need_dbias=need_b, param_dtype=ctx.param_dtype)
        return dx if need_x else None, dresidual if need_residual else None, dw, db, None, None, None


class EfficientMemoryDropoutAddLayerNorm(torch.nn.LayerNorm):
    """``LayerNorm(residual + dropout(x))`` in one kernel, with an uncompressed saved sum and the gradients of weight and
    bias (the compressing norm above gives none for its bias).

    ``forward(x, residual=None, rng=None)`` returns y, with ``return_sum=True`` ``(y, z)`` -- z being the sum in front of the
    norm, which a pre-norm block carries on.  The dropout's state and ``rng`` are those of
    :class:`~.efficient_dropout.EfficientMemoryCounterDropout`."""

    def __init__(self, normalized_shape, p: float = 0.0, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 *, seed=None, return_sum: bool = False, device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("only the last dimension can be normalised")
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability has to be between 0 and 1, got {p}")
        self.p, self.return_sum = p, return_sum
        if p > 0.0:
            self.register_buffer("rng_state", new_rng_state(seed, device))

    def take(self) -> torch.Tensor:
        return rowops.rng_take(self.rng_state)

    def forward(self, x, residual=None, rng=None):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"the last dimension has {x.shape[-1]} values, expected {self.normalized_shape[0]}")
        p = self.p if self.training else 0.0
        if p > 0.0 and rng is None:
            rng = self.take()
        y, z = DropoutAddLayerNormFunc.apply(x, residual, self.weight, self.bias, self.eps, p, rng if p > 0.0 else None)
        if not self.return_sum:
            return y
        return y, x if z is None else z

    def extra_repr(self):
        return f"{super().extra_repr()}, p={self.p}"
