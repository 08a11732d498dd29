"""Differentiable fronts of the operators for categorical states: classes looked up in a table on the way into a network, and the softmax
cross entropy over classes on the way out (the counterpart of ppgn_simple.loss_func_bce and ppgn_vlb.loss_func_kld where a state has more
than two values).  The reference's states are binary; nothing in it corresponds."""
import torch

from . import ops


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = weight.shape[0], scale
        return ops.embedding_fwd(weight, ids, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        return ops.embedding_wgrad(g.contiguous(), ids, ctx.rows, ctx.scale), None, None


def embedding(weight, ids, scale=1.0):
    """scale * weight[ids], differentiable with respect to weight [V, D] (float32 or bfloat16); an id outside [0, V) gives zeros and no
    gradient."""
    return _Embedding.apply(weight.contiguous(), ids.contiguous(), float(scale))


class _ClassLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, row_weight, denom, grad):
        # needs_input_grad says which inputs require one, also where none are recorded
        loss, _, dx, dweight = ops.loss_ce(x, weight, target, row_weight, denom, want_grad=grad and any(ctx.needs_input_grad[:2]))
        ctx.save_for_backward(dx, dweight)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        dx, dweight = ctx.saved_tensors
        return (_times(dx, g) if ctx.needs_input_grad[0] else None, _times(dweight, g) if ctx.needs_input_grad[1] else None, None, None, None, None)


def _times(t, g):
    """t * g with the float32 scalar g as it is: a product in bfloat16 would round g, too"""
    return t * g if t.dtype is torch.float32 else (t.float() * g).to(t.dtype)


def loss_func_ce(x, weight, target, row_weight=None, denom=None):
    """Softmax cross entropy of the classes' rows weight [V, D] against the last hidden layer x [..., D] (float32 scalar, differentiable
    with respect to x and weight): ops.loss_ce over the flattened positions; target [...] int64, outside [0, V): no class.  The gradients are
    computed with the loss, and not at all under torch.no_grad() or inference_mode.  row_weight [...] and denom are constants: a row_weight that
    requires a gradient is refused where gradients are recorded."""
    if row_weight is not None and row_weight.requires_grad and torch.is_grad_enabled():
        raise ValueError("row_weight: requires a gradient, which the class loss does not give; detach it")
    d = x.shape[-1]
    return _ClassLoss.apply(x.reshape(-1, d).contiguous(), weight.contiguous(), target.reshape(-1).contiguous(),
                            None if row_weight is None else row_weight.reshape(-1).contiguous(), denom, torch.is_grad_enabled())
