import torch

from .. import ops


class ComputeCrossAttention(torch.autograd.Function):
    """Cross attention between packed clouds with gradients (no counterpart in the reference).  backward returns gradients
    in the positional order of forward's inputs: (queries, keys, values, None, None, None); the scale has none, and backward
    refuses one that requires it."""

    @staticmethod
    def forward(ctx, p_queries, p_keys, p_values, p_query_ends, p_key_ends, p_scale=None):
        out, lse = ops.cross_attention(p_queries, p_keys, p_values, p_query_ends, p_key_ends, p_scale)
        ctx.save_for_backward(p_queries, p_keys, p_values, p_query_ends, p_key_ends, out, lse)
        ctx.scale_ = p_scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, p_grads):
        if any(ctx.needs_input_grad[5:]):
            raise RuntimeError("cross attention has no gradient for its scale: pass a number")
        query_grads, key_grads, value_grads = ops.cross_attention_grads(*ctx.saved_tensors, p_grads, ctx.scale_)
        return query_grads, key_grads, value_grads, None, None, None
