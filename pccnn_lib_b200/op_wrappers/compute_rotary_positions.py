import torch

from .. import ops


class ComputeRotaryPositions(torch.autograd.Function):
    """Rotary positions from point coordinates with gradients for features and points (no counterpart in the reference).
    backward returns gradients in the positional order of forward's inputs: (features, pts, None, None); frequencies have
    none, and backward refuses ones that require it."""

    @staticmethod
    def forward(ctx, p_features, p_pts, p_frequencies, p_axis_pairs):
        # only the points' gradient reads the features
        ctx.save_for_backward(p_features if ctx.needs_input_grad[1] else None, p_pts, p_frequencies)
        ctx.axis_pairs_ = p_axis_pairs
        return ops.rotary_positions(p_features, p_pts, p_frequencies, p_axis_pairs)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, p_grads):
        if ctx.needs_input_grad[2]:
            raise RuntimeError("rotary positions have no gradient for their frequencies: pass them without requires_grad")
        features, pts, frequencies = ctx.saved_tensors
        feat_grads, pt_grads = ops.rotary_positions_grads(features, pts, frequencies, ctx.axis_pairs_, p_grads,
                                                          with_pts=ctx.needs_input_grad[1])
        return feat_grads, pt_grads, None, None
