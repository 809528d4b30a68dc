import math

import torch

from ...op_wrappers import ComputeRotaryPositions


class RotaryPositions(torch.nn.Module):
    """Rotary positions of point features [N, heads, size] from the points' coordinates (no counterpart in the reference).

    Every axis gets the same number of feature pairs, size // (2 * dims); their wavelengths run geometrically from
    p_wavelengths[0] to p_wavelengths[1], in the unit of the coordinates.  Features left over are not turned.  The
    frequencies stay float32 when the module is cast: an angle at a far coordinate is many turns of a rounded one."""

    def __init__(self, p_dims, p_head_size, p_wavelengths=(0.1, 10.0)):
        super(RotaryPositions, self).__init__()
        pairs = p_head_size // (2 * p_dims)
        if pairs < 1:
            raise RuntimeError("a head of %d features has no pair for each of %d axes" % (p_head_size, p_dims))
        low, high = float(p_wavelengths[0]), float(p_wavelengths[1])
        if not 0.0 < low <= high:
            raise RuntimeError("p_wavelengths must be two ascending positive lengths")
        self.axis_pairs_ = [pairs] * p_dims
        steps = torch.arange(pairs, dtype=torch.float64) / max(pairs - 1, 1)
        frequencies = 2.0 * math.pi / (low * (high / low) ** steps)
        self.register_buffer('frequencies_', frequencies.to(torch.float32).repeat(p_dims))

    def _apply(self, p_fn, *p_args, **p_kwargs):
        frequencies = self.frequencies_
        super(RotaryPositions, self)._apply(p_fn, *p_args, **p_kwargs)
        if self.frequencies_.dtype != frequencies.dtype:  # a cast (and perhaps a move): the move alone
            self.frequencies_ = frequencies.to(self.frequencies_.device)
        return self

    def forward(self, p_features, p_pts):
        return ComputeRotaryPositions.apply(p_features, p_pts, self.frequencies_.float(), self.axis_pairs_)
