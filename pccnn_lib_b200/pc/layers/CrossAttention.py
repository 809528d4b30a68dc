import math

import torch

from ...op_wrappers import ComputeCrossAttention
from .LayerNorm import LayerNorm
from .RotaryPositions import RotaryPositions


class CrossAttention(torch.nn.Module):
    """Residual attention of the points of one point cloud batch to those of another, cloud by cloud (no counterpart in
    the reference): a decoder level that reads a coarser level, latents that read a scene, one query that pools a cloud.

    forward(pc_in, pc_out, in_features, out_features, cloud_ends=None) takes the features [N, p_in_features] of pc_in and
    [M, p_out_features] of pc_out and returns the new features of pc_out, and also the end offsets (in, out) of the clouds
    when none were passed in.  Both inputs are normalised, projected to heads (p_num_heads of p_head_size for the queries,
    p_num_kv_heads for keys and values), turned by their coordinates, attended, projected back and added.  Parameters are
    cast to the type of the features; float32 and bfloat16 are supported."""

    def __init__(self, p_dims, p_in_features, p_out_features, p_num_heads, p_head_size, p_num_kv_heads=None,
                 p_wavelengths=(0.1, 10.0)):
        super(CrossAttention, self).__init__()
        self.num_heads_, self.head_size_ = p_num_heads, p_head_size
        self.num_kv_heads_ = p_num_heads if p_num_kv_heads is None else p_num_kv_heads
        if self.num_kv_heads_ < 1 or p_num_heads % self.num_kv_heads_:
            raise RuntimeError("%d query heads cannot share %d key heads" % (p_num_heads, self.num_kv_heads_))
        self.norm_in_, self.norm_out_ = LayerNorm(p_in_features), LayerNorm(p_out_features)
        self.positions_ = RotaryPositions(p_dims, p_head_size, p_wavelengths)
        self.query_weights_ = torch.nn.Parameter(torch.empty(p_out_features, p_num_heads * p_head_size))
        self.key_value_weights_ = torch.nn.Parameter(torch.empty(p_in_features, 2 * self.num_kv_heads_ * p_head_size))
        self.out_weights_ = torch.nn.Parameter(torch.empty(p_num_heads * p_head_size, p_out_features))
        self.reset_parameters()

    def reset_parameters(self):
        for weights in (self.query_weights_, self.key_value_weights_, self.out_weights_):
            weights.data.normal_(0.0, math.sqrt(1.0 / weights.shape[0]))

    def forward(self, p_pc_in, p_pc_out, p_in_features, p_out_features, p_cloud_ends=None):
        ends = p_cloud_ends
        if ends is None:
            clouds = max(p_pc_in.batch_size_host(), p_pc_out.batch_size_host())
            ends = (p_pc_in.get_batch_ends(clouds), p_pc_out.get_batch_ends(clouds))
        dtype, n, m = p_out_features.dtype, p_in_features.shape[0], p_out_features.shape[0]
        queries = torch.matmul(self.norm_out_(p_out_features), self.query_weights_.to(dtype))
        queries = self.positions_(queries.view(m, self.num_heads_, self.head_size_), p_pc_out.pts_)
        keys_values = torch.matmul(self.norm_in_(p_in_features), self.key_value_weights_.to(p_in_features.dtype))
        keys_values = keys_values.view(n, 2, self.num_kv_heads_, self.head_size_)
        keys = self.positions_(keys_values[:, 0], p_pc_in.pts_)
        heads = ComputeCrossAttention.apply(queries, keys, keys_values[:, 1], ends[1], ends[0])
        out = p_out_features + torch.matmul(heads.view(m, self.num_heads_ * self.head_size_), self.out_weights_.to(dtype))
        return (out, ends) if p_cloud_ends is None else out
