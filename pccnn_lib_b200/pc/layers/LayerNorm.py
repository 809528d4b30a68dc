import torch

from ...op_wrappers import ComputeLayerNorm


class LayerNorm(torch.nn.Module):
    """Layer norm over the channels of point features [N, C] (no counterpart in the reference).  Parameters ``weights_``
    and ``bias_`` are float32; features are float32 or bfloat16 and keep their type."""

    def __init__(self, p_num_features, p_eps=1e-5):
        super(LayerNorm, self).__init__()
        self.eps_ = p_eps
        self.weights_ = torch.nn.Parameter(torch.ones(p_num_features))
        self.bias_ = torch.nn.Parameter(torch.zeros(p_num_features))

    def forward(self, p_features):
        return ComputeLayerNorm.apply(p_features, self.weights_.float(), self.bias_.float(), self.eps_)
