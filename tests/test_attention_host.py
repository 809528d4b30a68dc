"""Refusals and workspace queries of the attention entry points that end before any CUDA call (no GPU here)."""
import ctypes

import pytest
import torch


def strides(*s):
    return (ctypes.c_int64 * 2)(*s)


def test_attention_entry_points_refuse_bad_arguments_before_any_launch():
    from pccnn_lib_b200 import _capi
    lib, s = _capi.lib, strides(64, 32)

    def forward(m=4, n=4, clouds=1, heads=2, kv_heads=2, size=32, q=16, ws=16, nbytes=1 << 30, ends=16):
        return lib.pccnn_cross_attention(m, n, clouds, heads, kv_heads, size, 0, q, s, 16, s, 16, s, ends, 16, 1.0, 16, 16, ws, nbytes, None)
    for bad, word in ((dict(m=-1), "rows"), (dict(n=1 << 31), "rows"), (dict(heads=3), "share"), (dict(kv_heads=0), "share"), (dict(heads=2048), "share"),
                      (dict(size=257), "head size"), (dict(size=0), "head size"), (dict(q=None), "null"), (dict(ends=None), "null"),
                      (dict(ws=None), "workspace")):
        assert forward(**bad) != 0 and word in _capi.last_error(), bad
    assert forward(m=0, q=None, ws=None) == 0  # nothing to do
    assert lib.pccnn_layer_norm(4, 0, 16, 1, 0, 16, 16, 1e-5, 16, 16, 16, None) == 1 and "shape" in _capi.last_error()
    assert lib.pccnn_layer_norm(4, 8, 16, 7, 0, 16, 16, 1e-5, 16, 16, 16, None) == 1 and "stride" in _capi.last_error()
    assert lib.pccnn_layer_norm(4, 8, None, 8, 0, 16, 16, 1e-5, 16, 16, 16, None) == 1 and "null" in _capi.last_error()
    assert lib.pccnn_layer_norm(4, 8, 16, 8, 0, 16, 16, -1.0, 16, 16, 16, None) == 1 and "eps" in _capi.last_error()
    assert lib.pccnn_layer_norm_grads(4, 8, 16, 8, 0, 16, 16, 16, 16, 8, 16, 16, 16, None, 0, None) != 0 and "workspace" in _capi.last_error()
    pairs = (ctypes.c_int32 * 7)(*[1] * 7)
    for axes, size, word in ((7, 32, "axes"), (0, 32, "axes"), (3, 4, "do not fit"), (1, 1, "pairs"), (1, 2000, "shape")):
        assert lib.pccnn_rotary_positions(4, 2, size, 16, 64, 32, 0, axes, 16, 16, pairs, 16, None) == 1 and word in _capi.last_error()


def test_attention_workspaces_grow_with_the_splits_only():
    from pccnn_lib_b200 import _capi
    lib = _capi.lib
    # one query per cloud and many keys: the keys are split, the parts are kept in 32 bits
    assert lib.pccnn_cross_attention_workspace_bytes(16, 400000, 16, 8, 8, 64, 1) >= 2 * 16 * 8 * 64 * 4
    # more queries than the GPU has room for: no split
    assert lib.pccnn_cross_attention_workspace_bytes(100000, 100000, 4, 8, 8, 64, 1) <= 1 << 20
    for m, n in ((0, 10), (10, 0), (0, 0)):
        assert lib.pccnn_cross_attention_workspace_bytes(m, n, 1, 2, 2, 32, 0) >= 256
        assert lib.pccnn_cross_attention_grads_workspace_bytes(m, n, 1, 2, 2, 32, 0) >= 256
    assert lib.pccnn_layer_norm_grads_workspace_bytes(1000, 128) >= 2 * 128 * 4


def test_attention_operators_refuse_cpu_tensors():
    from pccnn_lib_b200 import ops
    x, e = torch.zeros(4, 2, 32), torch.tensor([4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.cross_attention(x, x, x, e, e)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.layer_norm(torch.zeros(4, 8), torch.ones(8), torch.zeros(8))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.rotary_positions(x, torch.zeros(4, 3), torch.ones(15), [5, 5, 5])


def test_layers_refuse_sizes_that_do_not_fit():
    from pccnn_lib_b200.pc import CrossAttention, RotaryPositions
    with pytest.raises(RuntimeError, match="share"):
        CrossAttention(3, 8, 8, 4, 32, p_num_kv_heads=3)
    with pytest.raises(RuntimeError, match="no pair"):
        RotaryPositions(3, 4)
    with pytest.raises(RuntimeError, match="ascending"):
        RotaryPositions(3, 32, (1.0, 0.5))
    layer = RotaryPositions(3, 32, (0.5, 8.0))
    assert layer.axis_pairs_ == [5, 5, 5] and layer.frequencies_.shape == (15,)
