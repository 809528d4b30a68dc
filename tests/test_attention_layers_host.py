"""Module casts of the attention layers (no GPU)."""
import copy

import torch


def test_frequencies_of_the_rotary_layer_survive_casts_of_the_module():
    from pccnn_lib_b200.pc import CrossAttention, RotaryPositions
    plain = RotaryPositions(3, 64, (0.1, 10.0))
    want = plain.frequencies_.clone()
    for cast in (lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double().bfloat16().float(),
                 lambda m: copy.deepcopy(m).bfloat16()):
        layer = cast(RotaryPositions(3, 64, (0.1, 10.0)))
        assert layer.frequencies_.dtype == torch.float32 and torch.equal(layer.frequencies_, want)
    inside = CrossAttention(3, 8, 8, 4, 64).bfloat16()
    assert torch.equal(inside.positions_.frequencies_, want)
    assert inside.query_weights_.dtype == torch.bfloat16 and inside.norm_in_.weights_.dtype == torch.bfloat16
    assert "frequencies_" in plain.state_dict() and list(plain.state_dict()) == list(inside.positions_.state_dict())
    other = RotaryPositions(3, 64, (0.2, 20.0)).bfloat16()
    other.load_state_dict(plain.state_dict())
    assert torch.equal(other.frequencies_, want)
    assert RotaryPositions(3, 64).to("meta").bfloat16().frequencies_.device.type == "meta"
