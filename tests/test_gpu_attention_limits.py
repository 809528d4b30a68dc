"""Where the attention operators could go wrong quietly: rounding that hides in a small cloud or adds up in a long one,
strides that only the C interface can pass, overflow in places that no result depends on, casts of modules."""
import ctypes
import math

import pytest
import torch

from attention_helpers import BF16, U, attention, check, check_attention, ends_of
from test_gpu_attention import TYPES, attention_case, draw

pytestmark = pytest.mark.gpu


# ---- row sums of the gradients ---------------------------------------------------------------------
def few_keys_reference(q, k, v, g, scale):
    """Plain 64-bit gradients of one cloud and their bounds with row sums (delta) from unrounded probabilities: no term
    for the rounding of the bf16 output."""
    d = q.shape[2]
    group = q.shape[1] // k.shape[1]
    r = {n: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for n, t in (("dq", q), ("dk", k))}
    off = {n: torch.zeros_like(t) for n, t in r.items()}
    for h in range(q.shape[1]):
        Q, K, V, G = q[:, h].double(), k[:, h // group].double(), v[:, h // group].double(), g[:, h].double()
        s = Q @ K.t() * scale
        p = torch.softmax(s, 1)
        dp = G @ V.t()
        delta = (p * dp).sum(1, keepdim=True)
        ds = p * (dp - delta)
        # a logit: d products and a few roundings; a probability: two such errors in its exponent and the rounding of the exponential
        # and of the row's lse; dp and delta: sums of d and of the keys' terms
        rel = 2 * ((d + 8) * U * ((Q.abs() @ K.abs().t()) * abs(scale) + s.abs().amax(1, keepdim=True) + 1)).amax(1, keepdim=True) + (len(K) + 8) * U
        mass = G.abs() @ V.abs().t()
        mass = mass + (p * mass).sum(1, keepdim=True)
        ds_off = p * mass * (rel + (d + len(K) + 8) * U) + p * BF16 * (dp - delta).abs()  # e is rounded to bf16 for the last products
        r["dq"][:, h] = scale * ds @ K
        r["dk"][:, h // group] += scale * ds.t() @ Q
        more = (group * len(Q) + len(K) + 8) * U * (ds.abs() + ds_off)
        off["dq"][:, h] = abs(scale) * ((ds_off + more) @ K.abs())
        off["dk"][:, h // group] += abs(scale) * ((ds_off + more).t() @ Q.abs())
    return r, {n: (1 + 4 * U + BF16) * t + BF16 * r[n].abs() + 1e-30 for n, t in off.items()}


@pytest.mark.parametrize("size", [64, 128, 36, 200], ids=["tiles64", "tiles128", "rows36", "rows200"])
def test_gradients_of_a_small_cloud_do_not_depend_on_the_clouds_beside_it(size):
    """Two keys with nearly the same values: dp - delta is 2^-8 of its terms, and a delta from the rounded output would be most of it."""
    from pccnn_lib_b200 import ops
    lengths, scale = ([3, 300], [2, 5000]), size ** -0.5
    q, k, v, qe, ke, g = attention_case(lengths, (4, 2), size, torch.bfloat16, seed=5)
    v[1] = (v[0].float() * (1 + 2.0 ** -7)).to(torch.bfloat16)
    out, lse = ops.cross_attention(q, k, v, qe, ke)
    beside = ops.cross_attention_grads(q, k, v, qe, ke, out, lse, g)
    alone = ops.cross_attention_grads(q[:3], k[:2], v[:2], qe[:1], ke[:1], out[:3].contiguous(), lse[:, :3].contiguous(), g[:3])
    ops.check_status()
    want, bound = few_keys_reference(q[:3], k[:2], v[:2], g[:3], scale)
    for name, x, y, rows in (("dq", alone[0], beside[0], 3), ("dk", alone[1], beside[1], 2), ("dv", alone[2], beside[2], 2)):
        if name in want:
            check(x, want[name], bound[name], name + " alone")
            check(y[:rows], want[name], bound[name], name + " beside a large cloud")
        assert torch.equal(x, y[:rows]), name
