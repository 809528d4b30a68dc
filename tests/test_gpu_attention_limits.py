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


# ---- layer norm ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("channels", [1, 7, 20, 33, 60, 100, 120])
def test_layer_norm_gradients_of_large_constant_rows_are_finite(channels, dtype):
    """mean * rstd overflows, but every x - mean is zero: the normalised row is zero and the gradient is that of its mean alone."""
    from pccnn_lib_b200 import ops
    value = 2.0 ** 121  # up to 127 of them add up to an exact 32-bit number
    x = draw((9, channels), 1, dtype)
    x[2], x[5] = value, -value
    w, b, g = 1 + draw((channels,), 2, scale=0.3), draw((channels,), 3), draw((9, channels), 4, dtype)
    out, mean, rstd = ops.layer_norm(x, w, b)
    assert mean[2] == value and mean[5] == -value and bool(torch.isinf(mean[2] * rstd[2]))
    assert bool(torch.isfinite(out).all())
    dx, dw, db = ops.layer_norm_grads(x, w, mean, rstd, g)
    gw = (g.double() * w.double())[[2, 5]]
    want = (gw - gw.mean(1, keepdim=True)) / math.sqrt(1e-5)
    size = (gw.abs() + gw.abs().mean(1, keepdim=True)) / math.sqrt(1e-5)
    check(dx[[2, 5]], want, (channels + 16) * U * size + (BF16 if dtype == torch.bfloat16 else 2 * U) * want.abs() + 1e-30, "dx")
    rest = [0, 1, 3, 4, 6, 7, 8]
    for got, other in zip((dx[rest], dw), ops.layer_norm_grads(x[rest], w, mean[rest], rstd[rest], g[rest])):
        # the two rows add exact zeros to the weights' gradient; its terms (a normalised value is at most sqrt(channels)) may be added in
        # another order
        check(got, other.double(), 34 * U * math.sqrt(channels) * g[rest].double().abs().sum(0) if got.dim() == 1 else 0 * other.double(), "other rows")


# ---- layers ----------------------------------------------------------------------------------------
def test_a_layer_cast_to_bf16_turns_by_the_same_angles():
    from pccnn_lib_b200.pc import RotaryPositions
    x, pts = draw((40, 4, 64), 1, torch.bfloat16), draw((40, 3), 2, scale=500.0)
    layer = RotaryPositions(3, 64, (0.1, 10.0)).cuda()
    want = layer(x, pts)
    assert torch.equal(layer.bfloat16()(x, pts), want)
    assert torch.equal(RotaryPositions(3, 64, (0.1, 10.0)).to("cuda", torch.bfloat16)(x, pts), want)


# ---- wrappers ----------------------------------------------------------------------------------------------
def test_a_gradient_that_no_operator_computes_is_refused_instead_of_left_out():
    from pccnn_lib_b200.op_wrappers import ComputeCrossAttention, ComputeLayerNorm, ComputeRotaryPositions
    x, pts, freq = draw((20, 2, 32), 1).requires_grad_(), draw((20, 3), 2), torch.exp(draw((15,), 3)).requires_grad_()
    out = ComputeRotaryPositions.apply(x, pts, freq, [5, 5, 5])
    with pytest.raises(RuntimeError, match="frequencies"):
        out.backward(torch.ones_like(out))
    q, k, v, qe, ke, g = attention_case(([20], [30]), (2, 2), 32, torch.float32)
    out = ComputeCrossAttention.apply(q.requires_grad_(), k, v, qe, ke, torch.tensor(0.3, requires_grad=True))
    with pytest.raises(RuntimeError, match="scale"):
        out.backward(g)
    f, w = draw((20, 32), 1).requires_grad_(), draw((32,), 2)
    out = ComputeLayerNorm.apply(f, w, w, torch.tensor(1e-5, requires_grad=True))
    with pytest.raises(RuntimeError, match="eps"):
        out.backward(torch.ones_like(out))
    with torch.no_grad():  # nothing to differentiate, nothing to refuse
        ComputeRotaryPositions.apply(x, pts, freq, [5, 5, 5])


# ---- strides that the C interface allows -------------------------------------------------------------
def strided(t, how):
    """(storage, address, strides) of a layout that torch itself cannot pass on, and the dense tensor it stands for."""
    rows, heads, size = t.shape
    e = t.element_size()
    if how == "rows reversed":
        return t, t.data_ptr() + (rows - 1) * heads * size * e, (-heads * size, size), t.flip(0)
    if how == "heads reversed":
        return t, t.data_ptr() + (heads - 1) * size * e, (heads * size, -size), t.flip(1)
    if how == "one head for all":
        return t, t.data_ptr(), (heads * size, 0), t[:, :1].expand(rows, heads, size)
    return t, t.data_ptr(), (0, size), t[:1].expand(rows, heads, size)  # one row for all


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("how", ["rows reversed", "heads reversed", "one head for all", "one row for all"])
@pytest.mark.parametrize("which", ["queries", "keys", "values", "grads"])
def test_attention_takes_zero_and_negative_strides_through_the_c_interface(which, how, dtype):
    from pccnn_lib_b200 import _capi, ops
    lib, lengths = _capi.lib, ([300, 40], [260, 200])  # large enough for tiles
    q, k, v, qe, ke, g = attention_case(lengths, (4, 4), 64, dtype, seed=7)
    tensors = {"queries": q, "keys": k, "values": v, "grads": g}
    passed = {n: (t, t.data_ptr(), (256, 64), t) for n, t in tensors.items()}
    passed[which] = strided(tensors[which], how)
    dense = [passed[n][3] for n in ("queries", "keys", "values", "grads")]
    m, n = q.shape[0], k.shape[0]
    shape = (m, n, 2, 4, 4, 64, int(dtype == torch.bfloat16))
    pair = lambda s: (ctypes.c_int64 * 2)(*s)  # noqa: E731
    inputs = [x for name in ("queries", "keys", "values") for x in (passed[name][1], pair(passed[name][2]))]
    inputs += [qe.data_ptr(), ke.data_ptr(), 0.125]
    out, lse = torch.empty_like(q), torch.empty((4, m), device="cuda")
    grads = [torch.empty_like(t) for t in (q, k, v)]
    stream = torch.cuda.current_stream().cuda_stream
    ws = torch.empty(lib.pccnn_cross_attention_workspace_bytes(*shape), dtype=torch.uint8, device="cuda")
    _capi.check(lib.pccnn_cross_attention(*shape, *inputs, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws.numel(), stream), "forward")
    ws = torch.empty(lib.pccnn_cross_attention_grads_workspace_bytes(*shape), dtype=torch.uint8, device="cuda")
    _capi.check(lib.pccnn_cross_attention_grads(*shape, *inputs, out.data_ptr(), lse.data_ptr(), passed["grads"][1], pair(passed["grads"][2]),
                                                *[t.data_ptr() for t in grads], ws.data_ptr(), ws.numel(), stream), "gradients")
    ops.check_status()
    check_attention([out, lse], attention(*dense[:3], *lengths, 0.125, dense[3]), grads)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("how", ["rows reversed", "heads reversed", "one head for all", "one row for all"])
def test_rotary_positions_take_zero_and_negative_strides_through_the_c_interface(how, dtype):
    from pccnn_lib_b200 import _capi, ops
    x, g, pts = draw((50, 4, 32), 1, dtype), draw((50, 4, 32), 2, dtype), draw((50, 3), 3)
    freq, pairs = torch.exp(draw((15,), 4)), (ctypes.c_int32 * 3)(5, 5, 5)
    _, px, sx, dense_x = strided(x, how)
    _, pg, sg, dense_g = strided(g, how)
    out, dx, dp = torch.empty_like(x), torch.empty_like(x), torch.empty_like(pts)
    bf16, stream = int(dtype == torch.bfloat16), torch.cuda.current_stream().cuda_stream
    _capi.check(_capi.lib.pccnn_rotary_positions(50, 4, 32, px, *sx, bf16, 3, pts.data_ptr(), freq.data_ptr(), pairs, out.data_ptr(), stream), "forward")
    _capi.check(_capi.lib.pccnn_rotary_positions_grads(50, 4, 32, px, *sx, bf16, 3, pts.data_ptr(), freq.data_ptr(), pairs, pg, *sg, dx.data_ptr(),
                                                       dp.data_ptr(), stream), "gradients")
    assert torch.equal(out, ops.rotary_positions(dense_x.contiguous(), pts, freq, [5, 5, 5]))
    want = ops.rotary_positions_grads(dense_x.contiguous(), pts, freq, [5, 5, 5], dense_g.contiguous())
    assert torch.equal(dx, want[0]) and torch.equal(dp, want[1])


# ---- splits of the keys' gradient ----------------------------------------------------------------------
@pytest.mark.parametrize("queries,heads", [(1000, (8, 1)), (1000, (8, 2)), (3000, (8, 1)), (600, (4, 1)), (2500, (3, 3)), (70, (32, 1)), (500, (48, 2))], ids=str)
def test_every_split_of_the_keys_gradients_has_queries_of_its_own(queries, heads):
    """One cloud: the parts in the workspace, one per split, are all written and none of them is only zeros."""
    from pccnn_lib_b200 import _capi, ops
    lib, keys = _capi.lib, 300
    q, k, v, qe, ke, g = attention_case(([queries], [keys]), heads, 64, torch.bfloat16, seed=3)
    out, lse = ops.cross_attention(q, k, v, qe, ke)
    shape = (queries, keys, 1, heads[0], heads[1], 64, 1)
    need, count = lib.pccnn_cross_attention_grads_workspace_bytes(*shape), keys * heads[1] * 64
    ws = torch.full((need // 4,), float("nan"), device="cuda")
    pair = lambda t: (ctypes.c_int64 * 2)(*t.stride()[:2])  # noqa: E731
    grads = [torch.empty_like(t) for t in (q, k, v)]
    _capi.check(lib.pccnn_cross_attention_grads(
        *shape, q.data_ptr(), pair(q), k.data_ptr(), pair(k), v.data_ptr(), pair(v), qe.data_ptr(), ke.data_ptr(), 0.125, out.data_ptr(), lse.data_ptr(),
        g.data_ptr(), pair(g), *[t.data_ptr() for t in grads], ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream), "gradients")
    ops.check_status()
    check_attention([out, lse], attention(q, k, v, [queries], [keys], 0.125, g), grads)
    delta = (queries * heads[0] * 4 + 256 + 255) // 256 * 256  # the row sums lie in front of the parts
    parts = ws[delta // 4:]
    parts = parts[:len(parts) // count * count].view(-1, count)
    written = ~torch.isnan(parts).any(1)
    splits = int(written.sum())
    assert splits % 2 == 0 and bool(written[:splits].all())  # dK's parts, then dV's
    assert splits <= 2 or bool((parts[:splits] != 0).any(1).all()), (parts[:splits] != 0).any(1).tolist()
    assert need <= delta + splits * count * 4 + 4096  # nothing is asked for that no split uses


# ---- long clouds -----------------------------------------------------------------------------------------
# The tensor cores truncate when they add to an accumulator: up to 2^-23 of it for every 16 rows.  Emptied every 65536 rows, that
# stays below (65536 / 16) 2^-23 = 2^-11 whatever the length; the sums of the emptied parts are rounded to nearest.
LONG_DRIFT = 2.0 ** -11
# The probabilities' roundings to bf16 (2^-8 of each at most) are independent and of mean zero: 2^-8 sqrt(sum p^2) / sum p of a sum, which is
# 2^-8 e^(s^2 / 2) / sqrt(n) for logits of spread s, here below 1.5: 7e-6 for three million.  Fourteen of them, with the
# 32-bit roundings of logits and sums (below 1e-5).
LONG_SPREAD = 1e-4


def half_step(x):
    """Half the distance of bf16 numbers at x."""
    return 2.0 ** (math.floor(math.log2(abs(x))) - 8)


@pytest.mark.parametrize("size", [64, 128])
def test_bf16_outputs_of_a_cloud_of_three_million_keys_do_not_drift(size):
    """All values of a feature are the same, so the output is that value whatever the probabilities are."""
    from pccnn_lib_b200 import ops
    n, m, heads = 3000000, 9600, 8  # enough blocks that the keys are not split
    q, k = draw((m, heads, size), 1, torch.bfloat16), draw((n, 1, size), 2, torch.bfloat16)
    v = torch.ones((n, 1, size), dtype=torch.bfloat16, device="cuda")
    value = 1.9921875  # 255 / 128: half a step of bf16 is 2^-8 of 2
    v[:, :, 1::2] = -value
    v[:, :, 0::2] = value
    out, lse = ops.cross_attention(q, k, v, ends_of([m]), ends_of([n]))
    ops.check_status()
    bound = half_step(value) + value * (LONG_DRIFT + LONG_SPREAD)
    assert float((out[..., 0::2].double() - value).abs().max()) <= bound
    assert float((out[..., 1::2].double() + value).abs().max()) <= bound


def test_bf16_value_gradients_of_a_cloud_of_three_million_queries_do_not_drift():
    from pccnn_lib_b200 import ops
    n, m, size = 49056, 3000000, 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    q, k, v = draw((m, 1, size), 1, torch.bfloat16, 0.5), draw((n, 1, size), 2, torch.bfloat16), draw((n, 1, size), 3, torch.bfloat16)
    g = torch.full((m, 1, size), 1.3359375, dtype=torch.bfloat16, device="cuda")
    qe, ke = ends_of([m]), ends_of([n])
    out, lse = ops.cross_attention(q, k, v, qe, ke)
    dv = ops.cross_attention_grads(q, k, v, qe, ke, out, lse, g)[2]
    ops.check_status()
    some = torch.arange(0, n, 1531, device="cuda")
    total = torch.zeros(len(some), dtype=torch.float64, device="cuda")
    for a in range(0, m, 250000):  # lse is a 32-bit result, tested elsewhere: off by some 2^-22
        logits = q[a:a + 250000, 0].double() @ k[some, 0].double().t() / math.sqrt(size)
        total += torch.exp(logits - lse[0, a:a + 250000].double()[:, None]).sum(0)
    want = (1.3359375 * total)[:, None].expand(-1, size)
    off = torch.tensor([half_step(float(x)) for x in want[:, 0]], device="cuda", dtype=torch.float64)[:, None]
    check(dv[some, 0], want, off + want * (LONG_DRIFT + LONG_SPREAD), "dv")


@pytest.mark.parametrize("size", [64, 128])
def test_bf16_rounds_of_a_long_cloud_fade_as_the_maximum_grows(size):
    """Logits that grow by 12 along 300000 keys, whose first values are positive and last ones negative: the output and the queries'
    gradient tell how much each part weighs."""
    from pccnn_lib_b200 import ops
    n, m, heads, scale = 300000, 9600, 8, size ** -0.5
    q, k = draw((m, heads, size), 1, torch.bfloat16, 0.1), draw((n, 1, size), 2, torch.bfloat16, 0.1)
    q[..., 0] = 1 / scale
    k[:, 0, 0] = torch.linspace(0, 12, n, device="cuda").to(torch.bfloat16)
    v, g = torch.full((n, 1, size), 1.3359375, dtype=torch.bfloat16, device="cuda"), torch.zeros_like(q)
    v[n - 20000:], g[..., 0] = -1.3359375, 1.0
    qe, ke = ends_of([m]), ends_of([n])
    out, lse = ops.cross_attention(q, k, v, qe, ke)
    dq = ops.cross_attention_grads(q, k, v, qe, ke, out, lse, g)[0]
    ops.check_status()
    Q, K, V = q[::1200].double(), k[:, 0].double(), v[:, 0, 0].double()
    s = Q @ K.t() * scale
    p = torch.softmax(s, -1)
    # 25000 keys weigh 1 / e of the largest or more: the probabilities' roundings add up to 2^-8 * 3 / sqrt(25000) = 7e-5 of the sums;
    # fourteen of them.  A logit of up to 12 is summed in 32 bits: 100 U of a probability.
    spread = 1e-3 + 200 * U
    want = (p * V).sum(-1)
    check(out[::1200], want[..., None].expand(-1, -1, size), (BF16 * want.abs() + 1.3359375 * (LONG_DRIFT + spread))[..., None].expand(-1, -1, size), "out")
    ds = p * (V - want[..., None])
    # delta comes from the rounded output
    bound = scale * ((ds.abs() * (LONG_DRIFT + spread) + p * (BF16 * want.abs() + 1.3359375 * (LONG_DRIFT + spread))[..., None]) @ K.abs())
    check(dq[::1200], scale * ds @ K, bound + BF16 * ((scale * ds @ K).abs() + bound), "dq")


def test_rotary_positions_keep_their_features_only_for_the_points_gradient():
    from pccnn_lib_b200 import ops
    from pccnn_lib_b200.op_wrappers import ComputeRotaryPositions
    x, pts, freq, g = draw((50, 3, 32), 1).requires_grad_(), draw((50, 3), 2), torch.exp(draw((15,), 3)), draw((50, 3, 32), 4)
    out = ComputeRotaryPositions.apply(x, pts, freq, [5, 5, 5])
    assert all(t is None or t.shape != x.shape for t in out.grad_fn.saved_tensors)
    out.backward(g)
    dx, none = ops.rotary_positions_grads(None, pts, freq, [5, 5, 5], g, with_pts=False)
    assert none is None and torch.equal(x.grad, dx) and torch.equal(dx, ops.rotary_positions_grads(x.detach(), pts, freq, [5, 5, 5], g)[0])
    with pytest.raises(RuntimeError, match="features"):
        ops.rotary_positions_grads(None, pts, freq, [5, 5, 5], g)
    with pytest.raises(RuntimeError, match="in_grads"):
        ops.rotary_positions_grads(x.detach(), pts, freq, [5, 5, 5], g[:, :2])
    wide = draw((50, 3, 48), 5)[:, :, 8:40]  # a view as the gradient
    assert torch.equal(ops.rotary_positions_grads(None, pts, freq, [5, 5, 5], wide, with_pts=False)[0],
                       ops.rotary_positions_grads(x.detach(), pts, freq, [5, 5, 5], wide)[0])


# ---- 32-bit accuracy -------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,size", [((4, 2), 64), ((4, 4), 32), ((3, 3), 128), ((2, 1), 36), ((2, 2), 200)], ids=str)
@pytest.mark.parametrize("lengths", [([700, 300], [900, 1400]), ([1, 1], [3000, 5000]), ([130, 9], [20000, 64])], ids=["tiles", "rows", "split"])
def test_32_bit_results_are_right_to_22_bits_in_norm(lengths, heads, size):
    """The worst-case bounds of the other tests are some 1e-4 wide for heads of 64; what the three planes of a 32-bit feature and the
    emptied accumulators are for shows in the norm of the error.  Two planes would leave 2^-17 of every product (1e-5 in the gradients),
    one accumulator for 1000 keys a bias of 64 truncations (4e-6).  Logits of spread 1.5 reach about 7 and are summed in 32 bits:
    their rounding is 2^-24 * 7, which two of them bring into a probability; sums and the last rounding add a few 2^-24: 2^-19 in all."""
    from pccnn_lib_b200 import ops
    q, k, v, qe, ke, g = attention_case(lengths, heads, size, torch.float32, seed=30)
    want = attention(q, k, v, *lengths, size ** -0.5, g)
    out, lse = ops.cross_attention(q, k, v, qe, ke)
    grads = ops.cross_attention_grads(q, k, v, qe, ke, out, lse, g)
    ops.check_status()
    for name, got in zip(("out", "dq", "dk", "dv"), [out] + grads):
        error = float((got.double() - want[name]).norm() / want[name].norm())
        assert error <= 2.0 ** -19, (name, error)


# ---- infinities ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths,size", [(([300, 20], [500, 40]), 64), (([2, 1], [700, 90]), 64), (([300, 20], [500, 40]), 36)],
                         ids=["tiles", "few", "rows"])
def test_an_infinity_reaches_only_the_results_that_depend_on_it(lengths, size, dtype):
    """A query's infinity stays in the row of its head, a value's in its feature of its cloud; what they reach is the formula's
    infinity or NaN (the route decides), everything else is as right as ever."""
    from pccnn_lib_b200 import ops
    q, k, v, qe, ke, g = attention_case(lengths, (4, 2), size, dtype)
    scale, (m, n) = size ** -0.5, (lengths[0][0], lengths[1][0])
    clean = attention(q, k, v, *lengths, scale)

    def check_rest(got, reached):
        out, lse = got
        hit = reached.to(out.device)
        check(torch.where(hit, 0, out.double()), clean["out"].masked_fill(hit, 0), clean["out_bound"], "out")
        assert not bool(torch.isfinite(out[hit]).any())
    for bad in (float("inf"), -float("inf")):
        spoiled = q.clone()
        spoiled[1, 2, 5] = bad
        got = ops.cross_attention(spoiled, k, v, qe, ke)
        reached = torch.zeros(q.shape, dtype=torch.bool)
        reached[1, 2] = True
        check_rest(got, reached)  # among random keys some logit is +infinity, so the formula itself gives NaN
        assert bool(torch.isnan(got[0][1, 2]).all())
        spoiled = v.clone()
        spoiled[7, 1, 9] = bad
        reached = torch.zeros(q.shape, dtype=torch.bool)
        reached[:m, 2:, 9] = True
        check_rest(ops.cross_attention(q, k, spoiled, qe, ke), reached)
    ops.check_status()
