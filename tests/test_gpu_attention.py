"""Layer norm, rotary positions and cross attention against plain forms in 64 bits."""
import math

import pytest
import torch

from attention_helpers import BF16, U, attention, check, check_attention, ends_of

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def draw(shape, seed, dtype=torch.float32, scale=1.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


# ---- layer norm ----------------------------------------------------------------------------------
def norm_reference(x, w, b, eps, g):
    """Plain 64-bit form and bounds: the sums of C terms are off by C U of their absolute values at most; what a row's
    mean and spread are off by enters the normalised value relative to the row's largest."""
    out_round = BF16 if x.dtype == torch.bfloat16 else 2 * U
    x, w, b, g = x.double(), w.double(), b.double(), g.double()
    c = x.shape[1]
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    hat = (x - mean) * rstd
    hat_off = ((c + 4) * U * x.abs().amax(1, keepdim=True) * rstd) * (2 + hat.abs()) + (c + 8) * U * hat.abs() + 1e-30
    out = hat * w + b
    r = {"out": out, "out_bound": hat_off * w.abs() + 4 * U * (hat * w).abs() + 2 * U * b.abs() + out_round * out.abs() + 1e-30}
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - hat * (gw * hat).mean(1, keepdim=True))
    size = gw.abs() + gw.abs().mean(1, keepdim=True) + hat.abs() * (gw * hat).abs().mean(1, keepdim=True)
    off = (c + 16) * U * size + hat_off * (gw * hat).abs().mean(1, keepdim=True) + hat.abs() * (gw.abs() * hat_off).mean(1, keepdim=True)
    off = off * rstd + dx.abs() * hat_off.amax(1, keepdim=True)
    r.update(dx=dx, dx_bound=off + out_round * dx.abs() + 1e-30)
    n = x.shape[0]
    r.update(dw=(g * hat).sum(0), dw_bound=((n + 8) * U * (g * hat).abs() + g.abs() * hat_off).sum(0) + 1e-30)
    r.update(db=g.sum(0), db_bound=(n + 8) * U * g.abs().sum(0) + 1e-30)
    return r


NORM_SHAPES = [(1, 1), (3, 1), (1, 7), (37, 64), (65, 31), (129, 33), (7, 100), (300, 128), (51, 130), (40, 256), (33, 257), (90, 511),
               (19, 512), (21, 1000), (21, 1001), (9, 1024), (5, 2048), (6, 4095), (6, 4096), (5, 4097), (4, 8192), (3, 9000), (5000, 48)]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=lambda s: "%dx%d" % s)
def test_layer_norm_and_its_gradients(shape, dtype):
    from pccnn_lib_b200 import ops
    n, c = shape
    x = (draw((n, c), 1) * (0.2 + 3 * torch.rand(n, 1, device="cuda")) + 0.7).to(dtype)
    w, b, g = 1 + draw((c,), 2, scale=0.3), draw((c,), 3, scale=0.3), draw((n, c), 4, dtype)
    want = norm_reference(x, w, b, 1e-5, g)
    out, mean, rstd = ops.layer_norm(x, w, b, 1e-5)
    check(out, want["out"], want["out_bound"], "out")
    for got, name in zip(ops.layer_norm_grads(x, w, mean, rstd, g), ("dx", "dw", "db")):
        check(got, want[name], want[name + "_bound"], name)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_layer_norm_reads_strided_and_unaligned_rows(dtype):
    from pccnn_lib_b200 import ops
    wide = draw((50, 300), 5, dtype)
    w, b = 1 + draw((128,), 2, scale=0.3), draw((128,), 3, scale=0.3)
    for x in (wide[:, 16:144], wide[:, 3:131], wide[::3, :128], wide[:, ::2][:, :128], wide.t()[:50, :].t()[:, :0].new_zeros((0, 128)),
              wide[0, :128].expand(9, 128)):
        g = draw(tuple(x.shape), 7, dtype)
        want = norm_reference(x, w, b, 1e-5, g)
        out, mean, rstd = ops.layer_norm(x, w, b, 1e-5)
        check(out, want["out"], want["out_bound"], "out")
        for got, name in zip(ops.layer_norm_grads(x, w, mean, rstd, g), ("dx", "dw", "db")):
            check(got, want[name], want[name + "_bound"], name)
        unaligned = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape).copy_(g)
        for got, other in zip(ops.layer_norm_grads(x, w, mean, rstd, unaligned), ops.layer_norm_grads(x, w, mean, rstd, g)):
            check(got, other.double(), 2 * (BF16 if dtype == torch.bfloat16 else 300 * U) * (other.double().abs() + other.double().abs().amax(-1, keepdim=True))
                  if other.numel() else other.double(), "unaligned")


@pytest.mark.parametrize("channels", [64, 100, 130])
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_layer_norm_with_weights_off_any_vector_boundary(channels, dtype):
    from pccnn_lib_b200 import ops
    x, g = draw((70, channels), 1, dtype), draw((70, channels), 2, dtype)
    for shift_w, shift_b in ((1, 0), (0, 1), (2, 3), (3, 2)):
        w, b = (1 + draw((channels + 4,), 3))[shift_w:shift_w + channels], draw((channels + 4,), 4)[shift_b:shift_b + channels]
        want = norm_reference(x, w, b, 1e-5, g)
        out, mean, rstd = ops.layer_norm(x, w, b, 1e-5)
        check(out, want["out"], want["out_bound"], "out")
        for got, name in zip(ops.layer_norm_grads(x, w, mean, rstd, g), ("dx", "dw", "db")):
            check(got, want[name], want[name + "_bound"], name)


def test_layer_norm_of_constant_rows_and_of_rows_with_infinities():
    from pccnn_lib_b200 import ops
    x = torch.full((4, 96), 3.25, device="cuda")
    x[1], x[2, 5], x[3, 7] = 0.0, float("inf"), float("nan")
    w, b = torch.ones(96, device="cuda"), draw((96,), 1)
    out, mean, rstd = ops.layer_norm(x, w, b, 1e-5)
    assert torch.equal(out[0], b) and torch.equal(out[1], b)  # the mean of equal values is that value here: 96 * 3.25 is exact
    assert bool(torch.isnan(out[2:]).all())
    g = draw((4, 96), 2)
    dx = ops.layer_norm_grads(x, w, mean, rstd, g)[0]
    assert bool(torch.isfinite(dx[:2]).all()) and bool(torch.isnan(dx[2:]).all())


def test_layer_norm_gradients_are_the_same_bits_on_every_run_and_stream():
    from pccnn_lib_b200 import ops
    x, w, g = draw((30001, 128), 1), 1 + draw((128,), 2), draw((30001, 128), 3)
    _, mean, rstd = ops.layer_norm(x, w, w)
    first = ops.layer_norm_grads(x, w, mean, rstd, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = ops.layer_norm_grads(x, w, mean, rstd, g)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


# ---- rotary positions ----------------------------------------------------------------------------
def rotary_reference(x, pts, freq, axis_pairs, g):
    out_round = BF16 if x.dtype == torch.bfloat16 else 2 * U
    x = x.double().requires_grad_()
    p = pts.double().requires_grad_()
    axis = torch.repeat_interleave(torch.arange(len(axis_pairs), device="cuda"), torch.tensor(axis_pairs, device="cuda"))
    angle = (p[:, axis] * freq.double())[:, None, :]
    turned = 2 * angle.shape[-1]
    a, b = x[..., 0:turned:2], x[..., 1:turned:2]
    ya, yb = a * torch.cos(angle) - b * torch.sin(angle), a * torch.sin(angle) + b * torch.cos(angle)
    out = torch.cat([torch.stack([ya, yb], -1).flatten(-2), x[..., turned:]], -1)
    dx, dp = torch.autograd.grad(out, (x, p), g.double(), allow_unused=True)
    dp = torch.zeros_like(p) if dp is None else dp

    def pair_size(t):  # |x0| + |x1| of the pair a feature belongs to
        t = t.detach().double().abs()
        s = t[..., 0:turned:2] + t[..., 1:turned:2]
        return torch.cat([torch.stack([s, s], -1).flatten(-2), 0 * t[..., turned:]], -1)
    # sine and cosine are off by 4 U (the angle's fraction of a turn rounded to 32 bits, and sincospi), two products and a sum
    r = {"out": out.detach(), "out_bound": 8 * U * pair_size(x) + out_round * out.detach().abs() + 1e-30,
         "dx": dx, "dx_bound": 8 * U * pair_size(g) + out_round * dx.abs() + 1e-30, "dp": dp.detach()}
    terms = (pair_size(g)[..., 0:turned:2] * pair_size(x)[..., 0:turned:2]).sum(1) * freq.double().abs()
    count = x.shape[1] * angle.shape[-1]
    r["dp_bound"] = torch.zeros_like(p.detach()).index_add_(1, axis, terms) * (count + 24) * U + 1e-30
    return r


ROTARY_CASES = [  # rows, heads, size, pairs per axis
    (1, 1, 2, [1]), (1, 1, 1, [0]), (5, 1, 7, [1, 1]), (61, 4, 32, [5, 5, 5]), (33, 3, 16, [2, 3, 1]), (100, 8, 64, [10, 10, 10]), (17, 2, 65, [32]),
    (40, 5, 24, [0, 4, 0, 8]), (12, 12, 128, [10, 11, 12, 13, 9, 8]), (3, 1, 1024, [512]), (7, 2, 1022, [100, 400]), (1000, 1, 8, [1, 1]),
    (9, 2, 96, [16, 16, 16])]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", ROTARY_CASES, ids=lambda c: "%dx%dx%d_%s" % (c[0], c[1], c[2], "_".join(map(str, c[3]))))
def test_rotary_positions_and_their_gradients(case, dtype):
    from pccnn_lib_b200 import ops
    n, h, d, pairs = case
    x, g = draw((n, h, d), 1, dtype), draw((n, h, d), 2, dtype)
    pts = draw((n, len(pairs)), 3, scale=50.0)
    freq = torch.exp(draw((sum(pairs),), 4))
    want = rotary_reference(x, pts, freq, pairs, g)
    check(ops.rotary_positions(x, pts, freq, pairs), want["out"], want["out_bound"], "out")
    dx, dp = ops.rotary_positions_grads(x, pts, freq, pairs, g)
    check(dx, want["dx"], want["dx_bound"], "dx")
    check(dp, want["dp"], want["dp_bound"], "dp")
    dx_alone, none = ops.rotary_positions_grads(x, pts, freq, pairs, g, with_pts=False)
    assert none is None and torch.equal(dx, dx_alone)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_rotary_positions_far_away_strided_and_with_infinities(dtype):
    from pccnn_lib_b200 import ops
    wide = draw((40, 3, 5, 80), 1, dtype)
    pts = draw((40, 3), 2, scale=3e6)  # a 32-bit product of coordinate and frequency would be wrong in every digit
    pts[0] = torch.tensor([0.0, -1e9, 2.0 ** 30], device="cuda")
    freq = torch.exp(draw((18,), 3))
    for x in (wide[:, 1, :, :48], wide[:, 1, :, 3:43], wide[:, 2, ::2, 8:72], wide[:, :, 0, :36]):
        g = draw(tuple(x.shape), 4, dtype)
        want = rotary_reference(x, pts, freq, [6, 6, 6], g)
        check(ops.rotary_positions(x, pts, freq, [6, 6, 6]), want["out"], want["out_bound"], "out")
        dx, dp = ops.rotary_positions_grads(x, pts, freq, [6, 6, 6], g)
        check(dx, want["dx"], want["dx_bound"], "dx")
        check(dp, want["dp"], want["dp_bound"], "dp")
    x = draw((4, 2, 40), 5, dtype)
    x[1, 0, 38], x[2, 1, 37] = float("inf"), float("nan")  # behind the last pair: passed, nothing else touched
    out = ops.rotary_positions(x, pts[:4], freq, [6, 6, 6])
    assert bool(torch.isinf(out[1, 0, 38])) and bool(torch.isnan(out[2, 1, 37])) and int(torch.isfinite(out).sum()) == out.numel() - 2
    empty = ops.rotary_positions(x[:0], pts[:0], freq, [6, 6, 6])
    assert empty.shape == (0, 2, 40)


# ---- cross attention -----------------------------------------------------------------------------
LENGTHS = {
    "single": ([1], [1]),
    "ragged": ([1, 7, 0, 130, 64], [300, 0, 5, 129, 1]),
    "pool": ([1, 1, 1], [3000, 1, 257]),
    "tiles": ([257, 128, 1, 31], [128, 127, 640, 65]),
    "long": ([520], [1500]),
    "few_keys": ([700, 3], [2, 9]),
}
HEADS = [(1, 1), (4, 4), (6, 2), (5, 1)]


def attention_case(lengths, heads, size, dtype, seed=0, behind=(0, 0), scale_q=1.5):
    q_lens, k_lens = lengths
    m, n = sum(q_lens) + behind[0], sum(k_lens) + behind[1]
    q, g = draw((m, heads[0], size), seed + 1, dtype, scale_q), draw((m, heads[0], size), seed + 4, dtype)
    k, v = draw((n, heads[1], size), seed + 2, dtype), draw((n, heads[1], size), seed + 3, dtype)
    return q, k, v, ends_of(q_lens), ends_of(k_lens), g


def run_and_check(q, k, v, qe, ke, g, lengths, scale=None):
    from pccnn_lib_b200 import ops
    want = attention(q, k, v, *lengths, 1 / math.sqrt(q.shape[2]) if scale is None else scale, g)
    got = ops.cross_attention(q, k, v, qe, ke, scale)
    check_attention(got, want)
    grads = ops.cross_attention_grads(q, k, v, qe, ke, *got, g, scale)
    ops.check_status()
    check_attention(got, want, grads)
    return got, grads


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [1, 5, 8, 16, 24, 32, 33, 40, 64, 65, 72, 80, 96, 104, 128, 129, 136, 200, 256])
def test_cross_attention_of_every_head_size(size, dtype):
    case = attention_case(LENGTHS["tiles"], (2, 1), size, dtype)
    run_and_check(*case, LENGTHS["tiles"])


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "%dof%d" % h)
@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("size", [32, 64, 128])
def test_cross_attention_of_ragged_clouds_and_shared_heads(size, lengths, heads, dtype):
    case = attention_case(LENGTHS[lengths], heads, size, dtype, seed=10)
    run_and_check(*case, LENGTHS[lengths])


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths", [([300, 40], [500, 300]), ([2, 1], [700, 90])], ids=["tiles", "rows"])
def test_rows_of_other_clouds_and_behind_the_last_never_reach_a_cloud(lengths, dtype):
    """NaN and infinities in the rows of the second cloud and behind it: the first cloud's results are unchanged, bit for bit."""
    from pccnn_lib_b200 import ops
    q, k, v, qe, ke, g = attention_case(lengths, (4, 2), 64, dtype, behind=(70, 90))
    clean = ops.cross_attention(q, k, v, qe, ke)
    clean_grads = ops.cross_attention_grads(q, k, v, qe, ke, *clean, g)
    check_attention(clean, attention(q, k, v, *lengths, 0.125, g), clean_grads)
    a, b = lengths[0][0], lengths[1][0]
    assert not bool(clean[0][sum(lengths[0]):].any()) and bool((clean[1][:, sum(lengths[0]):] == -float("inf")).all())
    assert not bool(clean_grads[0][sum(lengths[0]):].any()) and not bool(clean_grads[1][sum(lengths[1]):].any())
    for bad in (float("nan"), float("inf"), -float("inf")):
        for t, first in ((q, a), (g, a), (k, b), (v, b)):
            t[first:] = bad
        got = ops.cross_attention(q, k, v, qe, ke)
        grads = ops.cross_attention_grads(q, k, v, qe, ke, *got, g)
        assert torch.equal(got[0][:a], clean[0][:a]) and torch.equal(got[1][:, :a], clean[1][:, :a])
        for x, y, first in zip(grads, clean_grads, (a, b, b)):
            assert torch.equal(x[:first], y[:first])
        for x, last in ((got[0], sum(lengths[0])), (grads[0], sum(lengths[0])), (grads[1], sum(lengths[1])), (grads[2], sum(lengths[1]))):
            assert not bool(x[last:].any())


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_clouds_without_keys_queries_or_rows(dtype):
    from pccnn_lib_b200 import ops
    for lengths in (([5, 200], [0, 0]), ([0, 0], [5, 200]), ([0], [0]), ([], []), ([0, 3, 0], [4, 0, 9])):
        q, k, v, qe, ke, g = attention_case(lengths, (2, 2), 64, dtype, behind=(3, 2))
        got, grads = run_and_check(q, k, v, qe, ke, g, lengths)
        assert not bool(got[0].any()) and not any(bool(x.any()) for x in grads)
    q, k, v, qe, ke, g = attention_case(([4], [6]), (2, 2), 64, dtype)
    out, lse = ops.cross_attention(q[:0], k, v, qe * 0, ke)
    assert out.shape == (0, 2, 64) and lse.shape == (2, 0)
    dq, dk, dv = ops.cross_attention_grads(q[:0], k, v, qe * 0, ke, out, lse, g[:0])
    assert dq.numel() == 0 and not bool(dk.any()) and not bool(dv.any())
    out, lse = ops.cross_attention(q, k[:0], v[:0], qe, ke * 0)
    assert not bool(out.any())
    assert not bool(ops.cross_attention_grads(q, k[:0], v[:0], qe, ke * 0, out, lse, g)[0].any())


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_cross_attention_reads_views_in_place_and_unaligned_ones(dtype):
    lengths = LENGTHS["tiles"]
    m, n = sum(lengths[0]), sum(lengths[1])
    qe, ke, g = ends_of(lengths[0]), ends_of(lengths[1]), draw((m, 4, 64), 9, dtype)
    fused = draw((n, 2, 2, 64), 1, dtype)
    wide = draw((m, 4, 80), 2, dtype)
    run_and_check(wide[:, :, 8:72], fused[:, 0], fused[:, 1], qe, ke, g, lengths)
    run_and_check(wide[:, :, 3:67], fused[:, 0], fused[:, 1], qe, ke, g, lengths)  # rows start off any 16-byte boundary
    shuffled = draw((64, 4, m), 3, dtype).permute(2, 1, 0)
    run_and_check(shuffled, fused[:, 0], fused[:, 1], qe, ke, g[:1].expand(m, 4, 64), lengths)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("scale_q", [0.0, 20.0], ids=["flat", "peaked"])
def test_cross_attention_of_flat_and_peaked_rows_and_other_scales(scale_q, dtype):
    case = attention_case(LENGTHS["tiles"], (2, 2), 64, dtype, scale_q=scale_q)
    run_and_check(*case, LENGTHS["tiles"])
    run_and_check(*case, LENGTHS["tiles"], scale=0.03)
    run_and_check(*case, LENGTHS["tiles"], scale=-0.05)
    run_and_check(*case, LENGTHS["tiles"], scale=0.0)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [64, 104])
@pytest.mark.parametrize("lengths", [([40, 3, 5], [9000, 100, 700]), ([20, 0, 28], [3400, 3300, 3100]), ([300, 1], [5000, 0])],
                         ids=["one-large", "equal", "one-empty"])
def test_keys_split_between_blocks_for_clouds_of_all_sizes(lengths, size, dtype):
    """Few queries on many keys: a split goes by the mean cloud, so clouds have more, fewer or no splits."""
    run_and_check(*attention_case(lengths, (4, 2), size, dtype, behind=(3, 200)), lengths)


@pytest.mark.parametrize("heads", [(3, 3), (8, 8), (6, 2), (5, 1), (14, 2)], ids=str)
@pytest.mark.parametrize("size", [24, 32, 40, 64])
def test_single_queries_in_bf16_with_logits_from_products_of_16_keys(size, heads):
    """One query per cloud and key counts around 8 and 16, with one, two, three, four and five heads to a part of four columns."""
    keys = [0, 1, 7, 8, 9, 15, 16, 17, 31, 33, 255, 257, 1000]
    lengths = ([1] * len(keys), keys)
    run_and_check(*attention_case(lengths, heads, size, torch.bfloat16, behind=(2, 5)), lengths)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_logits_that_grow_along_the_keys(dtype):
    """Every block of keys raises the maximum, so all that was summed before has to fade."""
    lengths = ([140, 3], [900, 1000])
    q, k, v, qe, ke, g = attention_case(lengths, (2, 1), 64, dtype)
    ramp = torch.cat([torch.linspace(0, 40, 900, device="cuda"), torch.linspace(0, 60, 1000, device="cuda")])
    q[:, :, 0], k[:, 0, 0] = 8.0, ramp.to(dtype)  # the logit gains 8 * ramp / 8
    run_and_check(q, k, v, qe, ke, g, lengths)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_cross_attention_gradients_against_differences(dtype):
    """Along a direction, the gradients' product equals central differences of the plain 64-bit form."""
    from pccnn_lib_b200 import ops
    lengths = ([70, 33], [90, 150])
    q, k, v, qe, ke, g = attention_case(lengths, (4, 2), 32, dtype)
    out, lse = ops.cross_attention(q, k, v, qe, ke)
    grads = ops.cross_attention_grads(q, k, v, qe, ke, out, lse, g)
    scale, h = 1 / math.sqrt(32), 1e-5
    bounds = attention(q, k, v, *lengths, scale, g)
    for i, (name, grad) in enumerate(zip(("dq", "dk", "dv"), grads)):
        way = draw(tuple(grad.shape), 20 + i).double()
        loss = []
        for sign in (1, -1):
            moved = [t.double() + (sign * h * way if j == i else 0) for j, t in enumerate((q, k, v))]
            loss.append(float((attention(*moved, *lengths, scale)["out"] * g.double()).sum()))
        slope = (loss[0] - loss[1]) / (2 * h)
        bound = float((bounds[name + "_bound"] * way.abs()).sum())
        assert abs(float((grad.double() * way).sum()) - slope) <= bound + 1e-6 * max(1.0, abs(slope))


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_cross_attention_repeats_bit_for_bit_on_any_stream(dtype):
    from pccnn_lib_b200 import ops
    for lengths in (LENGTHS["tiles"], LENGTHS["pool"], ([2500], [40])):
        q, k, v, qe, ke, g = attention_case(lengths, (4, 2), 64, dtype)
        first = ops.cross_attention(q, k, v, qe, ke)
        first = list(first) + ops.cross_attention_grads(q, k, v, qe, ke, *first, g)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = ops.cross_attention(q, k, v, qe, ke)
            second = list(second) + ops.cross_attention_grads(q, k, v, qe, ke, *second, g)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths", ["tiles", "pool"])
def test_captured_calls_follow_new_inputs_and_lengths(lengths, dtype):
    """Two graphs of the same call, replayed in turn with other values and other cloud sizes in the same buffers."""
    from pccnn_lib_b200 import ops
    case = [t.clone() for t in attention_case(LENGTHS[lengths], (4, 2), 64, dtype)]
    q, k, v, qe, ke, g = case

    def step():
        out, lse = ops.cross_attention(q, k, v, qe, ke)
        return [out, lse] + ops.cross_attention_grads(q, k, v, qe, ke, out, lse, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    q_lens, k_lens = LENGTHS[lengths]
    for turn, other in enumerate(((q_lens, k_lens), (q_lens[::-1], k_lens[::-1]), ([sum(q_lens)] + [0] * (len(q_lens) - 1), k_lens))):
        fresh = attention_case(other, (4, 2), 64, dtype, seed=40 * turn)
        for kept, new in zip(case, fresh):
            kept.copy_(new)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = attention(q, k, v, *other, 0.125, g)
        for _, held in graphs:
            check_attention(held[:2], want, held[2:])


EDGES = [(1, 127), (127, 1), (128, 128), (129, 129), (255, 64), (256, 63), (257, 65), (7, 8), (8, 7), (9, 9), (31, 33), (32, 32), (33, 31), (64, 255),
         (65, 257), (63, 256), (3, 0), (0, 3), (130, 16), (16, 130)]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [24, 64, 120])
def test_clouds_that_end_at_and_around_the_borders_of_tiles(size, dtype):
    lengths = ([q for q, _ in EDGES], [k for _, k in EDGES])
    run_and_check(*attention_case(lengths, (4, 2), size, dtype, seed=70), lengths)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_thousands_of_tiny_clouds(dtype):
    gen = torch.Generator()
    gen.manual_seed(4)
    lengths = tuple(torch.randint(0, 5, (1500,), generator=gen).tolist() for _ in range(2))
    run_and_check(*attention_case(lengths, (2, 1), 32, dtype, seed=80), lengths)


@pytest.mark.parametrize("queries", [1, 300], ids=["rows", "tiles"])
def test_keys_beyond_32_bits_of_offset(queries):
    """The last cloud's keys lie behind 2^31 elements (and 2^32 bytes)."""
    from pccnn_lib_b200 import ops
    n, tail = (1 << 31) // (8 * 128) + 1000, 700
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    keys, values = (torch.randn((n, 8, 128), generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q, g = draw((queries + 1, 8, 128), 2, torch.bfloat16, 1.5), draw((queries + 1, 8, 128), 3, torch.bfloat16)
    qe, ke = ends_of([1, queries]), ends_of([n - tail, tail])
    out, lse = ops.cross_attention(q, keys, values, qe, ke)
    dq, dk, dv = ops.cross_attention_grads(q, keys, values, qe, ke, out, lse, g)
    ops.check_status()
    want = attention(q[1:], keys[-tail:], values[-tail:], [queries], [tail], 128 ** -0.5, g[1:])
    check_attention([out[1:], lse[:, 1:].contiguous()], want, [dq[1:], dk[-tail:], dv[-tail:]])


def test_norm_and_positions_beyond_32_bits_of_offset():
    from pccnn_lib_b200 import ops
    n = (1 << 31) // 128 + 64
    x = torch.zeros((n, 128), dtype=torch.bfloat16, device="cuda")
    tail, g = draw((64, 128), 1, torch.bfloat16), torch.zeros((n, 128), dtype=torch.bfloat16, device="cuda")
    x[-64:], g[-64:] = tail, draw((64, 128), 2, torch.bfloat16)
    w, b = 1 + draw((128,), 3, scale=0.3), draw((128,), 4)
    want = norm_reference(tail, w, b, 1e-5, g[-64:])
    out, mean, rstd = ops.layer_norm(x, w, b)
    check(out[-64:], want["out"], want["out_bound"], "out")
    dx, dw, db = ops.layer_norm_grads(x, w, mean, rstd, g)
    check(dx[-64:], want["dx"], want["dx_bound"], "dx")
    check(dw, want["dw"], want["dw_bound"], "dw")  # the other rows' gradients are zeros, exactly
    check(db, want["db"], want["db_bound"], "db")
    del out, dx
    pts, freq = torch.zeros((n, 3), device="cuda"), torch.exp(draw((15,), 5))
    pts[-64:] = draw((64, 3), 6, scale=20.0)
    want = rotary_reference(tail.view(64, 4, 32), pts[-64:], freq, [5, 5, 5], g[-64:].view(64, 4, 32))
    check(ops.rotary_positions(x.view(n, 4, 32), pts, freq, [5, 5, 5])[-64:], want["out"], want["out_bound"], "out")
    dx, dp = ops.rotary_positions_grads(x.view(n, 4, 32), pts, freq, [5, 5, 5], g.view(n, 4, 32))
    check(dx[-64:], want["dx"], want["dx_bound"], "dx")
    check(dp[-64:], want["dp"], want["dp_bound"], "dp")


class short_waits_and_a_silent_loader(object):
    """The loader issues nothing from its second tile on and the poll limit is lowered, so the waits of the other roles run
    out with no copy in flight."""

    def __enter__(self):
        from pccnn_lib_b200 import _capi
        _capi.check(_capi.lib.pccnn_gemm_set_test_hooks(4000, 1), "set_test_hooks")

    def __exit__(self, *exc):
        from pccnn_lib_b200 import _capi
        torch.cuda.synchronize()
        _capi.check(_capi.lib.pccnn_gemm_set_test_hooks(0, -1), "set_test_hooks")
        return False


@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_attention_reports_a_wait_that_ran_out_and_recovers(dtype, size):
    from pccnn_lib_b200 import ops
    lengths = ([500, 300], [900, 1100])
    q, k, v, qe, ke, g = attention_case(lengths, (4, 2), size, dtype)
    out, lse = ops.cross_attention(q, k, v, qe, ke)
    ops.check_status()
    with short_waits_and_a_silent_loader():
        ops.cross_attention(q, k, v, qe, ke)  # asynchronous: the call itself cannot know yet
        with pytest.raises(RuntimeError, match="cross attention .* gave up"):
            ops.check_status(synchronize=True)
    ops.check_status()  # the record was consumed
    if dtype == torch.bfloat16 or size <= 64:  # larger 32-bit heads take the kernels without tensor cores
        with short_waits_and_a_silent_loader():
            ops.cross_attention_grads(q, k, v, qe, ke, out, lse, g)
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="gave up"):
                ops.cross_attention(q, k, v, qe, ke)  # found by the next call
    run_and_check(q, k, v, qe, ke, g, lengths)


def test_the_first_call_of_a_process_can_be_a_captured_one():
    """In a fresh process, without a call in front of the capture: kernels and the pinned status word are set up inside."""
    import subprocess
    import sys
    from conftest import ROOT
    code = """
import sys; sys.path[:0] = [%r, %r]
import torch, test_gpu_attention as t
from pccnn_lib_b200 import ops
cases = [t.attention_case(t.LENGTHS["tiles"], (4, 2), 64, dtype) for dtype in t.TYPES]
x, w = torch.ones(9, 64, device="cuda"), torch.ones(64, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.layer_norm(x, w, w)
    held = [ops.cross_attention(*c[:5]) for c in cases]
    held = [h + ops.cross_attention_grads(*c[:5], *h, c[5]) for c, h in zip(cases, held)]
graph.replay()
torch.cuda.synchronize()
for (q, k, v, _, _, g), h in zip(cases, held):
    t.check_attention(h[:2], t.attention(q, k, v, *t.LENGTHS["tiles"], 0.125, g), h[2:])
ops.check_status()
print("captured")
""" % (ROOT, ROOT + "/tests")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-3000:]


def test_strides_of_single_rows_and_heads_mean_nothing():
    lengths = ([300], [400])
    q, k, v, qe, ke, g = attention_case(lengths, (1, 1), 64, torch.bfloat16)
    odd = [torch.as_strided(x, x.shape, (64, 3, 1)) for x in (q, k, v, g)]  # one head: any head stride
    run_and_check(*odd[:3], qe, ke, odd[3], lengths)
    one = ([1], [400])
    q, k, v, qe, ke, g = attention_case(one, (4, 4), 64, torch.bfloat16)
    run_and_check(torch.as_strided(q, q.shape, (5, 64, 1)), k, v, qe, ke, torch.as_strided(g, g.shape, (5, 64, 1)), one)


def test_attention_on_two_streams_at_once():
    from pccnn_lib_b200 import ops
    cases = [attention_case(LENGTHS["tiles"], (4, 2), 64, dtype, seed=90 + i) for i, dtype in enumerate(TYPES * 2)]
    want = [attention(q, k, v, *LENGTHS["tiles"], 0.125, g) for q, k, v, _, _, g in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    held = []
    for _ in range(5):
        for stream, (q, k, v, qe, ke, g) in zip(streams, cases):
            with torch.cuda.stream(stream):
                out, lse = ops.cross_attention(q, k, v, qe, ke)
                held.append((out, lse, ops.cross_attention_grads(q, k, v, qe, ke, out, lse, g)))
    torch.cuda.synchronize()
    ops.check_status()
    for i, (out, lse, grads) in enumerate(held):
        check_attention([out, lse], want[i % len(cases)], grads)


# ---- autograd and the layer ----------------------------------------------------------------------
def test_autograd_wrappers_return_the_operators_gradients():
    from pccnn_lib_b200 import ops
    from pccnn_lib_b200.op_wrappers import ComputeCrossAttention, ComputeLayerNorm, ComputeRotaryPositions
    x, w, b = (t.requires_grad_() for t in (draw((50, 96), 1), draw((96,), 2), draw((96,), 3)))
    g = draw((50, 96), 4)
    ComputeLayerNorm.apply(x, w, b).backward(g)
    _, mean, rstd = ops.layer_norm(x.detach(), w.detach(), b.detach())
    for t, want in zip((x, w, b), ops.layer_norm_grads(x.detach(), w.detach(), mean, rstd, g)):
        assert torch.equal(t.grad, want)
    x, pts = draw((50, 3, 32), 1).requires_grad_(), draw((50, 3), 2).requires_grad_()
    freq, g = torch.exp(draw((15,), 3)), draw((50, 3, 32), 4)
    ComputeRotaryPositions.apply(x, pts, freq, [5, 5, 5]).backward(g)
    for t, want in zip((x, pts), ops.rotary_positions_grads(x.detach(), pts.detach(), freq, [5, 5, 5], g)):
        assert torch.equal(t.grad, want)
    q, k, v, qe, ke, g = attention_case(LENGTHS["tiles"], (4, 2), 32, torch.float32)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    ComputeCrossAttention.apply(*leaves, qe, ke, 0.3).backward(g)
    plain = [t.detach() for t in leaves]
    out, lse = ops.cross_attention(*plain, qe, ke, 0.3)
    for t, want in zip(leaves, ops.cross_attention_grads(*plain, qe, ke, out, lse, g, 0.3)):
        assert torch.equal(t.grad, want)


def layer_reference(layer, pts_in, pts_out, f_in, f_out, lens_in, lens_out):
    """The layer in float64 torch operations, differentiable."""
    def norm(n, x):
        mean = x.mean(1, keepdim=True)
        return (x - mean) / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + n.eps_) * n.weights_.double() + n.bias_.double()

    def turn(x, pts):
        pairs = layer.positions_.axis_pairs_
        axis = torch.repeat_interleave(torch.arange(len(pairs), device="cuda"), torch.tensor(pairs, device="cuda"))
        angle = (pts[:, axis] * layer.positions_.frequencies_.double())[:, None, :]
        t = 2 * angle.shape[-1]
        a, b = x[..., 0:t:2], x[..., 1:t:2]
        return torch.cat([torch.stack([a * torch.cos(angle) - b * torch.sin(angle), a * torch.sin(angle) + b * torch.cos(angle)], -1).flatten(-2),
                          x[..., t:]], -1)
    h, hk, d = layer.num_heads_, layer.num_kv_heads_, layer.head_size_
    q = turn((norm(layer.norm_out_, f_out) @ layer.query_weights_.double()).view(-1, h, d), pts_out)
    kv = (norm(layer.norm_in_, f_in) @ layer.key_value_weights_.double()).view(-1, 2, hk, d)
    k, v = turn(kv[:, 0], pts_in), kv[:, 1]
    rows, a, b = [], 0, 0
    for lo, li in zip(lens_out, lens_in):
        heads = [torch.softmax(q[a:a + lo, i] @ k[b:b + li, i // (h // hk)].t() / math.sqrt(d), 1) @ v[b:b + li, i // (h // hk)] for i in range(h)]
        rows.append(torch.stack(heads, 1))
        a, b = a + lo, b + li
    return f_out + torch.cat(rows).reshape(-1, h * d) @ layer.out_weights_.double()


def make_layer_case(dtype):
    from pccnn_lib_b200.pc import CrossAttention, Pointcloud
    lens_in, lens_out = [200, 31, 90], [60, 140, 7]
    ids = lambda lens: torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(lens, device="cuda")).to(torch.int32)  # noqa: E731
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    pts = [torch.rand((sum(n), 3), generator=gen, device="cuda") for n in (lens_in, lens_out)]
    clouds = [Pointcloud(p, ids(n)) for p, n in zip(pts, (lens_in, lens_out))]
    torch.manual_seed(1)
    layer = CrossAttention(3, 48, 72, 4, 32, p_num_kv_heads=2).cuda()
    return layer, clouds, draw((sum(lens_in), 48), 5, dtype), draw((sum(lens_out), 72), 6, dtype), lens_in, lens_out


def test_cross_attention_layer_runs_norm_positions_and_attention_together():
    layer, clouds, f_in, f_out, lens_in, lens_out = make_layer_case(torch.float32)
    for c in clouds:
        c.pts_.requires_grad_()
    f_in.requires_grad_(), f_out.requires_grad_()
    out, ends = layer(clouds[0], clouds[1], f_in, f_out)
    again = layer(clouds[0], clouds[1], f_in, f_out, ends)
    assert torch.equal(out, again)
    g = draw(tuple(out.shape), 8)
    leaves = [f_in, f_out, clouds[0].pts_, clouds[1].pts_] + list(layer.parameters())
    got = torch.autograd.grad(out, leaves, g)
    wide = [t.detach().double().requires_grad_() for t in (f_in, f_out, clouds[0].pts_, clouds[1].pts_)]
    want = layer_reference(layer, wide[2], wide[3], wide[0], wide[1], lens_in, lens_out)
    # a chain of five operators on values of order one, sums of up to 200 terms: the framework's tolerance for convolutions
    assert float((out.detach().double() - want.detach()).abs().max()) <= 1e-4 * float(want.detach().abs().max())
    for x, y in zip(got, torch.autograd.grad(want, wide + list(layer.parameters()), g.double())):
        assert float((x.double() - y).abs().max()) <= 2e-4 * float(y.abs().max())


def test_cross_attention_layer_infers_in_bf16_and_trains_in_a_graph():
    layer, clouds, f_in, f_out, lens_in, lens_out = make_layer_case(torch.bfloat16)
    with torch.no_grad():
        out, ends = layer(clouds[0], clouds[1], f_in, f_out)
        want = layer_reference(layer, clouds[0].pts_.double(), clouds[1].pts_.double(), f_in.double(), f_out.double(), lens_in, lens_out)
    assert out.dtype == torch.bfloat16
    # six roundings to bf16 along the chain, each 2^-8 of values up to the largest, through projections of unit gain
    assert float((out.double() - want).abs().max()) <= 6 * BF16 * float(want.abs().max()) * 2
    out = layer(clouds[0], clouds[1], f_in, f_out, ends)
    grads = torch.autograd.grad(out, list(layer.parameters()), torch.ones_like(out))
    assert all(bool(torch.isfinite(x).all()) for x in grads)


def test_point_clouds_whose_rows_are_not_grouped_are_refused():
    from pccnn_lib_b200.pc import Pointcloud
    pts = torch.rand((4, 3), device="cuda")
    cloud = Pointcloud(pts, torch.tensor([0, 2, 2, 5], dtype=torch.int32, device="cuda"))
    assert cloud.get_batch_ends().tolist() == [1, 1, 3, 3, 3, 4]
    assert cloud.get_batch_ends(8).tolist() == [1, 1, 3, 3, 3, 4, 4, 4]
    with pytest.raises(RuntimeError, match="not grouped"):
        Pointcloud(pts, torch.tensor([0, 1, 0, 1], dtype=torch.int32, device="cuda")).get_batch_ends()


# ---- refusals ------------------------------------------------------------------------------------
def test_attention_operators_refuse_what_they_cannot_take():
    from pccnn_lib_b200 import ops
    q, k, v, qe, ke, g = attention_case(([4], [6]), (4, 2), 32, torch.float32)
    refused = [
        ((q.double(), k, v, qe, ke), "dtype"), ((q, k.bfloat16(), v, qe, ke), "dtype"), ((q.half(), k, v, qe, ke), "dtype"),
        ((q[0], k, v, qe, ke), "dimensions"), ((q, k[:, :, :16], v, qe, ke), "keys and values"), ((q, k, v[:3], qe, ke), "keys and values"),
        ((q[:, :3], k, v, qe, ke), "share"), ((q, k, v, qe.long(), ke), "dtype"), ((q, k, v, qe, ke.repeat(2)), "one entry per cloud"),
        ((q.cpu(), k, v, qe, ke), "CUDA tensor"), ((q, k, v, qe.cpu(), ke), "CUDA tensor"),
        ((q, k, v, qe - 10, ke), "decrease"), ((q, k, v, qe, ke + 1), "beyond"),
    ]
    for args, match in refused:
        with pytest.raises(RuntimeError, match=match):
            ops.cross_attention(*args)
    big = draw((2, 1, 257), 1)
    with pytest.raises(RuntimeError, match="head size"):
        ops.cross_attention(big, big, big, ends_of([2]), ends_of([2]))
    out, lse = ops.cross_attention(q, k, v, qe, ke)
    for bad in ((out[:3], lse, g), (out, lse[:, :3], g), (out, lse, g[:, :2]), (out, lse, g.bfloat16()), (out.bfloat16(), lse, g)):
        with pytest.raises(RuntimeError):
            ops.cross_attention_grads(q, k, v, qe, ke, *bad)
    x, w = draw((5, 8), 1), draw((8,), 2)
    for bad in ((x, w[:7], w), (x, w, w.bfloat16()), (x.half(), w, w), (x[0], w, w), (x[:, :0], w[:0], w[:0]), (x, w, w.cpu())):
        with pytest.raises(RuntimeError):
            ops.layer_norm(*bad)
    with pytest.raises(RuntimeError, match="negative"):
        ops.layer_norm(x, w, w, -1.0)
    pts, freq = draw((4, 3), 3), draw((15,), 4)
    for bad in ((q, pts, freq, [5, 5]), (q, pts, freq, [5, 5, 4]), (q, pts[:3], freq, [5, 5, 5]), (q, pts, draw((18,), 1), [6, 6, 6]),
                (q, draw((4, 7), 1), freq[:7], [1] * 7), (q, pts, freq, [-1, 8, 8]), (q, draw((4, 0), 1), freq[:0], [])):
        with pytest.raises(RuntimeError):
            ops.rotary_positions(*bad)
