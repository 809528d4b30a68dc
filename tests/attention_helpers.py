"""Plain 64-bit forms of the attention operators and the error bounds their tests hold the kernels to.

Every bound is worst-case rounding arithmetic.  A rounding to bf16 is off by at most 2^-8 of the value.  For 32-bit arithmetic the unit is
U = 2^-23 (one step: it covers rounding to nearest and the tensor cores' truncating sums): a sum of n terms is off by at most
n U of the sum of their absolute values."""
import torch

U = 2.0 ** -23
BF16 = 2.0 ** -8


def ends_of(lengths, device="cuda"):
    total, out = 0, []
    for n in lengths:
        total += n
        out.append(total)
    return torch.tensor(out, dtype=torch.int32, device=device)


def check(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), "%s: %d values beyond the bound, worst %.3g of it, first at %s" % (
        what, int(bad.sum()), float((off / bound.clamp_min(1e-300)).nan_to_num(1e9).max()), bad.nonzero()[0].tolist())


def attention(q, k, v, q_lens, k_lens, scale, g=None):
    """dict of float64 results and `*_bound` tensors.  Rows outside every cloud are zero (lse minus infinity)."""
    bf16 = q.dtype == torch.bfloat16
    q, k, v = q.double(), k.double(), v.double()
    m, h, d = q.shape
    n, hk = k.shape[:2]
    zero = lambda t: torch.zeros_like(t)  # noqa: E731
    r = {"out": zero(q), "out_bound": zero(q), "lse": q.new_full((h, m), -float("inf")), "lse_bound": q.new_zeros((h, m))}
    if g is not None:
        g = g.double()
        for name, t in (("dq", q), ("dk", k), ("dv", v)):
            r[name], r[name + "_bound"] = zero(t), zero(t)
    q0 = k0 = 0
    for lq, lk in zip(q_lens, k_lens):
        qs, ks = slice(q0, q0 + lq), slice(k0, k0 + lk)
        q0, k0 = q0 + lq, k0 + lk
        if lq == 0 or lk == 0:
            continue
        for a in range(h):
            b = a // (h // hk)
            Q, K, V = q[qs, a], k[ks, b], v[ks, b]
            s = Q @ K.t() * scale
            lse = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[:, None])
            # a logit: d products and a few roundings of the scaled sum; a probability: two such errors in its exponent,
            # the exponential (2 U) and the sum of lk terms
            ds_abs = (d + 8) * U * ((Q.abs() @ K.abs().t()) * abs(scale) + s.abs().amax(1, keepdim=True) + 1)
            rel = 2 * ds_abs.amax(1, keepdim=True) + (lk + 8) * U
            if bf16:
                rel_pv = rel + BF16  # the probability is rounded to bf16 for its product with the values
            else:
                rel_pv = rel + 8 * U
            out = p @ V
            r["out"][qs, a] = out
            r["out_bound"][qs, a] = (rel_pv + (lk + 8) * U) * (p @ V.abs()) + (BF16 * out.abs() if bf16 else 0)
            r["lse"][a, qs] = lse
            r["lse_bound"][a, qs] = (rel[:, 0] + 4 * U * (1 + lse.abs()))
            if g is None:
                continue
            G = g[qs, a]
            dp, delta = G @ V.t(), (G * out).sum(1, keepdim=True)
            ds = p * (dp - delta)
            mass = G.abs() @ V.abs().t() + (G.abs() * out.abs()).sum(1, keepdim=True)  # what dp - delta is a difference of
            ds_off = p * mass * (rel + (d + 8) * U)
            p_off = p * rel
            if bf16:
                # delta is taken from the rounded output: off by BF16 of its terms, and by what that output was off before
                ds_off = ds_off + p * ((G.abs() * r["out_bound"][qs, a]).sum(1, keepdim=True) + BF16 * (dp - delta).abs())
                p_off = p_off + p * BF16
            else:
                ds_off = ds_off + p * (G.abs() * r["out_bound"][qs, a]).sum(1, keepdim=True) + 8 * U * p * mass
                p_off = p_off + 8 * U * p
            r["dq"][qs, a] = scale * ds @ K
            r["dk"][ks, b] += scale * ds.t() @ Q
            r["dv"][ks, b] += p.t() @ G
            r["dq_bound"][qs, a] = abs(scale) * ((ds_off + (lk + 8) * U * (ds.abs() + ds_off)) @ K.abs())
            r["dk_bound"][ks, b] += abs(scale) * ((ds_off + (h * lq + 8) * U * (ds.abs() + ds_off)).t() @ Q.abs())
            r["dv_bound"][ks, b] += (p_off + (h * lq + 8) * U * p).t() @ G.abs()
    if g is not None:
        for name in ("dq", "dk", "dv"):
            r[name + "_bound"] = r[name + "_bound"] * (1 + 4 * U) + (BF16 * (r[name].abs() + r[name + "_bound"]) if bf16 else 0) + 1e-30
    r["out_bound"] = r["out_bound"] + 1e-30
    return r


def check_attention(got, want, grads=None):
    check(got[0], want["out"], want["out_bound"], "out")
    empty = torch.isinf(want["lse"])
    assert torch.equal(got[1] == -float("inf"), empty)
    check(got[1].double().masked_fill(empty, 0), want["lse"].masked_fill(empty, 0), want["lse_bound"] + 1e-30, "lse")
    for name, x in zip(("dq", "dk", "dv"), grads or ()):
        check(x, want[name], want[name + "_bound"], name)
