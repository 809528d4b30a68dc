"""Measured cases of the attention operators on packed point clouds: layer norm, rotary positions from point
coordinates, and cross attention between the points of two levels of the same clouds.

Features of a batch of clouds are packed: cloud b owns the rows [ends[b-1], ends[b]) of a tensor, as the rows of
``Pointcloud.pts_`` do.  Every pass is one operator in one direction; a training pass runs the forward operator and the
gradient operator and returns the outputs and all gradients."""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # a handful of pooled points in a small layer: the call's latency
        {"name": "norm_37x64_f32", "op": "norm", "rows": 37, "channels": 64, "type": "f32", "train": False},
        # inference over the points of a batch of surface clouds at a middle encoder width
        {"name": "norm_200000x256_bf16", "op": "norm", "rows": 200000, "channels": 256, "type": "bf16", "train": False},
        # training step of a large scene at the width of its convolutions
        {"name": "norm_train_500000x128_f32", "op": "norm", "rows": 500000, "channels": 128, "type": "f32", "train": True},
        # training on a coarse level: few rows, wide and odd
        {"name": "norm_train_20011x1001_bf16", "op": "norm", "rows": 20011, "channels": 1001, "type": "bf16", "train": True},
        # a few queries of one small cloud
        {"name": "rotary_61x4x32_f32", "op": "rotary", "rows": 61, "heads": 4, "size": 32, "axes": 3, "pairs": 5,
         "type": "f32", "train": False},
        # training step over the points of several scenes, with the gradient of the coordinates
        {"name": "rotary_train_150000x8x64_f32", "op": "rotary", "rows": 150000, "heads": 8, "size": 64, "axes": 3, "pairs": 10,
         "type": "f32", "train": True},
        # a small layer in training precision: two clouds, latency
        {"name": "attend_150x301x4x32_f32", "op": "attend", "clouds": 2, "queries": 150, "keys": 301, "heads": 4, "kv_heads": 4,
         "size": 32, "type": "f32", "train": False},
        # one learned query per cloud pools all its points: a long key axis with a single row
        {"name": "attend_pool_16x400000x8x64_bf16", "op": "attend", "clouds": 16, "queries": 16, "keys": 400000, "heads": 8,
         "kv_heads": 8, "size": 64, "type": "bf16", "train": False},
        # a decoder level reads the next coarser level, heads share keys and values, ragged clouds
        {"name": "attend_40001x20003x8of2x128_bf16", "op": "attend", "clouds": 16, "queries": 40001, "keys": 20003, "heads": 8,
         "kv_heads": 2, "size": 128, "type": "bf16", "train": False},
        # a few hundred latents per cloud read all its points
        {"name": "attend_latents_1024x120007x8x64_bf16", "op": "attend", "clouds": 4, "queries": 1024, "keys": 120007,
         "heads": 8, "kv_heads": 8, "size": 64, "type": "bf16", "train": False},
        # training step between two levels in reduced precision
        {"name": "attend_train_30011x30011x8x64_bf16", "op": "attend", "clouds": 8, "queries": 30011, "keys": 30011, "heads": 8,
         "kv_heads": 8, "size": 64, "type": "bf16", "train": True},
        # the same in the precision the layers train in
        {"name": "attend_train_16001x8003x8of4x64_f32", "op": "attend", "clouds": 8, "queries": 16001, "keys": 8003, "heads": 8,
         "kv_heads": 4, "size": 64, "type": "f32", "train": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Another case of the ranges above: rows, clouds and lengths over their logarithm, any channel count, every head
    layout; sizes whose work passes the largest listed case are drawn again."""
    op = rng.choice(["norm", "rotary", "attend", "attend"])
    kind, train = rng.choice(["f32", "bf16"]), rng.random() < 0.5
    if op == "norm":
        channels = _log_int(rng, 16, 1500)
        return {"op": "norm", "rows": _log_int(rng, 17, 40000000 // channels), "channels": channels, "type": kind, "train": train}
    if op == "rotary":
        size, heads, axes = rng.choice([16, 32, 64, 96, 128]), rng.randint(1, 12), rng.randint(2, 4)
        return {"op": "rotary", "rows": _log_int(rng, 17, 60000000 // (size * heads)), "heads": heads, "size": size, "axes": axes,
                "pairs": rng.randint(1, size // (2 * axes)), "type": kind, "train": train}
    while True:
        kv_heads = rng.randint(1, 6)
        case = {"op": "attend", "clouds": _log_int(rng, 1, 24), "queries": _log_int(rng, 24, 30000), "keys": _log_int(rng, 24, 100000),
                "heads": kv_heads * rng.randint(1, 3), "kv_heads": kv_heads, "size": rng.choice([16, 32, 40, 64]) if kind == "f32"
                else rng.choice([16, 32, 40, 64, 80, 96, 128]), "type": kind, "train": train}
        if work(case)["flops"] < (1.5e11 if kind == "f32" else 4e11):
            return case


# ---- inputs --------------------------------------------------------------------------------------
def _lengths(total, clouds):
    """Uneven cloud sizes that add up to `total`: between a fifth and nine fifths of the mean."""
    share = np.cumsum(1.0 + 0.8 * np.cos(2.4 * np.arange(clouds) + 0.3))
    return np.diff(np.rint(total * share / share[-1]).astype(int), prepend=0).tolist()


def _ends(lengths):
    return torch.tensor(np.cumsum(lengths), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    dtype = TYPES[case["type"]]
    state = {"case": dict(case)}
    if case["op"] == "norm":
        n, c = case["rows"], case["channels"]
        # activations of a convolution: every channel with its own spread, rows of different size, a mean away from zero
        x = normal(n, c) * (0.5 + torch.rand(c, generator=gen, device="cuda")) * (0.2 + torch.rand(n, 1, generator=gen, device="cuda") * 3.0)
        state["features"] = (x + 0.5).to(dtype)
        state["weights"], state["bias"] = 1.0 + normal(c, scale=0.2), normal(c, scale=0.2)
        state["grads"] = normal(n, c, dtype=dtype)
        return state
    if case["op"] == "rotary":
        n, h, d = case["rows"], case["heads"], case["size"]
        state["features"] = normal(n, h, d, dtype=dtype)
        # coordinates of a scene in units of its cells, the largest cells counted in hundreds
        state["pts"] = torch.rand((n, case["axes"]), generator=gen, device="cuda") * 400.0 - 100.0
        pairs = torch.arange(case["pairs"], dtype=torch.float64, device="cuda") / case["pairs"]
        state["frequencies"] = (100.0 ** -pairs).to(torch.float32).repeat(case["axes"])
        state["axis_pairs"] = [case["pairs"]] * case["axes"]
        state["grads"] = normal(n, h, d, dtype=dtype)
        return state
    m, n, d = case["queries"], case["keys"], case["size"]
    q_lens, k_lens = _lengths(m, case["clouds"]), _lengths(n, case["clouds"])
    state["queries"] = normal(m, case["heads"], d, scale=1.5, dtype=dtype)
    state["keys"] = normal(n, case["kv_heads"], d, dtype=dtype)
    state["values"] = normal(n, case["kv_heads"], d, dtype=dtype)
    state["grads"] = normal(m, case["heads"], d, dtype=dtype)
    state["query_ends"], state["key_ends"] = _ends(q_lens), _ends(k_lens)
    state["longest"] = (max(q_lens), max(k_lens))
    return state


# ---- one pass ------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    return {"norm": _plain_norm, "rotary": _plain_rotary, "attend": _plain_attend}[case["op"]](case, state)


def _own(case, s):
    from pccnn_lib_b200 import ops
    if case["op"] == "norm":
        out, mean, rstd = ops.layer_norm(s["features"], s["weights"], s["bias"], EPS)
        if not case["train"]:
            return {"out": out}
        feat, weight, bias = ops.layer_norm_grads(s["features"], s["weights"], mean, rstd, s["grads"])
        return {"out": out, "features": feat, "weights": weight, "bias": bias}
    if case["op"] == "rotary":
        out = ops.rotary_positions(s["features"], s["pts"], s["frequencies"], s["axis_pairs"])
        if not case["train"]:
            return {"out": out}
        feat, pts = ops.rotary_positions_grads(s["features"], s["pts"], s["frequencies"], s["axis_pairs"], s["grads"])
        return {"out": out, "features": feat, "pts": pts}
    args = (s["queries"], s["keys"], s["values"], s["query_ends"], s["key_ends"])
    out, lse = ops.cross_attention(*args)
    if not case["train"]:
        return {"out": out, "lse": lse}
    q, k, v = ops.cross_attention_grads(*args, out, lse, s["grads"])
    return {"out": out, "lse": lse, "queries": q, "keys": k, "values": v}


def _plain_norm(case, s):
    dtype = s["features"].dtype
    x = s["features"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    hat = centred * rstd
    out = (hat * s["weights"] + s["bias"]).to(dtype)
    if not case["train"]:
        return {"out": out}
    g = s["grads"].float()
    gw = g * s["weights"]
    feat = rstd * (gw - gw.mean(1, keepdim=True) - hat * (gw * hat).mean(1, keepdim=True))
    return {"out": out, "features": feat.to(dtype), "weights": (g * hat).sum(0), "bias": g.sum(0)}


def _rotation(s, rows):
    """cos and sin [rows, 1, pairs] of every pair's angle; the angles of far positions need 64 bits."""
    axis = torch.repeat_interleave(torch.arange(len(s["axis_pairs"]), device="cuda"), torch.tensor(s["axis_pairs"], device="cuda"))
    angle = s["pts"].double()[:, axis] * s["frequencies"].double()
    return torch.cos(angle).float().reshape(rows, 1, -1), torch.sin(angle).float().reshape(rows, 1, -1), axis


def _plain_rotary(case, s):
    dtype, n = s["features"].dtype, case["rows"]
    turned = 2 * case["pairs"] * case["axes"]
    cos, sin, axis = _rotation(s, n)
    x = s["features"].float()
    a, b = x[..., 0:turned:2], x[..., 1:turned:2]
    ya, yb = a * cos - b * sin, a * sin + b * cos
    out = torch.cat([torch.stack([ya, yb], -1).reshape(n, case["heads"], turned), x[..., turned:]], -1).to(dtype)
    if not case["train"]:
        return {"out": out}
    g = s["grads"].float()
    ga, gb = g[..., 0:turned:2], g[..., 1:turned:2]
    feat = torch.cat([torch.stack([ga * cos + gb * sin, gb * cos - ga * sin], -1).reshape(n, case["heads"], turned), g[..., turned:]], -1)
    turn = (gb * ya - ga * yb).sum(1) * s["frequencies"]
    pts = torch.zeros_like(s["pts"]).index_add_(1, axis, turn)
    return {"out": out, "features": feat.to(dtype), "pts": pts}


def _padded(x, ends, longest):
    """[clouds, heads, longest, size] in 32 bits with zeros behind each cloud's rows."""
    starts = torch.cat([ends.new_zeros(1), ends[:-1]])
    row = starts[:, None] + torch.arange(longest, device="cuda")
    valid = row < ends[:, None]
    rows = x[torch.where(valid, row, 0).long()].float()
    return torch.where(valid[:, :, None, None], rows, 0.0).transpose(1, 2), valid


def _packed(x, valid):
    """The rows of `_padded` back in their packed order."""
    return x.transpose(1, 2)[valid]


def _plain_attend(case, s):
    dtype, scale = s["queries"].dtype, 1.0 / math.sqrt(case["size"])
    group, (longest_q, longest_k) = case["heads"] // case["kv_heads"], s["longest"]
    q, q_valid = _padded(s["queries"], s["query_ends"], longest_q)
    k, k_valid = _padded(s["keys"], s["key_ends"], longest_k)
    v, _ = _padded(s["values"], s["key_ends"], longest_k)
    clouds, heads = q.shape[0], case["heads"]
    q = q.reshape(clouds, case["kv_heads"], group * longest_q, case["size"])  # heads that share keys are more rows
    logits = torch.matmul(q, k.transpose(-1, -2)) * scale
    logits = torch.where(k_valid[:, None, None, :], logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = torch.exp(logits - top)
    del logits
    total = p.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    p = p / torch.where(total > 0, total, 1.0)
    out = torch.matmul(p, v)
    unfold = lambda x: x.reshape(clouds, heads, longest_q, -1)  # noqa: E731
    result = {"out": _packed(unfold(out), q_valid).to(dtype), "lse": _packed(unfold(lse), q_valid)[..., 0].t().contiguous()}
    if not case["train"]:
        return result
    g, _ = _padded(s["grads"], s["query_ends"], longest_q)
    g = g.reshape(q.shape)
    dv = torch.matmul(p.transpose(-1, -2), g)
    ds = p * (torch.matmul(g, v.transpose(-1, -2)) - (g * out).sum(-1, keepdim=True)) * scale
    del p
    result["queries"] = _packed(unfold(torch.matmul(ds, k)), q_valid).to(dtype)
    result["keys"] = _packed(torch.matmul(ds.transpose(-1, -2), q), k_valid).to(dtype)
    result["values"] = _packed(dv, k_valid).to(dtype)
    return result


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    size = {"f32": 4, "bf16": 2}[case["type"]]
    if case["op"] == "norm":
        n, c = case["rows"], case["channels"]
        elements = n * c
        moved, flops = elements * size * 2 + 8 * c, 8 * elements
        if case["train"]:  # the gradient is read, the features' gradient written
            moved, flops = moved + elements * size * 2 + 8 * c, flops + 14 * elements
        return {"bytes": moved, "flops": flops}
    if case["op"] == "rotary":
        elements = case["rows"] * case["heads"] * case["size"]
        moved, flops = elements * size * 2 + case["rows"] * case["axes"] * 4, 3 * elements
        if case["train"]:
            moved, flops = moved + elements * size * 2 + case["rows"] * case["axes"] * 4, flops + 6 * elements
        return {"bytes": moved, "flops": flops}
    pairs = sum(a * b for a, b in zip(_lengths(case["queries"], case["clouds"]), _lengths(case["keys"], case["clouds"])))
    q, kv = case["queries"] * case["heads"] * case["size"] * size, case["keys"] * case["kv_heads"] * case["size"] * size
    moved, flops = 2 * q + 2 * kv + 4 * case["queries"] * case["heads"], 4 * pairs * case["heads"] * case["size"]
    if case["train"]:  # four more products of the same size: the probabilities' gradient and the three inputs'
        moved, flops = moved + 2 * q + 2 * kv, 3 * flops
    return {"bytes": moved, "flops": flops}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.double().requires_grad_() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "norm":
        x, w, b = wide["features"], wide["weights"], wide["bias"]
        with torch.set_grad_enabled(case["train"]):
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            out = (x - mean) * torch.rsqrt(var + EPS) * w + b
        result = {"out": out.detach()}
        if case["train"]:
            result["features"], result["weights"], result["bias"] = torch.autograd.grad(out, (x, w, b), wide["grads"].detach())
        return result
    if case["op"] == "rotary":
        x, pts = wide["features"], wide["pts"]
        with torch.set_grad_enabled(case["train"]):
            per_axis = [pts[:, a:a + 1] * f for a, f in enumerate(wide["frequencies"].detach().reshape(case["axes"], -1))]
            angle = torch.cat(per_axis, 1)[:, None, :]
            turned = 2 * angle.shape[-1]
            z = torch.view_as_complex(x[..., :turned].reshape(x.shape[0], x.shape[1], -1, 2)) * torch.polar(torch.ones_like(angle), angle)
            out = torch.cat([torch.view_as_real(z).flatten(-2), x[..., turned:]], -1)
        result = {"out": out.detach()}
        if case["train"]:
            result["features"], result["pts"] = torch.autograd.grad(out, (x, pts), wide["grads"].detach())
        return result
    result = {"out": torch.empty_like(wide["queries"]), "lse": torch.empty(wide["queries"].shape[1::-1], dtype=torch.float64, device="cuda")}
    grads = {k: torch.zeros_like(wide[k]) for k in ("queries", "keys", "values")}
    group, q0, k0 = case["heads"] // case["kv_heads"], 0, 0
    for q1, k1 in zip(s["query_ends"].tolist(), s["key_ends"].tolist()):
        for h in range(case["heads"]):  # one head of one cloud at a time
            q = wide["queries"].detach()[q0:q1, h].clone().requires_grad_()
            k, v = (wide[n].detach()[k0:k1, h // group].clone().requires_grad_() for n in ("keys", "values"))
            with torch.set_grad_enabled(case["train"]):
                logits = q @ k.t() / math.sqrt(case["size"])
                out = torch.softmax(logits, -1) @ v
            result["out"].data[q0:q1, h], result["lse"][h, q0:q1] = out.detach(), torch.logsumexp(logits.detach(), -1)
            if case["train"]:
                got = torch.autograd.grad(out, (q, k, v), wide["grads"].detach()[q0:q1, h])
                grads["queries"][q0:q1, h] += got[0]
                grads["keys"][k0:k1, h // group] += got[1]
                grads["values"][k0:k1, h // group] += got[2]
        q0, k0 = q1, k1
    result = {n: v.detach() for n, v in result.items()}
    if case["train"]:
        result.update({n: v.detach() for n, v in grads.items()})
    return result
