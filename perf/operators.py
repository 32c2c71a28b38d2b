"""Measured cases of the mixture-of-experts block operators: routing tokens to experts and back, the experts'
products, and the norms before and after the block.

``run`` computes an operator either in its plain form (elementary torch operations in 32 bits, ``own`` false) or by
the calls of ``torch.ops.npu`` (``own`` true); ``exact`` computes the same outputs in 64 bits from the definitions.

The operators, by a case's ``op``:

route      ``npu_moe_init_routing_v2`` with dynamic quantisation: the rows of x sorted by expert, each multiplied by its
           expert's smooth scales and quantised to int8 with a scale of its own.  Serving.
permute    ``npu_moe_token_permute``: the rows sorted by expert; with ``grad`` also the gradient of the tokens.
unpermute  ``npu_moe_token_unpermute``: every token's rows gathered, weighted and added; with ``grad`` also the
           gradients of the rows and of the weights.
experts    ``npu_grouped_matmul``: int8 rows times their expert's int8 weight, scaled per channel and per row.
norm       ``npu_gated_add_rms_norm`` (and its ``_dynamic_quant`` form): the norm after one block, its gate and residual
           scale, and the norm before the next.

``experts``: an index of -1 is a token's padding; it has no row, and the rows past the last expert's are zero.
"""
import math

import numpy as np
import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # A decode step of sixteen sequences: one launch's latency.
        dict(name="route_decode", op="route", tokens=16, topk=8, experts=64, hidden=4096, dtype="bf16", padded=False),
        # A prefill chunk whose last eighth is padding, with sizes that fill no tile.
        dict(name="route_ragged", op="route", tokens=4099, topk=6, experts=60, hidden=5120, dtype="f16", padded=True),
        # A long prefill with many small experts: eight rows out for one in.
        dict(name="permute_prefill", op="permute", tokens=8192, topk=8, experts=64, hidden=4096, dtype="bf16", grad=False, padded=False),
        # A training step with few large experts.
        dict(name="permute_train", op="permute", tokens=8192, topk=2, experts=8, hidden=8192, dtype="bf16", grad=True, padded=False),
        # The way back of a decode step.
        dict(name="unpermute_decode", op="unpermute", tokens=16, topk=8, experts=64, hidden=4096, dtype="bf16", weights="f32", grad=False, padded=False),
        # A training step with many small experts: rows, weights and both gradients.
        dict(name="unpermute_train", op="unpermute", tokens=8192, topk=8, experts=64, hidden=4096, dtype="bf16", weights="f32", grad=True, padded=False),
        # A decode step: two rows for an expert, so all of it is reading the weights.
        dict(name="experts_decode", op="experts", rows=128, experts=64, k=4096, n=4096, dtype="bf16", skew=0.5, tail=0),
        # A long prefill through few large experts: all of it is the int8 products.
        dict(name="experts_prefill", op="experts", rows=16384, experts=8, k=4096, n=22016, dtype="bf16", skew=0.3, tail=0),
        # A short prefill with very unequal experts, some of them empty, and rows past the last one.
        dict(name="experts_ragged", op="experts", rows=1531, experts=24, k=5120, n=1416, dtype="f16", skew=2.0, tail=77),
        # The block boundary of a decode step, quantised for the next int8 matmul.
        dict(name="norm_decode", op="norm", rows=16, hidden=8192, dtype="bf16", params="bf16", gate="channel", post=True, mode="quant"),
        # The block boundary of a training step.
        dict(name="norm_train", op="norm", rows=8192, hidden=4096, dtype="bf16", params="bf16", gate="channel", post=True, mode="train"),
        # Four samples with a gate of their own each, a width that no vector divides, 32-bit parameters.
        dict(name="norm_ragged", op="norm", rows=4 * 1531, hidden=1111, dtype="f16", params="f32", gate="sample", post=True, mode="train"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of 64 as in a model, else a multiple of 8, else any."""
    w, r = _log(rng, lo, hi), rng.random()
    step = 64 if r < 0.6 else 8 if r < 0.85 else 1
    return max(lo, w // step * step)


def draw(rng):
    op = rng.choice(["route", "permute", "unpermute", "experts", "norm"])
    if op == "norm":
        hidden = _width(rng, 128, 8192)
        rows = _log(rng, 1, min(8192, (8192 * 4096) // hidden))
        gate = rng.choice(["none", "channel", "row", "sample", "full"])
        if gate == "sample":
            rows = max(4, rows // 4 * 4)
        return dict(op=op, rows=rows, hidden=hidden, dtype=rng.choice(["bf16", "f16"]), params=rng.choice(["same", "f32"]), gate=gate,
                    post=rng.random() < 0.7, mode=rng.choice(["plain", "quant", "train"]))
    if op == "experts":
        # Widths that the tensor-core path takes (multiples of 16) and, for small calls, any.
        rows, experts = _log(rng, 1, 8192), rng.choice([1, 2, 4, 8, 16, 24, 32, 60, 64])
        k, n = _log(rng, 256, 8192) // 16 * 16, _log(rng, 256, 8192) // 8 * 8
        while experts * k * n > 8 * 4096 * 22016 or rows * k * n > 16384 * 4096 * 4096:
            k, n, rows = max(256, k // 32 * 16), max(256, n // 16 * 8), max(1, rows // 2)
        return dict(op=op, rows=rows, experts=experts, k=k, n=n, dtype=rng.choice(["bf16", "f16"]), skew=round(rng.uniform(0, 2), 3),
                    tail=rng.choice([0, 0, rng.randrange(64)]))
    experts = rng.choice([4, 8, 16, 60, 64, 128, 256])
    topk = min(experts, rng.choice([1, 2, 4, 6, 8]))
    hidden = _width(rng, 256, 8192)
    tokens = _log(rng, 1, min(8192, (8192 * 8 * 4096) // (hidden * topk)))
    c = dict(op=op, tokens=tokens, topk=topk, experts=experts, hidden=hidden, dtype=rng.choice(["bf16", "f16"]), padded=rng.random() < 0.3)
    if op != "route":
        c["grad"] = rng.random() < 0.5
    if op == "unpermute":
        c["weights"] = rng.choice(["f32", "same"])
    return c


def _dtype(case, key):
    return DTYPE[case["dtype"] if case[key] == "same" else case[key]]


def work(case):
    op, s = case["op"], SIZE[case["dtype"]]
    if op == "norm":
        r, h, p = case["rows"], case["hidden"], SIZE[case["dtype"] if case["params"] == "same" else case["params"]]
        gates = {"none": 0, "channel": h, "row": r, "sample": 4 * h, "full": r * h}[case["gate"]] * p
        params = (2 if case["post"] else 1) * h * p
        read, wrote = 2 * r * h * s + params + gates, r * h * s + r * h * (1 if case["mode"] == "quant" else s) + 4 * r
        if case["mode"] == "train":  # x, residual, both gradients and the parameters again; two gradients and the parameters' out
            read, wrote = read + 4 * r * h * s + params + gates, wrote + 2 * r * h * s + params + gates
        return {"bytes": read + wrote, "flops": r * h * (40 if case["mode"] == "train" else 12)}
    if op == "experts":
        r, e, k, n = case["rows"], case["experts"], case["k"], case["n"]
        used = e * (1 - (1 - 1 / e) ** r) if e > 1 else 1.0
        return {"bytes": r * k + 4 * r + used * (k * n + 4 * n) + (r + case["tail"]) * n * s, "flops": 2 * r * k * n}
    t, k, h = case["tokens"], case["topk"], case["hidden"]
    rows = k * (t - _padding(case))
    full, wide = t * k * h, rows * h
    if op == "route":
        used = min(case["experts"], rows) if rows else 0
        return {"bytes": t * h * s + used * h * 4 + full + 4 * t * k * 3, "flops": 4 * wide}
    if op == "permute":
        b = t * h * s + full * s + 4 * t * k * 2
        return {"bytes": b + (wide * s + t * h * s + 4 * t * k if case["grad"] else 0), "flops": wide if case["grad"] else t * k}
    b = wide * s + t * h * s + 8 * t * k
    return {"bytes": b + (t * h * s + wide * s + full * s + 12 * t * k if case["grad"] else 0), "flops": 2 * wide * (3 if case["grad"] else 1)}


# ------------------------------------------------------------------------------------------------ the inputs
def _padding(case):
    return case["tokens"] // 8 if case["padded"] else 0


def _router(case, g):
    """Expert indices [tokens, topk] and weights of a router: the top scores, some experts liked better than others."""
    t, e = case["tokens"], case["experts"]
    scores = torch.randn((t, e), generator=g, device="cuda") + 0.5 * torch.randn((e,), generator=g, device="cuda")
    top, idx = torch.topk(scores, case["topk"], dim=1)
    weights = torch.softmax(top, dim=1)
    idx = idx.to(torch.int32)
    if _padding(case):
        idx[t - _padding(case):] = -1
    return idx, weights


def _sorted(idx, experts):
    """For every (token, slot) the row it goes to, or -1; and the cumulative rows of the experts."""
    flat = idx.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = torch.argsort(key, stable=True)
    row = torch.empty_like(order)
    row[order] = torch.arange(order.numel(), device=order.device)
    ends = (key[None, :] <= torch.arange(experts, device=key.device)[:, None]).sum(1)
    return torch.where(flat < 0, -1, row).to(torch.int32), order, ends


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, dt = case["op"], DTYPE[case["dtype"]]

    def randn(*shape, dtype=dt, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)

    s = dict(case=case)
    if op == "norm":
        r, h, p = case["rows"], case["hidden"], _dtype(case, "params")
        s.update(x=randn(r, h, std=3.0), residual=randn(r, h), gamma=randn(h, dtype=p, std=0.2, mean=1.0), gate=None, post=None, smooth=None)
        if case["post"]:
            s["post"] = randn(h, dtype=p, std=0.2, mean=1.0)
        if case["gate"] == "sample":  # [samples, length, hidden] with one gate for each sample
            s["x"], s["residual"] = s["x"].reshape(4, r // 4, h), s["residual"].reshape(4, r // 4, h)
        shape = {"none": None, "channel": (h,), "row": (r, 1), "sample": (4, 1, h), "full": (r, h)}[case["gate"]]
        if shape:
            s["gate"] = randn(*shape, dtype=p, std=0.5, mean=0.5)
        if case["mode"] == "quant":
            s["smooth"] = torch.rand((h,), generator=g, device="cuda") * 1.5 + 0.5
        if case["mode"] == "train":
            s["dy"], s["dh"] = randn(*s["x"].shape), randn(*s["x"].shape, std=0.3)
        return s
    if op == "experts":
        r, e, k, n = case["rows"], case["experts"], case["k"], case["n"]
        rng = np.random.default_rng(seed)
        p = np.exp(case["skew"] * rng.standard_normal(e))
        counts = rng.multinomial(r, p / p.sum())
        s.update(x=torch.randint(-127, 128, (r + case["tail"], k), generator=g, device="cuda", dtype=torch.int8),
                 weight=torch.randint(-127, 128, (e, n, k), generator=g, device="cuda", dtype=torch.int8).transpose(1, 2),
                 scale=torch.rand((e, n), generator=g, device="cuda") * 9e-3 + 1e-3,
                 row_scale=torch.rand((r + case["tail"],), generator=g, device="cuda") * 9e-3 + 1e-3,
                 ends=torch.from_numpy(np.cumsum(counts)).cuda(), most=int(counts.max()))
        return s
    t, k, h, e = case["tokens"], case["topk"], case["hidden"], case["experts"]
    s["idx"], weights = _router(case, g)
    if op == "route":
        s.update(x=randn(t, h), smooth=torch.rand((e, h), generator=g, device="cuda") * 1.5 + 0.5)
    elif op == "permute":
        s.update(x=randn(t, h))
        if case["grad"]:
            s["dy"] = randn(t * k, h)
    else:
        s.update(rows=randn(t * k, h), weights=weights.to(_dtype(case, "weights")), place=_sorted(s["idx"], e)[0])
        if case["grad"]:
            s["dy"] = randn(t, h)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        import pytorch_b200  # noqa: F401  (registers torch.ops.npu)
    return (_own if own else _plain)[case["op"]](s, case)


def _values(q, scale, dtype):
    """What int8 rows with a scale each stand for, in the activations' type."""
    return torch.mul(q, scale[..., None], out=torch.empty(q.shape, dtype=dtype, device=q.device))


def _quantised(x):
    """Symmetric int8 per row: x / (max|x| / 127), to the nearest."""
    scale = x.abs().amax(-1) / torch.full((1,), 127.0, device=x.device, dtype=x.dtype)
    q = torch.where(scale[..., None] > 0, torch.round(x / scale[..., None]).clamp(-128, 127), 0)
    return q, scale


def _plain_route(s, case):
    x, idx = s["x"], s["idx"]
    place, order, ends = _sorted(idx, case["experts"])
    expert = idx.reshape(-1)[order].long()
    rows = torch.where((expert >= 0)[:, None], x.to(F32)[order // case["topk"]] * s["smooth"][expert.clamp(min=0)], 0)
    q, scale = _quantised(rows)
    return _values(q.to(torch.int8), scale, x.dtype), place, ends, scale


def _own_route(s, case):
    q, place, ends, scale = torch.ops.npu.npu_moe_init_routing_v2(
        s["x"], s["idx"], scale=s["smooth"], expert_num=case["experts"], expert_tokens_num_type=0, expert_tokens_num_flag=True, quant_mode=1)
    return _values(q, scale, s["x"].dtype), place, ends, scale


def _plain_permute(s, case):
    x, idx, k = s["x"], s["idx"], case["topk"]
    place, order, _ = _sorted(idx, case["experts"])
    y = torch.where((idx.reshape(-1)[order] >= 0)[:, None], x[order // k], 0)
    if not case["grad"]:
        return y, place
    at = place.long()
    dx = torch.where((at >= 0)[:, None], s["dy"].to(F32)[at.clamp(min=0)], 0).reshape(case["tokens"], k, -1).sum(1)
    return y, place, dx.to(x.dtype)


def _own_permute(s, case):
    if not case["grad"]:
        return torch.ops.npu.npu_moe_token_permute(s["x"], s["idx"])
    x = s["x"].detach().requires_grad_()
    y, place = torch.ops.npu.npu_moe_token_permute(x, s["idx"])
    return y.detach(), place, *torch.autograd.grad(y, x, s["dy"])


def _plain_unpermute(s, case):
    t, k, rows = case["tokens"], case["topk"], s["rows"]
    at, w = s["place"].long(), s["weights"].to(F32)
    there = (at >= 0)[:, None]
    parts = torch.where(there, rows.to(F32)[at.clamp(min=0)], 0).reshape(t, k, -1)
    y = (parts * w[:, :, None]).sum(1).to(rows.dtype)
    if not case["grad"]:
        return y
    dy = s["dy"].to(F32)
    dw = (parts * dy[:, None, :]).sum(2).to(s["weights"].dtype)
    # Each row belongs to one (token, slot) at most; slots without a row go to one row more, which is cut off.
    drows = torch.zeros((rows.shape[0] + 1, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    drows[torch.where(at < 0, rows.shape[0], at)] = (dy[:, None, :] * w[:, :, None]).reshape(t * k, -1).to(rows.dtype)
    return y, drows[:-1], dw


def _own_unpermute(s, case):
    if not case["grad"]:
        return torch.ops.npu.npu_moe_token_unpermute(s["rows"], s["place"], s["weights"])
    rows, w = s["rows"].detach().requires_grad_(), s["weights"].detach().requires_grad_()
    y = torch.ops.npu.npu_moe_token_unpermute(rows, s["place"], w)
    return y.detach(), *torch.autograd.grad(y, (rows, w), s["dy"])


def _plain_experts(s, case):
    # The experts' rows side by side, padded to the largest expert's.  The products' sums stay far below 2^24 for these
    # lengths (a sum of k products of uniform int8 values has a deviation of 5400 sqrt(k)), where 32 bits are exact.
    x, ends = s["x"], s["ends"]
    starts = torch.cat([ends.new_zeros(1), ends[:-1]])
    at = torch.arange(max(1, s["most"]), device=x.device)[None, :] + starts[:, None]
    acc = torch.bmm(x[at.clamp(max=x.shape[0] - 1)].to(F32), s["weight"].to(F32)) * s["scale"][:, None, :]
    row = torch.arange(x.shape[0], device=x.device)
    expert = (row[:, None] >= ends[None, :]).sum(1)
    live = expert < ends.numel()
    expert = expert.clamp(max=ends.numel() - 1)
    y = acc[expert, (row - starts[expert]).clamp(max=max(1, s["most"]) - 1)] * s["row_scale"][:, None]
    return torch.where(live[:, None], y, 0).to(DTYPE[case["dtype"]])


def _own_experts(s, case):
    return torch.ops.npu.npu_grouped_matmul([s["x"]], [s["weight"]], scale=[s["scale"]], per_token_scale=[s["row_scale"]], group_list=s["ends"],
                                            split_item=3, group_type=0, group_list_type=0, output_dtype=DTYPE[case["dtype"]])[0]


def _plain_norm(s, case):
    x, gamma, gate = s["x"].to(F32), s["gamma"].to(F32), None if s["gate"] is None else s["gate"].to(F32)
    dt = s["x"].dtype
    if s["post"] is None:
        z = x
    else:
        r1 = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xn = x * r1
        z = xn * s["post"].to(F32)
    h = s["residual"].to(F32) * 0.5 + (z if gate is None else gate * z)
    r2 = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    hn = h * r2
    y = hn * gamma
    if case["mode"] == "quant":
        q, scale = _quantised(y * s["smooth"])
        return _values(q.to(torch.int8), scale, dt), scale, h.to(dt)
    if case["mode"] == "plain":
        return y.to(dt), h.to(dt)
    dy = s["dy"].to(F32)
    u = dy * gamma
    dh = s["dh"].to(F32) + r2 * (u - hn * (u * hn).mean(-1, keepdim=True))
    out = {"y": y.to(dt), "h": h.to(dt), "residual": (dh * 0.5).to(dt), "gamma": (dy * hn).reshape(-1, gamma.numel()).sum(0).to(s["gamma"].dtype)}
    dz = dh
    if gate is not None:
        dz = dh * gate
        out["gate"] = (dh * z).sum_to_size(gate.shape).to(s["gate"].dtype)
    if s["post"] is None:
        out["x"] = dz.to(dt)
    else:
        out["post"] = (dz * xn).reshape(-1, gamma.numel()).sum(0).to(s["post"].dtype)
        v = dz * s["post"].to(F32)
        out["x"] = (r1 * (v - xn * (v * xn).mean(-1, keepdim=True))).to(dt)
    return out


def _own_norm(s, case):
    if case["mode"] == "quant":
        q, scale, h = torch.ops.npu.npu_gated_add_rms_norm_dynamic_quant(s["x"], s["residual"], s["gamma"], post_gamma=s["post"], gate=s["gate"],
                                                                         smooth_scales=s["smooth"], residual_scale=0.5, epsilon=EPS)
        return _values(q, scale, s["x"].dtype), scale, h
    names = [n for n in ("x", "residual", "gamma", "post", "gate") if s[n] is not None]
    at = {n: s[n].detach().requires_grad_(case["mode"] == "train") for n in names}
    y, _, h, _ = torch.ops.npu.npu_gated_add_rms_norm(at["x"], at["residual"], at["gamma"], post_gamma=at.get("post"), gate=at.get("gate"),
                                                      residual_scale=0.5, epsilon=EPS)
    if case["mode"] == "plain":
        return y, h
    grads = torch.autograd.grad((y, h), [at[n] for n in names], (s["dy"], s["dh"]))
    return {"y": y.detach(), "h": h.detach(), **dict(zip(names, grads))}


_plain = {"route": _plain_route, "permute": _plain_permute, "unpermute": _plain_unpermute, "experts": _plain_experts, "norm": _plain_norm}
_own = {"route": _own_route, "permute": _own_permute, "unpermute": _own_unpermute, "experts": _own_experts, "norm": _own_norm}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "norm":
        return _exact_norm(s, case)
    if op == "experts":
        x, ends = s["x"], [0] + s["ends"].tolist()
        y = torch.zeros((x.shape[0], case["n"]), dtype=F64, device="cuda")
        for e in range(case["experts"]):
            a, b = ends[e], ends[e + 1]
            if b > a:
                y[a:b] = x[a:b].to(F64) @ s["weight"][e].to(F64) * s["scale"][e].to(F64) * s["row_scale"][a:b, None].to(F64)
        return y
    t, k, h = case["tokens"], case["topk"], case["hidden"]
    flat = s["idx"].reshape(-1).cpu().numpy()
    order = [int(i) for i in np.argsort(flat, kind="stable") if flat[i] >= 0]  # the (token, slot) of every row
    slot = torch.tensor(order, dtype=torch.long, device="cuda")
    token = slot // k
    n = len(order)
    if op == "route":
        values = torch.zeros((t * k, h), dtype=F64, device="cuda")
        scale = torch.zeros((t * k,), dtype=F64, device="cuda")
        for a in range(0, n, 4096):
            b = min(n, a + 4096)
            xs = s["x"][token[a:b]].to(F64) * s["smooth"][s["idx"].reshape(-1)[slot[a:b]].long()].to(F64)
            step = xs.abs().max(dim=1).values / 127
            scale[a:b] = step
            values[a:b] = torch.round(xs / torch.where(step > 0, step, 1.0)[:, None]) * step[:, None]
        return values, None, None, scale
    if op == "permute":
        y = torch.zeros((t * k, h), dtype=F64, device="cuda")
        y[:n] = s["x"][token].to(F64)
        if not case["grad"]:
            return y, None
        dx = torch.zeros((t, h), dtype=F64, device="cuda")
        dx.index_add_(0, token, s["dy"][:n].to(F64))
        return y, None, dx
    w = s["weights"].reshape(-1)[slot].to(F64)
    rows = s["rows"][:n].to(F64)
    y = torch.zeros((t, h), dtype=F64, device="cuda").index_add_(0, token, rows * w[:, None])
    if not case["grad"]:
        return y
    dy = s["dy"][token].to(F64)
    drows = torch.zeros((t * k, h), dtype=F64, device="cuda")
    drows[:n] = dy * w[:, None]
    dw = torch.zeros((t * k,), dtype=F64, device="cuda")
    dw[slot] = torch.linalg.vecdot(rows, dy)
    return y, drows, dw.reshape(t, k)


def _exact_norm(s, case):
    names = [n for n in ("x", "residual", "gamma", "post", "gate") if s[n] is not None]
    at = {n: s[n].to(F64).requires_grad_() for n in names}
    z = at["x"]
    if "post" in at:
        z = z / torch.sqrt(torch.mean(z ** 2, dim=-1, keepdim=True) + EPS) * at["post"]
    h = 0.5 * at["residual"] + at.get("gate", 1.0) * z
    y = h / torch.sqrt(torch.mean(h ** 2, dim=-1, keepdim=True) + EPS) * at["gamma"]
    if case["mode"] == "plain":
        return y.detach(), h.detach()
    if case["mode"] == "quant":
        v = (y * s["smooth"].to(F64)).detach()
        step = v.abs().amax(-1) / 127
        return torch.round(v / step[..., None]) * step[..., None], step, h.detach()
    loss = (y * s["dy"].to(F64)).sum() + (h * s["dh"].to(F64)).sum()
    return {"y": y.detach(), "h": h.detach(), **dict(zip(names, torch.autograd.grad(loss, [at[n] for n in names])))}
