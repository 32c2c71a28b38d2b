"""Plain 64-bit CPU implementations of the mixture-of-experts block operators: the definitions the kernels are tested
against.  Integers (rows, counts) are exact; floating results come back in float64, not rounded to the output type."""
from __future__ import annotations

import numpy as np
import torch

from . import quant_oracle

F64 = torch.float64


def sorted_rows(expert_idx: torch.Tensor, begin: int, end: int):
    """``(row of every assignment or -1, assignment of every row or -1, rows of each expert)`` of a stable sort by
    expert; an expert outside ``[begin, end)`` has no row."""
    flat = expert_idx.reshape(-1).to(torch.int64).numpy()
    live = (flat >= begin) & (flat < end)
    order = np.argsort(np.where(live, flat, end), kind="stable")[:int(live.sum())]
    row = np.full(flat.size, -1, dtype=np.int32)
    row[order] = np.arange(order.size, dtype=np.int32)
    src = np.full(flat.size, -1, dtype=np.int32)
    src[:order.size] = order
    counts = np.bincount(flat[live] - begin, minlength=end - begin).astype(np.int64)
    return torch.from_numpy(row), torch.from_numpy(src), torch.from_numpy(counts)


def gather_rows(x: torch.Tensor, row_src: torch.Tensor, topk: int) -> torch.Tensor:
    """``x[assignment // topk]`` for every row, zero for rows without one; x's dtype."""
    out = torch.zeros((row_src.numel(), x.shape[1]), dtype=x.dtype)
    live = row_src >= 0
    out[live] = x[(row_src[live] // topk).long()]
    return out


def route_quantised(x: torch.Tensor, expert_idx: torch.Tensor, smooth: torch.Tensor | None, begin: int, end: int):
    """int8 rows and their scales, as ``quant_oracle.dynamic_quant`` of the gathered rows with each expert's smooth row."""
    _, src, counts = sorted_rows(expert_idx, begin, end)
    n = int(counts.sum())
    q = torch.zeros((src.numel(), x.shape[1]), dtype=torch.int8)
    scale = torch.zeros((src.numel(),), dtype=torch.float32)
    if n:
        rows = gather_rows(x, src, expert_idx.shape[1])[:n]
        if smooth is None or smooth.shape[0] == 1:
            q[:n], scale[:n] = quant_oracle.dynamic_quant(rows, None if smooth is None else smooth[0])
        else:
            q[:n], scale[:n] = quant_oracle.dynamic_quant(rows, smooth, torch.cumsum(counts, 0).to(torch.int32))
    return q, scale


def combine(rows: torch.Tensor, row_idx: torch.Tensor, weights: torch.Tensor | None, tokens: int, topk: int):
    """``(sum over k of weights[t,k] * rows[row_idx[t,k]], sum of the magnitudes)``; a row index out of range adds nothing."""
    idx = row_idx.reshape(tokens, topk).long()
    live = (idx >= 0) & (idx < rows.shape[0])
    parts = torch.zeros((tokens, topk, rows.shape[1]), dtype=F64)
    parts[live] = rows.to(F64)[idx[live]]
    if weights is not None:
        parts = parts * torch.where(live, weights.to(F64), torch.zeros((), dtype=F64))[:, :, None]
    return parts.sum(1), parts.abs().sum(1)


def combine_grad(dy: torch.Tensor, rows: torch.Tensor, row_idx: torch.Tensor, weights: torch.Tensor | None, tokens: int, topk: int):
    """``(drows, dweights, bound on the magnitude of dweights' terms)``."""
    idx = row_idx.reshape(tokens, topk).long()
    live = (idx >= 0) & (idx < rows.shape[0])
    t, k = torch.nonzero(live, as_tuple=True)
    w = torch.ones((tokens, topk), dtype=F64) if weights is None else weights.to(F64)
    drows = torch.zeros(rows.shape, dtype=F64)
    drows[idx[t, k]] = dy.to(F64)[t] * w[t, k][:, None]
    dw, size = torch.zeros((tokens, topk), dtype=F64), torch.zeros((tokens, topk), dtype=F64)
    terms = rows.to(F64)[idx[t, k]] * dy.to(F64)[t]
    dw[t, k], size[t, k] = terms.sum(1), terms.abs().sum(1)
    return drows, dw, size


def gated_add_rms_norm(x, residual, gamma, post_gamma, gate, residual_scale, epsilon):
    """``(y, h, rstd, post_rstd)`` of the norm after a block, its gate and residual scale, and the norm before the next."""
    z = x.to(F64)
    post_rstd = None
    if post_gamma is not None:
        post_rstd = 1 / torch.sqrt((z * z).mean(-1) + epsilon)
        z = z * post_rstd[..., None] * post_gamma.to(F64)
    h = residual_scale * residual.to(F64) + (z if gate is None else gate.to(F64) * z)
    rstd = 1 / torch.sqrt((h * h).mean(-1) + epsilon)
    return h * rstd[..., None] * gamma.to(F64), h, rstd, post_rstd


def gated_add_rms_norm_grad(x, residual, gamma, post_gamma, gate, residual_scale, epsilon, dy, dh):
    """``(gradients, bounds)`` by name.  The gradients are autograd's of the definition; a bound is the sum of the magnitudes
    of the terms that the gradient's formula adds for one element (over rows too, where the gradient sums over rows)."""
    named = [(n, t) for n, t in (("x", x), ("residual", residual), ("gamma", gamma), ("post_gamma", post_gamma), ("gate", gate)) if t is not None]
    at = {n: t.detach().to(F64).requires_grad_() for n, t in named}
    y, h, rstd, post_rstd = gated_add_rms_norm(at["x"], at["residual"], at["gamma"], at.get("post_gamma"), at.get("gate"), residual_scale, epsilon)
    loss = (y * dy.to(F64)).sum() + (h * dh.to(F64)).sum()
    grads = dict(zip(at, torch.autograd.grad(loss, list(at.values()))))
    with torch.no_grad():
        w2, hn = gamma.to(F64), h * rstd[..., None]
        u = dy.to(F64) * w2
        m2 = (u * hn).abs().mean(-1, keepdim=True)
        dhs = dh.to(F64).abs() + rstd[..., None] * (u.abs() + hn.abs() * m2)
        xn = x.to(F64) if post_gamma is None else x.to(F64) * post_rstd[..., None]
        z = xn if post_gamma is None else xn * post_gamma.to(F64)
        dz = dhs if gate is None else dhs * gate.to(F64).abs()
        flat = lambda t: t.reshape(-1, x.shape[-1]).sum(0)  # noqa: E731
        bounds = {"gamma": flat((dy.to(F64) * hn).abs()), "residual": abs(residual_scale) * dhs}
        if gate is not None:
            bounds["gate"] = (dhs * z.abs()).sum_to_size(gate.shape)
        if post_gamma is None:
            bounds["x"] = dz
        else:
            bounds["post_gamma"] = flat(dz * xn.abs())
            v = dz * post_gamma.to(F64).abs()
            bounds["x"] = post_rstd[..., None] * (v + xn.abs() * (v * xn.abs()).mean(-1, keepdim=True))
    return grads, bounds


def grouped_matmul(x, weight, group_ends, scale, row_scale, bias, out_dtype):
    """Rows of ``x`` times their group's ``weight [groups, k, n]`` with ``quant_oracle.quant_matmul``'s epilogue (the same fp32
    steps as the kernel's, so the result is bit-exact); rows past the last group are zero."""
    out = torch.zeros((x.shape[0], weight.shape[2]), dtype=out_dtype)
    start = 0
    for g in range(weight.shape[0]):
        end = min(max(int(group_ends[g]), start), x.shape[0])
        if end > start:
            out[start:end] = quant_oracle.quant_matmul(
                x[start:end], weight[g], torch.ones(1) if scale is None else scale[g],
                pertoken_scale=None if row_scale is None else row_scale[start:end], bias=None if bias is None else bias[g], output_dtype=out_dtype)
        start = end
    return out
