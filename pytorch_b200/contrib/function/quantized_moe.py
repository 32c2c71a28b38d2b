"""A W8A8 SwiGLU mixture of experts as a chain of the operators.

The reference tree has no function of this name; it names the pieces (``npu_moe_init_routing``, ``npu_grouped_matmul``,
``npu_swiglu_quant``, ``npu_moe_token_unpermute``) and leaves the chaining to the model code.  Between the router and the
result, HBM holds the int8 rows sorted by expert, the 16-bit gate/up products, the int8 activations and the 16-bit rows of
the down projection; nothing is padded to a capacity and nothing waits for the host to learn how many rows an expert has."""
from __future__ import annotations

import torch


def w8a8_swiglu_moe(x: torch.Tensor, expert_idx: torch.Tensor, expert_weight: torch.Tensor, smooth_in: torch.Tensor | None,
                    w_gate_up: torch.Tensor, scale_gate_up: torch.Tensor, smooth_act: torch.Tensor | None, w_down: torch.Tensor,
                    scale_down: torch.Tensor, expert_range: tuple[int, int] | None = None, expert_num: int | None = None) -> torch.Tensor:
    """``sum over slots of expert_weight * down_e( quant( silu(gate_e(x)) * up_e(x) ) )``.

    ``x`` ``[tokens, K]`` float16 or bfloat16; ``expert_idx`` ``[tokens, topk]`` int32 or int64 (-1: no expert, a padded token) and
    ``expert_weight`` of its shape from the router; ``w_gate_up`` ``[E, 2F, K]`` (gate rows first) and ``w_down`` ``[E, H, F]`` int8 with
    per-channel scales ``[E, 2F]`` / ``[E, H]``; ``smooth_in`` ``[E, K]`` (or ``[1, K]``) and ``smooth_act`` ``[F]`` are optional smooth-quant
    vectors.  With ``expert_range`` (and the whole number of experts, ``expert_num``) the weights are those of these experts only, as on a
    rank of expert parallelism: the result is then this rank's part of the sum."""
    ops = torch.ops.npu
    experts = w_gate_up.shape[0] if expert_num is None else expert_num
    q, row_idx, ends, s = ops.npu_moe_init_routing_v2(x, expert_idx, scale=smooth_in, expert_num=experts, quant_mode=1,
                                                      active_expert_range=None if expert_range is None else list(expert_range))
    gu = ops.npu_grouped_matmul([q], [w_gate_up.transpose(1, 2)], scale=[scale_gate_up], per_token_scale=[s], group_list=ends, split_item=3,
                                output_dtype=x.dtype)[0]
    qa, sa = ops.npu_swiglu_quant(gu, smooth_scales=smooth_act, activate_left=True, quant_mode=1)
    y = ops.npu_grouped_matmul([qa], [w_down.transpose(1, 2)], scale=[scale_down], per_token_scale=[sa], group_list=ends, split_item=3,
                               output_dtype=x.dtype)[0]
    return ops.npu_moe_token_unpermute(y, row_idx, expert_weight)
