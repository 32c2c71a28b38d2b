"""Derivatives that the mixture-of-experts block operators do not have: a tangent of forward mode is refused, never lost, and a backward
pass through an operator without a gradient goes on behind PyTorch's warning.  On fake tensors, which need no GPU."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.fixture(scope="module")
def pkg():
    import pytorch_b200
    return pytorch_b200


def tensor(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def calls(pkg):
    """Every operator of one float argument, the others fixed; whether the operator has a gradient."""
    idx, place = tensor(6, 2, dtype=torch.int32), tensor(12, dtype=torch.int32)
    x, w, rows, probs = tensor(6, 64), tensor(64), tensor(12, 64), tensor(6, 2, dtype=torch.float32)
    rstd = tensor(6, dtype=torch.float32)
    norm, quant, grad = pkg.npu_gated_add_rms_norm, pkg.npu_gated_add_rms_norm_dynamic_quant, pkg.npu_gated_add_rms_norm_grad
    q, weight, ends = tensor(12, 32, dtype=torch.int8), tensor(4, 32, 64, dtype=torch.int8), tensor(4, dtype=torch.int64)
    scale, row_scale = tensor(4, 64, dtype=torch.float32), tensor(12, dtype=torch.float32)
    product = lambda s, r: pkg.npu_grouped_matmul([q], [weight], scale=[s], per_token_scale=[r], group_list=ends, split_item=3)[0]  # noqa: E731
    return {
        "permute": (x, lambda t: pkg.npu_moe_token_permute(t, idx)[0], True),
        "unpermute rows": (rows, lambda t: pkg.npu_moe_token_unpermute(t, place, probs), True),
        "unpermute alone": (rows, lambda t: pkg.npu_moe_token_unpermute(t, place), True),
        "unpermute probs": (probs, lambda t: pkg.npu_moe_token_unpermute(rows, place, t), True),
        "norm x": (x, lambda t: norm(t, x, w)[0], True),
        "norm residual": (x, lambda t: norm(x, t, w)[2], True),
        "norm gamma": (w, lambda t: norm(x, x, t)[0], True),
        "norm post_gamma": (w, lambda t: norm(x, x, w, post_gamma=t)[0], True),
        "norm gate": (w, lambda t: norm(x, x, w, gate=t)[0], True),
        "routing": (x, lambda t: pkg.npu_moe_init_routing_v2(t, idx, expert_num=4)[0], False),
        "quantised norm": (x, lambda t: quant(t, x, w)[2], False),
        "permute_grad": (rows, lambda t: pkg.npu_moe_token_permute_grad(x, t, idx, place), False),
        "unpermute_grad": (x, lambda t: pkg.npu_moe_token_unpermute_grad(rows, t, place, probs)[0], False),
        "products' scale": (scale, lambda t: product(t, row_scale), False),
        "products' row scale": (row_scale, lambda t: product(scale, t), False),
        "norm_grad": (x, lambda t: grad(t, None, x, x, w, rstd)[0], False),
    }


NAMES = ("permute", "unpermute rows", "unpermute alone", "unpermute probs", "norm x", "norm residual", "norm gamma", "norm post_gamma", "norm gate",
         "routing", "quantised norm", "permute_grad", "unpermute_grad", "norm_grad",
         "products' scale", "products' row scale")


@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused(pkg, name):
    with FakeTensorMode():
        at, call, _ = calls(pkg)[name]
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(at, torch.ones_like(at))
            with pytest.raises(NotImplementedError):
                call(dual)
        with pytest.raises(NotImplementedError):
            torch.func.jvp(call, (at,), (torch.ones_like(at),))
        assert call(at).shape[-1] == 64                            # a plain tensor goes on as before


@pytest.mark.parametrize("name", NAMES)
def test_reverse_mode(pkg, name):
    """The operators with a gradient have their own node, the others PyTorch's that warns."""
    with FakeTensorMode():
        at, call, has_gradient = calls(pkg)[name]
        out = call(at.clone().requires_grad_())
        assert out.requires_grad
        with torch.no_grad():
            assert not call(at.clone().requires_grad_()).requires_grad
        with torch.inference_mode():
            assert call(at.clone()).shape == out.shape
        assert ("WarnNotImplemented" in out.grad_fn.name()) != has_gradient
