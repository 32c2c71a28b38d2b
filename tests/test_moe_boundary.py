"""Host-side checks of the mixture-of-experts block operators that need no GPU: shape contracts on meta tensors, refusals
of arguments, and the C ABI's argument checks (every call fails, or has nothing to do, before it touches the device)."""
import ctypes as C

import pytest
import torch

from pytorch_b200 import _cabi as cabi


@pytest.fixture(scope="module")
def pkg():
    import pytorch_b200
    return pytorch_b200


@pytest.fixture(scope="module")
def lib():
    return cabi.lib()


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


I32, I64, F32 = torch.int32, torch.int64, torch.float32


def test_routing_meta_contract(pkg):
    q, place, tokens, scale = pkg.npu_moe_init_routing_v2(meta(10, 64), meta(10, 4, dtype=I32), scale=meta(16, 64, dtype=F32), expert_num=16, quant_mode=1)
    assert q.shape == (40, 64) and q.dtype == torch.int8 and place.shape == (40,) and place.dtype == I32
    assert tokens.shape == (16,) and tokens.dtype == I64 and scale.shape == (40,) and scale.dtype == F32
    r, _, tokens, scale = pkg.npu_moe_init_routing_v2(meta(10, 64), meta(10, 4, dtype=I64), expert_num=16, active_expert_range=[4, 10])
    assert r.shape == (40, 64) and r.dtype == torch.bfloat16 and tokens.shape == (6,) and scale.shape == (0,)
    for kw, what in [(dict(expert_num=0), "expert_num"), (dict(expert_num=2000), "at most 1024"), (dict(expert_num=8, quant_mode=0), "quant_mode"),
                     (dict(expert_num=8, drop_pad_mode=1), "drop_pad_mode"), (dict(expert_num=8, expert_tokens_num_type=2), "expert_tokens_num_type"),
                     (dict(expert_num=8, active_num=7), "active_num"), (dict(expert_num=8, row_idx_type=2), "row_idx_type"),
                     (dict(expert_num=8, active_expert_range=[3, 9]), "active_expert_range"), (dict(expert_num=8, offset=meta(8)), "offset"),
                     (dict(expert_num=8, quant_mode=1, scale=meta(7, 64, dtype=F32)), "smooth scales"), (dict(expert_num=8, scale=meta(9, dtype=F32)), "scale must be")]:
        with pytest.raises(RuntimeError, match=what):
            pkg.npu_moe_init_routing_v2(meta(10, 64), meta(10, 4, dtype=I32), **kw)
    with pytest.raises(RuntimeError, match="tokens, topk"):
        pkg.npu_moe_init_routing_v2(meta(10, 64), meta(9, 4, dtype=I32), expert_num=8)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        pkg.npu_moe_init_routing_v2(meta(10, 64), meta(10, 4, dtype=F32), expert_num=8)


def test_permute_and_unpermute_meta_contract(pkg):
    rows, place = pkg.npu_moe_token_permute(meta(10, 64), meta(10, 4, dtype=I64))
    assert rows.shape == (40, 64) and place.shape == (40,) and place.dtype == I32
    assert pkg.npu_moe_token_permute(meta(10, 64), meta(10, dtype=I32), 7)[0].shape == (7, 64)
    assert pkg.npu_moe_token_permute(meta(10, 64), meta(10, 2, dtype=I32), 100)[0].shape == (20, 64)
    assert pkg.npu_moe_token_permute(meta(10, 64), meta(10, 2, dtype=I32), -3)[0].shape == (17, 64)
    y = pkg.npu_moe_token_unpermute(rows, place, meta(10, 4, dtype=F32))
    assert y.shape == (10, 64) and y.dtype == torch.bfloat16
    assert pkg.npu_moe_token_unpermute(rows, place).shape == (40, 64)
    d, w = pkg.npu_moe_token_unpermute_grad(rows, y, place, meta(10, 4, dtype=F32))
    assert d.shape == rows.shape and w.shape == (10, 4) and w.dtype == F32
    assert pkg.npu_moe_token_permute_grad(meta(10, 64), rows, meta(10, 4, dtype=I64), place).shape == (10, 64)
    with pytest.raises(RuntimeError, match="padded_mode"):
        pkg.npu_moe_token_permute(meta(10, 64), meta(10, 4, dtype=I64), None, True)
    with pytest.raises(RuntimeError, match="num_tokens"):
        pkg.npu_moe_token_permute(meta(10, 64), meta(11, 4, dtype=I64))
    with pytest.raises(RuntimeError, match="padded_mode"):
        pkg.npu_moe_token_unpermute(rows, place, None, False, [10, 64])
    with pytest.raises(RuntimeError, match="int32"):
        pkg.npu_moe_token_unpermute(rows, meta(40, dtype=I64))
    with pytest.raises(RuntimeError, match="do not match"):
        pkg.npu_moe_token_unpermute(rows, place, meta(10, 3, dtype=F32))
    with pytest.raises(RuntimeError, match="grad_unpermuted_tokens"):
        pkg.npu_moe_token_unpermute_grad(rows, meta(10, 32), place, meta(10, 4, dtype=F32))
    with pytest.raises(NotImplementedError):
        pkg.npu_moe_token_permute(torch.zeros(2, 8), torch.zeros(2, 1, dtype=I32))


def test_route_argument_checks(lib):
    last = lambda: lib.b200q_last_error().decode()  # noqa: E731
    assert lib.b200q_moe_route(None, None) == cabi.ERR_BAD_ARG
    buf = (C.c_uint8 * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256

    def args(**kw):
        a = cabi.MoeRouteArgs()
        a.x, a.x_dtype, a.expert_idx, a.idx_dtype, a.tokens, a.topk, a.hidden = p, cabi.BF16, p, cabi.I32, 4, 2, 8
        a.expert_begin, a.expert_end, a.out, a.out_rows, a.row_idx = 0, 8, p, 8, p
        for k, v in kw.items():
            setattr(a, k, v)
        return C.byref(a)

    for kw, status, what in [
            (dict(tokens=-1), cabi.ERR_BAD_ARG, "negative"), (dict(topk=2000), cabi.ERR_UNSUPPORTED, "1024 slots"),
            (dict(tokens=2 ** 31), cabi.ERR_UNSUPPORTED, "assignments"), (dict(idx_dtype=cabi.F32), cabi.ERR_UNSUPPORTED, "i32 or i64"),
            (dict(expert_end=2000), cabi.ERR_UNSUPPORTED, "1 to 1024"), (dict(expert_end=0), cabi.ERR_UNSUPPORTED, "1 to 1024"),
            (dict(out_rows=9), cabi.ERR_BAD_ARG, "out_rows"), (dict(x_dtype=cabi.I64), cabi.ERR_UNSUPPORTED, "dtype"),
            (dict(scale=p, scale_dtype=cabi.F32), cabi.ERR_BAD_ARG, "out_scale"), (dict(expert_idx=None), cabi.ERR_BAD_ARG, "NULL"),
            (dict(x=None), cabi.ERR_BAD_ARG, "NULL"), (dict(x=p + 1), cabi.ERR_BAD_ARG, "misaligned"), (dict(row_idx=p + 2), cabi.ERR_BAD_ARG, "misaligned"),
            (dict(quantise=1, x_dtype=cabi.F32), cabi.ERR_UNSUPPORTED, "bf16 or f16"), (dict(quantise=1, out_rows=7, out_scale=p), cabi.ERR_BAD_ARG, "every row"),
            (dict(quantise=1), cabi.ERR_BAD_ARG, "out_scale"),
            (dict(quantise=1, out_scale=p, scale=p, scale_dtype=cabi.F32, scale_rows=3), cabi.ERR_BAD_ARG, "one row"),
            (dict(tokens=2000, out_rows=4000), cabi.ERR_WORKSPACE, "workspace")]:
        assert lib.b200q_moe_route(args(**kw), None) == status and what in last(), (kw, last())
    assert lib.b200q_moe_route(args(tokens=0, out_rows=0), None) == cabi.OK
    assert lib.b200q_moe_route_workspace_bytes(2048, 1) == 0 and lib.b200q_moe_route_workspace_bytes(0, 1) == 0
    assert lib.b200q_moe_route_workspace_bytes(4096, 1) == 256 + 8 * 4096 and lib.b200q_moe_route_workspace_bytes(4096, 0) == 256


def test_combine_argument_checks(lib):
    last = lambda: lib.b200q_last_error().decode()  # noqa: E731
    buf = (C.c_uint8 * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256

    def fwd(rows=p, dtype=cabi.BF16, n=4, idx=p, w=None, wd=cabi.NONE, out=p, t=2, k=2, h=8):
        return lib.b200q_moe_combine(rows, dtype, n, idx, w, wd, out, t, k, h, None)

    assert fwd(dtype=cabi.I8) == cabi.ERR_UNSUPPORTED and fwd(k=0) == cabi.ERR_BAD_ARG and fwd(t=-1) == cabi.ERR_BAD_ARG
    assert fwd(w=p, wd=cabi.I32) == cabi.ERR_UNSUPPORTED and "weights" in last()
    assert fwd(k=2000) == cabi.ERR_UNSUPPORTED and fwd(rows=None) == cabi.ERR_BAD_ARG and fwd(out=p + 1) == cabi.ERR_BAD_ARG
    assert fwd(t=0) == cabi.OK and fwd(h=0) == cabi.OK

    def bwd(**kw):
        a = cabi.MoeCombineGradArgs()
        a.dy, a.dtype, a.rows, a.num_rows, a.row_idx, a.weight_dtype = p, cabi.BF16, p, 4, p, cabi.NONE
        a.tokens, a.topk, a.hidden, a.drows, a.workspace, a.workspace_bytes = 2, 2, 8, p, p, 256
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.b200q_moe_combine_grad(C.byref(a), None)

    assert lib.b200q_moe_combine_grad(None, None) == cabi.ERR_BAD_ARG
    assert bwd(dtype=cabi.I8) == cabi.ERR_UNSUPPORTED and bwd(topk=0) == cabi.ERR_BAD_ARG
    assert bwd(dweights=p) == cabi.ERR_UNSUPPORTED and bwd(dweights=p, weight_dtype=cabi.F32, rows=None) == cabi.ERR_BAD_ARG
    assert bwd(workspace_bytes=0) == cabi.ERR_WORKSPACE and bwd(workspace=p + 16) == cabi.ERR_WORKSPACE
    assert bwd(drows=None) == cabi.ERR_BAD_ARG and bwd(num_rows=0) == cabi.OK
    assert lib.b200q_moe_combine_grad_workspace_bytes(33) == 256 and lib.b200q_moe_combine_grad_workspace_bytes(0) == 0


def test_gated_norm_meta_contract(pkg):
    x, w = meta(4, 6, 64), meta(64)
    y, rstd, h, prstd = pkg.npu_gated_add_rms_norm(x, x, w, post_gamma=w, gate=meta(4, 1, 64))
    assert y.shape == h.shape == x.shape and rstd.shape == prstd.shape == (4, 6) and rstd.dtype == F32
    assert pkg.npu_gated_add_rms_norm(x, x, w)[3].shape == (0,)
    q, s, h = pkg.npu_gated_add_rms_norm_dynamic_quant(x, x, w, gate=meta(4, 6, 1), smooth_scales=meta(64, dtype=F32))
    assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == (4, 6) and h.dtype == torch.bfloat16
    g = pkg.npu_gated_add_rms_norm_grad(y, None, x, x, w, rstd, post_gamma=w, gate=meta(64, dtype=F32), post_rstd=prstd)
    assert [t.shape for t in g] == [x.shape, x.shape, w.shape, w.shape, (64,)] and g[4].dtype == F32
    for gate in (meta(6, 64), meta(1, 6, 64), meta(4, 1, 1), meta(1, 1, 1), meta(4, 6, 32), meta(1), meta(6, 1)):
        with pytest.raises(RuntimeError, match="gate"):
            pkg.npu_gated_add_rms_norm(x, x, w, gate=gate)
    for kw, what in [(dict(residual=meta(4, 64)), "residual"), (dict(residual=meta(4, 6, 64, dtype=F32)), "residual"), (dict(gamma=meta(32)), "gamma"),
                     (dict(post_gamma=meta(4, 64)), "post_gamma"), (dict(x=meta(4, 6, 64, dtype=I32)), "x must be"),
                     (dict(gate=meta(64, dtype=I32)), "gate must be")]:
        a = dict(x=x, residual=x, gamma=w) | kw
        with pytest.raises(RuntimeError, match=what):
            pkg.npu_gated_add_rms_norm(a.pop("x"), a.pop("residual"), a.pop("gamma"), **a)
    with pytest.raises(RuntimeError, match="smooth_scales"):
        pkg.npu_gated_add_rms_norm_dynamic_quant(x, x, w, smooth_scales=meta(32))
    with pytest.raises(RuntimeError, match="post_rstd"):
        pkg.npu_gated_add_rms_norm_grad(y, None, x, x, w, rstd, post_gamma=w)
    with pytest.raises(RuntimeError, match="rstd must be"):
        pkg.npu_gated_add_rms_norm_grad(y, None, x, x, w, meta(4, 5, dtype=F32))
    with pytest.raises(RuntimeError, match="grad_y"):
        pkg.npu_gated_add_rms_norm_grad(meta(4, 6, 32), None, x, x, w, rstd)


def test_gated_norm_argument_checks(lib):
    last = lambda: lib.b200q_last_error().decode()  # noqa: E731
    buf = (C.c_uint8 * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256

    def args(**kw):
        a = cabi.GatedNormArgs()
        a.x = a.residual = a.gamma = a.y = a.h = p
        a.dtype, a.param_dtype, a.rows, a.width, a.gate_rows = cabi.BF16, cabi.BF16, 2, 16, 1
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    fwd = lambda **kw: lib.b200q_gated_norm(C.byref(args(**kw)), None)  # noqa: E731
    assert lib.b200q_gated_norm(None, None) == cabi.ERR_BAD_ARG
    for kw, status, what in [
            (dict(rows=-1), cabi.ERR_BAD_ARG, "negative"), (dict(dtype=cabi.I8), cabi.ERR_UNSUPPORTED, "bf16, f16 or f32"),
            (dict(width=16385), cabi.ERR_UNSUPPORTED, "at most 16384"), (dict(param_dtype=cabi.F16), cabi.ERR_UNSUPPORTED, "gamma"),
            (dict(gate=p, gate_rows=0), cabi.ERR_BAD_ARG, "gate_rows"), (dict(gate=p, gate_rows=2, gate_per_row=1), cabi.ERR_UNSUPPORTED, "one row"),
            (dict(smooth=p), cabi.ERR_BAD_ARG, "quantised"), (dict(scale=p, smooth=p, smooth_dtype=cabi.I8), cabi.ERR_UNSUPPORTED, "smooth"),
            (dict(x=None), cabi.ERR_BAD_ARG, "NULL"), (dict(h=p + 1), cabi.ERR_BAD_ARG, "misaligned"), (dict(rstd=p + 2), cabi.ERR_BAD_ARG, "misaligned")]:
        assert fwd(**kw) == status and what in last(), (kw, last())
    assert fwd(rows=0) == cabi.OK and fwd(width=0) == cabi.OK

    def bwd(a=None, **kw):
        g = cabi.GatedNormGrads()
        g.dy = g.dx = g.dresidual = g.dgamma = g.workspace = p
        g.workspace_bytes = 4096
        for k, v in kw.items():
            setattr(g, k, v)
        return lib.b200q_gated_norm_grad(C.byref(a or args(rstd=p)), C.byref(g), None)

    assert bwd(a=args()) == cabi.ERR_BAD_ARG and "NULL" in last()
    assert bwd(dy=None) == cabi.ERR_BAD_ARG and bwd(dgamma=p + 1) == cabi.ERR_BAD_ARG
    assert bwd(workspace_bytes=64) == cabi.ERR_WORKSPACE and bwd(workspace=p + 16) == cabi.ERR_WORKSPACE
    assert bwd(a=args(rstd=p, gate=p)) == cabi.ERR_BAD_ARG                       # no place for the gate's gradient
    assert bwd(a=args(rstd=p, post_gamma=p, post_rstd=p)) == cabi.ERR_BAD_ARG
    assert lib.b200q_gated_norm_grad_workspace_bytes(C.byref(args())) == 2 * 2 * 16 * 4
    assert lib.b200q_gated_norm_grad_workspace_bytes(C.byref(args(gate=p, gate_rows=2))) == (2 * 2 + 2 + 1) * 16 * 4
    assert bwd(a=args(rstd=p, rows=70000 * 2, gate=p, gate_rows=2), dgate=p) == cabi.ERR_UNSUPPORTED and "65533" in last()


def test_grouped_matmul_meta_contract(pkg):
    x, w = meta(40, 64, dtype=torch.int8), meta(4, 64, 24, dtype=torch.int8)
    sc, rs, gl = meta(4, 24, dtype=F32), meta(40, dtype=F32), meta(4, dtype=I64)
    ok = dict(scale=[sc], per_token_scale=[rs], group_list=gl, split_item=3, output_dtype=torch.float16)
    out = pkg.npu_grouped_matmul([x], [w], **ok)
    assert len(out) == 1 and out[0].shape == (40, 24) and out[0].dtype == torch.float16
    assert pkg.npu_grouped_matmul([x], [w], group_list=gl, split_item=2, output_dtype=I32)[0].dtype == I32
    for kw, what in [(dict(split_item=0), "split_item"), (dict(group_type=2), "group_type"), (dict(group_list_type=2), "group_list_type"),
                     (dict(act_type=1), "act_type"), (dict(group_list=None), "group_list"), (dict(group_list=meta(3, dtype=I64)), "group_list"),
                     (dict(group_list=meta(4, dtype=F32)), "group_list"), (dict(scale=None), "scale is needed"), (dict(scale=[meta(4, 23, dtype=F32)]), "scale"),
                     (dict(scale=[sc, sc]), "one tensor"), (dict(per_token_scale=[meta(39, dtype=F32)]), "per_token_scale"),
                     (dict(bias=[meta(24, dtype=F32)]), "bias"), (dict(output_dtype=F32), "output_dtype"), (dict(offset=[sc]), "not implemented"),
                     (dict(antiquant_scale=[sc]), "not implemented")]:
        with pytest.raises(RuntimeError, match=what):
            pkg.npu_grouped_matmul([x], [w], **(ok | kw))
    with pytest.raises(RuntimeError, match="one x"):
        pkg.npu_grouped_matmul([x, x], [w], **ok)
    with pytest.raises(RuntimeError, match="int8"):
        pkg.npu_grouped_matmul([meta(40, 64)], [w], **ok)
    with pytest.raises(RuntimeError, match="inner dimensions"):
        pkg.npu_grouped_matmul([meta(40, 32, dtype=torch.int8)], [w], **ok)
    with pytest.raises(RuntimeError, match="bias"):
        pkg.npu_grouped_matmul([x], [w], group_list=gl, split_item=2, output_dtype=I32, bias=[meta(4, 24, dtype=F32)])


def test_grouped_matmul_argument_checks(lib):
    last = lambda: lib.b200q_last_error().decode()  # noqa: E731
    buf = (C.c_uint8 * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256

    def run(**kw):
        a = cabi.GroupedMatmulArgs()
        a.x = a.weight = a.group_list = a.scale = a.out = p
        a.m, a.k, a.n, a.groups, a.w_stride_g, a.w_stride_k, a.w_stride_n = 4, 16, 8, 2, 128, 1, 16
        a.scale_dtype, a.bias_dtype, a.out_dtype = cabi.F32, cabi.NONE, cabi.BF16
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.b200q_grouped_matmul(C.byref(a), None)

    assert lib.b200q_grouped_matmul(None, None) == cabi.ERR_BAD_ARG
    for kw, status, what in [
            (dict(m=-1), cabi.ERR_BAD_ARG, "negative"), (dict(groups=0), cabi.ERR_UNSUPPORTED, "groups"), (dict(groups=1025), cabi.ERR_UNSUPPORTED, "groups"),
            (dict(m=2 ** 31), cabi.ERR_UNSUPPORTED, "out of range"), (dict(out_dtype=cabi.I8), cabi.ERR_UNSUPPORTED, "output dtype"),
            (dict(scale_dtype=cabi.F16), cabi.ERR_UNSUPPORTED, "scale"), (dict(bias=p, bias_dtype=cabi.I8), cabi.ERR_UNSUPPORTED, "bias"),
            (dict(out_dtype=cabi.I32, bias=p, bias_dtype=cabi.F32), cabi.ERR_UNSUPPORTED, "bias"), (dict(group_list=None), cabi.ERR_BAD_ARG, "NULL"),
            (dict(scale=None), cabi.ERR_BAD_ARG, "NULL"), (dict(group_list=p + 4), cabi.ERR_BAD_ARG, "misaligned"),
            (dict(out=p + 1), cabi.ERR_BAD_ARG, "misaligned")]:
        assert run(**kw) == status and what in last(), (kw, last())
    assert run(m=0) == cabi.OK and run(n=0) == cabi.OK


def test_fake_tensors():
    """Under a dispatch mode the operators run on shapes alone, also where autograd is on (the backward pass itself needs a
    device for its thread)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    import pytorch_b200 as pkg
    with FakeTensorMode():
        def leaf(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda", requires_grad=True)

        x, res, w, post, gate = leaf(6, 64), leaf(6, 64), leaf(64), leaf(64), leaf(6, 1)
        y, rstd, h, post_rstd = pkg.npu_gated_add_rms_norm(x, res, w, post_gamma=post, gate=gate)
        assert y.requires_grad and h.requires_grad and not rstd.requires_grad and not post_rstd.requires_grad
        rows, sorted_idx = pkg.npu_moe_token_permute(y, torch.empty(6, 2, dtype=torch.int64, device="cuda"))
        assert rows.shape == (12, 64) and sorted_idx.shape == (12,) and sorted_idx.dtype == torch.int32
        probs = leaf(6, 2, dtype=torch.float32)
        out = pkg.npu_moe_token_unpermute(rows, sorted_idx, probs)
        assert out.shape == (6, 64) and out.dtype == torch.bfloat16
        assert out.requires_grad
        grads = torch.ops.npu.npu_gated_add_rms_norm_grad(torch.empty_like(y), None, x, res, w, rstd, post_gamma=post, gate=gate, post_rstd=post_rstd)
        assert [g.shape for g in grads] == [t.shape for t in (x, res, w, post, gate)]
        grads = torch.ops.npu.npu_moe_token_unpermute_grad(rows, torch.empty_like(out), sorted_idx, probs)
        assert grads[0].shape == rows.shape and grads[1].shape == probs.shape
        q, ri, et, sc = pkg.npu_moe_init_routing_v2(y.detach(), torch.empty(6, 2, dtype=torch.int32, device="cuda"), expert_num=4, active_num=12,
                                                    quant_mode=1, expert_tokens_num_flag=True, expert_tokens_num_type=0)
        assert q.shape == (12, 64) and q.dtype == torch.int8 and ri.shape == (12,) and et.shape == (4,) and sc.shape == (12,)
        got = pkg.npu_grouped_matmul([q], [torch.empty(4, 64, 32, dtype=torch.int8, device="cuda")], scale=[torch.empty(4, 32, device="cuda")],
                                     per_token_scale=[sc], group_list=et, split_item=3, group_type=0, group_list_type=0)
        assert got[0].shape == (12, 32) and got[0].dtype == torch.bfloat16
