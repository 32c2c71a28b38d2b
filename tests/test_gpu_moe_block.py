"""The mixture-of-experts block operators as they are used together: norm, router, routing with quantisation, the experts'
products, the way back and the next norm, against the same chain of CPU oracles fed with the kernels' own intermediate
results, and a training step through the differentiable operators against float64 autograd."""
import pytest
import torch

from oracle import moe_oracle as oracle
from oracle import quant_oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pb():
    import pytorch_b200
    import pytorch_b200.contrib.function  # noqa: F401
    assert torch.cuda.is_available()
    return pytorch_b200


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    from pytorch_b200 import _cabi
    torch.cuda.synchronize()
    assert _cabi.device_error() == 0


def router(x, w, topk):
    top, idx = torch.topk(x.float() @ w, topk, dim=1)
    return idx.to(torch.int32), torch.softmax(top, dim=1)


def parts(e, k, f, g):
    scale = lambda *s: torch.rand(s, generator=g) * 2e-3 + 1e-3  # noqa: E731
    return dict(w_gate_up=torch.randint(-127, 128, (e, 2 * f, k), generator=g).to(torch.int8), scale_gate_up=scale(e, 2 * f),
                w_down=torch.randint(-127, 128, (e, k, f), generator=g).to(torch.int8), scale_down=scale(e, k),
                smooth_in=torch.rand((e, k), generator=g) + 0.5, smooth_act=torch.rand(f, generator=g) + 0.5)


@pytest.mark.parametrize("tokens", [1, 5, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_block_forward(pb, tokens, dtype):
    e, k, f, topk = 8, 256, 128, 2
    g = torch.Generator().manual_seed(tokens)
    p = parts(e, k, f, g)
    c = {n: t.cuda() for n, t in p.items()}
    gamma, post = (torch.rand(k, generator=g) + 0.5).to(dtype), (torch.rand(k, generator=g) + 0.5).to(dtype)
    attn, res = torch.randn((tokens, k), generator=g).to(dtype), torch.randn((tokens, k), generator=g).to(dtype)
    npu = torch.ops.npu
    y, _, h, _ = npu.npu_gated_add_rms_norm(attn.cuda(), res.cuda(), gamma.cuda(), post_gamma=post.cuda())
    idx, weight = router(y, torch.randn((k, e), generator=g).cuda(), topk)
    if tokens > 4:
        idx[-2:] = -1                                              # padded tokens
    out = pb.contrib.function.w8a8_swiglu_moe(y, idx, weight, c["smooth_in"], c["w_gate_up"], c["scale_gate_up"], c["smooth_act"], c["w_down"],
                                              c["scale_down"])
    nxt, scale, h2 = npu.npu_gated_add_rms_norm_dynamic_quant(out, h, gamma.cuda(), post_gamma=post.cuda(), residual_scale=0.5)
    assert out.shape == (tokens, k) and torch.isfinite(out.float()).all() and (tokens <= 4 or float(out[-2:].abs().max()) == 0)
    # the integer parts bit for bit, each from the result before it
    row, src, counts = oracle.sorted_rows(idx.cpu(), 0, e)
    q, place, ends, s = npu.npu_moe_init_routing_v2(y, idx, scale=c["smooth_in"], expert_num=e, quant_mode=1)
    qo, so = oracle.route_quantised(y.cpu(), idx.cpu(), p["smooth_in"], 0, e)
    assert torch.equal(q.cpu(), qo) and torch.equal(s.cpu(), so) and torch.equal(place.cpu(), row) and torch.equal(ends.cpu(), torch.cumsum(counts, 0))
    gu = npu.npu_grouped_matmul([q], [c["w_gate_up"].transpose(1, 2)], scale=[c["scale_gate_up"]], per_token_scale=[s], group_list=ends, split_item=3,
                                output_dtype=dtype)[0]
    assert torch.equal(gu.cpu(), oracle.grouped_matmul(qo, p["w_gate_up"].transpose(1, 2), torch.cumsum(counts, 0), p["scale_gate_up"], so, None, dtype))
    qa, sa = npu.npu_swiglu_quant(gu, smooth_scales=c["smooth_act"], activate_left=True, quant_mode=1)
    rows = oracle.grouped_matmul(qa.cpu(), p["w_down"].transpose(1, 2), torch.cumsum(counts, 0), p["scale_down"], sa.cpu(), None, dtype)
    want, size = oracle.combine(rows, row, weight.cpu(), tokens, topk)
    tol = want.abs() * (torch.finfo(dtype).eps / 2) * (1 + 1e-6) + (topk + 1) * 2.0 ** -24 * size + torch.finfo(dtype).tiny
    assert bool(((out.cpu().double() - want).abs() <= tol).all())
    # the int8 activations against the CPU's: exp differs in its last bits, so a value next to a boundary may move by a step
    qs, ss = quant_oracle.swiglu_quant(gu.cpu(), p["smooth_act"], True)
    assert torch.allclose(sa.cpu(), ss, rtol=1e-5) and int((qa.cpu().int() - qs.int()).abs().max()) <= 1
    h64 = 0.5 * h.cpu().double() + oracle.gated_add_rms_norm(out.cpu(), h.cpu(), gamma, post, None, 0.0, 1e-6)[1]
    assert bool(((h2.cpu().double() - h64).abs() <= h64.abs() * (torch.finfo(dtype).eps / 2) + h64.abs().max() * 2.0 ** -24 * (24 + k)).all())
    assert nxt.dtype == torch.int8 and scale.shape == (tokens,)


def test_experts_split_over_two_ranks_add_up(pb):
    """Two halves of the experts, as on two ranks: each has its experts' rows only, and their results add up to the whole."""
    e, k, f, topk, tokens = 8, 128, 64, 3, 200
    g = torch.Generator().manual_seed(1)
    c = {n: t.cuda() for n, t in parts(e, k, f, g).items()}
    x = torch.randn((tokens, k), generator=g).to(torch.bfloat16).cuda()
    idx, weight = router(x, torch.randn((k, e), generator=g).cuda(), topk)
    run = pb.contrib.function.w8a8_swiglu_moe
    whole = run(x, idx, weight, c["smooth_in"], c["w_gate_up"], c["scale_gate_up"], c["smooth_act"], c["w_down"], c["scale_down"])
    halves = [run(x, idx, weight, c["smooth_in"][a:b], c["w_gate_up"][a:b], c["scale_gate_up"][a:b], c["smooth_act"], c["w_down"][a:b], c["scale_down"][a:b],
                  expert_range=(a, b), expert_num=e) for a, b in ((0, 4), (4, 8))]
    # three roundings to bf16 of values no larger than the parts' magnitudes
    size = halves[0].double().abs() + halves[1].double().abs()
    assert bool(((halves[0].double() + halves[1].double() - whole.double()).abs() <= size * 3 * 2.0 ** -8 + 1e-6).all())


def test_training_step(pb):
    """Norm, permute, a dense float product per expert, unpermute and norm: gradients of every leaf against float64 autograd of the
    definitions.  All in float32: some hundreds of fp32 operations on values of order ten, so 1e-4 of each gradient's largest value."""
    npu = torch.ops.npu
    e, k, topk, tokens = 4, 64, 2, 40
    g = torch.Generator().manual_seed(7)
    leaves = dict(x=torch.randn((tokens, k), generator=g), res=torch.randn((tokens, k), generator=g), gamma=torch.rand(k, generator=g) + 0.5,
                  post=torch.rand(k, generator=g) + 0.5, gate=torch.rand(k, generator=g) + 0.5, w=torch.randn((e, k, k), generator=g) / 8,
                  weight=torch.softmax(torch.randn((tokens, topk), generator=g), 1))
    idx = torch.stack([torch.randperm(e, generator=g)[:topk] for _ in range(tokens)]).to(torch.int32)
    idx[-3:] = -1
    row, src, counts = oracle.sorted_rows(idx, 0, e)
    dout = torch.randn((tokens, k), generator=g)

    def plain(a):
        def norm(x, res, gate):
            z = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * a["post"]
            h = 0.7 * res + gate * z
            return h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * a["gamma"], h
        y, h = norm(a["x"], a["res"], a["gate"])
        live = src >= 0
        rows = torch.zeros((tokens * topk, k), dtype=torch.float64)
        expert = idx.reshape(-1)[src[live].long()].long()
        out = torch.einsum("rk,rkn->rn", y[(src[live] // topk).long()], a["w"][expert])
        rows = rows.index_copy(0, torch.nonzero(live)[:, 0], out)
        t, s = torch.nonzero(idx >= 0, as_tuple=True)
        back = torch.zeros((tokens, k), dtype=torch.float64).index_add(0, t, rows[row.reshape(tokens, topk)[t, s].long()] * a["weight"][t, s][:, None])
        return norm(back, h, 1.0)[0]

    a64 = {n: v.double().requires_grad_() for n, v in leaves.items()}
    want = torch.autograd.grad((plain(a64) * dout.double()).sum(), list(a64.values()))
    a = {n: v.cuda().requires_grad_() for n, v in leaves.items()}
    y, _, h, _ = npu.npu_gated_add_rms_norm(a["x"], a["res"], a["gamma"], post_gamma=a["post"], gate=a["gate"], residual_scale=0.7)
    rows, place = npu.npu_moe_token_permute(y, idx.cuda())
    n = int(counts.sum())
    expert = torch.repeat_interleave(torch.arange(e), counts).cuda()
    prod = torch.cat([torch.einsum("rk,rkn->rn", rows[:n], a["w"][expert]), torch.zeros((tokens * topk - n, k), device="cuda")])
    back = npu.npu_moe_token_unpermute(prod, place, a["weight"])
    out, _, _, _ = npu.npu_gated_add_rms_norm(back, h, a["gamma"], post_gamma=a["post"], residual_scale=0.7)
    got = torch.autograd.grad((out * dout.cuda()).sum(), list(a.values()))
    for name, u, v in zip(leaves, got, want):
        # the padded tokens' last norm has a mean of squares of zero: epsilon makes its factor 1000
        assert bool(((u.cpu().double() - v).abs() <= 1e-4 * v.abs().max()).all()), name


def test_fake_tensors_in_both_directions(pb):
    """Under a dispatch mode a training step runs on shapes alone: the gradients are operators that the mode sees."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        def leaf(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda", requires_grad=True)

        x, res, w, post, gate, probs = leaf(6, 64), leaf(6, 64), leaf(64), leaf(64), leaf(6, 1), leaf(6, 2, dtype=torch.float32)
        y, _, h, _ = pb.npu_gated_add_rms_norm(x, res, w, post_gamma=post, gate=gate)
        rows, place = pb.npu_moe_token_permute(y, torch.empty(6, 2, dtype=torch.int64, device="cuda"))
        (pb.npu_moe_token_unpermute(rows, place, probs).sum() + h.sum()).backward()
        for t in (x, res, w, post, gate, probs):
            assert t.grad.shape == t.shape and t.grad.dtype == t.dtype and t.grad.device.type == "cuda"
