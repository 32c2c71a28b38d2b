"""The mixture-of-experts block operators on tensors of more than 2^31 elements: what lies behind the 32-bit range is
checked on its own, exactly where the result is a copy or an integer and against float64 where it is a sum."""
import gc

import pytest
import torch

from oracle import moe_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def npu():
    import pytorch_b200  # noqa: F401
    assert torch.cuda.is_available()
    return torch.ops.npu


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    from pytorch_b200 import _cabi
    torch.cuda.synchronize()
    assert _cabi.device_error() == 0
    gc.collect()
    torch.cuda.empty_cache()


def filled(shape, dtype, seed):
    """Values that differ from row to row without a 64-bit random tensor of the full size."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn((257, shape[1]), generator=g, device="cuda")
    t = torch.empty(shape, dtype=dtype, device="cuda")
    for a in range(0, shape[0], 257):
        b = min(shape[0], a + 257)
        t[a:b] = base[: b - a] * (1 + (a // 257) % 31)
    return t


ENDS = lambda n: torch.cat([torch.arange(40), torch.arange(n - 40, n)])  # noqa: E731


@pytest.mark.parametrize("hidden", [8192, 8195])
def test_permute_and_unpermute(npu, hidden):
    t, k, e = 33000, 8, 64
    assert t * k * hidden > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.topk(torch.rand((t, e), generator=g, device="cuda"), k).indices
    x = filled((t, hidden), torch.bfloat16, 2)
    rows, place = npu.npu_moe_token_permute(x, ids)
    at = place.view(t, k).long()
    assert torch.equal(at.flatten().sort().values, torch.arange(t * k, device="cuda"))
    ends = ENDS(t).cuda()
    assert torch.equal(rows[at[ends]], x[ends, None].expand(-1, k, -1))
    last = torch.arange(t * k - 64, t * k, device="cuda")                              # the rows furthest back
    owner = torch.empty(t * k, dtype=torch.int64, device="cuda").scatter_(0, place.long(), torch.arange(t * k, device="cuda"))
    assert torch.equal(rows[last], x[owner[last] // k])
    probs = torch.softmax(torch.randn((t, k), generator=g, device="cuda"), -1)
    leaf, weight = rows.clone().requires_grad_(), probs.clone().requires_grad_()
    out = npu.npu_moe_token_unpermute(leaf, place, weight)
    want = (rows[at[ends]].double() * probs[ends, :, None].double()).sum(1)
    size = (rows[at[ends]].double() * probs[ends, :, None].double()).abs().sum(1)
    assert bool(((out.detach()[ends].double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.0001 + size * 2.0 ** -24 * (k + 1)).all())
    dy = filled((t, hidden), torch.bfloat16, 3)
    out.backward(dy)
    want = dy[ends, None].double() * probs[ends, :, None].double()
    assert bool(((leaf.grad[at[ends]].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -23)).all())
    terms = rows[at[ends]].double() * dy[ends, None].double()
    assert bool(((weight.grad[ends].double() - terms.sum(-1)).abs() <= terms.abs().sum(-1) * 2.0 ** -24 * hidden).all())


@pytest.mark.parametrize("hidden", [8192, 8200])
def test_quantised_routing(npu, hidden):
    t, k, e = 33000, 8, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.topk(torch.rand((t, e), generator=g, device="cuda"), k).indices.int()
    x = filled((t, hidden), torch.bfloat16, 5)
    q, place, tokens, scale = npu.npu_moe_init_routing_v2(x, ids, expert_num=e, quant_mode=1, expert_tokens_num_flag=True)
    assert int(tokens[-1]) == t * k
    ends = ENDS(t)
    at = place.view(t, k).cpu().long()[ends]
    last = at.flatten().topk(16).indices                                              # among them the rows furthest back
    assert int(at.flatten()[last].max()) * hidden > 2 ** 31
    # One expert a token leaves the rows in their order.
    want, want_scale = oracle.route_quantised(x[ends.cuda()].cpu(), torch.zeros((len(ends), 1), dtype=torch.int32), None, 0, 1)
    assert torch.equal(q[at.cuda()].cpu(), want[:, None].expand(-1, k, -1))
    assert torch.equal(scale[at.cuda()].cpu(), want_scale[:, None].expand(-1, k))


@pytest.mark.parametrize("width,gate", [(16384, "channel"), (4092, "row")])
def test_norm_and_its_gradient(npu, width, gate):
    n = 2 ** 31 // width + 100
    x, res = filled((n, width), torch.bfloat16, 6), filled((n, width), torch.bfloat16, 7)
    g = torch.Generator(device="cuda").manual_seed(8)
    gamma = (torch.randn(width, generator=g, device="cuda") * 0.2 + 1).bfloat16()
    gt = torch.randn((width,) if gate == "channel" else (n, 1), generator=g, device="cuda").bfloat16()
    ends = ENDS(n).cuda()
    leaves = [t.requires_grad_() for t in (x, res, gamma, gt)]
    y, rstd, h, _ = npu.npu_gated_add_rms_norm(x, res, gamma, gate=gt, epsilon=1e-6)
    sub = [t.detach()[ends].cpu().double().requires_grad_() for t in (x, res)]
    w64 = gamma.detach().cpu().double().requires_grad_()
    g64 = (gt.detach() if gate == "channel" else gt.detach()[ends]).cpu().double().requires_grad_()
    h64 = sub[1] + sub[0] * g64
    y64 = h64 * torch.rsqrt((h64 * h64).mean(-1, keepdim=True) + 1e-6) * w64

    def close(got, want, size, terms):
        err = (got.cpu().double() - want).abs()
        assert bool((err <= want.abs() * 2.0 ** -8 * 1.0001 + size * 2.0 ** -24 * (24 + terms)).all()), float(err.max())

    close(h[ends].detach(), h64.detach(), h64.detach().abs().max(), 0)
    close(y[ends].detach(), y64.detach(), y64.detach().abs().max(), width)
    # Only the rows at both ends have a gradient: the sums over all rows are theirs.
    dy = torch.zeros_like(x)
    dy[ends] = torch.randn((80, width), generator=g, device="cuda").bfloat16()
    y.backward(dy)
    y64.backward(dy[ends].cpu().double())
    close(x.grad[ends], sub[0].grad, sub[0].grad.abs().max(), width)
    close(res.grad[ends], sub[1].grad, sub[1].grad.abs().max(), width)
    close(gamma.grad, w64.grad, (dy[ends].cpu().double() * y64.detach()).abs().sum(0).max(), width + 80)
    if gate == "channel":
        close(gt.grad, g64.grad, (sub[0].grad.abs().max() * sub[0].detach().abs().max()) * 80, width + 80)
    else:
        close(gt.grad[ends], g64.grad, (sub[0].detach() * sub[1].grad).abs().sum(-1, keepdim=True), 2 * width)
        assert int(torch.count_nonzero(gt.grad)) <= 80
    mid = slice(40, n - 40)
    assert int(torch.count_nonzero(x.grad[mid])) == 0 and int(torch.count_nonzero(res.grad[mid])) == 0
    del leaves


@pytest.mark.parametrize("m,k,n,groups", [(140000, 128, 16384, 6), (300, 8192, 8192, 40), (140001, 17, 16390, 3), (64, 4097, 8200, 70)])
def test_grouped_matmul(npu, m, k, n, groups):
    assert m * n > 2 ** 31 or groups * k * n > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (groups, n, k), generator=g, device="cuda", dtype=torch.int8).transpose(1, 2)
    ends = torch.linspace(0, m, groups + 1).long()[1:]
    (out,) = npu.npu_grouped_matmul([x], [w], group_list=ends.cuda(), split_item=3, group_type=0, output_dtype=torch.int32)
    for group in {0, groups // 2, groups - 1}:
        a, b = int(ends[group - 1]) if group else 0, int(ends[group])
        a = max(a, b - 48)
        want = x[a:b].double() @ w[group].double()                                    # integers below 2^53: exact
        assert torch.equal(out[a:b], want.int())
