"""Routing tokens to experts and back on the GPU against the 64-bit CPU oracle.  Rows, counts and copies are exact, the
quantised rows bit-exact; sums are held to the rounding of their type plus the fp32 accumulation's bound."""
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


def ids_of(tokens, topk, experts, g, padded=0, dtype=torch.int32):
    idx = torch.stack([torch.randperm(experts, generator=g)[:topk] for _ in range(tokens)]) if tokens else torch.zeros((0, topk), dtype=torch.int64)
    if padded:
        idx[tokens - padded:] = -1
    return idx.to(dtype)


def half_step(t, v):
    """Largest error of rounding v to type t: half a step of a normal value, half the smallest subnormal's step below."""
    fi = torch.finfo(t)
    return (v.abs() * (fi.eps / 2)).clamp(min=fi.tiny * fi.eps / 2)


# (tokens, topk, experts, hidden): one token, a decode step, the last size of the one-launch path (2048 assignments), the
# first of the sorted one, more than one CTA of the sort, odd widths, more slots than a register block holds.
SIZES = [(1, 1, 1, 8), (1, 8, 64, 4096), (16, 8, 64, 4096), (256, 8, 128, 256), (257, 8, 128, 264), (3001, 6, 60, 130),
         (2500, 12, 1024, 40), (9001, 2, 8, 72), (33, 3, 16, 1111), (700, 40, 96, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int8])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("padded", [False, True])
def test_permute_and_its_gradient(npu, size, dtype, padded):
    t, k, e, h = size
    g = torch.Generator().manual_seed(t * 31 + k)
    idx = ids_of(t, k, e, g, padded=(t + 3) // 4 if padded else 0, dtype=torch.int64 if t % 2 else torch.int32)
    x = torch.randint(-128, 128, (t, h), generator=g).to(dtype) if dtype == torch.int8 else torch.randn((t, h), generator=g).to(dtype)
    row, src, _ = oracle.sorted_rows(idx, 0, 1024)
    want = oracle.gather_rows(x, src, k)
    for keep in (None, 1, t * k - 1, -2):
        rows = t * k if keep is None else (min(t * k, keep) if keep > 0 else max(0, t * k + keep))
        rows = t * k if keep == 0 else rows
        got, place = npu.npu_moe_token_permute(x.cuda(), idx.cuda(), keep)
        assert place.dtype == torch.int32 and torch.equal(place.cpu(), row)
        assert got.shape == (rows, h) and torch.equal(got.cpu(), want[:rows])
    if dtype == torch.int8:
        return
    dy = torch.randn((t * k, h), generator=g).to(dtype)
    leaf = x.cuda().requires_grad_()
    got, place = npu.npu_moe_token_permute(leaf, idx.cuda())
    assert not place.requires_grad
    got.backward(dy.cuda())
    want, size_ = oracle.combine(dy, row, None, t, k)
    # k additions in fp32, then one rounding to the type
    assert bool(((leaf.grad.cpu().double() - want).abs() <= half_step(dtype, want) * (1 + 1e-6) + k * 2.0 ** -24 * size_).all())
    direct = npu.npu_moe_token_permute_grad(x.cuda(), dy.cuda(), idx.cuda(), place)
    assert torch.equal(direct, leaf.grad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("smooth", [None, "shared", "f32", "x"])
def test_routing_with_quantisation(npu, size, dtype, smooth):
    t, k, e, h = size
    g = torch.Generator().manual_seed(t * 7 + h)
    idx = ids_of(t, k, e, g, padded=t // 3)
    x = torch.randn((t, h), generator=g).to(dtype)
    x[t - t // 3:] = float("nan")                                  # padded tokens are not looked at
    sm = None if smooth is None else (torch.rand((1 if smooth == "shared" else e, h), generator=g) * 1.5 + 0.5).to(dtype if smooth == "x" else torch.float32)
    q, place, ends, scale = npu.npu_moe_init_routing_v2(x.cuda(), idx.cuda(), scale=None if sm is None else sm.cuda(), expert_num=e, quant_mode=1)
    row, src, counts = oracle.sorted_rows(idx, 0, e)
    qo, so = oracle.route_quantised(x, idx, sm, 0, e)
    assert torch.equal(place.cpu(), row) and torch.equal(ends.cpu(), torch.cumsum(counts, 0))
    assert torch.equal(scale.cpu().view(torch.int32), so.view(torch.int32)) and torch.equal(q.cpu(), qo)
    q, place, ends, _ = npu.npu_moe_init_routing_v2(x.cuda(), idx.cuda().long(), scale=None if sm is None else sm.cuda(), expert_num=e, quant_mode=1,
                                                    expert_tokens_num_type=1, row_idx_type=1)
    assert torch.equal(place.cpu(), src) and torch.equal(ends.cpu(), counts) and torch.equal(q.cpu(), qo)


@pytest.mark.parametrize("size", [(16, 8, 64, 96), (1024, 4, 64, 96)])
@pytest.mark.parametrize("quant", [False, True])
def test_a_range_of_the_experts_and_carried_scales(npu, size, quant):
    t, k, e, h = size
    g = torch.Generator().manual_seed(5)
    idx = ids_of(t, k, e, g)
    lo, hi = 13, 40
    row, src, counts = oracle.sorted_rows(idx, lo, hi)
    if quant:
        x = torch.randn((t, h), generator=g).to(torch.bfloat16)
        sm = torch.rand((hi - lo, h), generator=g) + 0.5
        q, place, n, scale = npu.npu_moe_init_routing_v2(x.cuda(), idx.cuda(), scale=sm.cuda(), expert_num=e, quant_mode=1, expert_tokens_num_type=1,
                                                         active_expert_range=[lo, hi])
        qo, so = oracle.route_quantised(x, idx, sm, lo, hi)
        assert torch.equal(q.cpu(), qo) and torch.equal(scale.cpu(), so)
    else:
        x = torch.randint(-128, 128, (t, h), generator=g).to(torch.int8)
        s = torch.rand((t,), generator=g)
        q, place, n, scale = npu.npu_moe_init_routing_v2(x.cuda(), idx.cuda(), scale=s.cuda(), expert_num=e, quant_mode=-1, expert_tokens_num_type=1,
                                                         active_expert_range=[lo, hi])
        assert torch.equal(q.cpu(), oracle.gather_rows(x, src, k))
        assert torch.equal(scale.cpu(), oracle.gather_rows(s[:, None], src, k)[:, 0])
    assert torch.equal(place.cpu(), row) and torch.equal(n.cpu(), counts)


@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32),
                                         (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("size", SIZES)
def test_unpermute_and_its_gradients(npu, size, dtype, wtype):
    t, k, e, h = size
    g = torch.Generator().manual_seed(t + h)
    idx = ids_of(t, k, e, g, padded=t // 5)
    row, _, counts = oracle.sorted_rows(idx, 0, e)
    live = int(counts.sum())
    rows = torch.randn((t * k, h), generator=g).to(dtype)
    rows[live:] = float("nan")                                    # rows behind the last expert's are not read
    w = torch.rand((t, k), generator=g).to(wtype)
    w[t - t // 5:] = float("nan")                                 # nor the weights of padded tokens
    dy = torch.randn((t, h), generator=g).to(dtype)
    a, b = rows.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = npu.npu_moe_token_unpermute(a, row.cuda(), b)
    want, size_ = oracle.combine(rows, row, w, t, k)
    assert bool(((y.detach().cpu().double() - want).abs() <= half_step(dtype, want) * (1 + 1e-6) + (k + 1) * 2.0 ** -24 * size_).all())
    y.backward(dy.cuda())
    drows, dw, terms = oracle.combine_grad(dy, rows, row, w, t, k)
    # one product in fp32, rounded to the type
    assert bool(((a.grad.cpu().double() - drows).abs() <= half_step(dtype, drows) * (1 + 1e-6) + 2.0 ** -24 * drows.abs()).all())
    # h products and additions in fp32 in some order: each term meets at most h roundings
    assert bool(((b.grad.cpu().double() - dw).abs() <= half_step(wtype, dw) * (1 + 1e-6) + (h + 1) * 2.0 ** -24 * terms).all())
    d2, w2 = npu.npu_moe_token_unpermute_grad(rows.cuda(), dy.cuda(), row.cuda(), w.cuda())
    assert torch.equal(d2, a.grad) and torch.equal(w2, b.grad)
    # without weights: one row a token
    y1 = npu.npu_moe_token_unpermute(rows.cuda(), row.cuda())
    assert torch.equal(y1.cpu(), oracle.combine(rows, row, None, t * k, 1)[0].to(dtype))


def test_gradients_against_differences(npu):
    """The fp32 gradients against differences of the operators' own values (linear in each operand, so exact but for
    rounding: the loss is a sum of 5*3*24 terms of order one)."""
    g = torch.Generator().manual_seed(2)
    idx = ids_of(5, 3, 6, g, padded=1)
    x, w = torch.randn((5, 24), generator=g).cuda(), torch.rand((5, 3), generator=g).cuda()
    dy = torch.randn((5, 24), generator=g).cuda()

    def f(x, w):
        rows, place = npu.npu_moe_token_permute(x, idx.cuda())
        return npu.npu_moe_token_unpermute(rows, place, w)

    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    f(a, b).backward(dy)
    for which, (leaf, grad) in enumerate(((x, a.grad), (w, b.grad))):
        d = torch.randn(leaf.shape, generator=g).cuda()
        up = f(x + d if which == 0 else x, w + d if which == 1 else w)
        diff = ((up.double() - f(x, w).double()) * dy.double()).sum()
        assert abs(float(diff) - float((grad.double() * d.double()).sum())) < 1e-3


def test_strides_empty_calls_and_streams(npu):
    g = torch.Generator().manual_seed(9)
    idx = ids_of(40, 4, 16, g)
    x = torch.randn((40, 256), generator=g).to(torch.bfloat16)
    row, src, _ = oracle.sorted_rows(idx, 0, 1024)
    want = oracle.gather_rows(x, src, 4)
    wide = torch.zeros((40, 300), dtype=torch.bfloat16, device="cuda")
    wide[:, 7:263] = x.cuda()
    cols = torch.zeros((4, 40), dtype=torch.int32, device="cuda").copy_(idx.t().cuda()).t()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, place = npu.npu_moe_token_permute(wide[:, 7:263], cols)
        back = npu.npu_moe_token_unpermute(got, place, torch.full((40, 4), 0.25, device="cuda"))
    side.synchronize()
    assert torch.equal(got.cpu(), want) and torch.equal(place.cpu(), row)
    assert torch.equal(back.cpu(), x)                              # a quarter of each, four times: exact
    # storage that no 16-byte vector fits
    odd = torch.zeros(40 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].reshape(40, 256)
    odd.copy_(x)
    assert torch.equal(npu.npu_moe_token_permute(odd, idx.cuda())[0].cpu(), want)
    for t, k, h in ((0, 4, 64), (5, 0, 64), (5, 4, 0)):
        xe = torch.zeros((t, h), dtype=torch.bfloat16, device="cuda", requires_grad=True)
        ie = torch.zeros((t, k), dtype=torch.int32, device="cuda")
        rows, place = npu.npu_moe_token_permute(xe, ie)
        assert rows.shape == (t * k, h) and place.shape == (t * k,)
        rows.sum().backward()
        assert xe.grad.shape == (t, h) and float(xe.grad.abs().sum()) == 0
        q, _, ends, s = npu.npu_moe_init_routing_v2(xe.detach(), ie, expert_num=3, quant_mode=1)
        assert q.shape == (t * k, h) and s.shape == (t * k,) and ends.tolist() == [t * k] * 3 and float(s.sum()) == 0
    y = npu.npu_moe_token_unpermute(torch.zeros((0, 64), device="cuda"), torch.full((6,), -1, dtype=torch.int32, device="cuda"),
                                    torch.ones((3, 2), device="cuda"))
    assert y.shape == (3, 64) and float(y.abs().sum()) == 0


def test_captured_graphs_replay_with_new_inputs(npu):
    """Two captured passes over one memory pool, replayed with other inputs, beside an eager call."""
    g = torch.Generator().manual_seed(11)
    x = torch.zeros((600, 512), dtype=torch.bfloat16, device="cuda")
    idx = torch.zeros((600, 8), dtype=torch.int32, device="cuda")
    dy = torch.zeros((600, 512), dtype=torch.bfloat16, device="cuda")
    w = torch.full((600, 8), 0.125, device="cuda")

    def step():
        rows, place = npu.npu_moe_token_permute(x, idx)
        y = npu.npu_moe_token_unpermute(rows, place, w)
        return (rows, place, y, *npu.npu_moe_token_unpermute_grad(rows, dy, place, w))

    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    pool = torch.cuda.graph_pool_handle()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(step())
        graphs.append(graph)
    for r in range(3):
        x.copy_(torch.randn((600, 512), generator=g))
        dy.copy_(torch.randn((600, 512), generator=g))
        idx.copy_(ids_of(600, 8, 64, g, padded=r * 50))
        want = step()
        for graph, out in zip(graphs, outs):
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_device_errors_are_reported(npu):
    from pytorch_b200 import _cabi
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    idx = torch.tensor([[0], [1024], [2], [-7]], dtype=torch.int32, device="cuda")
    rows, place = npu.npu_moe_token_permute(x, idx)
    torch.cuda.synchronize()
    assert place.tolist() == [0, -1, 1, -1]
    with pytest.raises(RuntimeError, match="1024 or more"):
        npu.npu_moe_token_permute(x, idx)
    big = torch.zeros((4000, 1), dtype=torch.int64, device="cuda")
    big[7] = 2 ** 40
    npu.npu_moe_token_permute(torch.zeros((4000, 8), device="cuda"), big)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="1024 or more"):
        npu.npu_moe_token_permute(x, idx)
    npu.npu_moe_token_unpermute_grad(x, x, torch.tensor([0, 1, 1, 3], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="twice"):
        npu.npu_moe_token_permute(x, idx)
    assert _cabi.device_error() == 0


def test_refusals(npu):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    i = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="same device"):
        npu.npu_moe_token_permute(x, i.cpu())
    with pytest.raises(RuntimeError, match="create_graph"):
        a = x.float().requires_grad_()
        y, _ = npu.npu_moe_token_permute(a, i)
        torch.autograd.grad(y.sum(), a, create_graph=True)


def test_expanded_inputs_and_one_set_of_rows_twice(npu):
    """One token's row and one row of weights expanded over all tokens; the rows of one permute used by two unpermutes."""
    g = torch.Generator().manual_seed(12)
    t, k, h = 700, 4, 264
    idx = ids_of(t, k, 16, g)
    x, w, dy = torch.randn((1, h), generator=g), torch.rand((1, k), generator=g), torch.randn((t, h), generator=g)
    row, _, _ = oracle.sorted_rows(idx, 0, 1024)
    lx, lw = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    rows, place = npu.npu_moe_token_permute(lx.expand(t, h), idx.cuda())
    assert torch.equal(place.cpu(), row) and torch.equal(rows.detach().cpu(), x.expand(t * k, h))
    first = npu.npu_moe_token_unpermute(rows, place, lw.expand(t, k))
    second = npu.npu_moe_token_unpermute(rows, place, lw.expand(t, k).flip(1))
    (first + second).backward(dy.cuda())
    sum_w = float(w.double().sum())
    # y = 2 * sum(w) * x for every token, through fp32 sums of k products, added up over t tokens and 2 k slots
    assert bool(((lx.grad.cpu().double() - 2 * sum_w * dy.double().sum(0)).abs() <= dy.double().abs().sum(0) * 2 * sum_w * (t + 4 * k) * 2.0 ** -24).all())
    dots = (dy.double() @ x.double().t()).sum()
    size = (dy.double().abs() @ x.double().abs().t()).sum()
    assert bool(((lw.grad.cpu().double() - 2 * dots).abs() <= 2 * size * (t + h) * 2.0 ** -24).all())
