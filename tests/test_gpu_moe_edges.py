"""The mixture-of-experts block operators in places where memory, parameters or values lie at an edge: buffers that touch one
another, parameters and values that are not finite, rows of no width."""
import ctypes as C

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


@pytest.mark.parametrize("hidden", [20, 24, 30])
@pytest.mark.parametrize("repeat", range(3))
def test_rows_next_to_their_indices(npu, hidden, repeat):
    """x ends and row_idx begins in one 32-byte sector.  The copy kernel loads x while the sort still runs and reads the rows
    afterwards: they are the sort's, not what the sector held when x came in (-1, which would leave the row out)."""
    from pytorch_b200 import _cabi as cabi
    tokens, topk, experts = 3, 1024, 64
    n = tokens * topk
    g = torch.Generator().manual_seed(hidden + repeat)
    idx = torch.randint(0, experts, (tokens, topk), generator=g, dtype=torch.int32)
    x = torch.randn((tokens, hidden), generator=g).to(torch.bfloat16)
    raw = x.view(torch.uint8).numel()
    assert raw % 4 == 0
    buf = torch.full((raw + 4 * n,), 0xFF, dtype=torch.uint8, device="cuda")
    buf[:raw] = x.view(torch.uint8).reshape(-1).cuda()
    ids, out = idx.cuda(), torch.zeros((n, hidden), dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(256, dtype=torch.uint8, device="cuda")
    a = cabi.MoeRouteArgs()
    a.x, a.x_dtype, a.expert_idx, a.idx_dtype = buf.data_ptr(), cabi.BF16, ids.data_ptr(), cabi.I32
    a.tokens, a.topk, a.hidden, a.expert_begin, a.expert_end = tokens, topk, hidden, 0, experts
    a.out, a.out_rows, a.row_idx = out.data_ptr(), n, buf.data_ptr() + raw
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    torch.cuda.synchronize()
    assert cabi.lib().b200q_moe_route(C.byref(a), torch.cuda.current_stream().cuda_stream) == cabi.OK
    torch.cuda.synchronize()
    row, src, _ = oracle.sorted_rows(idx, 0, experts)
    assert torch.equal(buf[raw:].view(torch.int32).cpu(), row)
    assert torch.equal(out.cpu(), oracle.gather_rows(x, src, topk))


def norm_inputs(rows, width, g):
    x, res = (torch.randn((rows, width), generator=g) + 4).to(torch.bfloat16), torch.randn((rows, width), generator=g).to(torch.bfloat16)
    param = lambda: torch.rand(width, generator=g) + 0.5  # noqa: E731
    return x, res, param(), param(), param()


# Rows in full vectors; rows of other widths, a handful and many of them (which pass through shared memory).
WIDTHS = [(3, 256), (3, 8), (5, 17), (4, 1111), (2, 4097), (1300, 1111), (1250, 520), (1300, 768)]


@pytest.mark.parametrize("which", ["post_gamma", "gate"])
@pytest.mark.parametrize("rows,width", WIDTHS)
def test_an_infinite_parameter_in_the_last_column(npu, rows, width, which):
    """h is infinite in that column, so the row's factor is 0: y is 0 in every other column, and 0 * infinity there.  Lanes behind
    the row's end take no part."""
    g = torch.Generator().manual_seed(width)
    x, res, gamma, post, gate = norm_inputs(rows, width, g)
    (post if which == "post_gamma" else gate)[-1] = float("inf")
    y, rstd, h, post_rstd = npu.npu_gated_add_rms_norm(x.cuda(), res.cuda(), gamma.cuda(), post_gamma=post.cuda(), gate=gate.cuda())
    assert float(rstd.abs().max()) == 0 and bool(torch.isfinite(post_rstd).all())
    assert bool(torch.isinf(h[:, -1]).all()) and bool(torch.isfinite(h[:, :-1]).all())
    assert float(y[:, :-1].abs().max()) == 0 and bool(torch.isnan(y[:, -1]).all())


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("rows,width", [(10, 256), (10, 64), (12, 8192), (1300, 1111), (1300, 512)])
def test_rows_that_are_not_finite_keep_a_scale_that_is_not(npu, rows, width, post):
    """int8 cannot hold what is not finite, so the row's scale says it: a row of y with an infinity or a NaN does not leave as zeros
    with scale 0, which would look like a row of zeros.  The other rows keep their bits."""
    g = torch.Generator().manual_seed(width + post)
    x, res, gamma, pg, gate = norm_inputs(rows, width, g)
    smooth = torch.rand(width, generator=g) + 0.5
    bad = [1, 4, 5, rows - 1]
    x[1, 2], res[4, width - 1], x[5, 0], res[rows - 1, 1] = float("inf"), float("-inf"), float("nan"), float("nan")
    kw = dict(post_gamma=pg.cuda() if post else None, gate=gate.cuda())
    for sm in (None, smooth.cuda()):
        q, scale, h = npu.npu_gated_add_rms_norm_dynamic_quant(x.cuda(), res.cuda(), gamma.cuda(), smooth_scales=sm, **kw)
        assert not bool(torch.isfinite(scale[bad]).any())
        clean = torch.ones(rows, dtype=torch.bool)
        clean[bad] = False
        zeroed = [torch.where(clean[:, None], t, 0).cuda() for t in (x, res)]
        q2, scale2, h2 = npu.npu_gated_add_rms_norm_dynamic_quant(*zeroed, gamma.cuda(), smooth_scales=sm, **kw)
        assert torch.equal(q[clean.cuda()], q2[clean.cuda()]) and torch.equal(scale[clean.cuda()], scale2[clean.cuda()])
        assert torch.equal(h[clean.cuda()], h2[clean.cuda()]) and bool((scale2[clean.cuda()] > 0).all())


@pytest.mark.parametrize("shape", [(4, 0), (2, 3, 0)])
def test_statistics_of_rows_without_columns(npu, shape):
    """The mean over nothing is NaN, and so is its root's reciprocal: no statistic is left as the memory had it."""
    w = torch.ones(0, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.zeros(shape, dtype=dtype, device="cuda")
        for fill in (0.0, 1.0):
            torch.full(shape[:-1], fill, device="cuda")                 # what the allocator hands out next
            _, rstd, _, post_rstd = npu.npu_gated_add_rms_norm(x, x, w, post_gamma=w)
            assert rstd.shape == post_rstd.shape == shape[:-1]
            assert bool(torch.isnan(rstd).all()) and bool(torch.isnan(post_rstd).all())


@pytest.mark.parametrize("tokens", [40, 3000])
def test_a_strict_range_past_32_bits(npu, tokens):
    """Experts numbered from 2^31 on: an index before the range has no row and is no error, also where the range's end does not fit into
    32 bits."""
    from pytorch_b200 import _cabi as cabi
    begin, experts, h = 2 ** 31, 8, 16
    g = torch.Generator().manual_seed(tokens)
    local = torch.randint(-1, experts, (tokens, 1), generator=g)
    idx = torch.where(local < 0, torch.full_like(local, 7), local + begin)
    idx[3] = -2 ** 63
    x = torch.randn((tokens, h), generator=g)
    cx, ids, out = x.cuda(), idx.cuda(), torch.full((tokens, h), 7.0, device="cuda")
    place, ends = torch.empty(tokens, dtype=torch.int32, device="cuda"), torch.empty(experts, dtype=torch.int64, device="cuda")
    ws = torch.empty(256, dtype=torch.uint8, device="cuda")
    a = cabi.MoeRouteArgs()
    a.x, a.x_dtype, a.expert_idx, a.idx_dtype = cx.data_ptr(), cabi.F32, ids.data_ptr(), cabi.I64
    a.tokens, a.topk, a.hidden, a.expert_begin, a.expert_end, a.strict = tokens, 1, h, begin, begin + experts, 1
    a.out, a.out_rows, a.row_idx, a.expert_tokens = out.data_ptr(), tokens, place.data_ptr(), ends.data_ptr()
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    assert cabi.lib().b200q_moe_route(C.byref(a), torch.cuda.current_stream().cuda_stream) == cabi.OK
    torch.cuda.synchronize()
    assert cabi.device_error() == 0
    row, src, counts = oracle.sorted_rows(idx, begin, begin + experts)
    assert torch.equal(place.cpu(), row) and torch.equal(ends.cpu(), counts) and torch.equal(out.cpu(), oracle.gather_rows(x, src, 1))


def test_router_weights_learn_through_the_quantised_block(npu):
    """The quantised part of the block has no gradient.  A backward pass through the whole gives the router's weights theirs, with and
    without a gradient asked for x (then behind a warning)."""
    import pytorch_b200.contrib.function as function
    g = torch.Generator().manual_seed(1)
    t, k, e, h, f = 40, 2, 4, 64, 32
    x, idx = torch.randn((t, h), generator=g).to(torch.bfloat16).cuda(), torch.topk(torch.rand((t, e), generator=g), k).indices.int().cuda()
    w_in, w_out = (torch.randint(-127, 128, s, generator=g).to(torch.int8).cuda() for s in ((e, 2 * f, h), (e, h, f)))
    s_in, s_out = (torch.rand(s, generator=g).cuda() * 1e-3 for s in ((e, 2 * f), (e, h)))
    probs, dy = torch.rand((t, k), generator=g).cuda(), torch.randn((t, h), generator=g).to(torch.bfloat16).cuda()
    grads = []
    for asked in (False, True):
        a, p = x.clone().requires_grad_(asked), probs.clone().requires_grad_()
        function.w8a8_swiglu_moe(a, idx, p, None, w_in, s_in, None, w_out, s_out).backward(dy)
        assert a.grad is None
        grads.append(p.grad)
    assert torch.equal(grads[0], grads[1]) and float(grads[0].abs().min()) > 0
