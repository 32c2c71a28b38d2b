"""npu_gated_add_rms_norm, its gradient and its quantised form on the GPU against the definitions in float64 (autograd of
the plain formula for the gradients)."""
import pytest
import torch

from oracle import moe_oracle as oracle

pytestmark = pytest.mark.gpu

EPS = 1e-6


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


def inputs(shape, dtype, ptype, gate, post, g):
    h = shape[-1]
    x, res = (torch.randn(shape, generator=g) * 3).to(dtype), torch.randn(shape, generator=g).to(dtype)
    gamma = (torch.randn(h, generator=g) * 0.2 + 1).to(ptype)
    pg = (torch.randn(h, generator=g) * 0.2 + 1).to(ptype) if post else None
    gs = {None: None, "channel": (h,), "row": (*shape[:-1], 1), "full": shape, "sample": (shape[0], *([1] * (len(shape) - 2)), h)}[gate]
    gt = (torch.randn(gs, generator=g) * 0.5 + 0.5).to(ptype) if gs is not None else None
    return x, res, gamma, pg, gt


def within(got, want, width, what, rows=1, terms=None):
    """A value rounded to its type after fp32 arithmetic.  Every row passes two sums of `width` squares (each within
    width * 2^-24 relative, halved by the root) and about twenty elementary operations on terms no larger than the
    largest of the tensor; a sum over rows adds one rounding of its terms per row."""
    t = got.dtype
    fi = torch.finfo(t)
    want = want.to(torch.float64)
    err = (got.cpu().to(torch.float64) - want).abs()
    size = want.abs().max() if terms is None else terms
    tol = (want.abs() * (fi.eps / 2)).clamp(min=fi.tiny * fi.eps / 2) * (1 + 1e-6) + size * (2.0 ** -24) * (24 + width + rows)
    assert bool((err <= tol).all()), (what, float((err - tol).max()), float(size))


CASES = [((1, 8), "channel", True), ((3, 4096), "channel", True), ((5, 7, 1111), "sample", True), ((300, 128), "full", True),
         ((129, 8192), "row", True), ((2, 16384), "channel", True), ((1000, 40), None, False), ((64, 520), "channel", False),
         ((4, 3, 5, 264), "sample", True), ((700, 1), "channel", True), ((33, 4104), "row", False), ((9, 2056), "full", False),
         ((2, 200, 96), "sample", False), ((5, 16383), "channel", True)]


@pytest.mark.parametrize("dtype,ptype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32),
                                         (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("case", CASES)
def test_values_and_gradients(npu, case, dtype, ptype):
    shape, gate, post = case
    g = torch.Generator().manual_seed(shape[-1] + len(shape))
    x, res, gamma, pg, gt = inputs(shape, dtype, ptype, gate, post, g)
    dy, dh = torch.randn(shape, generator=g).to(dtype), (torch.randn(shape, generator=g) * 0.3).to(dtype)
    y64, h64, r64, p64 = oracle.gated_add_rms_norm(x, res, gamma, pg, gt, 0.5, EPS)
    leaves = [t.cuda().requires_grad_() if t is not None else None for t in (x, res, gamma, pg, gt)]
    y, rstd, h, prstd = npu.npu_gated_add_rms_norm(leaves[0], leaves[1], leaves[2], post_gamma=leaves[3], gate=leaves[4], residual_scale=0.5, epsilon=EPS)
    width = shape[-1]
    within(y.detach(), y64, width, "y")
    within(h.detach(), h64, width, "h")
    within(rstd, r64, width, "rstd")
    assert rstd.shape == shape[:-1] and not rstd.requires_grad and prstd.shape == (shape[:-1] if post else (0,))
    if post:
        within(prstd, p64, width, "post_rstd")
    names = [n for n, t in zip(("x", "residual", "gamma", "post_gamma", "gate"), leaves) if t is not None]
    have = [t for t in leaves if t is not None]
    want, terms = oracle.gated_add_rms_norm_grad(x, res, gamma, pg, gt, 0.5, EPS, dy, dh)
    for k, t in enumerate(torch.autograd.grad((y, h), have, (dy.cuda(), dh.cuda()))):
        n = names[k]
        assert t.shape == have[k].shape and t.dtype == have[k].dtype
        rows = x.numel() // width
        within(t, want[n], width, n, rows=rows if n in ("gamma", "post_gamma", "gate") else 1, terms=terms[n])
    # the same gradients without autograd, the same bits
    with torch.no_grad():
        again = npu.npu_gated_add_rms_norm_grad(dy.cuda(), dh.cuda(), leaves[0], leaves[1], leaves[2], rstd, post_gamma=leaves[3], gate=leaves[4],
                                                post_rstd=prstd if post else None, residual_scale=0.5)
    y, rstd, h, prstd = npu.npu_gated_add_rms_norm(leaves[0], leaves[1], leaves[2], post_gamma=leaves[3], gate=leaves[4], residual_scale=0.5, epsilon=EPS)
    ref = torch.autograd.grad((y, h), have, (dy.cuda(), dh.cuda()))
    kept = [t for t, leaf in zip(again, leaves) if leaf is not None]
    assert all(torch.equal(a, b) for a, b in zip(kept, ref))


def test_only_one_of_the_outputs_is_used(npu):
    g = torch.Generator().manual_seed(3)
    x, res, gamma, pg, gt = inputs((12, 256), torch.float32, torch.float32, "channel", True, g)
    zero = torch.zeros_like(x)
    d = torch.randn(x.shape, generator=g)
    for which in (0, 1):
        leaves = [t.cuda().requires_grad_() for t in (x, res, gamma, pg, gt)]
        y, _, h, _ = npu.npu_gated_add_rms_norm(leaves[0], leaves[1], leaves[2], post_gamma=leaves[3], gate=leaves[4])
        (y if which == 0 else h).backward(d.cuda())
        want, terms = oracle.gated_add_rms_norm_grad(x, res, gamma, pg, gt, 1.0, EPS, d if which == 0 else zero, zero if which == 0 else d)
        for n, t in zip(("x", "residual", "gamma", "post_gamma", "gate"), leaves):
            within(t.grad, want[n], 256, n, rows=12, terms=terms[n].clamp(min=1e-6) if n != "gamma" else terms[n] + 1e-6)


def test_gradients_against_differences(npu):
    """fp32 gradients against central differences of the operator's own values along random directions.  The values are
    sums of 6 * 96 terms of order one in fp32 (each off by at most 2^-20 or so), the step 2^-6: the difference quotient is
    off by 576 * 2^-20 * 2^6 = 0.04 from rounding at the very most, and by order 2^-12 times third derivatives."""
    g = torch.Generator().manual_seed(4)
    x, res, gamma, pg, gt = (t.cuda() for t in inputs((6, 96), torch.float32, torch.float32, "row", True, g))
    dy, dh = torch.randn((6, 96), generator=g).cuda(), torch.randn((6, 96), generator=g).cuda()

    def f(*a):
        y, _, h, _ = npu.npu_gated_add_rms_norm(a[0], a[1], a[2], post_gamma=a[3], gate=a[4], residual_scale=0.7)
        return float((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum())

    leaves = [t.clone().requires_grad_() for t in (x, res, gamma, pg, gt)]
    y, _, h, _ = npu.npu_gated_add_rms_norm(leaves[0], leaves[1], leaves[2], post_gamma=leaves[3], gate=leaves[4], residual_scale=0.7)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    base = [t.detach() for t in leaves]
    for k in range(5):
        d = torch.randn(base[k].shape, generator=g).cuda()
        d = d / d.norm()
        step = 2.0 ** -6
        up, down = [*base], [*base]
        up[k], down[k] = base[k] + step * d, base[k] - step * d
        quotient = (f(*up) - f(*down)) / (2 * step)
        assert abs(quotient - float((grads[k].double() * d.double()).sum())) < 0.05, k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", [((16, 8192), "channel", True, "f32"), ((5, 7, 1111), "sample", True, "p"), ((300, 128), None, False, None),
                                  ((2, 16384), "row", True, "f32"), ((200, 2048), "full", False, "f32")])
def test_quantised_form(npu, case, dtype):
    """The quantised values are those of the operator's own fp32 row to within the rounding of that row: a value may move by
    one step where it lies next to a boundary, and by none elsewhere."""
    shape, gate, post, smooth = case
    g = torch.Generator().manual_seed(17)
    ptype = torch.float32 if dtype == torch.float16 else dtype
    x, res, gamma, pg, gt = inputs(shape, dtype, ptype, gate, post, g)
    sm = None if smooth is None else (torch.rand(shape[-1], generator=g) * 1.5 + 0.5).to(ptype if smooth == "p" else torch.float32)
    cu = [t.cuda() if t is not None else None for t in (x, res, gamma, pg, gt, sm)]
    q, scale, h = npu.npu_gated_add_rms_norm_dynamic_quant(cu[0], cu[1], cu[2], post_gamma=cu[3], gate=cu[4], smooth_scales=cu[5], residual_scale=0.5)
    _, _, h2, _ = npu.npu_gated_add_rms_norm(cu[0], cu[1], cu[2], post_gamma=cu[3], gate=cu[4], residual_scale=0.5)
    assert torch.equal(h, h2) and q.dtype == torch.int8 and scale.shape == shape[:-1]
    y64, _, _, _ = oracle.gated_add_rms_norm(x, res, gamma, pg, gt, 0.5, EPS)
    v = y64 if sm is None else y64 * sm.double()
    s64 = v.abs().amax(-1) / 127
    width = shape[-1]
    rel = (width + 40) * 2.0 ** -24                # two means of squares and the elementary operations, as above
    assert bool(((scale.cpu().double() - s64).abs() <= s64 * rel).all())
    steps = v / s64[..., None]
    near = (steps - torch.floor(steps) - 0.5).abs() <= 127 * 2 * rel
    d = (q.cpu().double() - torch.round(steps)).abs()
    assert float(d.max()) <= 1 and bool((d[~near] == 0).all())


def test_zero_rows_infinities_and_strides(npu):
    g = torch.Generator().manual_seed(6)
    x, res, gamma, pg, gt = inputs((10, 64), torch.bfloat16, torch.bfloat16, "channel", True, g)
    x[3], res[3] = 0, 0
    x[5, 2] = float("inf")
    x[6, 1] = float("nan")
    args = [t.cuda() for t in (x, res, gamma)]
    kw = dict(post_gamma=pg.cuda(), gate=gt.cuda())
    y, rstd, h, _ = npu.npu_gated_add_rms_norm(*args, **kw)
    assert float(y[3].abs().max()) == 0 and float(h[3].abs().max()) == 0 and float(rstd[3]) == pytest.approx(1e3, rel=1e-5)
    clean = [0, 1, 2, 4, 7, 8, 9]                                  # other rows do not see the bad ones
    y2, _, h2, _ = npu.npu_gated_add_rms_norm(args[0][clean], args[1][clean], args[2], **kw)
    assert torch.equal(y[clean], y2) and torch.equal(h[clean], h2)
    q, scale, _ = npu.npu_gated_add_rms_norm_dynamic_quant(*args, **kw)
    assert float(scale[3]) == 0 and int(q[3].abs().max()) == 0
    # columns of a wider matrix, expanded rows, storage off the vector grid
    wide = torch.zeros((10, 100), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:67] = args[0]
    y3, _, h3, _ = npu.npu_gated_add_rms_norm(wide[:, 3:67], args[1], args[2], **kw)
    assert torch.equal(y3[clean], y2) and torch.equal(h3[clean], h2)
    one = args[1][:1].expand(10, 64)
    assert torch.equal(npu.npu_gated_add_rms_norm(args[0], one, args[2])[2][clean], npu.npu_gated_add_rms_norm(args[0], one.contiguous(), args[2])[2][clean])
    odd = torch.zeros(641, dtype=torch.bfloat16, device="cuda")[1:].reshape(10, 64)
    odd.copy_(args[0])
    y4, _, h4, _ = npu.npu_gated_add_rms_norm(odd, args[1], args[2], **kw)
    assert torch.equal(h4[clean], h2)
    for shape in ((0, 64), (4, 0)):
        e = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        gate = torch.ones(shape[-1], device="cuda", requires_grad=True)
        y, r, h, p = npu.npu_gated_add_rms_norm(e, e, w, post_gamma=w, gate=gate)
        assert y.shape == shape and r.shape == shape[:1]
        (y.sum() + h.sum()).backward()
        assert w.grad.shape == (shape[-1],) and float(w.grad.abs().sum()) == 0 and float(gate.grad.abs().sum()) == 0
        q, s, _ = npu.npu_gated_add_rms_norm_dynamic_quant(e.detach(), e.detach(), w.detach())
        assert q.shape == shape and float(s.sum()) == 0


def test_captured_step_replays(npu):
    g = torch.Generator().manual_seed(8)
    x, res, gamma, pg, gt = (t.cuda() for t in inputs((300, 1024), torch.bfloat16, torch.bfloat16, "channel", True, g))
    dy = torch.randn((300, 1024), generator=g).cuda().to(torch.bfloat16)

    def step():
        y, rstd, h, prstd = npu.npu_gated_add_rms_norm(x, res, gamma, post_gamma=pg, gate=gt)
        return (y, h, *npu.npu_gated_add_rms_norm_grad(dy, None, x, res, gamma, rstd, post_gamma=pg, gate=gt, post_rstd=prstd),
                *npu.npu_gated_add_rms_norm_dynamic_quant(x, res, gamma, post_gamma=pg, gate=gt))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        x.copy_(torch.randn((300, 1024), generator=g))
        dy.copy_(torch.randn((300, 1024), generator=g))
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


# Many rows, where the rows of a CTA overlap: full vectors of one, two and four a thread with one or several rows at a time, rows
# that are not full vectors through shared memory (with odd starts, a last row that ends off the 16-byte grid, groups of
# rows), gates that change within a CTA's rows, and storage off the vector grid.
MANY = [((700, 256), "channel", True), ((1200, 512), "row", True), ((600, 768), "full", True), ((40, 31, 1024), "sample", True), ((333, 4096), "channel", True),
        ((301, 5632), "channel", True), ((310, 8192), "sample2", True), ((299, 9216), "channel", True), ((150, 16384), "channel", True), ((905, 1111), "channel", True),
        ((7, 131, 333), "sample", True), ((2500, 8), "sample2", True), ((777, 17), None, False), ((301, 4095), "full", False), ((300, 4097), "row", True),
        ((1301, 1111), "channel", True), ((3, 431, 555), "sample", False), ((1250, 2047), "full", True), ((6, 200, 513), "sample", True),
        ((1500, 700), "sample2", True), ((1600, 256), "sample2", True), ((905, 2048), "sample2", False)]


@pytest.mark.parametrize("dtype,ptype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("case", range(len(MANY)))
def test_many_rows(npu, case, dtype, ptype):
    shape, gate, post = MANY[case]
    g = torch.Generator().manual_seed(case)
    if gate == "sample2":                                          # a gate for every five rows
        shape, gate = (shape[0] // 5, 5, shape[1]), "sample"
    x, res, gamma, pg, gt = inputs(shape, dtype, ptype, gate, post, g)
    dy, dh = torch.randn(shape, generator=g).to(dtype), (torch.randn(shape, generator=g) * 0.3).to(dtype)
    width = shape[-1]
    y64, h64, _, _ = oracle.gated_add_rms_norm(x, res, gamma, pg, gt, 0.5, EPS)
    want, terms = oracle.gated_add_rms_norm_grad(x, res, gamma, pg, gt, 0.5, EPS, dy, dh)
    for offset in (0, 1):
        def place(t):                                              # the same values, one element off the allocation's start
            if t is None or not offset:
                return t if t is None else t.cuda()
            wide = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
            wide[1:] = t.reshape(-1).cuda()
            return wide[1:].reshape(t.shape)
        leaves = [place(t).requires_grad_() if t is not None else None for t in (x, res, gamma, pg, gt)]
        y, _, h, _ = npu.npu_gated_add_rms_norm(leaves[0], leaves[1], leaves[2], post_gamma=leaves[3], gate=leaves[4], residual_scale=0.5, epsilon=EPS)
        within(y.detach(), y64, width, "y")
        within(h.detach(), h64, width, "h")
        q, s, hq = npu.npu_gated_add_rms_norm_dynamic_quant(*(t.detach() for t in leaves[:3]), post_gamma=None if pg is None else leaves[3].detach(),
                                                            gate=None if gt is None else leaves[4].detach(), residual_scale=0.5, epsilon=EPS)
        s64 = y64.abs().amax(-1) / 127
        assert torch.equal(hq, h) and bool(((s.cpu().double() - s64).abs() <= s64 * (width + 40) * 2.0 ** -24).all())
        assert float((q.cpu().double() - y64 / s64[..., None]).abs().max()) <= 0.5 + 127 * (width + 40) * 2.0 ** -23
        names = [n for n, t in zip(("x", "residual", "gamma", "post_gamma", "gate"), leaves) if t is not None]
        have = [t for t in leaves if t is not None]
        for n, t in zip(names, torch.autograd.grad((y, h), have, (place(dy), place(dh)))):
            rows = x.numel() // width
            within(t, want[n], width, n, rows=rows if n in ("gamma", "post_gamma", "gate") else 1, terms=terms[n])


def test_one_tensor_twice_and_expanded_inputs(npu):
    """x as its own residual, one row expanded over all rows, one gamma for both norms: the gradients of what is shared are the sums
    that autograd adds up; nothing is written through an expanded input."""
    g = torch.Generator().manual_seed(11)
    for width, dtype in ((512, torch.float32), (77, torch.float32)):
        x, res, gamma, _, gt = inputs((40, width), dtype, torch.float32, "channel", True, g)
        dy, dh = torch.randn((40, width), generator=g), torch.randn((40, width), generator=g)
        a, w = x.cuda().requires_grad_(), gamma.cuda().requires_grad_()
        y, _, h, _ = npu.npu_gated_add_rms_norm(a, a, w, post_gamma=w, gate=gt.cuda(), residual_scale=0.5, epsilon=EPS)
        torch.autograd.backward((y, h), (dy.cuda(), dh.cuda()))
        want, terms = oracle.gated_add_rms_norm_grad(x, x, gamma, gamma, gt, 0.5, EPS, dy, dh)
        within(a.grad, want["x"] + want["residual"], width, "x", terms=terms["x"] + terms["residual"])
        within(w.grad, want["gamma"] + want["post_gamma"], width, "gamma", rows=40, terms=terms["gamma"] + terms["post_gamma"])
        row = x[:1].clone()
        leaf = row.cuda().requires_grad_()
        y, _, h, _ = npu.npu_gated_add_rms_norm(leaf.expand(40, width), res.cuda(), gamma.cuda(), gate=gt.cuda(), residual_scale=0.5, epsilon=EPS)
        torch.autograd.backward((y, h), (dy.cuda(), dh.cuda()[:1].expand(40, width)))
        want, terms = oracle.gated_add_rms_norm_grad(row.expand(40, width).contiguous(), res, gamma, None, gt, 0.5, EPS, dy,
                                                     dh[:1].expand(40, width).contiguous())
        assert torch.equal(leaf.detach().cpu(), row)
        within(leaf.grad, want["x"].sum(0, keepdim=True), width, "row", rows=40, terms=terms["x"].max() * 40)
