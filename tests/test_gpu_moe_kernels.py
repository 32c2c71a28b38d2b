"""The mixture-of-experts block operators against the oracle at sizes that reach each kernel behind an entry point: which kernel
a call takes goes by its sizes, so every form of the larger ones has cases of its own here.  Copies, counts and quantised rows are
exact; sums are held to the rounding of their type plus the bound of an fp32 accumulation."""
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


def ids_of(tokens, topk, experts, g, padded):
    idx = torch.topk(torch.rand((tokens, experts), generator=g), topk, dim=1).indices.to(torch.int32)
    if padded:
        idx[tokens - padded:] = -1
        idx[1, topk // 2] = -1                                     # one slot without an expert among others that have one
    return idx


def half_step(t, v):
    fi = torch.finfo(t)
    return (v.abs() * (fi.eps / 2)).clamp(min=fi.tiny * fi.eps / 2)


# ------------------------------------------------------------------------------------------------ the way back as a pipeline
# From two tokens an SM (296) and rows of 1024 bytes on, up to eight slots: (tokens, topk, experts, hidden).  One to eight slots; rows
# that end inside a stage of 4096 bytes, on it and behind it; one or several tokens a CTA.
RING = [(400, 1, 8, 512), (301, 2, 8, 2056), (400, 3, 16, 2560), (296, 4, 16, 520), (500, 5, 16, 1032), (350, 6, 60, 5120), (300, 7, 64, 4104),
        (900, 8, 64, 1024)]
TYPES = [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32)]


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("size", RING)
@pytest.mark.parametrize("padded", [False, True])
def test_unpermute_and_its_gradients(npu, size, dtype, wtype, padded):
    t, k, e, h = size
    g = torch.Generator().manual_seed(t + h)
    idx = ids_of(t, k, e, g, t // 5 if padded else 0)
    row, _, counts = oracle.sorted_rows(idx, 0, e)
    live, there = int(counts.sum()), (row >= 0).reshape(t, k)
    rows = torch.randn((t * k + 3, h), generator=g).to(dtype)
    rows[live:] = float("nan")                                    # rows that nothing names are not read
    w = torch.where(there, torch.rand((t, k), generator=g), float("nan")).to(wtype)      # nor the weights of missing ones
    dy = torch.randn((t, h), generator=g).to(dtype)
    a, b = rows.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = npu.npu_moe_token_unpermute(a, row.cuda(), b)
    want, size_ = oracle.combine(rows, row, w, t, k)
    assert bool(((y.detach().cpu().double() - want).abs() <= half_step(dtype, want) * (1 + 1e-6) + (k + 1) * 2.0 ** -24 * size_).all())
    y.backward(dy.cuda())
    drows, dw, terms = oracle.combine_grad(dy, rows, row, w, t, k)
    assert bool(((a.grad.cpu().double() - drows).abs() <= half_step(dtype, drows) * (1 + 1e-6) + 2.0 ** -24 * drows.abs()).all())
    assert bool((a.grad[live:] == 0).all()) and bool((b.grad.cpu()[~there] == 0).all())
    assert bool(((b.grad.cpu().double() - dw).abs() <= half_step(wtype, dw) * (1 + 1e-6) + (h + 1) * 2.0 ** -24 * terms).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("size", RING)
@pytest.mark.parametrize("padded", [False, True])
def test_gradient_of_permute(npu, size, dtype, padded):
    """The pipeline without weights: a token's gradient is the sum of its rows', also where the last rows were dropped."""
    t, k, e, h = size
    g = torch.Generator().manual_seed(t * 3 + h)
    idx = ids_of(t, k, e, g, t // 5 if padded else 0)
    row, src, counts = oracle.sorted_rows(idx, 0, e)
    x = torch.randn((t, h), generator=g).to(dtype)
    for keep in (t * k, t * k - t // 2):
        leaf = x.cuda().requires_grad_()
        got, place = npu.npu_moe_token_permute(leaf, idx.cuda(), keep)
        assert torch.equal(place.cpu(), row) and torch.equal(got.detach().cpu(), oracle.gather_rows(x, src, k)[:keep])
        dy = torch.randn((keep, h), generator=g).to(dtype)
        dy[int(counts.sum()):] = float("nan")
        got.backward(dy.cuda())
        want, size_ = oracle.combine(dy, row, None, t, k)
        assert bool(((leaf.grad.cpu().double() - want).abs() <= half_step(dtype, want) * (1 + 1e-6) + k * 2.0 ** -24 * size_).all())


# Without weights a row is a token's only one: (rows, hidden), of full vectors and of others, few and many.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,h", [(1, 8), (40, 4096), (33, 17), (500, 1024), (700, 130), (5000, 40)])
def test_gradient_of_unpermute_without_weights(npu, rows, h, dtype):
    """A copy in either direction: exact, and zero for rows that nothing names."""
    g = torch.Generator().manual_seed(rows + h)
    order = torch.randperm(rows + 5, generator=g)[:rows].to(torch.int32)
    order[::7] = -1
    values = torch.randn((rows + 5, h), generator=g).to(dtype)
    dy = torch.randn((rows, h), generator=g).to(dtype)
    leaf = values.cuda().requires_grad_()
    y = npu.npu_moe_token_unpermute(leaf, order.cuda())
    assert torch.equal(y.detach().cpu(), oracle.combine(values, order, None, rows, 1)[0].to(dtype))
    y.backward(dy.cuda())
    want = oracle.combine_grad(dy, values, order, None, rows, 1)[0].to(dtype)
    assert torch.equal(leaf.grad.cpu(), want)
    drows, dprobs = npu.npu_moe_token_unpermute_grad(values.cuda(), dy.cuda(), order.cuda())
    assert torch.equal(drows.cpu(), want) and dprobs.numel() == 0


# ------------------------------------------------------------------------------------------------ quantised rows behind a sort
# More than 2048 assignments: (tokens, topk, experts, hidden).  Two vectors a thread below 1024 columns, four from there on; widths
# whose threads' vectors all lie inside the row (the next row's loads then wait for this row's products) and widths with a remainder;
# widths that eight does not divide.
SORTED = [(350, 6, 60, 5120), (300, 7, 64, 4104), (600, 8, 64, 1024), (700, 4, 8, 512), (1100, 2, 300, 520), (2100, 1, 5, 2048), (300, 8, 16, 1111),
          (260, 8, 24, 16384), (3000, 2, 64, 2056)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SORTED)
@pytest.mark.parametrize("smooth", [None, "shared", "f32", "x"])
@pytest.mark.parametrize("padded", [False, True])
def test_quantised_routing(npu, size, dtype, smooth, padded):
    t, k, e, h = size
    assert t * k > 2048
    g = torch.Generator().manual_seed(t * 7 + h)
    idx = ids_of(t, k, e, g, t // 3 if padded else 0)
    x = torch.randn((t, h), generator=g).to(dtype)
    if padded:
        x[t - t // 3:] = float("nan")                              # padded tokens are not looked at
    x[5] = 0
    sm = None if smooth is None else (torch.rand((1 if smooth == "shared" else e, h), generator=g) * 1.5 + 0.5).to(dtype if smooth == "x" else torch.float32)
    q, place, ends, scale = npu.npu_moe_init_routing_v2(x.cuda(), idx.cuda(), scale=None if sm is None else sm.cuda(), expert_num=e, quant_mode=1)
    row, _, counts = oracle.sorted_rows(idx, 0, e)
    qo, so = oracle.route_quantised(x, idx, sm, 0, e)
    assert torch.equal(place.cpu(), row) and torch.equal(ends.cpu(), torch.cumsum(counts, 0))
    assert torch.equal(scale.cpu().view(torch.int32), so.view(torch.int32)) and torch.equal(q.cpu(), qo)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("size", [(600, 8, 64, 1024), (700, 6, 60, 2056)])
def test_a_range_of_the_experts_behind_a_sort(npu, size, quant):
    """Most assignments belong to other ranks' experts: their rows are zero, the range's scales are its own."""
    t, k, e, h = size
    lo, hi = 13, 29
    g = torch.Generator().manual_seed(h)
    idx = ids_of(t, k, e, g, 50)
    x = torch.randn((t, h), generator=g).to(torch.float16)
    row, src, counts = oracle.sorted_rows(idx, lo, hi)
    if quant:
        sm = torch.rand((hi - lo, h), generator=g) + 0.5
        q, place, n, scale = npu.npu_moe_init_routing_v2(x.cuda(), idx.cuda(), scale=sm.cuda(), expert_num=e, quant_mode=1, active_expert_range=[lo, hi])
        qo, so = oracle.route_quantised(x, idx, sm, lo, hi)
        assert torch.equal(q.cpu(), qo) and torch.equal(scale.cpu(), so)
    else:
        q, place, n, _ = npu.npu_moe_init_routing_v2(x.cuda(), idx.cuda(), expert_num=e, quant_mode=-1, active_expert_range=[lo, hi])
        assert torch.equal(q.cpu(), oracle.gather_rows(x, src, k))
    assert torch.equal(place.cpu(), row) and torch.equal(n.cpu(), torch.cumsum(counts, 0))


# ------------------------------------------------------------------------------------------------ products on pairs of CTAs
# From 1536 rows a group (on average) on: (counts, tail, k, n).  One group, empty groups, rows behind the last, groups of one row
# next to large ones, tiles of 32 to 256 rows; k of a part of a block, of several and of more than the ring holds; n that leaves the
# second CTA of the last pair without channels, with some, with an odd number.
PAIRS = [([1700], 0, 144, 130), ([3100, 0, 1800], 33, 1040, 264), ([0, 4700, 1, 0], 1600, 2048, 200), ([1537, 1600], 0, 128, 520), ([3300, 31], 5, 400, 384),
         ([2048], 0, 16, 8), ([4609, 255], 17, 272, 333)]


def grouped(npu, x, w, ends, out, **kw):
    lists = {k: [v] for k, v in kw.items() if v is not None}
    return npu.npu_grouped_matmul([x], [w.transpose(1, 2)], group_list=ends, split_item=3, group_type=0, output_dtype=out, **lists)[0]


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.int32])
@pytest.mark.parametrize("case", range(len(PAIRS)))
def test_grouped_matmul_of_large_groups(npu, case, out):
    counts, tail, k, n = PAIRS[case]
    e, m = len(counts), sum(counts) + tail
    assert m >= 1536 * e
    g = torch.Generator().manual_seed(case)
    x = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int64).to(torch.int8)
    w = torch.randint(-128, 128, (e, n, k), generator=g, dtype=torch.int64).to(torch.int8)
    ends = torch.cumsum(torch.tensor(counts), 0)
    if out == torch.int32:
        biases = [None, torch.randint(-1000, 1000, (e, n), generator=g).to(torch.int32)]
        scale = row_scale = None
    else:
        scale, row_scale = torch.rand((e, n), generator=g) * 9e-3 + 1e-3, torch.rand((m,), generator=g) * 9e-3 + 1e-3
        row_scale[sum(counts):] = float("nan")                     # rows behind the last group are zero whatever their scale
        biases = [None, torch.randn((e, n), generator=g)]
    for bias in biases:
        for rs in (row_scale, None) if row_scale is not None else (None,):
            want = oracle.grouped_matmul(x, w.transpose(1, 2), ends, scale, rs, bias, out)
            put = lambda t: None if t is None else t.cuda()  # noqa: E731
            got = grouped(npu, x.cuda(), w.cuda(), ends.cuda(), out, scale=put(scale), per_token_scale=put(rs), bias=put(bias))
            assert torch.equal(got.cpu(), want)
