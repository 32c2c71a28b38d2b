"""npu_grouped_matmul (int8 rows sorted by expert times their expert's weight) against the CPU oracle, bit for bit."""
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


def operands(counts, tail, k, n, g):
    e, m = len(counts), sum(counts) + tail
    x = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int64).to(torch.int8)
    w = torch.randint(-128, 128, (e, n, k), generator=g, dtype=torch.int64).to(torch.int8)
    scale = torch.rand((e, n), generator=g) * 9e-3 + 1e-3
    row_scale = torch.rand((m,), generator=g) * 9e-3 + 1e-3
    return x, w, scale, row_scale, torch.cumsum(torch.tensor(counts), 0)


def call(npu, x, w_ekn, ends, out, **kw):
    lists = {k: [v] for k, v in kw.items() if k in ("scale", "per_token_scale", "bias") and v is not None}
    rest = {k: v for k, v in kw.items() if k not in ("scale", "per_token_scale", "bias")}
    return npu.npu_grouped_matmul([x], [w_ekn], group_list=ends, split_item=3, group_type=0, output_dtype=out, **lists, **rest)[0]


# counts, tail, k, n: one row; empty groups at both ends and between; a tile's edges (16, 64, 256 and one more); several
# tiles of a group; widths that fill no tile; k of one block, a part of one, many; rows behind the last group; one group.
CASES = [([1], 0, 16, 8), ([0, 1, 0, 2, 0], 3, 128, 130), ([16, 17, 64, 65], 0, 256, 128), ([15, 0, 48, 33], 1, 144, 264),
         ([256, 257, 1], 0, 128, 256), ([512, 513, 300, 0], 5, 384, 520), ([100, 1000, 40, 7], 0, 1040, 200), ([0, 0, 0], 9, 64, 64),
         ([700], 0, 4096, 384), ([3] * 64, 0, 512, 384), ([2, 0] * 512, 0, 128, 136), ([5, 400, 0, 31], 0, 2048, 1416)]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.int32])
def test_matches_the_oracle(npu, case, out):
    counts, tail, k, n = CASES[case]
    g = torch.Generator().manual_seed(case)
    x, w, scale, row_scale, ends = operands(counts, tail, k, n, g)
    row_scale[sum(counts):] = float("nan")                 # rows behind the last group are zero whatever their scale
    acc = out == torch.int32
    want = oracle.grouped_matmul(x, w.transpose(1, 2), ends, None if acc else scale, None if acc else row_scale, None, out)
    kw = {} if acc else dict(scale=scale.cuda(), per_token_scale=row_scale.cuda())
    got = call(npu, x.cuda(), w.cuda().transpose(1, 2), ends.cuda(), out, **kw)
    assert got.dtype == out and torch.equal(got.cpu(), want)
    got = call(npu, x.cuda(), w.cuda().transpose(1, 2), torch.tensor(counts, dtype=torch.int32).cuda(), out, group_list_type=1, **kw)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("bias", [torch.int32, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sdtype", [torch.float32, torch.bfloat16, torch.int64])
@pytest.mark.parametrize("counts", [[3, 0, 20], [300, 0, 77]])
def test_bias_and_scale_types(npu, bias, sdtype, counts):
    g = torch.Generator().manual_seed(3)
    x, w, scale, row_scale, ends = operands(counts, 0, 256, 192, g)
    b = torch.randint(-1000, 1000, (3, 192), generator=g).to(bias)
    s = scale.view(torch.int32).to(torch.int64) if sdtype == torch.int64 else scale.to(sdtype)
    for rs in (row_scale, None):
        want = oracle.grouped_matmul(x, w.transpose(1, 2), ends, s, rs, b, torch.float16)
        got = call(npu, x.cuda(), w.cuda().transpose(1, 2), ends.cuda(), torch.float16, scale=s.cuda(), bias=b.cuda(),
                   per_token_scale=None if rs is None else rs.cuda())
        assert torch.equal(got.cpu(), want)
    if bias == torch.int32:
        want = oracle.grouped_matmul(x, w.transpose(1, 2), ends, None, None, b, torch.int32)
        assert torch.equal(call(npu, x.cuda(), w.cuda().transpose(1, 2), ends.cuda(), torch.int32, bias=b.cuda()).cpu(), want)


def test_layouts(npu):
    """Weights that the tensor cores do not take (n-major, k not a multiple of 16, off the 16-byte grid) and ones with gaps
    between rows and experts, which they do."""
    g = torch.Generator().manual_seed(4)
    for counts, k, n in (([5, 0, 40], 96, 72), ([5, 300, 40], 96, 72), ([5, 0, 40], 37, 19), ([5, 0, 40], 40, 16)):
        x, w, scale, row_scale, ends = operands(counts, 2, k, n, g)
        want = oracle.grouped_matmul(x, w.transpose(1, 2), ends, scale, row_scale, None, torch.bfloat16)
        kw = dict(scale=scale.cuda(), per_token_scale=row_scale.cuda())
        gaps = torch.zeros((3, n + 3, (k + 15) // 16 * 16 + 32), dtype=torch.int8, device="cuda")
        gaps[:, :n, :k] = w.cuda()
        off = torch.zeros(w.numel() + 1, dtype=torch.int8, device="cuda")[1:].reshape(w.shape)
        off.copy_(w)
        wide = torch.zeros((x.shape[0], k + 16), dtype=torch.int8, device="cuda")
        wide[:, 8:k + 8] = x.cuda()
        for weight, rows in ((w.cuda().transpose(1, 2), x.cuda()), (w.cuda().transpose(1, 2).contiguous(), x.cuda()),
                             (gaps[:, :n, :k].transpose(1, 2), x.cuda()), (off.transpose(1, 2), x.cuda()), (w.cuda().transpose(1, 2), wide[:, 8:k + 8])):
            assert torch.equal(call(npu, rows, weight, ends.cuda(), torch.bfloat16, **kw).cpu(), want)


def test_bad_lists_stay_inside(npu):
    """Ends that go down, are negative or past the rows are clamped; counts past the rows too."""
    g = torch.Generator().manual_seed(5)
    x, w, scale, row_scale, _ = operands([10, 10, 10, 10], 0, 128, 64, g)
    kw = dict(scale=scale.cuda(), per_token_scale=row_scale.cuda())
    for listed, kind, ends in (([20, 10, 2 ** 40, 30], 0, [20, 20, 40, 40]), ([-5, -1, 12, 12], 0, [0, 0, 12, 12]),
                               ([30, -7, 2 ** 40, 5], 1, [30, 30, 40, 40]), ([0, 0, 0, 0], 1, [0, 0, 0, 0])):
        want = oracle.grouped_matmul(x, w.transpose(1, 2), ends, scale, row_scale, None, torch.float16)
        got = call(npu, x.cuda(), w.cuda().transpose(1, 2), torch.tensor(listed).cuda(), torch.float16, group_list_type=kind, **kw)
        assert torch.equal(got.cpu(), want)


def test_empty_calls_streams_and_captured_graphs(npu):
    g = torch.Generator().manual_seed(6)
    x, w, scale, row_scale, ends = operands([40, 0, 300, 5], 3, 256, 320, g)
    cx, cw, cs, cr, ce = x.cuda(), w.cuda().transpose(1, 2), scale.cuda(), row_scale.cuda(), ends.cuda()
    e = call(npu, cx[:0], cw, torch.zeros(4, dtype=torch.int64, device="cuda"), torch.bfloat16, scale=cs, per_token_scale=cr[:0])
    assert e.shape == (0, 320)
    e = call(npu, cx, cw[:, :, :0], ce, torch.bfloat16, scale=cs[:, :0], per_token_scale=cr)
    assert e.shape == (348, 0)
    e = call(npu, cx[:, :0], cw[:, :0], ce, torch.bfloat16, scale=cs, per_token_scale=cr)
    assert e.shape == (348, 320) and float(e.abs().sum()) == 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = call(npu, cx, cw, ce, torch.bfloat16, scale=cs, per_token_scale=cr)
    b = call(npu, cx, cw, ce, torch.bfloat16, scale=cs, per_token_scale=cr)   # at the same time as the other stream's
    side.synchronize()
    assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(npu, cx, cw, ce, torch.bfloat16, scale=cs, per_token_scale=cr)
    for new in ([348, 348, 348, 348], [0, 0, 0, 1], [100, 101, 200, 340]):
        ce.copy_(torch.tensor(new))
        cx.copy_(torch.randint(-128, 128, x.shape, generator=g).to(torch.int8))
        graph.replay()
        assert torch.equal(out, call(npu, cx, cw, ce, torch.bfloat16, scale=cs, per_token_scale=cr))
        want = oracle.grouped_matmul(cx.cpu(), w.transpose(1, 2), new, scale, row_scale, None, torch.bfloat16)
        assert torch.equal(out.cpu(), want)
