"""8-bit rows and their product on the HIP kernels, against 64-bit formulas.

Tolerances: q is a nearest whole number: off by at most half, plus 127 * 2^-22 where fp32 scales 16-bit values (two roundings of
a number up to 127) and 2^-40 where fp64 scales fp32 values; the scale is the fp32 quotient, exactly.  Given q and scales the
sum is exact; the result has one rounding of its type and at most 4 of fp32 (sum to fp32, two products, bias), and 8 more relative
to the pre-activation through silu."""
import ctypes as C

import pytest
import torch

from norm_ref import E32, GroupNormRef, act as act_ref, close
from yolo_amd import _lib
from yolo_amd.groupnorm import group_norm_rows
from yolo_amd.int8 import Int8Conv1x1, Int8Linear, Int8Rows, Int8Weight, conv1x1_i8, linear_i8, quantize_rows, quantize_weight, row_bytes
from test_gpu_groupnorm import cl, make

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def check_rows(rows, x, lead):
    """rows against the values x (n, k) in fp64 that were quantised, on the CPU."""
    k = x.shape[1]
    assert rows.q.dtype is torch.int8 and rows.q.shape == (x.shape[0], row_bytes(k)) and rows.lead == tuple(lead) and rows.k == k
    q = rows.q.cpu().double()
    assert not bool(q[:, k:].any()), 'padding'
    a = x.abs().amax(1, keepdim=True)
    some = a >= 2.0 ** -120
    t = torch.where(some, x * 127 / torch.where(some, a, 1.0), 0.0)
    off = 127 * 2.0 ** -22 if rows.dtype is not F32 else 2.0 ** -40
    assert float((q[:, :k] - t).abs().max()) <= 0.5 + off
    assert torch.equal(rows.scale.cpu(), torch.where(some, a, 0.0)[:, 0].float() / 127)


ROWS = [(1, 1), (1, 16), (3, 17), (5, 8), (257, 31), (1000, 64), (4099, 80), (33, 512), (7, 1000), (2, 4096), (130, 4095), (3, 4097), (2, 20000), (5000, 255)]


@pytest.mark.parametrize('dtype', [F16, BF16, F32], ids=['fp16', 'bf16', 'fp32'])
@pytest.mark.parametrize('m,k', ROWS)
def test_quantize_rows(dev, m, k, dtype):
    g = torch.Generator().manual_seed(m * k)
    x = (torch.randn(m, k, generator=g) * (2 * torch.randn(m, 1, generator=g)).exp()).to(dtype)
    if m > 4:
        x[3] = 0
        x[1] = 1e-7  # subnormal in fp16
    check_rows(quantize_rows(x.to(dev)), x.double(), (m,))
    # a pitch, rows that start off alignment, and a lead of two dimensions
    wide = torch.full((m, k + 5), 1e4, dtype=dtype)
    wide[:, 3:3 + k] = x
    got = quantize_rows(wide.to(dev)[:, 3:3 + k])
    want = quantize_rows(x.to(dev).reshape(1, m, k))
    assert torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale) and want.lead == (1, m)


def test_quantize_rows_extremes(dev):
    inf, nan, big = float('inf'), float('nan'), torch.finfo(F32).max
    x = torch.tensor([[0, 0, 0], [1, inf, 2], [nan, 1, 2], [big, -big, 1], [1e-45, 0, 0], [-2.0 ** -120, 0, 2.0 ** -121], [2.0 ** -121, 0, 0], [-inf, nan, 0]], dtype=F32)
    r = quantize_rows(x.to(dev))
    q, s = r.q.cpu()[:, :3], r.scale.cpu()
    assert s[0] == 0 and s[4] == 0 and s[6] == 0 and not bool(q[[0, 1, 2, 4, 6, 7]].any())
    assert bool(s[[1, 2, 7]].isnan().all())
    assert q[3].tolist() == [127, -127, 0] and q[5].tolist() in ([-127, 0, 63], [-127, 0, 64]) and s[3] == torch.tensor(big) / 127
    y = linear_i8(x.to(dev), Int8Weight(torch.ones(2, 3, dtype=torch.int8, device=dev), torch.ones(2, device=dev)), torch.tensor([0.5, 1.5], device=dev))
    assert bool(y[[1, 2, 7]].isnan().all()) and y[0].tolist() == [0.5, 1.5] and bool(y[[0, 3, 4, 5, 6]].isfinite().all())


def product_ref(q, scale, w, wscale, bias, act, slope):
    whole = q.double() @ w.double().t()  # exact
    s = whole.cpu() * (scale.cpu().double()[:, None] * wscale.cpu().double())
    b = torch.zeros(w.shape[0]).double() if bias is None else bias.cpu().double()
    z = s + b
    return act_ref(z, act, slope), 4 * E32 * (s.abs() + b.abs()) + (8 * E32 * z.abs() if act == 'silu' else 0)


# rows x values x channels: one of each; every edge of a 16-value vector, a 64-value fragment and a tile; the head's 255 channels; rows of
# one token up to several tiles; long rows with few channels and the reverse
PRODUCTS = [(1, 1, 1), (1, 16, 16), (2, 17, 3), (1, 4096, 512), (3, 1000, 255), (16, 64, 64), (17, 65, 33), (64, 128, 128), (65, 129, 257), (333, 1000, 255),
            (300, 80, 72), (1000, 32, 64), (515, 256, 256), (129, 2048, 130), (8, 20000, 24), (4, 640, 4100), (2049, 63, 40), (1030, 520, 392), (700, 1280, 700),
            (20, 2048, 2064), (4100, 60, 130), (66000, 128, 72), (66000, 240, 80), (66000, 500, 33), (2000, 500, 2040), (4090, 512, 2048), (16300, 2000, 1000), (1200000, 144, 1), (1060000, 16, 2)]


@pytest.mark.parametrize('dtype', [F16, BF16, F32], ids=['fp16', 'bf16', 'fp32'])
@pytest.mark.parametrize('m,k,n', PRODUCTS)
def test_product(dev, m, k, n, dtype):
    g = torch.Generator().manual_seed(m + k + n)
    act = (None, 'leaky', 'silu')[(m + k + n) % 3]
    q = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    if m > 2:  # the largest sums there are
        q[0] = 127
        w[0] = -128
    s, ws = torch.rand(m, generator=g) * 0.02 + 1e-3, (torch.rand(n, generator=g) + 0.1) * 0.02 / k ** 0.5
    bias = None if n % 2 else torch.randn(n, generator=g)
    want, err = product_ref(q.to(dev), s, w.to(dev), ws, bias, act, 0.2)
    rows = Int8Rows(torch.nn.functional.pad(q, (0, row_bytes(k) - k)).to(dev), s.to(dev), (m,), k, dtype)
    y = linear_i8(rows, Int8Weight(w.to(dev), ws.to(dev)), None if bias is None else bias.to(dev), act=act, slope=0.2)
    assert y.dtype is dtype
    close(y, want, err, 'y')


@pytest.mark.parametrize('dtype', [F16, BF16, F32], ids=['fp16', 'bf16', 'fp32'])
@pytest.mark.parametrize('m,k,n', [(1, 4096, 96), (2, 30, 7), (5, 257, 300), (13, 1024, 64), (16, 640, 255), (31, 96, 17), (77, 200, 64), (900, 64, 64), (1111, 72, 24), (513, 512, 130), (640, 250, 256),
                                   (4100, 48, 130), (17000, 128, 80), (16500, 240, 33), (16400, 512, 64), (16400, 256, 200), (16400, 272, 20), (4, 16384, 24), (3, 21848, 40)])
def test_linear_from_floating_point(dev, m, k, n, dtype):
    """linear_i8 of a tensor is the product of its quantised rows: the same bits as in two calls, and those within tolerance."""
    g = torch.Generator().manual_seed(m * 7 + k + n)
    x = (torch.randn(m, k, generator=g) * (0.5 * torch.randn(m, 1, generator=g)).exp()).to(dtype)
    if m > 3:
        x[2] = 0
    w = quantize_weight((torch.randn(n, k, generator=g) * k ** -0.5).to(dev))
    bias = torch.randn(n, generator=g).to(dev)
    act = (None, 'leaky', 'silu')[(m + n) % 3]
    rows = quantize_rows(x.to(dev))
    y = linear_i8(x.to(dev), w, bias, act=act)
    assert torch.equal(y, linear_i8(rows, w, bias, act=act))
    want, err = product_ref(rows.q[:, :k], rows.scale, w.q[:, :k], w.scale, bias, act, 0.1)
    close(y, want, err, 'y')
    for other in (F16, F32):
        close(linear_i8(x.to(dev), w, bias, act=act, dtype=other), want, err, 'y as %s' % other)
    wide = torch.zeros(m, k + 3, dtype=dtype, device=dev)
    wide[:, 1:1 + k] = x.to(dev)
    assert torch.equal(y, linear_i8(wide[:, 1:1 + k], w, bias, act=act))
    assert torch.equal(y.reshape(1, m, n), linear_i8(x.to(dev).reshape(1, m, k), w, bias, act=act))


@pytest.mark.parametrize('dtype', [F16, BF16, F32], ids=['fp16', 'bf16', 'fp32'])
@pytest.mark.parametrize('shape,groups', [((1, 16, 1, 1), 4), ((2, 13, 5, 3), 13), ((3, 75, 15, 9), 5), ((1, 512, 20, 20), 32), ((2, 64, 80, 80), 32),
                                          ((1, 4096, 3, 3), 32), ((2, 1280, 7, 5), 32), ((1, 5, 199, 201), 1), ((2, 24, 9), 3), ((1, 2048, 9, 3), 16)],
                         ids=lambda v: str(v).replace(' ', ''))
def test_group_norm_rows(dev, shape, groups, dtype):
    act = (None, 'leaky', 'silu')[sum(shape) % 3]
    x, w, b, _ = make(shape, dtype, sum(shape))
    ref = GroupNormRef(x, groups, w, b, 1e-5, act)
    r = group_norm_rows(x.to(dev), groups, w.to(dev), b.to(dev), act=act)
    c = shape[1]
    z, err = (v.movedim(1, -1).reshape(-1, c) for v in (ref.y, ref.err_y))
    assert r.lead == (shape[0], *shape[2:]) and r.k == c and r.dtype is dtype
    q, s = r.q.cpu().double(), r.scale.cpu().double()[:, None]
    assert not bool(q[:, c:].any())
    a = z.abs().amax(1, keepdim=True)
    assert bool(((s * 127 - a).abs() <= err.amax(1, keepdim=True) + 2 * E32 * a).all())
    far = (q[:, :c] * s - z).abs() - (0.5 * s * (1 + 2.0 ** -14) + err)
    assert float(far.max()) <= 0


@pytest.mark.parametrize('hw', [(5, 3), (90, 81)])
def test_chain_of_norm_and_convolution(dev, hw):
    """norm -> activation -> 8-bit 1x1 convolution, as a half model runs it, against the same in 64 bits: an 8-bit row is off by half
    a step of its largest value / 127 a value, independently, so a sum over c values by that times sqrt(c / 12) |w| (5 deviations)."""
    c, n = 64, 40
    x, w, b, _ = make((2, c, *hw), F16, 23)
    g = torch.Generator().manual_seed(2)
    conv = torch.nn.Conv2d(c, n, 1)
    conv.weight.data = torch.randn(n, c, 1, 1, generator=g) * c ** -0.5
    layer = Int8Conv1x1.from_conv(conv).to(dev).half()
    assert layer.scale.dtype is F32 and layer.bias.dtype is F32
    rows = group_norm_rows(x.to(dev), 8, w.to(dev), b.to(dev), act='silu')
    y = layer(rows)
    assert y.shape == (2, n, *hw) and y.movedim(1, -1).is_contiguous() and y.dtype is F16
    z = GroupNormRef(x, 8, w, b, 1e-5, 'silu').y
    wq = layer.q[:, :c].cpu().double() * layer.scale.cpu().double()[:, None]
    want = torch.einsum('bchw,nc->bnhw', z, wq) + conv.bias.detach().double()[:, None, None]
    step = z.abs().amax(1, keepdim=True) / 127
    slack = 5 * step * (wq ** 2).sum(1).sqrt()[:, None, None] / 12 ** 0.5 + 1e-3 * step
    close(y, want, slack, 'y')
    # the same rows one image at a time
    one = layer(group_norm_rows(x[1:].to(dev), 8, w.to(dev), b.to(dev), act='silu'))
    assert torch.equal(one[0], y[1])


def test_layers_of_the_model(dev):
    """models.common.Conv blocks and linear layers as 8-bit layers; maps and channel slices as their input."""
    from yolo_amd.models.common import Conv
    torch.manual_seed(0)
    block = Conv(48, 56, 1, 1).eval()
    block.bn.running_mean.normal_()
    block.bn.running_var.uniform_(0.5, 2)
    layer = Int8Conv1x1.from_conv(block).to(dev)
    assert layer.act == 'leaky' and layer.slope == pytest.approx(0.1)
    x, *_ = make((2, 48, 9, 7), F16, 29)
    want = block(x.float())
    got = layer(x.to(dev)).float().cpu()
    assert float((got - want).norm() / want.norm()) < 0.02  # two 8-bit roundings: 1 / 254 of the largest, over values of a third of it
    wide = torch.zeros(2, 9, 7, 100, dtype=F16, device=dev).permute(0, 3, 1, 2)
    wide[:, 24:72] = x.to(dev)
    assert torch.equal(layer(wide[:, 24:72]), layer(x.to(dev))) and torch.equal(layer(x.to(dev).contiguous()), layer(x.to(dev)))
    lin = torch.nn.Linear(48, 10)
    q = Int8Linear.from_linear(lin).to(dev)
    t = torch.randn(3, 5, 48)
    assert float((q(t.to(dev)).cpu() - lin(t)).norm() / lin(t).norm()) < 0.02
    again = Int8Linear(Int8Weight(torch.zeros(10, 48, dtype=torch.int8), torch.ones(10)), torch.zeros(10)).to(dev)
    again.load_state_dict(q.state_dict())
    assert torch.equal(again(t.to(dev)), q(t.to(dev)))


def test_graphs_streams_and_neighbours(dev):
    """Two captured graphs in turn with eager work between them, two streams at once, and memory behind the output left alone."""
    g = torch.Generator().manual_seed(31)
    for m, k, n in ((1, 512, 96), (70, 200, 255), (600, 96, 64), (1000, 512, 512)):
        w = quantize_weight(torch.randn(n, k, generator=g).to(dev))
        bias = torch.randn(n, generator=g).to(dev)
        xs = [torch.randn(m, k, generator=g).half().to(dev) for _ in range(2)]
        want = [linear_i8(x, w, bias, act='silu') for x in xs]
        x = xs[0].clone()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = linear_i8(x, w, bias, act='silu')
            graphs.append((graph, out))
        for turn in range(3):
            x.copy_(xs[turn % 2])
            linear_i8(xs[1], w, bias)
            for graph, out in graphs:
                graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(out, want[turn % 2]) for _, out in graphs)
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s, v in zip(streams, xs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(linear_i8(v, w, bias, act='silu'))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        # through the C entry point: rows of a wider buffer
        rows = quantize_rows(xs[0])
        wide = torch.full((m + 2, n + 7), 9.0, dtype=F16, device=dev)
        d = _lib.GemmI8Desc(a=rows.q.data_ptr(), a_scale=rows.scale.data_ptr(), w=w.q.data_ptr(), w_scale=w.scale.data_ptr(), bias=bias.data_ptr(),
                            y=wide.data_ptr() + 2 * (n + 7 + 3), m=m, y_ld=n + 7, n=n, k=k, ld=rows.q.shape[1], dtype=_lib.F16, act=_lib.ACT_SILU)
        _lib.check(_lib.lib().y5_gemm_i8(C.byref(d), _lib.current_stream()))
        assert torch.equal(wide[1:m + 1, 3:n + 3], want[0])
        wide[1:m + 1, 3:n + 3] = 9
        assert bool((wide == 9).all())


def test_many_rows(dev):
    """More than 2^31 bytes of rows and of outputs: offsets beyond 32 bits."""
    k, n, m = 64, 64, 36_000_000
    w = Int8Weight(torch.eye(n, k, device=dev).to(torch.int8), torch.ones(n, device=dev))
    q = torch.zeros((m, k), dtype=torch.int8, device=dev)
    idx = torch.tensor([0, 1, 127, 128, 16_777_216, 33_554_431, 33_554_432, 33_554_500, m - 129, m - 1], device=dev)
    vals = torch.randint(-127, 128, (len(idx), k), device=dev, dtype=torch.int8)
    q[idx] = vals
    y = linear_i8(Int8Rows(q, torch.ones(m, device=dev), (m,), k, F16), w)
    assert torch.equal(y[idx], vals.half())
    assert int((y != 0).any(1).sum()) == int((vals != 0).any(1).sum())


def test_one_row_and_scalars(dev):
    w = quantize_weight(torch.randn(24, 40, generator=torch.Generator().manual_seed(1)).to(dev))
    x = torch.randn(3, 40, generator=torch.Generator().manual_seed(2)).half().to(dev)
    y = linear_i8(x, w)
    assert torch.equal(linear_i8(x[1], w), y[1]) and linear_i8(x[1], w).shape == (24,)
    assert torch.equal(linear_i8(quantize_rows(x[1]), w), y[1])
    assert torch.equal(linear_i8(x[1].expand(5, 40), w), y[1].expand(5, 24))  # a pitch of zero
    assert torch.equal(linear_i8(x.t().contiguous().t(), w), y)
    one = Int8Weight(torch.full((3, 1), 5, dtype=torch.int8, device=dev), torch.ones(3, device=dev))
    t = torch.tensor([[2.0], [-3.0], [0.0]], device=dev)
    assert torch.allclose(linear_i8(t, one), (5 * t).expand(3, 3), rtol=1e-6)


def test_empty(dev):
    w = Int8Weight(torch.ones(4, 8, dtype=torch.int8, device=dev), torch.ones(4, device=dev))
    assert linear_i8(torch.zeros(0, 8, device=dev), w).shape == (0, 4)
    assert conv1x1_i8(torch.zeros(2, 8, 0, 3, device=dev), w).shape == (2, 4, 0, 3)
    assert group_norm_rows(torch.zeros(0, 8, 2, 2, device=dev), 2).shape == (0, 2, 2, 8)
