"""Channels-last group norm with an activation on the HIP kernels, against 64-bit formulas (tests/norm_ref.py).

Tolerances: one rounding to the output type (half a step) plus 64 fp32 roundings of the largest value each sum or difference
handles - a serial chain of the kernels is at most ~64 additions long before partial sums meet pairwise or in short rows."""
import ctypes as C

import pytest
import torch

from norm_ref import GroupNormRef, close
from yolo_amd import _lib
from yolo_amd.groupnorm import GroupNormAct, group_norm

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def cl(x):
    return x.movedim(1, -1).contiguous().movedim(-1, 1)


def make(shape, dtype, seed, param=None, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    c = shape[1]
    per = (1, c) + (1,) * (len(shape) - 2)
    x = torch.randn(shape, generator=g) * (0.5 * torch.randn(per, generator=g)).exp() + 0.5 * torch.randn(per, generator=g) + shift
    w, b = 1 + 0.2 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g)
    return cl(x.to(dtype)), w.to(param or dtype), b.to(param or dtype), cl(torch.randn(shape, generator=g).to(dtype))


# (batch, channels, *spatial), groups: one value a group and image; groups of every alignment against a 16-byte vector; odd
# channel counts (several pixels a vector, images that start off alignment, rows cut short); one pixel; maps beyond one
# workgroup (the two-pass form) in each of those; the widest channel counts
SHAPES = [
    ((1, 1, 1, 1), 1), ((2, 4, 1, 1), 4), ((2, 4, 3), 2), ((3, 6), 2), ((2, 13, 5, 3), 13), ((1, 25, 7, 1), 5), ((3, 75, 45, 27), 5),
    ((1, 512, 20, 20), 32), ((2, 32, 64, 64), 1), ((2, 64, 17, 19), 32), ((2, 24, 9, 5), 8), ((3, 3, 181, 179), 1), ((2, 160, 13, 11), 32),
    ((2, 64, 80, 80), 32), ((1, 128, 80, 81), 32), ((1, 96, 101, 99), 4), ((1, 160, 90, 80), 32), ((2, 5, 199, 201), 5), ((2, 2, 300, 301), 1),
    ((1, 4096, 3, 3), 32), ((1, 4096, 2, 30), 4096), ((2, 511, 3, 5), 7), ((1, 1280, 25, 40), 32), ((1, 2, 2, 3, 4), 2), ((2, 16, 40, 33), 1),
    ((1, 1024, 1, 1), 32), ((5, 8, 1, 37), 8), ((1, 4000, 40, 41), 1), ((1, 4096, 40, 41), 4096), ((1, 4096, 33, 31), 512), ((2, 512, 90, 3), 512), ((300, 24, 1, 2), 3),
]


@pytest.mark.parametrize('dtype', [F16, BF16, F32], ids=['fp16', 'bf16', 'fp32'])
@pytest.mark.parametrize('shape,groups', SHAPES, ids=lambda v: str(v).replace(' ', ''))
def test_forward_and_gradient(dev, shape, groups, dtype):
    act = (None, 'leaky', 'silu')[sum(shape) % 3]
    x, w, b, dy = make(shape, dtype, sum(shape), F32 if groups % 2 else dtype)
    z = GroupNormRef(x, groups, w, b, 1e-5, act).z
    if act == 'leaky':
        dy = dy * (z.abs() > 1e-3).to(dtype)  # the activation's kink: either side is right there
    ref = GroupNormRef(x, groups, w, b, 1e-5, act, dy=dy)
    with torch.enable_grad():
        xd, wd, bd = (v.to(dev).requires_grad_() for v in (x, w, b))
        y = group_norm(xd, groups, wd, bd, act=act)
        dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.to(dev))
    assert y.dtype is dtype and dx.dtype is dtype and dw.dtype is w.dtype and y.movedim(1, -1).is_contiguous()
    close(y, ref.y, ref.err_y, 'y')
    close(dx, ref.dx, ref.err_dx, 'dx')
    close(dw, ref.dgamma, ref.err_dgamma, 'dgamma')
    close(db, ref.dbeta, ref.err_dbeta, 'dbeta')
    assert torch.equal(y, group_norm(x.to(dev), groups, w.to(dev), b.to(dev), act=act)), 'the same call without gradients'


@pytest.mark.parametrize('act', [None, 'leaky', 'silu'])
@pytest.mark.parametrize('affine', [(True, False), (False, True), (False, False)])
def test_without_parameters(dev, act, affine):
    x, w, b, dy = make((2, 24, 9, 7), F32, 3)
    w, b = w if affine[0] else None, b if affine[1] else None
    ref = GroupNormRef(x, 4, w, b, 1e-3, act, 0.25, dy)
    with torch.enable_grad():
        leaves = [v.to(dev).requires_grad_() for v in (x, w, b) if v is not None]
        it = iter(leaves[1:])
        y = group_norm(leaves[0], 4, next(it) if w is not None else None, next(it) if b is not None else None, 1e-3, act, 0.25)
        grads = torch.autograd.grad(y, leaves, dy.to(dev))
    close(y, ref.y, ref.err_y, 'y')
    close(grads[0], ref.dx, ref.err_dx, 'dx')
    if w is not None:
        close(grads[1], ref.dgamma, ref.err_dgamma, 'dgamma')
    if b is not None:
        close(grads[-1], ref.dbeta, ref.err_dbeta, 'dbeta')


def test_gradient_against_differences(dev):
    """The gradient in a random direction against central differences of the fp32 kernel's own output: step h changes the loss by
    h |grad| with an error of h^2 and of roundings / h."""
    x, w, b, dy = (v.to(dev) for v in make((2, 16, 6, 5), F32, 9))
    d = [torch.randn(v.shape, generator=torch.Generator().manual_seed(1)).to(dev) for v in (x, w, b)]
    d[0] = d[0].to(memory_format=torch.channels_last)
    with torch.enable_grad():
        leaves = [v.clone().requires_grad_() for v in (x, w, b)]
        grads = torch.autograd.grad(group_norm(leaves[0], 4, leaves[1], leaves[2], act='silu'), leaves, dy)

    def loss(h, i):
        v = [x, w, b]
        v[i] = v[i] + h * d[i]
        return (group_norm(v[0], 4, v[1], v[2], act='silu').double() * dy.double()).sum()

    for i in range(3):
        h = 1e-2
        numeric = float((loss(h, i) - loss(-h, i)) / (2 * h))
        want = float((grads[i].double() * d[i].double()).sum())
        # h^2 / 6 times the third derivative (O(10) of the terms' sum) + 960 roundings of 2^-24 * 4 / h
        slack = float((grads[i].double() * d[i].double()).abs().sum()) * 10 * h * h + 960 ** 0.5 * 2.0 ** -22 / h
        assert abs(numeric - want) <= slack, (i, numeric, want, slack)


@pytest.mark.parametrize('hw', [(6, 5), (150, 141)])
def test_mean_far_from_zero(dev, hw):
    x, w, b, _ = make((2, 32, *hw), F32, 5, shift=300.0)
    ref = GroupNormRef(x, 8, w, b, 1e-5, None)
    close(group_norm(x.to(dev), 8, w.to(dev), b.to(dev)), ref.y, ref.err_y, 'y')


@pytest.mark.parametrize('dtype', [F16, F32])
@pytest.mark.parametrize('hw', [(9, 7), (120, 113)])
def test_layouts(dev, dtype, hw):
    """Channel slices of wider maps (on and off 16 bytes), batch slices, torch's contiguous layout, permuted views, a broadcast
    gradient: the same bits as the channels_last tensor."""
    x, w, b, dy = (v.to(dev) for v in make((2, 16, *hw), dtype, 7))
    wide = cl(torch.full((3, 64, *hw), 5.0, dtype=dtype, device=dev))

    def both(x, dy):
        with torch.enable_grad():
            x = x.detach().requires_grad_()
            y = group_norm(x, 4, w, b, act='silu')
            return y.detach(), torch.autograd.grad(y, x, dy)[0]

    want = both(x, dy)
    for name, at in (('slice', 16), ('slice off 16 bytes', 3)):
        v = wide.clone(memory_format=torch.preserve_format)
        v[1:, at:at + 16] = x
        v = v[1:, at:at + 16]
        assert v.stride(1) == 1 and v.data_ptr() % 16 == (0 if at == 16 else 3 * v.element_size() % 16)
        got = both(v, dy)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), name
    got = both(x.contiguous(), dy.contiguous())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = both(x.transpose(2, 3).contiguous().transpose(2, 3), dy)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = torch.ones((), dtype=dtype, device=dev).expand(x.shape)
    assert torch.equal(both(x, one)[1], both(x, one.clone())[1])


@pytest.mark.parametrize('hw', [(6, 5), (160, 121)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_not_finite_stays_in_its_group(dev, hw, bad):
    x, w, b, _ = (v.to(dev) for v in make((2, 64, *hw), F16, 11))
    want = group_norm(x, 8, w, b, act='leaky')
    x[1, 19, hw[0] // 2, 1] = bad
    got = group_norm(x, 8, w, b, act='leaky')
    assert bool(got[1, 16:24].isnan().all())
    got[1, 16:24] = want[1, 16:24]
    assert torch.equal(got, want)


@pytest.mark.parametrize('c,hw', [(64, (9, 5)), (64, (160, 120)), (5, (300, 201))])
def test_bits_do_not_depend_on_batch_stream_or_replay(dev, c, hw):
    x, w, b, dy = (v.to(dev) for v in make((3, c, *hw), F16, 13))
    groups = 5 if c == 5 else 32

    def step(x, dy):
        with torch.enable_grad():
            leaves = [v.detach().requires_grad_() for v in (x, w, b)]
            y = group_norm(leaves[0], groups, leaves[1], leaves[2], act='silu')
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = step(x, dy)
    torch.cuda.synchronize()
    for i in range(3):
        one = step(x[i:i + 1], dy[i:i + 1])
        assert torch.equal(one[0][0], want[0][i]) and torch.equal(one[1][0], want[1][i])
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:  # two calls at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(x, dy))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(g, want))
    graphs = []
    xs, ds = x.clone(memory_format=torch.preserve_format), dy.clone(memory_format=torch.preserve_format)
    for _ in range(2):  # two graphs of the same call, replayed in turn, with eager work between
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(xs, ds)
        graphs.append((graph, out))
    for turn in range(3):
        flip = turn % 2 == 1
        xs.copy_(x.flip(0) if flip else x)
        ds.copy_(dy.flip(0) if flip else dy)
        expect = step(xs, ds)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, expect)), turn


def test_writes_only_its_own_channels(dev):
    """Through the C entry point: output slices of wider buffers, and y over x."""
    lib = _lib.lib()
    for hw in ((7, 5), (130, 121)):
        x, w, b, _ = (v.to(dev) for v in make((2, 16, *hw), F16, 17))
        want = group_norm(x, 2, w, b, act='leaky')
        wide = torch.full((2, *hw, 40), 7.0, dtype=F16, device=dev)
        wide[..., 8:24] = x.permute(0, 2, 3, 1)
        d = _lib.GroupNormDesc(x=wide.data_ptr() + 16, y=wide.data_ptr() + 16, weight=w.data_ptr(), bias=b.data_ptr(), batch=2,
                               pixels=hw[0] * hw[1], c=16, groups=2, x_ld=40, y_ld=40, act=_lib.ACT_LEAKY, slope=0.1, eps=1e-5)
        n = C.c_size_t()
        _lib.check(lib.y5_group_norm_workspace(C.byref(d), _lib.GN_FORWARD, C.byref(n)))
        ws = torch.empty(max(n.value, 16), dtype=torch.uint8, device=dev)
        d.workspace, d.workspace_bytes = ws.data_ptr(), n.value
        if n.value:
            d.workspace_bytes -= 1
            assert lib.y5_group_norm(C.byref(d), _lib.current_stream()) == _lib.EWORKSPACE
            d.workspace_bytes += 1
        _lib.check(lib.y5_group_norm(C.byref(d), _lib.current_stream()))
        assert torch.equal(wide[..., 8:24].permute(0, 3, 1, 2), want)
        assert bool((wide[..., :8] == 7).all()) and bool((wide[..., 24:] == 7).all())


def test_differentiable_once(dev):
    x, w, b, dy = (v.to(dev) for v in make((1, 8, 3, 2), F32, 41))
    with torch.enable_grad():
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        plain = torch.autograd.grad(group_norm(leaves[0], 2, leaves[1], leaves[2], act='silu'), leaves, dy)
        again = torch.autograd.grad(group_norm(leaves[0], 2, leaves[1], leaves[2], act='silu'), leaves, dy, create_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(plain, again))
        with pytest.raises(RuntimeError, match='differentiable once'):
            again[0].sum().backward()
        y = group_norm(leaves[0], 2, leaves[1], leaves[2])
        with torch.no_grad():
            leaves[0].mul_(2)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.sum().backward()


def test_errors_of_the_library_and_leaf_gradients(dev):
    with pytest.raises(_lib.Y5Error, match='channels'):
        group_norm(torch.zeros(1, 513, 2, 2, dtype=F16, device=dev), 1)
    with pytest.raises(_lib.Y5Error, match='batch'):
        group_norm(torch.zeros(65536, 8, dtype=F16, device=dev), 1)
    # gradients accumulate on leaves of several layouts; bias alone, weight alone
    x, w, b, dy = (v.to(dev) for v in make((2, 24, 5, 4), F16, 43))
    want = torch.autograd.grad
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)):
        with torch.enable_grad():
            leaves = [v.detach().clone().requires_grad_(bool(n)) for v, n in zip((x, w, b), need)]
            full = [v.detach().clone().requires_grad_() for v in (x, w, b)]
            grads = want(group_norm(full[0], 4, full[1], full[2], act='leaky'), full, dy)
            for _ in range(2):
                group_norm(leaves[0], 4, leaves[1], leaves[2], act='leaky').backward(dy.contiguous())
        for leaf, n, g in zip(leaves, need, grads):
            assert (leaf.grad is not None) == bool(n) and (not n or torch.equal(leaf.grad, g + g))


def test_empty_and_module(dev):
    for shape in ((0, 8, 3, 3), (2, 8, 0, 3)):
        with torch.enable_grad():
            x = torch.zeros(shape, device=dev, requires_grad=True)
            y = group_norm(x, 2, torch.ones(8, device=dev), None)
            y.sum().backward()
        assert y.shape == x.shape == x.grad.shape
    m = GroupNormAct(4, 16).to(dev)
    x, *_ = make((2, 16, 5, 4), F16, 19)
    m.load_state_dict(torch.nn.GroupNorm(4, 16).state_dict())
    ref = GroupNormRef(x, 4, None, None, 1e-5, 'leaky')
    close(m(x.to(dev)), ref.y, ref.err_y, 'y')  # fp32 parameters beside an fp16 map
    with torch.enable_grad():
        m.half()(x.to(dev).requires_grad_()).float().sum().backward()
    assert m.weight.grad.dtype is F16
    # only the parameters' gradients wanted
    with torch.enable_grad():
        y = m(x.to(dev))
        m.zero_grad()
        y.backward(torch.ones_like(y))
    ref = GroupNormRef(x, 4, None, None, 1e-5, 'leaky', dy=torch.ones(x.shape))
    close(m.weight.grad, ref.dgamma, ref.err_dgamma + 0.9 * (ref.z.abs() < 1e-5).sum((0, 2, 3)) * 1e-5, 'dgamma')


def test_capture_beside_a_live_graph_is_refused(dev):
    """A leaf whose accumulation node lives on the default stream cannot be reached by a captured gradient; the same leaf can once that graph
    is gone."""
    x, w, b, dy = (v.to(dev) for v in make((2, 16, 5, 4), F16, 47))
    with torch.enable_grad():
        leaves = [v.detach().clone().requires_grad_() for v in (x, w, b)]
        alive = group_norm(leaves[0], 4, leaves[1], leaves[2], act='silu')
        want = torch.autograd.grad(alive, leaves, dy, retain_graph=True)
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            y = group_norm(leaves[0], 4, leaves[1], leaves[2], act='silu')
            with pytest.raises(RuntimeError, match='live graph'):
                torch.autograd.grad(y, leaves, dy)
        del alive, y
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(group_norm(leaves[0], 4, leaves[1], leaves[2], act='silu'), leaves, dy)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize('shape,groups,reps,dtype', [((3, 64, 160, 160), 32, 16, F16), ((3, 256, 20, 20), 32, 22, F16), ((3, 256, 20, 20), 32, 171, BF16), ((3, 512, 10, 10), 32, 40, F32),
                                                     ((3, 75, 27, 27), 25, 667, BF16), ((3, 256, 40, 40), 32, 22, F16), ((3, 128, 40, 40), 32, 11, BF16)],
                         ids=lambda v: str(v).replace(' ', ''))
def test_large_batches(dev, shape, groups, reps, dtype):
    """Batches that take wide slices, more vectors a thread, the split form for a gradient alone, or stores past the cache: three images over and
    over, whose results are as right as those of the three and the same every time.  The parameters' gradients add up to 2001 rows in 16
    chains, of 126 + 16 additions: (142 + 64) / 64 times the bound of the three."""
    x, w, b, dy = make(shape, dtype, sum(shape), F32)
    ref = GroupNormRef(x, groups, w, b, 1e-5, 'silu', dy=dy)

    def over(v):
        v = v.to(dev).movedim(1, -1).contiguous()
        return v.repeat(reps, *[1] * (v.dim() - 1)).movedim(-1, 1)

    with torch.enable_grad():
        leaves = [v.requires_grad_() for v in (over(x), w.to(dev), b.to(dev))]
        y = group_norm(leaves[0], groups, leaves[1], leaves[2], act='silu')
        dx, dw, db = torch.autograd.grad(y, leaves, over(dy))
    y = y.detach()
    inference = group_norm(leaves[0].detach(), groups, leaves[1].detach(), leaves[2].detach(), act='silu')
    for got, want, err, name in ((y, ref.y, ref.err_y, 'y'), (dx, ref.dx, ref.err_dx, 'dx'), (inference, ref.y, ref.err_y, 'y without gradient')):
        close(got[-3:], want, err, name)
        for i in range(reps):
            assert torch.equal(got[3 * i:3 * i + 3], got[-3:]), (name, i)
    close(dw, reps * ref.dgamma, 4 * reps * ref.err_dgamma, 'dgamma')
    close(db, reps * ref.dbeta, 4 * reps * ref.err_dbeta, 'dbeta')
