"""Group norm with an activation over channels-last feature maps, its gradient, and its 8-bit form, on HIP kernels.

The reference's blocks normalise with BatchNorm2d (models/common.py:27), whose batch statistics need more images a step than
fine-tuning or the pruning search's short runs have; this is the normalisation for those: statistics over the pixels and
the channels of a group, image by image.

    y = group_norm(x, num_groups, weight, bias, eps, act='leaky')       # differentiable
    rows = group_norm_rows(x, num_groups, weight, bias, eps, act=...)   # 8-bit rows for yolo_amd.int8.conv1x1_i8

x is (batch, channels, *spatial), fp16 / bf16 / fp32, in channels_last memory (a channel slice of a wider channels_last tensor
included); another layout is copied to channels_last first.  The result is channels_last.  Arithmetic is fp32 with one
rounding at the end; sums are taken in a fixed order.  CPU tensors go through torch's own operators.

Channels: any number the groups divide, up to 4096 (multiples of 8; multiples of 4 in fp32); at a lesser divisibility up to
4096 / (8 / gcd(channels, 8)), e.g. 512 for odd counts in 16 bits.
"""
import ctypes as C

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from yolo_amd import _lib

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_ACTS = {None: _lib.ACT_NONE, 'leaky': _lib.ACT_LEAKY, 'silu': _lib.ACT_SILU}


def act_code(act):
    if act not in _ACTS:
        raise ValueError("act must be None, 'leaky' or 'silu', got %r" % (act,))
    return _ACTS[act]


def apply_act(z, act, slope):
    """The activation in torch operators (CPU tensors)."""
    if act == 'leaky':
        return torch.where(z > 0, z, z * slope)
    return z * torch.sigmoid(z) if act == 'silu' else z


def pixel_pitch(x):
    """Elements from one pixel of x (batch, channels, *spatial) to the next when its memory is (batch, pixels, channels) at one
    pitch, else None."""
    c = x.shape[1]
    if c != 1 and x.stride(1) != 1:
        return None
    pitch = expect = None
    for d in list(range(x.dim() - 1, 1, -1)) + [0]:
        if x.shape[d] == 1:
            continue
        if expect is None:
            pitch = expect = x.stride(d)
        elif x.stride(d) != expect:
            return None
        expect *= x.shape[d]
    return c if pitch is None else pitch if pitch >= c else None


def channels_last(x):
    """x itself where the kernels can walk it, else a channels_last copy; with its pixel pitch."""
    pitch = pixel_pitch(x)
    if pitch is None or (pitch != x.shape[1] and x.shape[1] * x.element_size() % 16):
        x = x.movedim(1, -1).contiguous().movedim(-1, 1)
        pitch = x.shape[1]
    return x, pitch


def empty_channels_last(shape, dtype, device):
    return torch.empty((shape[0], *shape[2:], shape[1]), dtype=dtype, device=device).movedim(-1, 1)


class on_device:
    """The launch context of a tensor: its device is current inside."""

    def __init__(self, x):
        self.guard = None if x.device.index == torch.cuda.current_device() else torch.cuda.device(x.device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _check(x, num_groups, weight, bias, eps, act):
    if x.dim() < 2:
        raise ValueError('group_norm expects (batch, channels, ...), got shape %s' % (tuple(x.shape),))
    if x.dtype not in _DTYPES:
        raise TypeError('group_norm expects fp16, bf16 or fp32, got %s' % x.dtype)
    c = x.shape[1]
    if num_groups < 1 or c % num_groups:
        raise ValueError('%d channels do not divide into %d groups' % (c, num_groups))
    if not eps >= 0:
        raise ValueError('eps must not be negative, got %r' % (eps,))
    act_code(act)
    for name, p in (('weight', weight), ('bias', bias)):
        if p is None:
            continue
        if p.shape != (c,):
            raise ValueError('%s must have shape (%d,), got %s' % (name, c, tuple(p.shape)))
        if p.dtype not in _DTYPES:
            raise TypeError('%s must be fp16, bf16 or fp32, got %s' % (name, p.dtype))
        if p.device != x.device:
            raise ValueError('%s is on %s, x on %s' % (name, p.device, x.device))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError('weight is %s, bias %s' % (weight.dtype, bias.dtype))


def _plain(x, num_groups, weight, bias, eps, act, slope):
    # torch.group_norm on fp32 values: CPU tensors, and tensors without elements
    p = [None if v is None else v.float() for v in (weight, bias)]
    y = torch.group_norm(x.float(), num_groups, p[0], p[1], eps)
    y = apply_act(y, act, slope).to(x.dtype)
    return y.movedim(1, -1).contiguous().movedim(-1, 1)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _desc(x, pitch, groups, weight, bias, eps, act, slope, y=None, dy=None, dy_ld=0, dx=None, dweight=None, dbias=None, mean=None, rstd=None):
    p = weight if weight is not None else bias
    n, c = x.shape[0], x.shape[1]
    return _lib.GroupNormDesc(x.data_ptr(), _ptr(y), _ptr(dy), _ptr(dx), _ptr(weight), _ptr(bias), _ptr(dweight), _ptr(dbias),
                              _ptr(mean), _ptr(rstd), None, 0, n, x.numel() // (n * c), c, groups, pitch, c, dy_ld, c,
                              _DTYPES[x.dtype], _lib.F32 if p is None else _DTYPES[p.dtype], _ACTS[act], slope, eps)


def _workspace(lib, d, what, device):
    n = C.c_size_t()
    _lib.check(lib.y5_group_norm_workspace(C.byref(d), what, C.byref(n)))
    if not n.value:
        return None
    ws = torch.empty(n.value, dtype=torch.uint8, device=device)
    d.workspace, d.workspace_bytes = ws.data_ptr(), n.value
    return ws


def _forward(x, num_groups, weight, bias, eps, act, slope, stats):
    """(y, mean, rstd, x as it was read, its pitch); mean and rstd where stats is true."""
    with on_device(x):
        lib = _lib.lib()
        x, pitch = channels_last(x)
        y = empty_channels_last(x.shape, x.dtype, x.device)
        mean = rstd = None
        if stats:
            both = torch.empty((2, x.shape[0], num_groups), dtype=torch.float32, device=x.device)
            mean, rstd = both[0], both[1]
        d = _desc(x, pitch, num_groups, weight, bias, eps, act, slope, y=y, mean=mean, rstd=rstd)
        ws = _workspace(lib, d, _lib.GN_FORWARD, x.device)  # noqa: F841 - held until the launch
        _lib.check(lib.y5_group_norm(C.byref(d), _lib.current_stream()))
    return y, mean, rstd, x


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, act, slope):
        y, mean, rstd, xl = _forward(x, num_groups, weight, bias, eps, act, slope, True)
        ctx.save_for_backward(xl, weight, bias, mean, rstd)
        ctx.args = (num_groups, eps, act, slope)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        num_groups, eps, act, slope = ctx.args
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        with on_device(x):
            lib = _lib.lib()
            dy, dy_ld = channels_last(dy)
            dx = empty_channels_last(x.shape, x.dtype, x.device) if need_x else None
            dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if need_w else None
            db = torch.empty_like(bias, memory_format=torch.contiguous_format) if need_b else None
            d = _desc(x, pixel_pitch(x), num_groups, weight, bias, eps, act, slope, dy=dy, dy_ld=dy_ld, dx=dx, dweight=dw, dbias=db,
                      mean=mean, rstd=rstd)
            ws = _workspace(lib, d, _lib.GN_BACKWARD, x.device)  # noqa: F841 - held until the launch
            _lib.check(lib.y5_group_norm_backward(C.byref(d), _lib.current_stream()))
        return dx, dw, db, None, None, None, None


def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, act=None, slope=0.1):
    """act(group_norm(x)) in x's type, channels_last.  weight, bias: (channels,) of one type (x's, or fp32 beside a 16-bit x),
    or None.  act: None, 'leaky' (with slope) or 'silu'.  Differentiable once in x, weight and bias; their gradients
    come in their own types, each sum rounded once."""
    _check(x, num_groups, weight, bias, eps, act)
    if not x.is_cuda or x.numel() == 0:
        return _plain(x, num_groups, weight, bias, eps, act, slope)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return _GroupNorm.apply(x, weight, bias, num_groups, eps, act, slope)
    return _forward(x, num_groups, weight, bias, eps, act, slope, False)[0]


def group_norm_rows(x, num_groups, weight=None, bias=None, eps=1e-5, act=None, slope=0.1):
    """group_norm(...) as 8-bit rows, one row a pixel (yolo_amd.int8.Int8Rows of shape (batch, *spatial)): the fp32 values before
    any rounding are quantised, with a scale a pixel.  Inference only."""
    from yolo_amd import int8
    _check(x, num_groups, weight, bias, eps, act)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        raise RuntimeError('group_norm_rows has no gradient: call it under torch.no_grad()')
    lead = (x.shape[0], *x.shape[2:])
    if not x.is_cuda or x.numel() == 0:
        p = [None if v is None else v.float() for v in (weight, bias)]
        z = apply_act(torch.group_norm(x.float(), num_groups, p[0], p[1], eps), act, slope)
        rows = int8.quantize_rows(z.movedim(1, -1))
        rows.dtype = x.dtype
        return rows
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    with on_device(x):
        lib = _lib.lib()
        x, pitch = channels_last(x)
        rows = int8.Int8Rows.empty(lead, x.shape[1], x.dtype, x.device)
        d = _desc(x, pitch, num_groups, weight, bias, eps, act, slope)
        ws = _workspace(lib, d, _lib.GN_ROWS, x.device)  # noqa: F841 - held until the launch
        _lib.check(lib.y5_group_norm_rows_i8(C.byref(d), rows.q.data_ptr(), rows.q.shape[1], rows.scale.data_ptr(), _lib.current_stream()))
    return rows


class GroupNormAct(nn.GroupNorm):
    """nn.GroupNorm followed by an activation, as one operator (parameters and state_dict of nn.GroupNorm)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, act='leaky', slope=0.1, device=None, dtype=None):
        super().__init__(num_groups, num_channels, eps=eps, affine=affine, device=device, dtype=dtype)
        act_code(act)
        self.act, self.slope = act, slope

    def forward(self, x):
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.act, self.slope)

    def extra_repr(self):
        return super().extra_repr() + ', act=%s, slope=%g' % (self.act, self.slope)
