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
4096 / (8 / gcd(channels, 8)), e.g. 512 for odd counts in 16 bits.  Up to 65535 images of up to 2^30 pixels.
"""
import torch
import torch.nn as nn

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
    if x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last):
        return x, x.shape[1]
    pitch = pixel_pitch(x)
    if pitch is None or (pitch != x.shape[1] and x.shape[1] * x.element_size() % 16):
        x = x.movedim(1, -1).contiguous().movedim(-1, 1)
        pitch = x.shape[1]
    return x, pitch


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


def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, act=None, slope=0.1):
    """act(group_norm(x)) in x's type, channels_last.  weight, bias: (channels,) of one type (x's, or fp32 beside a 16-bit x),
    or None.  act: None, 'leaky' (with slope) or 'silu'.  Differentiable once in x, weight and bias; their gradients
    come in their own types, each sum rounded once.  A captured gradient is refused for leaves of which a graph made on the
    default stream still lives: torch would have it wait for that stream."""
    _check(x, num_groups, weight, bias, eps, act)
    if not x.is_cuda or x.numel() == 0:
        return _plain(x, num_groups, weight, bias, eps, act, slope)
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    x, pitch = channels_last(x)
    return _lib.calls().group_norm(x, pitch, num_groups, weight, bias, eps, _ACTS[act], slope)


def group_norm_rows(x, num_groups, weight=None, bias=None, eps=1e-5, act=None, slope=0.1):
    """group_norm(...) as 8-bit rows, one row a pixel (yolo_amd.int8.Int8Rows of shape (batch, *spatial)): the fp32 values before
    any rounding are quantised, with a scale a pixel.  Inference only."""
    from yolo_amd import int8
    _check(x, num_groups, weight, bias, eps, act)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        raise RuntimeError('group_norm_rows has no gradient: call it under torch.no_grad()')
    lead = (x.shape[0], *x.shape[2:])
    if not x.is_cuda or x.numel() == 0:
        p = [None if v is None else v.float() for v in (weight, bias)]
        z = apply_act(torch.group_norm(x.float(), num_groups, p[0], p[1], eps), act, slope)
        rows = int8.quantize_rows(z.movedim(1, -1))
        rows.dtype = x.dtype
        return rows
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    xl, pitch = channels_last(x)
    q, scale = _lib.calls().group_norm_rows(xl, pitch, num_groups, weight, bias, eps, _ACTS[act], slope)
    return int8.Int8Rows.of(q, scale, lead, x.shape[1], x.dtype)


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
