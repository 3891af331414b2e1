"""Linear layers and 1x1 convolutions in 8-bit integers: weights with a scale an output channel, activations quantised on the
fly with a scale a row (token, pixel), exact int32 sums on the matrix cores.

The 8-bit form of the reference's 1x1 convolutions (models/common.py:26, :51-53) and of linear layers, for the step after
filter pruning.

    w = quantize_weight(conv.weight)                       # or Int8Weight(q, scale) from a quantisation of one's own
    y = conv1x1_i8(x, w, bias, act='leaky')                # x (batch, channels, h, w), channels_last
    y = linear_i8(t, w, bias)                              # t (..., features)
    layer = Int8Conv1x1.from_conv(block)                   # a models.common.Conv or nn.Conv2d as a module

A row x becomes whole numbers q = nearest(127 x / max|x|) and the scale max|x| / 127; a row of zeros (max|x| < 2^-120) has scale
0; a row with an infinity or a NaN gives NaN outputs.  y = act(sum(q w) * (scale_row * scale_channel) + bias) in fp32, rounded once.
Inference only.  CPU tensors go through torch's own operators (sums in fp64, exact too).
"""
import math

import torch
import torch.nn as nn

from yolo_amd import _lib
from yolo_amd.groupnorm import _ACTS, _DTYPES, act_code, apply_act, pixel_pitch

ZERO_ROW = 2.0 ** -120


def row_bytes(k):
    """Bytes of an 8-bit row of k values: padded with zeros to whole 16-byte vectors."""
    return (k + 15) // 16 * 16


def _check_k(k):
    if not 1 <= k <= _lib.I8_MAX_K:
        raise ValueError('rows must hold 1 to %d values, got %d' % (_lib.I8_MAX_K, k))


class Int8Rows:
    """Quantised rows: q (rows, row_bytes(k)) int8, scale (rows) fp32, for a tensor of shape (*lead, k) that was of type dtype."""

    __slots__ = ('q', 'scale', 'lead', 'k', 'dtype')

    def __init__(self, q, scale, lead, k, dtype):
        _check_k(k)
        n = math.prod(lead)
        if q.dtype is not torch.int8 or q.shape != (n, row_bytes(k)) or not q.is_contiguous():
            raise ValueError('Int8Rows expects q as %d contiguous int8 rows of %d bytes, got %s %s' % (n, row_bytes(k), tuple(q.shape), q.dtype))
        if scale.dtype is not torch.float32 or scale.shape != (n,) or not scale.is_contiguous() or scale.device != q.device:
            raise ValueError('Int8Rows expects %d contiguous fp32 scales beside q, got %s %s' % (n, tuple(scale.shape), scale.dtype))
        if dtype not in _DTYPES:
            raise TypeError('Int8Rows stands for fp16, bf16 or fp32, not %s' % dtype)
        self.q, self.scale, self.lead, self.k, self.dtype = q, scale, tuple(lead), k, dtype

    @classmethod
    def of(cls, q, scale, lead, k, dtype):
        """What the kernels wrote, unchecked."""
        self = cls.__new__(cls)
        self.q, self.scale, self.lead, self.k, self.dtype = q, scale, lead, k, dtype
        return self

    @property
    def shape(self):
        return (*self.lead, self.k)

    @property
    def device(self):
        return self.q.device

    def dequantize(self, dtype=None):
        return (self.q[:, :self.k].float() * self.scale[:, None]).reshape(self.shape).to(dtype or self.dtype)


class Int8Weight:
    """8-bit weights of a layer: q (n, k) int8 - (n, k, 1, 1) is taken too - and scale (n), so that row n stands for q[n] * scale[n].
    Rows are padded once, here, to whole 16-byte vectors."""

    __slots__ = ('q', 'scale', 'n', 'k')

    def __init__(self, q, scale):
        if q.dtype is not torch.int8:
            raise TypeError('Int8Weight expects int8 values, got %s' % q.dtype)
        if q.dim() == 4 and q.shape[2:] == (1, 1):
            q = q[:, :, 0, 0]
        if q.dim() != 2 or q.shape[0] < 1:
            raise ValueError('Int8Weight expects (n, k) or (n, k, 1, 1), got %s' % (tuple(q.shape),))
        _check_k(q.shape[1])
        if scale.shape != (q.shape[0],) or not scale.is_floating_point():
            raise ValueError('Int8Weight expects %d floating-point scales, got %s %s' % (q.shape[0], tuple(scale.shape), scale.dtype))
        if scale.device != q.device:
            raise ValueError('q is on %s, scale on %s' % (q.device, scale.device))
        self.n, self.k = q.shape
        pad = row_bytes(self.k) - self.k
        self.q = torch.nn.functional.pad(q, (0, pad)) if pad else q.contiguous()
        if self.q.data_ptr() % 16:
            self.q = self.q.clone()
        self.scale = scale.float().contiguous()

    @property
    def device(self):
        return self.q.device

    def dequantize(self, dtype=torch.float32):
        return (self.q[:, :self.k].float() * self.scale[:, None]).to(dtype)


def _refuse_grad(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError('%s has no gradient: call it under torch.no_grad()' % name)


def _quantize_plain(x, lead, k, dtype):
    v = x.reshape(-1, k).double()
    a = v.abs().amax(1, keepdim=True) if v.numel() else v[:, :1]
    fine = torch.isfinite(a)
    some = fine & (a >= ZERO_ROW)
    q = torch.where(some, v * (127 / torch.where(some, a, 1.0)), 0.0).round()
    scale = torch.where(fine, torch.where(some, a / 127, 0.0), float('nan'))
    return Int8Rows(torch.nn.functional.pad(q.to(torch.int8), (0, row_bytes(k) - k)), scale[:, 0].float(), lead, k, dtype)


def _rows_of(x):
    """x (..., k) as rows at one pitch: itself where its memory is that, else a copy."""
    k = x.shape[-1]
    if x.dim() != 2 or x.stride(1) != 1 or x.stride(0) < k:
        x = x.reshape(-1, k)
        if (k > 1 and x.stride(1) != 1) or x.stride(0) < k:
            x = x.contiguous()
    return x, max(x.stride(0), k)


def quantize_rows(x):
    """x (..., k), fp16 / bf16 / fp32 -> Int8Rows with a scale a row of the last dimension."""
    if x.dtype not in _DTYPES:
        raise TypeError('quantize_rows expects fp16, bf16 or fp32, got %s' % x.dtype)
    if x.dim() < 1:
        raise ValueError('quantize_rows expects (..., k)')
    _refuse_grad('quantize_rows', x)
    lead, k = tuple(x.shape[:-1]), x.shape[-1]
    _check_k(k)
    if not x.is_cuda or x.numel() == 0:
        return _quantize_plain(x, lead, k, x.dtype)
    r, pitch = _rows_of(x)
    return Int8Rows.of(*_lib.calls().quantize_rows(r, pitch, r.shape[0], k), lead, k, x.dtype)


def quantize_weight(w):
    """(n, k) or (n, k, 1, 1) floating-point weights -> Int8Weight, each output channel scaled by its own largest magnitude."""
    if w.dim() == 4 and w.shape[2:] == (1, 1):
        w = w[:, :, 0, 0]
    if w.dim() != 2 or w.shape[0] < 1:
        raise ValueError('quantize_weight expects (n, k) or (n, k, 1, 1), got %s' % (tuple(w.shape),))
    rows = quantize_rows(w.detach().float())
    return Int8Weight(rows.q[:, :rows.k], rows.scale)


def _plain_product(rows, weight, bias, act, slope, dtype):
    y = rows.q[:, :rows.k].double() @ weight.q[:, :weight.k].double().t()
    y = y.float() * (rows.scale[:, None] * weight.scale)
    y = y if bias is None else y + bias
    return apply_act(y, act, slope).to(dtype)


def _check(name, x, weight, bias, act, dtype):
    if not isinstance(weight, Int8Weight):
        raise TypeError('%s expects an Int8Weight, got %s' % (name, type(weight).__name__))
    act_code(act)
    if dtype not in _DTYPES:
        raise TypeError('%s gives fp16, bf16 or fp32, not %s' % (name, dtype))
    if x.device != weight.device:
        raise ValueError('x is on %s, the weight on %s' % (x.device, weight.device))
    if bias is None:
        return None
    if bias.shape != (weight.n,) or not bias.is_floating_point():
        raise ValueError('bias must be %d floating-point values, got %s %s' % (weight.n, tuple(bias.shape), bias.dtype))
    if bias.device != weight.device:
        raise ValueError('bias is on %s, the weight on %s' % (bias.device, weight.device))
    if bias.requires_grad:
        _refuse_grad(name, bias)
    return bias if bias.dtype is torch.float32 and bias.is_contiguous() else bias.float().contiguous()


def linear_i8(x, weight, bias=None, act=None, slope=0.1, dtype=None):
    """act(x @ weight.T + bias) with 8-bit operands.  x: (..., k) fp16 / bf16 / fp32, quantised here row by row, or Int8Rows.
    weight: Int8Weight; bias: (n) or None; act: None, 'leaky' (with slope) or 'silu'.  The result is (..., n) of type dtype
    (x's own by default)."""
    rows = isinstance(x, Int8Rows)
    dtype = dtype or x.dtype
    bias = _check('linear_i8', x, weight, bias, act, dtype)
    k = x.k if rows else x.shape[-1] if x.dim() else 0
    if k != weight.k:
        raise ValueError('rows of %d values, weights for %d' % (k, weight.k))
    if rows:
        if not x.q.is_cuda or x.q.shape[0] == 0:
            return _plain_product(x, weight, bias, act, slope, dtype).reshape(*x.lead, weight.n)
        return _lib.calls().product(x.q, x.scale, weight.q, weight.scale, k, bias, _ACTS[act], slope, dtype, (*x.lead, weight.n))
    if x.dtype not in _DTYPES:
        raise TypeError('linear_i8 expects fp16, bf16, fp32 or Int8Rows, got %s' % x.dtype)
    if x.requires_grad:
        _refuse_grad('linear_i8', x)
    if not x.is_cuda or x.numel() == 0:
        return _plain_product(quantize_rows(x), weight, bias, act, slope, dtype).reshape(*x.shape[:-1], weight.n)
    r, pitch = _rows_of(x)
    return _lib.calls().linear(r, pitch, r.shape[0], weight.q, weight.scale, k, bias, _ACTS[act], slope, dtype, (*x.shape[:-1], weight.n))


def conv1x1_i8(x, weight, bias=None, act=None, slope=0.1, dtype=None):
    """The 1x1 convolution of x (batch, channels, *spatial) - or of Int8Rows of shape (batch, *spatial, channels), as
    groupnorm.group_norm_rows gives them.  Arguments as linear_i8; the result is (batch, n, *spatial) in channels_last memory."""
    if isinstance(x, Int8Rows):
        if not x.lead:
            raise ValueError('conv1x1_i8 expects rows of shape (batch, *spatial, channels)')
        return linear_i8(x, weight, bias, act, slope, dtype).movedim(-1, 1)
    if x.dim() < 2:
        raise ValueError('conv1x1_i8 expects (batch, channels, ...), got %s' % (tuple(x.shape),))
    if x.dtype not in _DTYPES:
        raise TypeError('conv1x1_i8 expects fp16, bf16 or fp32, got %s' % x.dtype)
    if not x.is_cuda or x.numel() == 0:
        return linear_i8(x.movedim(1, -1), weight, bias, act, slope, dtype).movedim(-1, 1)
    pitch = pixel_pitch(x)
    if pitch is None:
        return linear_i8(x.movedim(1, -1).contiguous(), weight, bias, act, slope, dtype).movedim(-1, 1)
    dtype = dtype or x.dtype
    bias = _check('conv1x1_i8', x, weight, bias, act, dtype)
    if x.shape[1] != weight.k:
        raise ValueError('%d channels, weights for %d' % (x.shape[1], weight.k))
    _refuse_grad('conv1x1_i8', x)
    y = _lib.calls().linear(x, pitch, x.numel() // weight.k, weight.q, weight.scale, weight.k, bias, _ACTS[act], slope, dtype,
                            (x.shape[0], *x.shape[2:], weight.n))
    return y.movedim(-1, 1)


class Int8Linear(nn.Module):
    """A linear layer with 8-bit weights: buffers q (n, row_bytes(k)) int8, scale (n) and bias (n or None) fp32.  .half() and the like leave
    the buffers' types alone; the output has the input's type."""

    def __init__(self, weight, bias=None, act=None, slope=0.1):
        super().__init__()
        act_code(act)
        self.act, self.slope, self.k = act, slope, weight.k
        self.register_buffer('q', weight.q)
        self.register_buffer('scale', weight.scale)
        self.register_buffer('bias', None if bias is None else bias.detach().float().contiguous())

    @classmethod
    def from_linear(cls, linear, act=None, slope=0.1):
        with torch.no_grad():
            return cls(quantize_weight(linear.weight), linear.bias, act, slope)

    def _apply(self, fn, *args, **kwargs):
        scale, bias = self.scale, self.bias
        super()._apply(fn, *args, **kwargs)
        self.scale = scale.to(self.q.device)
        self.bias = None if bias is None else bias.to(self.q.device)
        return self

    def _weight(self):
        w = Int8Weight.__new__(Int8Weight)
        w.q, w.scale, w.n, w.k = self.q, self.scale, self.q.shape[0], self.k
        return w

    def forward(self, x):
        return linear_i8(x, self._weight(), self.bias, self.act, self.slope)

    def extra_repr(self):
        return 'in=%d, out=%d, act=%s' % (self.k, self.q.shape[0], self.act)


class Int8Conv1x1(Int8Linear):
    """A 1x1 convolution with 8-bit weights."""

    @classmethod
    def from_conv(cls, conv):
        """From a models.common.Conv block (its BatchNorm folded in, its LeakyReLU kept) or an nn.Conv2d: kernel 1, stride 1, no
        padding, one group."""
        from yolo_amd.utils.torch_utils import fuse_conv_and_bn
        act, slope = None, 0.1
        if not isinstance(conv, nn.Conv2d):
            block, conv = conv, conv.conv
            if isinstance(block.act, nn.LeakyReLU):
                act, slope = 'leaky', block.act.negative_slope
            elif isinstance(block.act, nn.SiLU):
                act = 'silu'
            elif not isinstance(block.act, nn.Identity):
                raise ValueError('Int8Conv1x1 knows LeakyReLU and SiLU, not %s' % type(block.act).__name__)
            if block.bn is not None:
                if conv.groups != 1:
                    raise ValueError('Int8Conv1x1 needs one group, got %d' % conv.groups)
                conv = fuse_conv_and_bn(conv, block.bn)
        if conv.kernel_size != (1, 1) or conv.stride != (1, 1) or conv.padding not in ((0, 0), 'valid', 'same') or conv.groups != 1:
            raise ValueError('Int8Conv1x1 needs kernel 1, stride 1, no padding and one group: %s' % conv)
        with torch.no_grad():
            return cls(quantize_weight(conv.weight), conv.bias, act, slope)

    def forward(self, x):
        return conv1x1_i8(x, self._weight(), self.bias, self.act, self.slope)
