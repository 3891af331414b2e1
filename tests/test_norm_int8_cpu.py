"""Group norm and the 8-bit layers without a GPU: the formulas on CPU tensors, layouts, and every refusal - those of the Python
functions and those of the C entry points, which come before anything is launched."""
import ctypes as C

import pytest
import torch

from norm_ref import GroupNormRef, close
from yolo_amd import _lib, groupnorm, int8


@pytest.mark.parametrize('act', [None, 'leaky', 'silu'])
def test_group_norm_on_the_cpu(act):
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = torch.randn(2, 12, 5, 3, generator=g), torch.randn(12, generator=g), torch.randn(12, generator=g), torch.randn(2, 12, 5, 3, generator=g)
    ref = GroupNormRef(x, 4, w, b, 1e-5, act, dy=dy)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    with torch.enable_grad():
        y = groupnorm.group_norm(x, 4, w, b, act=act)
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
    for got, want, err in ((y, ref.y, ref.err_y), (dx, ref.dx, ref.err_dx), (dw, ref.dgamma, ref.err_dgamma), (db, ref.dbeta, ref.err_dbeta)):
        close(got, want, err, str(act))
    with torch.no_grad():
        rows = groupnorm.group_norm_rows(x, 4, w, b, act=act)
    assert rows.shape == (2, 5, 3, 12)
    assert float((rows.dequantize().permute(0, 3, 1, 2) - y.detach()).abs().max()) <= float(y.detach().abs().max()) / 254 * 1.001


def test_product_on_the_cpu():
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(7, 19, generator=g), torch.randn(5, 19, generator=g)
    q = int8.quantize_weight(w)
    assert q.q.shape == (5, 32) and not bool(q.q[:, 19:].any()) and int(q.q.abs().max()) == 127
    rows = int8.quantize_rows(x)
    y = int8.linear_i8(x, q, torch.ones(5), act='leaky')
    z = (rows.dequantize(torch.float64) @ q.dequantize(torch.float64).t()) + 1
    assert torch.allclose(y.double(), torch.where(z > 0, z, 0.1 * z), atol=1e-5)
    assert float((y - torch.nn.functional.leaky_relu(x @ w.t() + 1, 0.1)).abs().max()) < 0.1
    m = int8.conv1x1_i8(x.reshape(1, 7, 19, 1).permute(0, 2, 1, 3), q)
    assert m.shape == (1, 5, 7, 1) and m.stride(1) == 1


def test_pixel_pitch():
    x = torch.zeros(2, 6, 4, 5)
    assert groupnorm.pixel_pitch(x) is None
    v = x.to(memory_format=torch.channels_last)
    assert groupnorm.pixel_pitch(v) == 6 and groupnorm.pixel_pitch(v[:, 1:4]) == 6 and groupnorm.pixel_pitch(v[1:]) == 6
    assert groupnorm.pixel_pitch(v[:, :, 1:]) is None and groupnorm.pixel_pitch(v[:, :, :, ::2]) is None  # no single pitch
    assert groupnorm.pixel_pitch(v[:1, :, 1:]) == 6
    assert groupnorm.pixel_pitch(torch.zeros(3, 6)) == 6 and groupnorm.pixel_pitch(torch.zeros(3, 6)[:, 2:5]) == 6
    assert groupnorm.pixel_pitch(torch.zeros(1, 6).expand(3, 6)) is None and groupnorm.pixel_pitch(torch.zeros(2, 6, 1, 1)) == 6
    assert groupnorm.pixel_pitch(torch.zeros(2, 1, 4, 5)) == 1
    y, pitch = groupnorm.channels_last(v[:, 1:4])  # three fp32 values are no whole vector: copied
    assert pitch == 3 and torch.equal(y, v[:, 1:4])


def test_refusals():
    x, gn = torch.zeros(2, 8, 3, 3), groupnorm.group_norm
    for call in (lambda: gn(x, 3), lambda: gn(x, 0), lambda: gn(x, 2, eps=-1.0), lambda: gn(x, 2, eps=float('nan')), lambda: gn(x, 2, act='relu'),
                 lambda: gn(x[0, 0, 0], 1), lambda: gn(x, 2, torch.ones(4)), lambda: groupnorm.GroupNormAct(2, 8, act='tanh')):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: gn(x.double(), 2), lambda: gn(x, 2, torch.ones(8, dtype=torch.int32)), lambda: gn(x, 2, torch.ones(8), torch.ones(8).half())):
        with pytest.raises(TypeError):
            call()
    w = int8.Int8Weight(torch.ones(4, 8, dtype=torch.int8), torch.ones(4))
    t = torch.zeros(3, 8)
    with pytest.raises(RuntimeError), torch.enable_grad():
        int8.linear_i8(t.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError), torch.enable_grad():
        groupnorm.group_norm_rows(x.clone().requires_grad_(), 2)
    for call in (lambda: int8.linear_i8(t[:, :7], w), lambda: int8.linear_i8(t, w, torch.ones(3)), lambda: int8.linear_i8(t, w, act='gelu'),
                 lambda: int8.Int8Weight(torch.ones(4, dtype=torch.int8), torch.ones(4)), lambda: int8.Int8Weight(torch.ones(4, 8, dtype=torch.int8), torch.ones(8)),
                 lambda: int8.quantize_rows(torch.zeros(2, 0)), lambda: int8.quantize_rows(torch.zeros(1, _lib.I8_MAX_K + 1)),
                 lambda: int8.Int8Conv1x1.from_conv(torch.nn.Conv2d(8, 8, 3)), lambda: int8.Int8Conv1x1.from_conv(torch.nn.Conv2d(8, 8, 1, groups=2))):
        with pytest.raises(ValueError):
            call()
    q = torch.zeros(3, 16, dtype=torch.int8)
    for args in ((q, torch.ones(4), (3,), 8), (q[:, :8], torch.ones(3), (3,), 8), (q, torch.ones(3), (2,), 8), (q, torch.ones(3), (3,), 17),
                 (q, torch.ones(3).half(), (3,), 8), (q.float(), torch.ones(3), (3,), 8)):
        with pytest.raises(ValueError):
            int8.Int8Rows(*args, torch.float16)
    for call in (lambda: int8.linear_i8(t, torch.ones(4, 8)), lambda: int8.linear_i8(t.long(), w), lambda: int8.linear_i8(t, w, dtype=torch.float64),
                 lambda: int8.Int8Weight(torch.ones(4, 8), torch.ones(4)), lambda: int8.quantize_rows(t.double())):
        with pytest.raises(TypeError):
            call()


def test_extension_is_there():
    """The host side of the calls is built with the library, next to it."""
    m = _lib.calls()
    assert m.__file__.startswith(_lib.os.path.dirname(_lib.LIB_PATH)) and callable(m.group_norm) and callable(m.linear)


def _gn(**kw):
    base = dict(x=0x1000, y=0x2000, dy=0x3000, dx=0x4000, mean=0x5000, rstd=0x6000, workspace=0x10000, workspace_bytes=1 << 40, batch=2, pixels=9, c=16,
                groups=4, x_ld=16, y_ld=16, dy_ld=16, dx_ld=16, eps=1e-5)
    base.update(kw)
    return _lib.GroupNormDesc(**base)


def test_c_entry_points_refuse_before_any_launch():
    lib = _lib.lib()

    def refused(rc, text, code=_lib.EINVAL):
        assert rc == code and text in lib.y5_last_error(), (rc, lib.y5_last_error())

    n = C.c_size_t()
    for fn in (lib.y5_group_norm, lib.y5_group_norm_backward):
        refused(fn(None, None), b'null descriptor')
        for kw, text in ((dict(groups=3), b'divide'), (dict(groups=0), b'divide'), (dict(batch=0), b'batch'), (dict(batch=65536), b'batch'), (dict(pixels=0), b'pixels'),
                         (dict(pixels=(1 << 30) + 1), b'pixels'), (dict(c=0), b'channels'),
                         (dict(dtype=5), b'dtype'), (dict(param_dtype=-1), b'param_dtype'), (dict(act=3), b'activation'), (dict(eps=-1.0), b'eps'),
                         (dict(eps=float('nan')), b'eps'), (dict(x=None), b'null x'), (dict(x=0x1001), b'misaligned x'), (dict(x_ld=15), b'pitch'),
                         (dict(c=12, x_ld=16), b'pitch'), (dict(c=4104, groups=1, x_ld=4104), b'channels'), (dict(c=513, groups=1, x_ld=513), b'channels')):
            refused(fn(C.byref(_gn(**kw)), None), text)
    refused(lib.y5_group_norm(C.byref(_gn(rstd=None)), None), b'go together')
    refused(lib.y5_group_norm(C.byref(_gn(y=None)), None), b'null y')
    refused(lib.y5_group_norm(C.byref(_gn(pixels=1 << 20, workspace_bytes=16)), None), b'workspace', _lib.EWORKSPACE)
    refused(lib.y5_group_norm(C.byref(_gn(pixels=1 << 20, workspace=0x10008)), None), b'misaligned workspace')
    refused(lib.y5_group_norm_backward(C.byref(_gn(dy=None)), None), b'null dy')
    refused(lib.y5_group_norm_backward(C.byref(_gn(dx_ld=8)), None), b'dx pitch')
    refused(lib.y5_group_norm_backward(C.byref(_gn(mean=None)), None), b'null mean')
    refused(lib.y5_group_norm_backward(C.byref(_gn(workspace=None)), None), b'workspace', _lib.EWORKSPACE)
    refused(lib.y5_group_norm_workspace(None, 0, C.byref(n)), b'null')
    refused(lib.y5_group_norm_workspace(C.byref(_gn()), 7, C.byref(n)), b'call 7')
    assert lib.y5_group_norm_workspace(C.byref(_gn(pixels=1 << 20)), _lib.GN_FORWARD, C.byref(n)) == 0 and n.value >= 2 * 4 * 8
    g = _gn(workspace_bytes=0)
    refused(lib.y5_group_norm_rows_i8(C.byref(g), 0x1000, 16, 0x2000, None), b'workspace', _lib.EWORKSPACE)
    refused(lib.y5_group_norm_rows_i8(C.byref(_gn()), 0x1000, 32, 0x2000, None), b'bytes')
    refused(lib.y5_group_norm_rows_i8(C.byref(_gn()), 0x1008, 16, 0x2000, None), b'misaligned')
    refused(lib.y5_group_norm_rows_i8(C.byref(_gn()), None, 16, 0x2000, None), b'null output')
    qr = lib.y5_quantize_rows_i8
    refused(qr(None, 16, 0, 4, 16, 0x1000, 16, 0x2000, None), b'null x')
    refused(qr(0x1000, 16, 3, 4, 16, 0x1000, 16, 0x2000, None), b'dtype')
    refused(qr(0x1000, 16, 0, 0, 16, 0x1000, 16, 0x2000, None), b'rows')
    refused(qr(0x1000, 8, 0, 4, 16, 0x1000, 16, 0x2000, None), b'pitch')
    refused(qr(0x1000, 16, 0, 4, 17, 0x1000, 16, 0x2000, None), b'bytes')
    refused(qr(0x1000, 16, 0, 4, 0, 0x1000, 0, 0x2000, None), b'values')
    refused(qr(0x1000, 1 << 20, 0, 4, _lib.I8_MAX_K + 1, 0x1000, _lib.I8_MAX_K + 16, 0x2000, None), b'values')
    refused(qr(0x1001, 16, 0, 4, 16, 0x1000, 16, 0x2000, None), b'misaligned x')
    refused(lib.y5_gemm_i8(None, None), b'null descriptor')
    base = dict(a=0x1000, a_scale=0x2000, w=0x3000, w_scale=0x4000, y=0x5000, m=4, y_ld=8, n=8, k=20, ld=32)
    for kw, text in ((dict(a=None), b'null'), (dict(y=None), b'null'), (dict(w_scale=None), b'null'), (dict(m=0), b'rows'), (dict(n=0), b'channels'), (dict(k=0), b'values'),
                     (dict(ld=20), b'bytes'), (dict(y_ld=7), b'pitch'), (dict(dtype=4), b'dtype'), (dict(act=9), b'activation'), (dict(a=0x1008), b'aligned'),
                     (dict(y=0x5001), b'misaligned'), (dict(m=1 << 32), b'rows')):
        refused(lib.y5_gemm_i8(C.byref(_lib.GemmI8Desc(**{**base, **kw})), None), text)
