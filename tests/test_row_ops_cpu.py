"""Operators on rows in few bits: what they refuse, checked before any device work, and their size functions."""
import ctypes as C

import pytest

A = 1 << 20   # an address that is aligned to everything; never read


def _refused(b200, call, text):
    with pytest.raises(b200.B200IdxError) as e:
        call()
    assert e.value.code == 2001 and text in e.value.msg, e.value


def test_sizes(b200):
    assert [b200.mx4_row_bytes(d) for d in (1, 32, 33, 128, 16384)] == [16, 16, 32, 64, 8192]
    assert [b200.mx4_scale_bytes(n, d) for n, d in ((1, 1), (128, 128), (129, 128), (1, 129))] == [512, 512, 1024, 1024]
    for bad in (0, -1, 16385):
        _refused(b200, lambda: b200.mx4_row_bytes(bad), "d in")
        _refused(b200, lambda: b200.mx4_scale_bytes(4, bad), "d in")
    _refused(b200, lambda: b200.mx4_scale_bytes(0, 32), "n must")


def _rms(b200, **kw):
    a = dict(n=2, d=32, dtype=b200.BF16, x_ptr=A, weight_ptr=A, eps=1e-6, q_ptr=A, scales_ptr=A)
    a.update(kw)
    b200.rms_norm_i8_device(**a)


@pytest.mark.parametrize("kw, text", [
    (dict(n=0), "n must"), (dict(n=1000000000), "n must"), (dict(d=0), "dims"), (dict(d=16385), "dims"),
    (dict(dtype=3), "dtype"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=2.0), "eps"),
    (dict(x_ptr=0), "Invalid x"), (dict(weight_ptr=0), "Invalid weight"), (dict(q_ptr=0), "Invalid q"),
    (dict(scales_ptr=0), "exactly one"), (dict(static_scale_ptr=A), "exactly one"),
    (dict(sum_ptr=A), "needs a residual"),
    (dict(ldx=31), "ldx"), (dict(ldq=31), "ldq"), (dict(ldr=-1), "ldr"),
    (dict(residual_ptr=A, sum_ptr=A, ldr=40), "same stride"),
    (dict(x_ptr=A + 1), "aligned"), (dict(scales_ptr=A + 2), "aligned"),
])
def test_rms_norm_refuses(b200, kw, text):
    _refused(b200, lambda: _rms(b200, **kw), text)


@pytest.mark.parametrize("kw, text", [
    (dict(n=0), "n must"), (dict(d=20000), "dims"), (dict(dtype=7), "dtype"), (dict(q_ptr=0), "Invalid q"),
    (dict(out_ptr=0), "Invalid out"), (dict(scales_ptr=0), "exactly one"), (dict(static_scale_ptr=A), "exactly one"),
    (dict(ldo=3), "ldo"), (dict(out_ptr=A + 2), "aligned"),
])
def test_i8_dequantize_refuses(b200, kw, text):
    a = dict(n=2, d=32, q_ptr=A, dtype=b200.F32, out_ptr=A, scales_ptr=A)
    a.update(kw)
    _refused(b200, lambda: b200.i8_dequantize_device(**a), text)


@pytest.mark.parametrize("kw, text", [
    (dict(n=0), "n must"), (dict(d=0), "dims"), (dict(dtype=3), "dtype"), (dict(x_ptr=0), "Invalid x"),
    (dict(codes_ptr=0), "Invalid codes"), (dict(scales_ptr=0), "Invalid scales"), (dict(codes_ptr=A + 8), "aligned"),
    (dict(scales_ptr=A + 4), "aligned"), (dict(ldx=8), "ldx"),
])
def test_mx4_quantize_refuses(b200, kw, text):
    a = dict(n=2, d=32, dtype=b200.F32, x_ptr=A, codes_ptr=A, scales_ptr=A)
    a.update(kw)
    _refused(b200, lambda: b200.mx4_quantize_device(**a), text)


@pytest.mark.parametrize("kw, text", [
    (dict(n=-5), "n must"), (dict(d=0), "dims"), (dict(dtype=3), "dtype"), (dict(out_ptr=0), "Invalid out"),
    (dict(codes_ptr=A + 4), "aligned"), (dict(ldo=31), "ldo"),
])
def test_mx4_dequantize_refuses(b200, kw, text):
    a = dict(n=2, d=32, codes_ptr=A, scales_ptr=A, dtype=b200.F32, out_ptr=A)
    a.update(kw)
    _refused(b200, lambda: b200.mx4_dequantize_device(**a), text)


@pytest.mark.parametrize("kw, text", [
    (dict(m=0), "m must"), (dict(n=0), "n must"), (dict(d=20000), "dims"), (dict(dtype=3), "dtype"),
    (dict(a_codes_ptr=0), "Invalid a_codes"), (dict(b_scales_ptr=A + 8), "aligned"), (dict(ldo=2), "ldo"),
    (dict(out_ptr=A + 1), "aligned"),
])
def test_mx4_product_refuses(b200, kw, text):
    a = dict(m=2, n=3, d=32, a_codes_ptr=A, a_scales_ptr=A, b_codes_ptr=A, b_scales_ptr=A, dtype=b200.F32, out_ptr=A)
    a.update(kw)
    _refused(b200, lambda: b200.mx4_product_device(**a), text)


def test_host_memory_is_refused_or_no_device_found(b200):
    import torch
    buf = (C.c_float * 64)()
    at = C.addressof(buf) + (-C.addressof(buf)) % 16
    with pytest.raises(b200.B200IdxError) as e:
        b200.mx4_quantize_device(1, 32, b200.F32, at, at, at)
    if torch.cuda.is_available():
        assert e.value.code == 2001 and "device pointer" in e.value.msg
    else:
        assert e.value.code == 2010 and "no CUDA device" in e.value.msg
