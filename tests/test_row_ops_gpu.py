"""Operators on rows in few bits against plain 64-bit statements (tests/row_reference.py)."""
import numpy as np
import pytest
import torch

import row_reference as ref

pytestmark = pytest.mark.gpu


def _rows(rng, n, d, dtype, wide=0.5):
    x = rng.standard_normal((n, d)) * np.exp(wide * rng.standard_normal(d))
    return torch.from_numpy(x).to("cuda", ref.TORCH[dtype])


def _strided(t, ld, offset=0):
    """A copy of t with row stride ld, starting `offset` elements into its memory."""
    n, d = t.shape
    big = torch.zeros(n * ld + offset + 8, dtype=t.dtype, device="cuda")
    v = big[offset:offset + n * ld].view(n, ld)[:, :d]
    v.copy_(t)
    return v


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ---- MX4 rounding ----
def quantize(b, x, canary=True):
    n, d = x.shape
    pitch, sb = b.mx4_row_bytes(d), b.mx4_scale_bytes(n, d)
    codes = torch.full((n * pitch + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    scales = torch.full((sb + 64,), 0xCD, dtype=torch.uint8, device="cuda")
    dt = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[x.dtype]
    b.mx4_quantize_device(n, d, dt, x.data_ptr(), codes.data_ptr(), scales.data_ptr(), ldx=x.stride(0) if n > 1 else 0,
                          stream_ptr=_stream())
    assert bool((codes[n * pitch:] == 0xAB).all()) and bool((scales[sb:] == 0xCD).all())
    return codes[:n * pitch].view(n, pitch), scales[:sb]


def check_quantize(b, x):
    n, d = x.shape
    codes, scales = quantize(b, x)
    rc, rs = ref.mx4_encode(x.double().cpu().numpy())
    pc, ps = ref.mx4_pack(rc, rs, fill=0xCD)   # scale bytes of rows behind n stay as they were
    np.testing.assert_array_equal(codes.cpu().numpy(), pc)
    np.testing.assert_array_equal(scales.cpu().numpy(), ps)
    return codes, scales, rc, rs


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("n, d", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 127), (130, 128), (129, 129), (7, 256), (33, 777),
                                  (1, 4096), (300, 96), (2, 16384), (1, 16383), (1000, 8)])
def test_mx4_quantize(b200, n, d, dtype):
    rng = np.random.default_rng(n * 1000 + d)
    check_quantize(b200, _rows(rng, n, d, dtype))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("ld, offset", [(100, 0), (104, 0), (101, 3), (128, 1)])
def test_mx4_quantize_strides(b200, ld, offset, dtype):
    x = _rows(np.random.default_rng(5), 37, 100, dtype)
    check_quantize(b200, _strided(x, ld, offset))


def test_mx4_quantize_borders_and_special_values(b200):
    # every border between two codes, its neighbours in fp32, and both signs, at several scales
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9999995], np.float32)
    near = np.concatenate([mids, np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(8))])
    near = np.minimum(near, np.float32(7.9999995))
    rows = []
    for e in (-126, -30, 0, 17, 125):
        for lo in range(0, len(near), 15):
            v = np.zeros(32, np.float32)
            v[0] = 4.0   # keeps the block's scale at 2^0 before shifting
            part = near[lo:lo + 15]
            v[1:1 + len(part)] = part
            v[16:16 + len(part)] = -part
            rows.append((v.astype(np.float64) * 2.0 ** e).astype(np.float32))
    tiny = np.float32(1e-45)
    big = np.finfo(np.float32).max
    for v in ([0.0], [-0.0, 0.0], [tiny], [2.0 ** -127, -tiny], [big, -big, 1.0], [np.nan, 1.0], [np.inf, 2.0], [-np.inf],
              [2.0 ** -126, 2.0 ** -128]):
        r = np.zeros(32, np.float32)
        r[:len(v)] = v
        rows.append(r)
    x = torch.from_numpy(np.stack(rows)).cuda()
    codes, scales, rc, rs = check_quantize(b200, x)
    out = torch.empty(x.shape, device="cuda")
    b200.mx4_dequantize_device(x.shape[0], 32, codes.data_ptr(), scales.data_ptr(), b200.F32, out.data_ptr())
    np.testing.assert_array_equal(out.cpu().numpy(), ref.mx4_values(rc, rs, 32).astype(np.float32))
    # a block that is not a number leaves its neighbours alone
    y = torch.ones(2, 96, device="cuda")
    y[1, 40] = float("nan")
    check_quantize(b200, y)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("n, d, ld", [(1, 1, 0), (9, 5, 0), (3, 33, 0), (130, 128, 0), (7, 777, 780), (5, 100, 101), (2, 4096, 0),
                                      (300, 777, 0), (6, 96, 104), (40, 9, 0)])
def test_mx4_dequantize(b200, n, d, ld, dtype):
    rng = np.random.default_rng(d)
    rc, rs = ref.random_mx4(rng, n, d, spread=9)
    pc, ps = ref.mx4_pack(rc, rs)
    codes, scales = torch.from_numpy(pc).cuda(), torch.from_numpy(ps).cuda()
    ld = ld or d
    out = torch.full((n, ld), -7.0, dtype=ref.TORCH[dtype], device="cuda")
    b200.mx4_dequantize_device(n, d, codes.data_ptr(), scales.data_ptr(), dtype, out.data_ptr(), ldo=ld, stream_ptr=_stream())
    want = torch.from_numpy(ref.mx4_values(rc, rs, d)).to(ref.TORCH[dtype])   # one rounding, none for fp32 and bf16
    assert torch.equal(out[:, :d].cpu(), want) and bool((out[:, d:] == -7.0).all())


# ---- RMS norm -> int8 ----
def rms(b, x, w, eps=1e-6, residual=None, static=None, in_place=None, ldq=0):
    n, d = x.shape
    dt = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[x.dtype]
    ld = lambda t: t.stride(0) if n > 1 else 0  # noqa: E731
    q = torch.full((n * (ldq or d) + 64,), 99, dtype=torch.int8, device="cuda")
    scales = None if static is not None else torch.full((n + 4,), -5.0, device="cuda")
    total = None
    if residual is not None:
        total = {"x": x, "residual": residual, None: torch.empty(n, d, dtype=x.dtype, device="cuda")}[in_place]
    b.rms_norm_i8_device(n, d, dt, x.data_ptr(), w.data_ptr(), eps, q.data_ptr(), ldx=ld(x), ldq=ldq,
                         residual_ptr=0 if residual is None else residual.data_ptr(),
                         ldr=0 if residual is None else ld(residual),
                         sum_ptr=0 if total is None else total.data_ptr(), lds=0 if total is None else ld(total),
                         scales_ptr=0 if scales is None else scales.data_ptr(),
                         static_scale_ptr=0 if static is None else static.data_ptr(), stream_ptr=_stream())
    torch.cuda.synchronize()
    assert bool((q[n * (ldq or d):] == 99).all()) and (scales is None or bool((scales[n:] == -5.0).all()))
    rows = q[:n * (ldq or d)].view(n, ldq or d)
    assert bool((rows[:, d:] == 99).all())
    return rows[:, :d], None if scales is None else scales[:n], total


def check_rms(x, w, eps, q, scales, total, residual=None, static=None):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    if total is not None:
        assert torch.equal(total, s)
    y = ref.rms_norm(s.double().cpu().numpy(), w.double().cpu().numpy(), eps)
    if static is None:
        want = np.abs(y).max(1) / 127
        # fp32: d squares added up in any order (d eps), root, quotient, products: under (d / 2 + 8) roundings,
        # half of the sum's error left by the root; blockwise sums keep it far below that
        tol = (s.shape[1] / 64 + 8) * ref.EPS[0]
        np.testing.assert_allclose(scales.double().cpu().numpy(), want, rtol=tol, atol=0)
        step = np.where(want > 0, want, 1.0)[:, None]
    else:
        step = float(static)
    exact = np.clip(y / step, -127, 127)
    # half a step, and the fp32 roundings of a value of at most 127 steps
    off = np.abs(q.double().cpu().numpy() - exact)
    assert off.max() <= 0.5 + 127 * (s.shape[1] / 64 + 8) * ref.EPS[0], off.max()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("static", [False, True])
@pytest.mark.parametrize("n, d", [(1, 1), (1, 768), (5, 31), (3, 256), (9, 257), (4, 512), (2, 1000), (6, 1024), (3, 2048),
                                  (2, 3001), (3, 4096), (2, 5000), (1, 8192), (2, 16384), (1, 16001)])
def test_rms_norm_i8(b200, n, d, static, residual, dtype):
    rng = np.random.default_rng(d + n)
    x, w = _rows(rng, n, d, dtype), _rows(rng, 1, d, dtype, 0.0).view(-1)
    r = _rows(rng, n, d, dtype) if residual else None
    s = torch.tensor([0.021], device="cuda") if static else None
    q, scales, total = rms(b200, x, w, residual=r, static=s)
    check_rms(x, w, 1e-6, q, scales, total, r, s)


@pytest.mark.parametrize("dtype", [0, 2])
@pytest.mark.parametrize("ld, offset, ldq", [(104, 0, 104), (101, 3, 0), (112, 1, 103)])
def test_rms_norm_strides(b200, ld, offset, ldq, dtype):
    rng = np.random.default_rng(3)
    x, r = (_strided(_rows(rng, 11, 100, dtype), ld, offset) for _ in range(2))
    w = _rows(rng, 1, 100, dtype).view(-1)
    q, scales, total = rms(b200, x, w, residual=r, ldq=ldq)
    check_rms(x, w, 1e-6, q, scales, total, r)


@pytest.mark.parametrize("place", ["x", "residual"])
@pytest.mark.parametrize("n, d, dtype", [(5, 64, 2), (5, 77, 2), (5, 4096, 2), (20000, 64, 2), (15001, 77, 1), (3000, 1024, 0), (1500, 4096, 2)])
def test_rms_norm_sum_in_place(b200, place, n, d, dtype):
    """(With many rows a thread's next row is on its way while it writes this one.)"""
    rng = np.random.default_rng(4)
    x, r, w = _rows(rng, n, d, dtype), _rows(rng, n, d, dtype), _rows(rng, 1, d, dtype).view(-1)
    x0, r0 = x.clone(), r.clone()
    q, scales, total = rms(b200, x, w, residual=r, in_place=place)
    check_rms(x0, w, 1e-6, q, scales, total, r0)
    assert torch.equal(r if place == "x" else x, r0 if place == "x" else x0)


def test_rms_norm_range(b200):
    """Rows whose squares leave fp32, tiny rows, rows of zeros, rows that hold no numbers."""
    d = 300
    rng = np.random.default_rng(9)
    base = rng.standard_normal((6, d)).astype(np.float32)
    x = np.stack([base[0] * 1e30, base[1] * 1e-30, np.zeros(d, np.float32), base[3], base[4], base[5] * 3e37])
    x[3, 7] = np.nan
    x[4, 290] = np.inf
    x = torch.from_numpy(x).cuda()
    w = torch.from_numpy((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)).cuda()
    for residual in (None, torch.zeros_like(x)):
        q, scales, total = rms(b200, x, w, residual=residual, in_place=None if residual is None else "x")
        good = [0, 1, 5]
        check_rms(x[good], w, 1e-6, q[good], scales[good], None)
        assert float(scales[2]) == 0.0 and bool((q[2] == 0).all())
        assert bool(torch.isnan(scales[3:5]).all()) and bool((q[3:5] == 0).all())
    for s in (0.0, -1.0, float("nan"), float("inf")):
        q, _, _ = rms(b200, x, w, static=torch.tensor([s], device="cuda"))
        assert bool((q == 0).all())


@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("static", [False, True])
@pytest.mark.parametrize("n, d, dtype", [(5, 20, 0), (7, 100, 1), (6, 128, 2), (3, 777, 2), (4, 900, 0), (3, 4096, 2), (2, 16384, 1)])
def test_rms_norm_weights_that_are_no_numbers(b200, n, d, dtype, static, bad):
    rng = np.random.default_rng(d)
    x = _rows(rng, n, d, dtype)
    x[n - 1, d // 2] = 0.0   # 0 * infinity
    w = torch.ones(d, dtype=ref.TORCH[dtype], device="cuda")
    w[d // 2] = float(bad)
    q, scales, _ = rms(b200, x, w, static=torch.full((1,), 0.03, device="cuda") if static else None)
    assert bool((q == 0).all())
    assert static or bool(torch.isnan(scales).all())


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("d, dtype", [(20, 0), (100, 1), (100, 2), (128, 0), (250, 2), (500, 1), (900, 2)])
def test_rms_norm_range_next_to_others(b200, d, dtype, residual):
    """Rows that leave the fast path between rows that do not, in one warp and in one block."""
    rng = np.random.default_rng(10)
    n = 700
    base = rng.standard_normal((n, d))
    huge, tiny = (3e4, 1e-6) if dtype == 1 else (1e36, 1e-33)
    kind = rng.integers(0, 8, n)
    base[kind == 0] *= huge / np.abs(base).max()
    base[kind == 1] *= tiny
    base[kind == 2] = 0
    x = torch.from_numpy(base).to("cuda", ref.TORCH[dtype])
    bad = torch.from_numpy((kind == 3) | (kind == 4)).cuda()
    x[torch.from_numpy(kind == 3).cuda(), d // 2] = float("nan")
    x[torch.from_numpy(kind == 4).cuda(), 0] = float("inf")
    w = _rows(rng, 1, d, dtype, 0.1).view(-1)
    r = torch.zeros_like(x) if residual else None
    q, scales, total = rms(b200, x, w, residual=r)
    assert bool(torch.isnan(scales[bad]).all()) and bool((q[bad] == 0).all())
    if dtype == 1:   # (fp16 rows of subnormal numbers: their values are exact, as every fp16 value is in 64 bits)
        assert float(x[torch.from_numpy(kind == 1).cuda()].abs().max()) < 1e-4
    good = ~bad
    check_rms(x[good], w, 1e-6, q[good], scales[good], None if total is None else total[good], None if r is None else r[good])


@pytest.mark.parametrize("static", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n, d, dtype", [(3, 20, 0), (700, 100, 2), (9, 128, 0), (5, 250, 2), (300, 777, 2), (4, 1024, 0), (3, 4096, 2),
                                         (2, 9000, 0), (2, 16384, 2)])
def test_rms_norm_products_below_fp32(b200, n, d, dtype, residual, static):
    """s w below fp32's least number, y above it (the root is at least 1e-6 with this eps): rows between zeros and others."""
    rng = np.random.default_rng(d)
    base = rng.uniform(0.25, 1.0, (n, d)) * rng.choice([-1.0, 1.0], (n, d))
    kind = np.arange(n) % 3
    base[kind == 0] *= 1e-23            # products of at most 5e-46: no fp32 number but 0 is as near
    base[kind == 1] = 0
    x = torch.from_numpy(base).to("cuda", ref.TORCH[dtype])
    w = torch.from_numpy(rng.uniform(0.5, 1.0, d) * 5e-23).to("cuda", ref.TORCH[dtype])
    r = torch.zeros_like(x) if residual else None
    s = torch.full((1,), 1e-41, device="cuda") if static else None
    q, scales, total = rms(b200, x, w, eps=1e-12, residual=r, static=s)
    y = ref.rms_norm(x.double().cpu().numpy(), w.double().cpu().numpy(), 1e-12)
    tiny = kind == 0
    assert 0 < np.abs(y[tiny]).max() < 2.0 ** -125 and bool((q[torch.from_numpy(kind == 1).cuda()] == 0).all())
    if static:
        step = np.full((n, 1), float(s.double()))
    else:
        top = np.abs(y).max(1) / 127
        # half of fp32's least number where the scale is that small
        np.testing.assert_allclose(scales.double().cpu().numpy(), top, rtol=(d / 64 + 8) * ref.EPS[0], atol=2.0 ** -150)
        step = np.where(top > 0, top, 1.0)[:, None]
    assert np.abs(np.clip(y / step, -127, 127)[tiny]).max() > 5
    off = np.abs(q.double().cpu().numpy() - np.clip(y / step, -127, 127))
    assert off.max() <= 0.5 + 127 * (d / 64 + 8) * ref.EPS[0], off.max()


@pytest.mark.parametrize("d, dtype", [(40, 0), (300, 2), (2048, 0)])
def test_rms_norm_given_scale_below_fp32(b200, d, dtype):
    """A given scale of 1e-41: elements of that size count next to large ones, which are cut."""
    rng = np.random.default_rng(d)
    x = rng.standard_normal((6, d))
    x[:, 1::2] = rng.uniform(-1, 1, (6, d // 2)) * 9e-40
    x = torch.from_numpy(x).to("cuda", ref.TORCH[dtype])
    w = torch.ones(d, dtype=ref.TORCH[dtype], device="cuda")
    s = torch.full((1,), 1e-41, device="cuda")
    q, scales, total = rms(b200, x, w, static=s)
    check_rms(x, w, 1e-6, q, scales, total, None, s)
    assert int((q.abs() < 127).sum()) > d


def test_rms_norm_ties(b200):
    """Products that lie exactly between two steps go to the even one: s w 254 / max is a whole odd number."""
    d = 64
    rng = np.random.default_rng(12)
    x = rng.integers(-254, 255, (500, d)).astype(np.float64)
    x[:, 0] = 254          # scale 2 after the norm's factor: every odd number is half way
    for dtype in (0, 1):   # (bf16 holds only some of these numbers)
        xt = torch.from_numpy(x).to("cuda", ref.TORCH[dtype])
        q, _, _ = rms(b200, xt, torch.ones(d, dtype=ref.TORCH[dtype], device="cuda"))
        np.testing.assert_array_equal(q.cpu().numpy(), np.rint(x / 2))   # (numpy rounds halves to even)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("n, d, ldq, ldo", [(1, 1, 0, 0), (3, 100, 104, 101), (65, 96, 0, 0), (7, 4096, 0, 0)])
def test_i8_dequantize(b200, n, d, ldq, ldo, dtype):
    rng = np.random.default_rng(1)
    q = torch.from_numpy(rng.integers(-128, 128, (n, ldq or d)).astype(np.int8)).cuda()
    scales = torch.from_numpy(rng.random(n).astype(np.float32)).cuda()
    out = torch.full((n, ldo or d), 3.0, dtype=ref.TORCH[dtype], device="cuda")
    b200.i8_dequantize_device(n, d, q.data_ptr(), dtype, out.data_ptr(), scales_ptr=scales.data_ptr(), ldq=ldq, ldo=ldo,
                              stream_ptr=_stream())
    want = (q[:, :d].float() * scales[:, None]).to(ref.TORCH[dtype])
    assert torch.equal(out[:, :d], want) and bool((out[:, d:] == 3.0).all())
    b200.i8_dequantize_device(n, d, q.data_ptr(), dtype, out.data_ptr(), static_scale_ptr=scales.data_ptr(), ldq=ldq,
                              ldo=ldo, stream_ptr=_stream())
    assert torch.equal(out[:, :d], (q[:, :d].float() * scales[0]).to(ref.TORCH[dtype]))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("n, d", [(1, 9), (5, 9), (33, 77), (4, 777), (7, 1001), (1000, 13), (2001, 8), (3, 15), (130, 100)])
def test_i8_dequantize_rows_without_gaps(b200, n, d, dtype):
    """Rows that end inside a thread's eight outputs, which then have the scales of two rows; a last piece of fewer than eight."""
    rng = np.random.default_rng(n + d)
    q = torch.from_numpy(rng.integers(-128, 128, (n, d)).astype(np.int8)).cuda()
    scales = torch.from_numpy(np.exp2(rng.integers(-3, 4, n)).astype(np.float32) * 1.25).cuda()
    for given in (False, True):
        out = torch.full((n * d + 16,), 3.0, dtype=ref.TORCH[dtype], device="cuda")
        b200.i8_dequantize_device(n, d, q.data_ptr(), dtype, out.data_ptr(), scales_ptr=0 if given else scales.data_ptr(),
                                  static_scale_ptr=scales.data_ptr() if given else 0, stream_ptr=_stream())
        want = (q.float() * (scales[0] if given else scales[:, None])).to(ref.TORCH[dtype])
        assert torch.equal(out[:n * d].view(n, d), want) and bool((out[n * d:] == 3.0).all())


# ---- MX4 product ----
def product(b, m, n, d, a, bb, dtype=0, ldo=0):
    out = torch.full((m * (ldo or n) + 16,), -3.0, dtype=ref.TORCH[dtype], device="cuda")
    b.mx4_product_device(m, n, d, a[0].data_ptr(), a[1].data_ptr(), bb[0].data_ptr(), bb[1].data_ptr(), dtype, out.data_ptr(),
                         ldo=ldo, stream_ptr=_stream())
    torch.cuda.synchronize()
    assert bool((out[m * (ldo or n):] == -3.0).all())
    rows = out[:m * (ldo or n)].view(m, ldo or n)
    assert bool((rows[:, n:] == -3.0).all())
    return rows[:, :n]


def random_operand(rng, n, d, spread=2, fill=127):
    c, s = ref.random_mx4(rng, n, d, spread)
    p, t = ref.mx4_pack(c, s, fill)
    return (torch.from_numpy(p).cuda(), torch.from_numpy(t).cuda()), ref.mx4_values(c, s, d)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("m, n, d", [(1, 1, 1), (1, 64, 32), (2, 300, 64), (3, 257, 33), (17, 1000, 128), (64, 129, 160),
                                     (65, 511, 256), (127, 256, 288), (128, 257, 1000), (129, 300, 96), (200, 70, 544),
                                     (1, 5000, 768), (16, 4096, 2048), (5, 130, 4096), (300, 600, 4100), (2, 40, 16384),
                                     (2100, 2300, 96), (700, 7000, 544), (2049, 2305, 4100), (4000, 1300, 33)])
def test_mx4_product(b200, m, n, d, dtype):
    """Sums that fp32 holds exactly: products are quarters times at least 2^-4, sums stay below 2^24 of those
    (|sum| <= 36 d 2^2, in steps of 2^-6: d <= 2^24 / (36 * 2^8) = 1820; longer rows use equal scales:
    d <= 2^24 / (36 * 4)).  Equality, then, or one rounding to 16 bits."""
    rng = np.random.default_rng(m * 7 + n + d)
    spread = 1 if d <= 1800 else 0
    # rows behind m and n have scale bytes that stand for NaN: nobody may see them
    if spread:
        a, va = random_operand(rng, m, d, spread, fill=255)
        bb, vb = random_operand(rng, n, d, spread, fill=255)
    else:
        ca, cb = ref.random_mx4(rng, m, d)[0], ref.random_mx4(rng, n, d)[0]
        nb = -(-d // 32)
        sa, sb = np.full((m, nb), 126, np.uint8), np.full((n, nb), 129, np.uint8)
        a = [torch.from_numpy(t).cuda() for t in ref.mx4_pack(ca, sa, 255)]
        bb = [torch.from_numpy(t).cuda() for t in ref.mx4_pack(cb, sb, 255)]
        va, vb = ref.mx4_values(ca, sa, d), ref.mx4_values(cb, sb, d)
    want = torch.from_numpy(va @ vb.T).to(ref.TORCH[dtype]).cuda()
    assert torch.equal(product(b200, m, n, d, a, bb, dtype), want)


@pytest.mark.parametrize("dtype", [0, 2])
@pytest.mark.parametrize("ldo", [301, 304, 512])
def test_mx4_product_output_stride(b200, ldo, dtype):
    rng = np.random.default_rng(2)
    for m in (3, 140):
        a, va = random_operand(rng, m, 96)
        bb, vb = random_operand(rng, 300, 96)
        want = torch.from_numpy(va @ vb.T).to(ref.TORCH[dtype]).cuda()
        assert torch.equal(product(b200, m, 300, 96, a, bb, dtype, ldo), want)


@pytest.mark.parametrize("m", [1, 7, 33, 150])
def test_mx4_product_wide_scales(b200, m):
    """Scales across the whole range of the format; sums round."""
    rng = np.random.default_rng(8)
    n, d = 200, 512
    ca, cb = ref.random_mx4(rng, m, d)[0], ref.random_mx4(rng, n, d)[0]
    sa = rng.integers(87, 168, (m, d // 32)).astype(np.uint8)
    sb = rng.integers(87, 168, (n, d // 32)).astype(np.uint8)
    a = [torch.from_numpy(t).cuda() for t in ref.mx4_pack(ca, sa)]
    bb = [torch.from_numpy(t).cuda() for t in ref.mx4_pack(cb, sb)]
    va, vb = ref.mx4_values(ca, sa, d), ref.mx4_values(cb, sb, d)
    got = product(b200, m, n, d, a, bb).double().cpu().numpy()
    # d additions of terms of that size, each off by at most a step (the tensor core may cut instead of round)
    tol = 2 * ref.EPS[0] * d * (np.abs(va) @ np.abs(vb).T)
    assert np.all(np.abs(got - va @ vb.T) <= tol)


@pytest.mark.parametrize("m", [1, 40, 200])
def test_mx4_product_nan_blocks(b200, m):
    """A block that stands for NaN makes its row's scores NaN and nobody else's."""
    rng = np.random.default_rng(6)
    n, d = 150, 100
    ca, sa = ref.random_mx4(rng, m, d)
    cb, sb = ref.random_mx4(rng, n, d)
    sa[0, 1], ca[0, 32:64] = 255, 0
    sb[149, 3], cb[149, 96:128] = 255, 0
    a = [torch.from_numpy(t).cuda() for t in ref.mx4_pack(ca, sa)]
    bb = [torch.from_numpy(t).cuda() for t in ref.mx4_pack(cb, sb)]
    got = product(b200, m, n, d, a, bb).cpu().numpy()
    bad = np.zeros((m, n), bool)
    bad[0], bad[:, 149] = True, True
    want = ref.mx4_values(ca, sa, d) @ ref.mx4_values(cb, sb, d).T
    np.testing.assert_array_equal(np.isnan(got), bad)
    np.testing.assert_array_equal(got[~bad], want[~bad].astype(np.float32))


@pytest.mark.parametrize("m, n, d", [(1, 3000, 768), (3, 260, 4096), (100, 700, 1000), (140, 300, 2048), (1500, 3500, 160)])
def test_mx4_product_captured_and_on_two_streams(b200, m, n, d):
    """Every kernel of the product (few rows, split K, 128 and 256 columns, pairs of CTAs): captured once, replayed on
    other operands in the same memory, while another stream computes a product of its own."""
    rng = np.random.default_rng(m)
    mk = lambda r: [torch.from_numpy(t).cuda() for t in ref.mx4_pack(*ref.random_mx4(rng, r, d, 1))]  # noqa: E731
    a, bb, a2 = mk(m), mk(n), mk(m)
    out, other = torch.zeros(m, n, device="cuda"), torch.zeros(n, m, device="cuda")
    call = lambda x, y, r, c, o, s: b200.mx4_product_device(r, c, d, x[0].data_ptr(), x[1].data_ptr(), y[0].data_ptr(),  # noqa: E731
                                                            y[1].data_ptr(), b200.F32, o.data_ptr(), stream_ptr=s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(a, bb, m, n, out, _stream())
    vals = lambda t, r: ref.mx4_values(*ref.mx4_unpack(t[0].cpu().numpy(), t[1].cpu().numpy(), r, -(-d // 32)), d)  # noqa: E731
    vb = vals(bb, n)
    side = torch.cuda.Stream()
    for new in (a, a2):
        if new is not a:
            for t, u in zip(a, new):
                t.copy_(u)
        torch.cuda.synchronize()
        for _ in range(3):
            g.replay()
            call(bb, a, n, m, other, side.cuda_stream)
        torch.cuda.synchronize()
        want = vals(a, m) @ vb.T
        tol = 2 * ref.EPS[0] * d * 36 * 4   # (d > 1800: sums may round)
        assert float((out.double().cpu() - torch.from_numpy(want)).abs().max()) <= (0 if d <= 1800 else tol)
        assert torch.equal(other.t(), out) or d > 1800


def test_offsets_beyond_32_bits(b200):
    """More than 2^32 elements of input and of output."""
    n, d = 70_000_000, 64
    x = torch.zeros(n, d, dtype=torch.bfloat16, device="cuda")
    ends = torch.from_numpy(np.random.default_rng(1).standard_normal((300, d))).to("cuda", torch.bfloat16)
    x[:300], x[-300:] = ends, ends
    x[33_554_400:33_554_700] = ends            # around element 2^31
    codes = torch.empty(n, 32, dtype=torch.uint8, device="cuda")
    scales = torch.empty(b200.mx4_scale_bytes(n, d), dtype=torch.uint8, device="cuda")
    b200.mx4_quantize_device(n, d, b200.BF16, x.data_ptr(), codes.data_ptr(), scales.data_ptr(), stream_ptr=_stream())
    rc, rs = ref.mx4_encode(ends.double().cpu().numpy())
    packed = torch.from_numpy(ref.mx4_pack(rc, rs)[0]).cuda()
    for lo in (0, 33_554_400, n - 300):
        assert torch.equal(codes[lo:lo + 300], packed)
    out = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    b200.mx4_dequantize_device(n, d, codes.data_ptr(), scales.data_ptr(), b200.BF16, out.data_ptr(), stream_ptr=_stream())
    want = torch.from_numpy(ref.mx4_values(rc, rs, d)).to("cuda", torch.bfloat16)
    for lo in (0, 33_554_400, n - 300):
        assert torch.equal(out[lo:lo + 300], want)
    w = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    q = torch.empty(n, d, dtype=torch.int8, device="cuda")
    sc = torch.empty(n, device="cuda")
    b200.rms_norm_i8_device(n, d, b200.BF16, x.data_ptr(), w.data_ptr(), 1e-6, q.data_ptr(), scales_ptr=sc.data_ptr(), stream_ptr=_stream())
    check_rms(ends, w, 1e-6, q[-300:], sc[-300:], None)
    b200.i8_dequantize_device(n, d, q.data_ptr(), b200.BF16, out.data_ptr(), scales_ptr=sc.data_ptr(), stream_ptr=_stream())
    assert torch.equal(out[-300:], (q[-300:].float() * sc[-300:, None]).bfloat16())
    del out, q, x
    # scores: 70 million rows against 70 of them
    m = 70
    res = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    b200.mx4_product_device(m, n, d, codes.data_ptr(), scales.data_ptr(), codes.data_ptr(), scales.data_ptr(), b200.BF16,
                            res.data_ptr(), stream_ptr=_stream())
    v = want.double()
    assert torch.equal(res[:, -300:], (v[:m] @ v.t()).bfloat16())
    assert torch.equal(res[:, :300], (v[:m] @ v.t()).bfloat16())


# ---- the operators as they are used ----
def test_states_to_scores(b200):
    """fp16 states -> RMS norm -> int8 -> values -> MX4 -> scores, one after the other on a stream of their own,
    while that stream is not the current one's default; then the same captured and replayed on new states."""
    rng = np.random.default_rng(11)
    n, m, d = 70, 9, 200
    st = torch.cuda.Stream()
    x = _rows(rng, n, d, 1)
    w = _rows(rng, 1, d, 1, 0.1).view(-1)
    q = torch.empty(n, d, dtype=torch.int8, device="cuda")
    sc = torch.empty(n, device="cuda")
    val = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    codes = torch.empty(n, b200.mx4_row_bytes(d), dtype=torch.uint8, device="cuda")
    scales = torch.empty(b200.mx4_scale_bytes(n, d), dtype=torch.uint8, device="cuda")
    out = torch.empty(m, n, device="cuda")

    def chain(s):
        b200.rms_norm_i8_device(n, d, b200.F16, x.data_ptr(), w.data_ptr(), 1e-6, q.data_ptr(), scales_ptr=sc.data_ptr(),
                                stream_ptr=s)
        b200.i8_dequantize_device(n, d, q.data_ptr(), b200.BF16, val.data_ptr(), scales_ptr=sc.data_ptr(), stream_ptr=s)
        b200.mx4_quantize_device(n, d, b200.BF16, val.data_ptr(), codes.data_ptr(), scales.data_ptr(), stream_ptr=s)
        b200.mx4_product_device(m, n, d, codes.data_ptr(), scales.data_ptr(), codes.data_ptr(), scales.data_ptr(), b200.F32,
                                out.data_ptr(), stream_ptr=s)

    def check():
        check_rms(x, w, 1e-6, q, sc, None)
        assert torch.equal(val, (q.float() * sc[:, None]).bfloat16())
        rc, rs = ref.mx4_encode(val.double().cpu().numpy())
        v = ref.mx4_values(rc, rs, d)
        np.testing.assert_allclose(out.double().cpu().numpy(), (v @ v.T)[:m], rtol=0,
                                   atol=2 * ref.EPS[0] * d * float((np.abs(v) @ np.abs(v).T).max()))

    torch.cuda.synchronize()
    chain(st.cuda_stream)
    torch.cuda.synchronize()
    check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chain(_stream())
    for seed in (12, 13):
        x.copy_(_rows(np.random.default_rng(seed), n, d, 1))
        g.replay()
        torch.cuda.synchronize()
        check()
