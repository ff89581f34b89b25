"""Operators on rows of vectors in few bits: what programs that build and search compressed exact indexes call.

``own`` false: ``run`` computes the operators in their plain form with elementary torch operations.
``own`` true : ``run`` makes the calls of ``indexsdk_b200`` that a user's program makes.

kind   : rms      residual addition, root-mean-square norm and rounding to int8 rows with scales, as the last
                  step of an embedding model before its rows go into an Int8Flat index
         quantize rows -> microscaled 4-bit floating point (blocks of 32 elements E2M1, one scale E8M0 a block)
         product  all scores of two sets of such rows, out[i][j] = sum_k a[i][k] b[j][k]
         search   k nearest rows of an index that stores such rows (queries are rounded the same way)

What is held in 8 or 4 bits comes back as the values it stands for: ``run`` ends with the reconstruction.

Layout of 4-bit rows: row r is ceil(d / 32) * 16 bytes, element 2 i in the low half of byte i, zeros behind
element d.  The scale of block c of row r is byte (r / 128 * ceil(ceil(d / 32) / 4) + c / 4) * 512 +
r % 32 * 16 + r % 128 / 32 * 4 + c % 4; blocks behind the last one have the scale 1 (127).
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # The last hidden state of one query on its way into a search: latency is all that counts.
        dict(name="rms_one", kind="rms", n=1, d=768, dtype="bf16", residual=True, static=False),
        # A ragged batch of fp32 states without a residual, rows of an odd length, one scale for the whole index.
        dict(name="rms_ragged", kind="rms", n=1003, d=1001, dtype="f32", residual=False, static=True),
        # Loading an index from an embedding model's batches: wide bf16 rows, the largest call of this kind.
        dict(name="rms_load", kind="rms", n=65_536, d=4096, dtype="bf16", residual=True, static=False),
        # One query rounded to 4 bits.
        dict(name="quantize_one", kind="quantize", n=1, d=128, dtype="f32"),
        # Loading a gallery of a million rows of the exact-search benchmark's width.
        dict(name="quantize_load", kind="quantize", n=1_000_000, d=128, dtype="f32"),
        # Half-precision rows of an odd length (the last block is short, rows start on odd addresses).
        dict(name="quantize_ragged", kind="quantize", n=20_011, d=777, dtype="bf16"),
        # All scores of one query against a gallery.
        dict(name="product_one", kind="product", m=1, n=100_003, d=768, out="f32"),
        # A ragged batch: rows, columns and depth divide nothing.
        dict(name="product_ragged", kind="product", m=100, n=20_011, d=1000, out="f32"),
        # All pairs of two large sets of wide rows, the largest amount of arithmetic here.
        dict(name="product_large", kind="product", m=4096, n=16_384, d=4096, out="bf16"),
        # One online query against an index of 4-bit rows.
        dict(name="search_one", kind="search", n=100_003, d=128, metric="l2", nq=1, k=10),
        # The exact-search benchmark's shape on 4-bit rows: 1 M x 128, k = 100, a batch of 64 queries.
        dict(name="search_1m", kind="search", n=1_000_000, d=128, metric="ip", nq=64, k=100),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges that the listed ones span."""
    kind = rng.choice(["rms", "quantize", "product", "product", "search"])
    if kind == "rms":
        d = rng.choice([_log(rng, 32, 4096), 16 * _log(rng, 2, 256)])
        return dict(kind=kind, n=_log(rng, 1, min(65_536, 100_000_000 // d)), d=d, dtype=rng.choice(list(DTYPES)),
                    residual=rng.random() < 0.6, static=rng.random() < 0.4)
    if kind == "quantize":
        d = rng.choice([_log(rng, 32, 4096), 32 * _log(rng, 1, 128)])
        return dict(kind=kind, n=_log(rng, 1, min(1_000_000, 100_000_000 // d)), d=d, dtype=rng.choice(list(DTYPES)))
    if kind == "product":
        d = rng.choice([_log(rng, 32, 4096), 32 * _log(rng, 1, 128)])
        m = _log(rng, 1, 4096)
        n = _log(rng, 64, min(1_000_000, 200_000_000 // d, 60_000_000 // m))
        return dict(kind=kind, m=m, n=n, d=d, out=rng.choice(list(DTYPES)))
    d = 16 * _log(rng, 4, 64)
    nq = _log(rng, 1, 256)
    n = _log(rng, 1000, min(1_000_000, 200_000_000 // d, 60_000_000 // nq))
    return dict(kind=kind, n=n, d=d, metric=rng.choice(["ip", "l2"]), nq=nq, k=_log(rng, 1, min(300, n)))


# ---- the 4-bit format in elementary operations ----
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _blocks(x):
    n, d = x.shape
    nb = (d + 31) // 32
    p = torch.zeros(n, nb * 32, device=x.device)
    p[:, :d] = x
    return p.view(n, nb, 32)


def _encode(x):
    """Codes (0 .. 15) and scale bytes of rows, both as integers: [n][nb][32], [n][nb]."""
    v = _blocks(x)
    amax = v.abs().amax(2)
    fine = torch.isfinite(v).all(2)
    _, e = torch.frexp(torch.where(fine & (amax > 0), amax, torch.ones_like(amax)))   # amax = m 2^e, 1/2 <= m < 1
    e = torch.where(amax > 0, (e - 3).clamp(-127, 125), torch.full_like(e, -127))
    u = torch.ldexp(v, -e.unsqueeze(2))
    a = u.abs()
    # nearest of the eight magnitudes; a value half way goes to the even code
    mag = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() +
           (a >= 3.5).int() + (a > 5.0).int())
    codes = torch.where(fine.unsqueeze(2), mag + 8 * torch.signbit(u).int(), torch.zeros_like(mag))
    return codes, torch.where(fine, e + 127, torch.full_like(e, 255))


def _values(codes, scales, d):
    """The values that codes and scale bytes stand for, fp32 [n][d]."""
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (table[codes.long()] * s.unsqueeze(2)).flatten(1)[:, :d]


def _pack(codes, scales):
    """The layout that programs keep: packed codes [n][nb * 16] and scale bytes in blocks of 128 rows."""
    n, nb = scales.shape
    flat = codes.flatten(1)
    packed = (flat[:, 0::2] | (flat[:, 1::2] << 4)).to(torch.uint8)
    rt, ct = (n + 127) // 128, (nb + 3) // 4
    s = torch.full((rt * 128, ct * 4), 127, device=scales.device, dtype=torch.uint8)
    s[:n, :nb] = scales.to(torch.uint8)
    s = s.view(rt, 4, 32, ct, 4).permute(0, 3, 2, 1, 4).contiguous()
    return packed, s.view(-1)


def _unpack(packed, scales, n):
    nb = packed.shape[1] // 16
    codes = torch.stack((packed & 15, packed >> 4), 2).view(n, nb, 32)
    rt, ct = (n + 127) // 128, (nb + 3) // 4
    s = scales.view(rt, ct, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, ct * 4)
    return codes, s[:n, :nb]


def _packed_rows(x):
    """Packed form of many rows, a stretch at a time."""
    n, d = x.shape
    step = max(128, 32_000_000 // d // 128 * 128)
    parts = [_pack(*_encode(x[lo:lo + step])) for lo in range(0, n, step)]
    return torch.cat([p for p, _ in parts]), torch.cat([s for _, s in parts])


# ---- inputs ----
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _states(n, d, g, dtype):
    """Hidden states: normal values, some channels wider than others."""
    wide = torch.exp(0.5 * torch.randn(d, generator=g, device="cuda"))
    return torch.randn(n, d, generator=g, device="cuda").mul_(wide).to(DTYPES[dtype])


def _embeddings(n, d, g):
    x = torch.randn(n, d, generator=g, device="cuda")
    return x.div_(x.norm(dim=1, keepdim=True))


def _inputs(case, seed):
    """The numbers of a case, in the types in which a program has them."""
    g, kind = _gen(seed), case["kind"]
    if kind == "rms":
        n, d, t = case["n"], case["d"], case["dtype"]
        x = _states(n, d, g, t)
        r = _states(n, d, g, t) if case["residual"] else None
        w = (1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(DTYPES[t])
        # one scale for the whole index, as a calibration gives it: a few values saturate
        s = torch.tensor([4.0 / 127], device="cuda") if case["static"] else None
        return dict(x=x, r=r, w=w, scale=s)
    if kind == "quantize":
        return dict(x=_states(case["n"], case["d"], g, case["dtype"]))
    if kind == "product":
        return dict(a=_embeddings(case["m"], case["d"], g), b=_embeddings(case["n"], case["d"], g))
    return dict(b=_embeddings(case["n"], case["d"], g), q=_embeddings(case["nq"], case["d"], g))


def prepare(case, seed):
    st = dict(_inputs(case, seed), case=case)
    if case["kind"] == "product":
        st["a"], st["b"] = _packed_rows(st["a"]), _packed_rows(st["b"])
    elif case["kind"] == "search":
        if own:
            import indexsdk_b200 as b
            metric = b.METRIC_L2 if case["metric"] == "l2" else b.METRIC_INNER_PRODUCT
            st["index"] = b.IndexFlat(case["d"], metric, b.MX4)
            torch.cuda.synchronize()
            st["index"].add_device(st["b"].data_ptr(), case["n"])
            st["D"] = torch.empty(case["nq"], case["k"], device="cuda")
            st["I"] = torch.empty(case["nq"], case["k"], device="cuda", dtype=torch.int64)
            del st["b"]
        else:
            st["b"] = _packed_rows(st["b"])
    torch.cuda.synchronize()
    return st


# ---- one pass, plain ----
def _plain(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "rms":
        x, r, w = st["x"], st["r"], st["w"]
        s = x if r is None else (x.float() + r.float()).to(x.dtype)
        f = s.double()   # (a rounding to whole numbers follows: values next to a border)
        y = f / torch.sqrt(f.square().mean(1, keepdim=True) + EPS) * w.double()
        scale = y.abs().amax(1, keepdim=True) / 127 if st["scale"] is None else st["scale"].double().view(1, 1)
        q = torch.round(y / torch.where(scale > 0, scale, torch.ones_like(scale))).clamp(-127, 127)
        scale = scale.float()
        values = (q.float() * scale).bfloat16()
        out = dict(values=values)
        if r is not None:
            out["sum"] = s
        if st["scale"] is None:
            out["scale"] = scale.view(-1)
        return out
    if kind == "quantize":
        codes, scales = _encode(st["x"].float())
        return _values(codes, scales, case["d"]).bfloat16()
    if kind == "product":
        a = _values(*_unpack(*st["a"], case["m"]), case["d"])
        b = _values(*_unpack(*st["b"], case["n"]), case["d"])
        return (a @ b.t()).to(DTYPES[case["out"]])
    q = _values(*_encode(st["q"]), case["d"])
    b = _values(*_unpack(*st["b"], case["n"]), case["d"])
    score = q @ b.t()
    if case["metric"] == "ip":
        key, pos = torch.sort(score, dim=1, descending=True, stable=True)   # ties: the lower position first
        return key[:, :case["k"]].contiguous(), pos[:, :case["k"]].contiguous()
    key, pos = torch.sort(b.square().sum(1) - 2 * score, dim=1, stable=True)
    dist = (key[:, :case["k"]] + q.square().sum(1, keepdim=True)).clamp(min=0)
    return dist, pos[:, :case["k"]].contiguous()


# ---- one pass, the framework's calls ----
def _framework(st):
    import indexsdk_b200 as b
    case, kind = st["case"], st["case"]["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    types = {"f32": b.F32, "f16": b.F16, "bf16": b.BF16}
    if kind == "rms":
        x, r, n, d = st["x"], st["r"], case["n"], case["d"]
        q = torch.empty(n, d, dtype=torch.int8, device="cuda")
        values = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
        out = dict(values=values)
        if r is not None:
            out["sum"] = torch.empty_like(x)
        if st["scale"] is None:
            out["scale"] = torch.empty(n, device="cuda")
        b.rms_norm_i8_device(n, d, types[case["dtype"]], x.data_ptr(), st["w"].data_ptr(), EPS, q.data_ptr(),
                             residual_ptr=r.data_ptr() if r is not None else 0,
                             sum_ptr=out["sum"].data_ptr() if r is not None else 0,
                             scales_ptr=out["scale"].data_ptr() if st["scale"] is None else 0,
                             static_scale_ptr=st["scale"].data_ptr() if st["scale"] is not None else 0,
                             stream_ptr=stream)
        b.i8_dequantize_device(n, d, q.data_ptr(), b.BF16, values.data_ptr(),
                               scales_ptr=out["scale"].data_ptr() if st["scale"] is None else 0,
                               static_scale_ptr=st["scale"].data_ptr() if st["scale"] is not None else 0,
                               stream_ptr=stream)
        return out
    if kind == "quantize":
        n, d = case["n"], case["d"]
        codes = torch.empty(n, b.mx4_row_bytes(d), dtype=torch.uint8, device="cuda")
        scales = torch.empty(b.mx4_scale_bytes(n, d), dtype=torch.uint8, device="cuda")
        values = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
        b.mx4_quantize_device(n, d, types[case["dtype"]], st["x"].data_ptr(), codes.data_ptr(), scales.data_ptr(),
                              stream_ptr=stream)
        b.mx4_dequantize_device(n, d, codes.data_ptr(), scales.data_ptr(), b.BF16, values.data_ptr(),
                                stream_ptr=stream)
        return values
    if kind == "product":
        m, n = case["m"], case["n"]
        out = torch.empty(m, n, dtype=DTYPES[case["out"]], device="cuda")
        b.mx4_product_device(m, n, case["d"], st["a"][0].data_ptr(), st["a"][1].data_ptr(), st["b"][0].data_ptr(),
                             st["b"][1].data_ptr(), types[case["out"]], out.data_ptr(), stream_ptr=stream)
        return out
    st["index"].search_device(st["q"].data_ptr(), case["nq"], case["k"], st["D"].data_ptr(), st["I"].data_ptr())
    return st["D"], st["I"]


def run(st):
    return _framework(st) if own else _plain(st)


def work(case):
    """Every input read once and every output written once, in their stored types; multiply-adds as two operations."""
    kind, d = case["kind"], case["d"]
    if kind in ("rms", "quantize"):
        n, size = case["n"], 4 if case["dtype"] == "f32" else 2
        if kind == "quantize":
            return dict(bytes=float(n * d * (size + 2)), flops=float(4 * n * d))
        moved = n * d * (size * (3 if case["residual"] else 1) + 2) + d * size + (0 if case["static"] else 4 * n)
        return dict(bytes=float(moved), flops=float(8 * n * d))
    row = (d + 31) // 32 * 17
    if kind == "product":
        m, n = case["m"], case["n"]
        return dict(bytes=float((m + n) * row + m * n * (4 if case["out"] == "f32" else 2)), flops=2.0 * m * n * d)
    nq, n = case["nq"], case["n"]
    return dict(bytes=float(n * row + nq * d * 4 + nq * case["k"] * 12), flops=2.0 * nq * n * d)


# ---- the definitions in 64 bits ----
def _exact_rows(x):
    """x rounded to 4-bit blocks, by distance to the 15 values instead of by borders."""
    n, d = x.shape
    nb = (d + 31) // 32
    v = torch.nn.functional.pad(x.double(), (0, nb * 32 - d)).view(n, nb, 32)
    top = v.abs().amax(2, keepdim=True)
    power = torch.floor(torch.log2(top))
    power = power - (torch.exp2(power) > top).double() + (torch.exp2(power + 1) <= top).double()
    step = torch.exp2(torch.where(top > 0, power - 2, torch.full_like(power, -127.0)).clamp(-127, 125))
    u = v / step
    best, out = torch.full_like(u, math.inf), torch.zeros_like(u)
    for value in (0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0):   # the even codes first: they win where two are as near
        gap = (u.abs() - value).abs()
        out = torch.where(gap < best, torch.full_like(u, value), out)
        best = torch.minimum(best, gap)
    return (out * torch.sign(u) * step).flatten(1)[:, :d]


def _exact_many(x):
    step = max(1, 8_000_000 // x.shape[1])
    return torch.cat([_exact_rows(x[lo:lo + step]) for lo in range(0, x.shape[0], step)])


def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "rms":
        parts = []
        step = max(1, 32_000_000 // case["d"])
        for lo in range(0, case["n"], step):
            s = t["x"][lo:lo + step].double()
            if t["r"] is not None:
                s = (t["x"][lo:lo + step].float() + t["r"][lo:lo + step].float()).to(t["x"].dtype).double()
            norm = (s * s).sum(1, keepdim=True).div(case["d"]).add(EPS).sqrt()
            y = s * t["w"].double() / norm
            scale = t["scale"].double().view(1, 1) if t["scale"] is not None else y.abs().amax(1, keepdim=True) / 127
            whole = torch.clamp(torch.round(y / scale), -127, 127)
            parts.append(((whole * scale).bfloat16(), s.to(t["x"].dtype), scale.view(-1)))
        out = dict(values=torch.cat([p[0] for p in parts]).double())
        if t["r"] is not None:
            out["sum"] = torch.cat([p[1] for p in parts]).double()
        if t["scale"] is None:
            out["scale"] = torch.cat([p[2] for p in parts])
        return out
    if kind == "quantize":
        return _exact_many(t["x"])
    if kind == "product":
        return _exact_many(t["a"]) @ _exact_many(t["b"]).t()
    q, b = _exact_many(t["q"]), _exact_many(t["b"])
    rows = []
    for i in range(case["nq"]):
        far = b @ q[i] if case["metric"] == "ip" else (b - q[i]).square().sum(1)
        best = torch.topk(far, case["k"], largest=case["metric"] == "ip").values
        rows.append(best)
    return torch.stack(rows), None
