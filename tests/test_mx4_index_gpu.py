"""Flat indexes that store microscaled 4-bit rows: search against a 64-bit statement on the rounded vectors.

Rows and queries are normal values: blocks have scales of 2^-3 .. 2^0, products are multiples of 2^-8 and sums stay
below |q| |x| < 2^13 for d <= 4096, so every fp32 sum is exact and distances and labels have to be equal."""
import os
import subprocess

import numpy as np
import pytest
import torch

import row_reference as ref

pytestmark = pytest.mark.gpu


def rounded(x):
    c, s = ref.mx4_encode(np.asarray(x, np.float64))
    return ref.mx4_values(c, s, x.shape[1])


def expected(b, metric, vb, vq, k, keep=None, labels=None):
    """(D, I) by key and position; rows that are no numbers, or filtered out, do not appear."""
    score = vq @ vb.T
    if metric == b.METRIC_L2:
        key = (vb * vb).sum(1)[None, :] - 2 * score
    else:
        key = -score
    ok = np.isfinite(key)
    if keep is not None:
        ok &= keep
    n, nq = vb.shape[0], vq.shape[0]
    D = np.full((nq, k), np.float32(3.402823466e+38), np.float32)
    I = np.full((nq, k), -1, np.int64)
    labels = np.arange(n) if labels is None else labels
    for q in range(nq):
        order = np.argsort(np.where(ok[q], key[q], np.inf), kind="stable")[:min(k, int(ok[q].sum()))]
        d = key[q][order] + (vq[q] * vq[q]).sum() if metric == b.METRIC_L2 else -key[q][order]
        D[q, :len(order)], I[q, :len(order)] = d, labels[order]
    return D, I


def check(got, want):
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[0], want[0])


def data(seed, n, nq, d):
    rng = np.random.default_rng(seed)
    return rng.standard_normal((n, d)).astype(np.float32), rng.standard_normal((nq, d)).astype(np.float32)


@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("n, nq, d, k", [(1, 1, 16, 1), (5, 3, 32, 8), (255, 1, 48, 10), (257, 130, 128, 5), (1000, 7, 256, 100),
                                         (20000, 1, 128, 10), (30000, 129, 64, 10), (3000, 20, 1024, 50), (700, 3, 4096, 20),
                                         (70000, 33, 96, 1), (9000, 5, 272, 1000), (200000, 65, 128, 100),
                                         (3000, 260, 2048, 10), (66000, 300, 512, 7), (40000, 1, 1040, 3)])
def test_search(b200, n, nq, d, k, metric):
    x, q = data(n + d, n, nq, d)
    ix = b200.IndexFlat(d, metric, b200.MX4)
    cut = n // 3
    if cut:
        ix.add(x[:cut])
    ix.add(x[cut:])
    assert ix.ntotal == n
    vb = rounded(x)
    np.testing.assert_array_equal(ix.get_base(), vb.astype(np.float32))
    check(ix.search(q, k), expected(b200, metric, vb, rounded(q), k))


def test_rows_and_queries_on_the_device(b200):
    x, q = data(1, 5000, 9, 160)
    a, c = b200.IndexFlat(160, dtype=b200.MX4), b200.IndexFlat(160, dtype=b200.MX4)
    a.add(x)
    xd, qd = torch.from_numpy(x).cuda(), torch.from_numpy(q).cuda()
    D, I = torch.empty(9, 30, device="cuda"), torch.empty(9, 30, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    ids = np.arange(5000, dtype=np.int64) * 3 + 7
    c.add_device(xd.data_ptr(), 5000, ids)
    c.search_device(qd.data_ptr(), 9, 30, D.data_ptr(), I.data_ptr())
    Dr, Ir = a.search(q, 30)
    check((D.cpu().numpy(), I.cpu().numpy()), (Dr, Ir * 3 + 7))
    np.testing.assert_array_equal(c.get_ids(), ids)


@pytest.mark.parametrize("metric", [0, 1])
def test_ties_go_to_the_lower_position(b200, metric):
    """A few distinct rows, each many times: candidate lists overflow and every query is searched again."""
    x, q = data(2, 8, 40, 64)
    x = np.tile(x, (5000, 1))
    ix = b200.IndexFlat(64, metric, b200.MX4)
    ix.add(x)
    check(ix.search(q, 20), expected(b200, metric, rounded(x), rounded(q), 20))


@pytest.mark.parametrize("metric", [0, 1])
def test_masks(b200, metric):
    x, q = data(3, 6000, 11, 128)
    ix = b200.IndexFlat(128, metric, b200.MX4)
    ix.add(x)
    rng = np.random.default_rng(0)
    keep = rng.random((11, 6000)) < 0.3
    keep[4] = False          # leaves nothing
    keep[5] = False
    keep[5, 5999] = True
    got = ix.search_with_masks(q, 15, np.packbits(keep, axis=1, bitorder="little"))
    check(got, expected(b200, metric, rounded(x), rounded(q), 15, keep))


@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("n, nq, d, k", [(140001, 16, 48, 10), (140001, 17, 32, 200), (140001, 64, 80, 3), (133000, 128, 64, 20),
                                         (30011, 2, 2064, 10), (30000, 40, 2064, 10)])
def test_few_queries_over_many_rows(b200, n, nq, d, k, metric):
    """Thresholds and two stretches of the base; rows that are no numbers; a filter; the same index twice in a row."""
    x, q = data(n + nq, n, nq, d)
    x[5, 0], x[n - 1, d - 1] = np.nan, np.inf
    q[nq - 1] = 0.0
    ix = b200.IndexFlat(d, metric, b200.MX4)
    ix.add(x)
    vb, vq = rounded(x), rounded(q)
    want = expected(b200, metric, vb, vq, k)
    check(ix.search(q, k), want)
    check(ix.search(q, k), want)
    rng = np.random.default_rng(n)
    keep = rng.random((nq, n)) < 0.6
    keep[0] = False
    keep[0, n - 2] = True
    check(ix.search_with_masks(q, k, np.packbits(keep, axis=1, bitorder="little")), expected(b200, metric, vb, vq, k, keep))


@pytest.mark.parametrize("metric", [0, 1])
def test_rows_that_are_no_numbers(b200, metric):
    x, q = data(4, 300, 5, 96)
    x[7, 3], x[299, 95], x[100] = np.nan, np.inf, -np.inf
    q[2, 40] = np.nan
    ix = b200.IndexFlat(96, metric, b200.MX4)
    ix.add(x)
    check(ix.search(q, 300), expected(b200, metric, rounded(x), rounded(q), 300))
    vb = rounded(x)
    np.testing.assert_array_equal(ix.get_base(), vb.astype(np.float32))


def test_remove_reset_and_add_again(b200):
    x, q = data(5, 1500, 6, 144)
    ix = b200.IndexFlat(144, b200.METRIC_L2, b200.MX4)
    ix.add(x)
    gone = [0, 1, 130, 131, 700, 1499]
    assert ix.remove_ids(gone + [99999]) == len(gone)
    order = list(range(1500))
    for p in sorted(gone, reverse=True):       # the last row takes the removed one's place
        order[p] = order[-1]
        order.pop()
    vb = rounded(x[order])
    np.testing.assert_array_equal(ix.get_base(), vb.astype(np.float32))
    check(ix.search(q, 40), expected(b200, b200.METRIC_L2, vb, rounded(q), 40, labels=np.array(order)))
    ix.reset()
    D, I = ix.search(q, 2)
    assert ix.ntotal == 0 and (I == -1).all()
    ix.add(x[:10])
    check(ix.search(q, 12), expected(b200, b200.METRIC_L2, rounded(x[:10]), rounded(q), 12))


def test_save_and_load(b200, tmp_path):
    x, q = data(6, 777, 4, 80)
    x[5, 2] = np.nan
    x[6] = 0
    ix = b200.IndexFlat(80, b200.METRIC_INNER_PRODUCT, b200.MX4)
    ix.add_with_ids(x, np.arange(777)[::-1])
    path = str(tmp_path / "mx4.b2ix")
    ix.save(path)
    again = b200.load_index(path)
    assert again.dtype == b200.MX4
    np.testing.assert_array_equal(again.get_base().view(np.uint32), ix.get_base().view(np.uint32))
    np.testing.assert_array_equal(again.get_ids(), ix.get_ids())
    check(again.search(q, 33), ix.search(q, 33))
    again.add(x[:3])
    assert again.ntotal == 780


def test_several_indexes_together(b200):
    parts, q = [data(10 + i, 400 + 50 * i, 1, 64)[0] for i in range(3)], data(9, 1, 7, 64)[1]
    ixs = []
    base = 0
    for p in parts:
        ix = b200.IndexFlat(64, b200.METRIC_L2, b200.MX4)
        ix.add_with_ids(p, base + np.arange(len(p)))
        base += len(p)
        ixs.append(ix)
    check(b200.search_multi(ixs, q, 25), expected(b200, b200.METRIC_L2, rounded(np.concatenate(parts)), rounded(q), 25))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("n, nq, d, ldo", [(1, 1, 16, 0), (3001, 5, 96, 3008), (700, 200, 1024, 0), (20000, 300, 64, 0)])
def test_scores(b200, n, nq, d, ldo, dtype):
    x, q = data(30, n, nq, d)
    ix = b200.IndexFlat(d, b200.METRIC_L2, b200.MX4)
    ix.add(x)
    qd = torch.from_numpy(q).cuda()
    out = torch.full((nq, ldo or n), -1.0, dtype=ref.TORCH[dtype], device="cuda")
    torch.cuda.synchronize()
    ix.scores_device(qd.data_ptr(), nq, dtype, out.data_ptr(), ldo)
    want = torch.from_numpy(rounded(q) @ rounded(x).T).to(ref.TORCH[dtype])
    assert torch.equal(out[:, :n].cpu(), want) and bool((out[:, n:] == -1.0).all())
    check(ix.search(q, 4), expected(b200, b200.METRIC_L2, rounded(x), rounded(q), 4))   # (the scratch is shared)


def test_refusals(b200):
    ix = b200.IndexFlat(64, b200.METRIC_L2, b200.MX4)
    x = np.zeros((2, 64), np.float32)
    ix.add(x)
    for call in (lambda: ix.add_f16(np.zeros((1, 64), np.uint16)), lambda: ix.search_f16(np.zeros((1, 64), np.uint16), 1),
                 lambda: b200.IndexFlat(64, b200.METRIC_L2, b200.BF16), lambda: b200.IndexFlat(50, b200.METRIC_L2, b200.MX4),
                 lambda: b200.IndexFlat(64, b200.METRIC_INT8_COSINE, b200.MX4)):
        with pytest.raises(b200.B200IdxError) as e:
            call()
        assert e.value.code == 2001
    d = torch.zeros(2, 64, device="cuda")
    for bad in (dict(n=0), dict(x_ptr=0), dict(dtype=b200.MX4), dict(out_ptr=0), dict(ldo=1)):
        with pytest.raises(b200.B200IdxError) as e:
            ix.scores_device(**dict(dict(x_ptr=d.data_ptr(), n=2, dtype=b200.F32, out_ptr=d.data_ptr()), **bad))
        assert e.value.code == 2001
    with pytest.raises(b200.B200IdxError) as e:
        b200.IndexFlat(64).scores_device(d.data_ptr(), 2, b200.F32, d.data_ptr())
    assert e.value.code == 2001 and "MX4" in e.value.msg
    D, I = torch.empty(2, 1, device="cuda"), torch.empty(2, 1, dtype=torch.int64, device="cuda")
    with pytest.raises(b200.B200IdxError) as e:
        ix.search_device_noalloc(d.data_ptr(), 2, 1, D.data_ptr(), I.data_ptr())
    assert e.value.code == 2001 and "MX4" in e.value.msg


def test_lists_that_come_short(b200, tmp_path):
    """Up to 128 queries, thresholds and candidates come from two kernels, which need not round alike."""
    from indexsdk_b200 import build
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    objects = [os.path.join(build.BUILD_DIR, s[:-3] + ".o") for s in build.SOURCES]
    if not all(map(os.path.exists, objects)):
        build.build(force=True)
    exe = str(tmp_path / "test_short_lists")
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-I", os.path.join(root, "include"), "-I", "/usr/local/cuda/include",
                    os.path.join(root, "tests", "cpp", "test_short_lists.cpp"), *objects, "-o", exe,
                    "-Wl,--wrap=_ZN4b20020launch_kth_thresholdEPKjiiiiPKfjPjRKNS_7TauFoldEP11CUstream_st",
                    "-L/usr/local/cuda/lib64", "-lcudart_static", "-lpthread", "-ldl", "-lrt"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "0 failed" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("n, nq, d, k", [(30000, 1, 128, 1), (30000, 64, 128, 20), (9000, 128, 1024, 100), (140001, 16, 64, 10),
                                         (30000, 129, 256, 20)])
def test_sums_that_round(b200, n, nq, d, k, metric):
    """Scales spread over 2^24 in rows and in queries: fp32 holds no sum exactly.  A key is off by at most
    2 eps d sum |q| |x| (half a step each of at most 2 d additions and cuts, relative to the largest partial sum), for L2
    twice that and the roundings of two norms and two additions; so is the j-th smallest of the keys against the j-th
    smallest of the exact ones, and so is the key of the row that a label names."""
    rng = np.random.default_rng(n + d)

    def wide(rows):
        c, s = rng.integers(0, 16, (rows, d)), rng.integers(-12, 12, (rows, d // 32))
        v = ref.MAGNITUDES[c & 7] * np.where(c & 8, -1.0, 1.0)
        v[:, ::32] = 6.0   # (a block that holds its largest value keeps its scale)
        return (v.reshape(rows, -1, 32) * np.exp2(s)[:, :, None]).reshape(rows, d)

    x, q = wide(n), wide(nq)
    ix = b200.IndexFlat(d, metric, b200.MX4)
    ix.add(x.astype(np.float32))
    np.testing.assert_array_equal(ix.get_base(), x)
    D, I = ix.search(q.astype(np.float32), k)
    assert I.min() >= 0 and all(len(set(r)) == k for r in I.tolist())
    exact = ((q * q).sum(1)[:, None] + (x * x).sum(1) - 2 * q @ x.T) if metric == b200.METRIC_L2 else q @ x.T
    bound = 2 * ref.EPS[0] * d * (np.abs(q) @ np.abs(x).T)
    if metric == b200.METRIC_L2:
        bound = 2 * bound + ref.EPS[0] * (d / 8 + 8) * ((q * q).sum(1)[:, None] + (x * x).sum(1))
    worst = bound.max(1, keepdims=True)
    best = np.sort(exact, 1)[:, :k] if metric == b200.METRIC_L2 else -np.sort(-exact, 1)[:, :k]
    assert (np.abs(D - best) <= worst).all()
    assert (np.abs(np.take_along_axis(exact, I, 1) - D) <= np.take_along_axis(bound, I, 1)).all()
    step = np.diff(D, axis=1) if metric == b200.METRIC_L2 else -np.diff(D, axis=1)
    assert (step >= 0).all()


def test_save_and_load_keeps_norms(b200, tmp_path):
    """L2 distances of a loaded index, bit for bit: norms are sums that round here."""
    rng = np.random.default_rng(7)
    n, d = 700, 528
    x = (rng.standard_normal((n, d)) * np.exp2(rng.integers(-12, 12, (n, d // 16))).repeat(16, 1)).astype(np.float32)
    ix = b200.IndexFlat(d, b200.METRIC_L2, b200.MX4)
    ix.add(x)
    path = str(tmp_path / "mx4.b2ix")
    ix.save(path)
    again = b200.load_index(path)
    for q in (x[:5], np.zeros((1, d), np.float32)):   # (distances from 0 are the norms themselves)
        check(again.search(q, n), ix.search(q, n))


# ---- hidden states into an Int8Flat index ----
@pytest.mark.parametrize("metric, static", [(0, True), (1, True), (2, False), (2, True)])
@pytest.mark.parametrize("residual", [False, True])
def test_states_into_int8flat(b200, metric, static, residual):
    """The states calls are the operator followed by add and search."""
    rng = np.random.default_rng(20)
    n, nq, d, k = 3000, 17, 192, 12
    mk = lambda r: torch.from_numpy(rng.standard_normal((r, d))).to("cuda", torch.bfloat16)  # noqa: E731
    x, q, w = mk(n), mk(nq), mk(1).view(-1)
    rx, rq = (mk(n), mk(nq)) if residual else (None, None)
    s = torch.tensor([0.03], device="cuda") if static else None
    sp = s.data_ptr() if static else 0
    ix = b200.IndexInt8Flat(d, metric)
    D, I = torch.empty(nq, k, device="cuda"), torch.empty(nq, k, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    ids = np.arange(n, dtype=np.int64) + 5
    for lo, hi in ((0, 1001), (1001, n)):
        ix.add_states_device(hi - lo, b200.BF16, x[lo:hi].data_ptr(), w.data_ptr(), 1e-5, static_scale_ptr=sp, ids=ids[lo:hi],
                             residual_ptr=rx[lo:hi].data_ptr() if residual else 0)
    ix.search_states_device(nq, b200.BF16, q.data_ptr(), w.data_ptr(), 1e-5, k, D.data_ptr(), I.data_ptr(),
                            residual_ptr=rq.data_ptr() if residual else 0, static_scale_ptr=sp)

    def rows(t, r):
        out = torch.empty(t.shape, dtype=torch.int8, device="cuda")
        sc = torch.empty(t.shape[0], device="cuda")
        b200.rms_norm_i8_device(t.shape[0], d, b200.BF16, t.data_ptr(), w.data_ptr(), 1e-5, out.data_ptr(),
                                residual_ptr=r.data_ptr() if residual else 0, static_scale_ptr=sp,
                                scales_ptr=0 if static else sc.data_ptr())
        return out.cpu().numpy()

    plain = b200.IndexInt8Flat(d, metric)
    plain.add_with_ids(rows(x, rx), ids)
    np.testing.assert_array_equal(ix.get_base(), plain.get_base())
    np.testing.assert_array_equal(ix.get_ids(), ids)
    Dr, Ir = plain.search(rows(q, rq), k)
    np.testing.assert_array_equal(I.cpu().numpy(), Ir)
    np.testing.assert_array_equal(D.cpu().numpy(), Dr)


def test_states_refusals(b200):
    x = torch.zeros(4, 64, device="cuda")
    D, I = torch.empty(4, 1, device="cuda"), torch.empty(4, 1, dtype=torch.int64, device="cuda")
    s = torch.ones(1, device="cuda")
    ip = b200.IndexInt8Flat(64, b200.METRIC_INNER_PRODUCT)
    ok = dict(n=4, dtype=b200.F32, x_ptr=x.data_ptr(), weight_ptr=x.data_ptr(), eps=1e-6)
    for bad, text in ((dict(), "static_scale"), (dict(n=0), "n must"), (dict(dtype=9), "dtype"), (dict(eps=0.0), "eps"),
                      (dict(x_ptr=0), "Invalid x"), (dict(weight_ptr=0), "Invalid weight")):
        a = dict(ok, **bad)
        for call in (lambda: ip.add_states_device(**a, static_scale_ptr=s.data_ptr() if bad else 0),
                     lambda: ip.search_states_device(**a, k=1, D_ptr=D.data_ptr(), I_ptr=I.data_ptr(),
                                                     static_scale_ptr=s.data_ptr() if bad else 0)):
            with pytest.raises(b200.B200IdxError) as e:
                call()
            assert e.value.code == 2001 and text in e.value.msg
    with pytest.raises(b200.B200IdxError):
        ip.search_states_device(**ok, k=0, D_ptr=D.data_ptr(), I_ptr=I.data_ptr(), static_scale_ptr=s.data_ptr())
    lib = b200.load()
    fl = b200.IndexFlat(64)
    assert lib.b200idx_add_states_device(fl.handle, 4, 0, x.data_ptr(), 0, x.data_ptr(), 1e-6, s.data_ptr(), None) == 2001
    assert ip.ntotal == 0
