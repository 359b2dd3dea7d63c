"""Matrices whose offsets pass 32 bits, in elements and in bytes: the rows at their far end hold
values, the rest zeros, and what is written there is checked against the plain definitions."""
import ctypes as C

import numpy as np
import pytest

import mxfp_ref as ref
from test_gpu_mxfp import _bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from paracel_amd import capi as m

    return m


class Big:
    """Zeroed device memory, read and written in pieces."""

    def __init__(self, nbytes):
        self.p, self.nbytes = C.c_void_p(), nbytes
        assert ref.hip().hipMalloc(C.byref(self.p), nbytes) == 0
        assert ref.hip().hipMemset(self.p, 0, C.c_size_t(nbytes)) == 0
        self.ptr = self.p.value

    def put(self, at, a):
        a = np.ascontiguousarray(a)
        assert 0 <= at and at + a.nbytes <= self.nbytes
        assert ref.hip().hipMemcpy(self.ptr + at, a.ctypes.data, a.nbytes, 1) == 0

    def get(self, at, shape, dtype):
        a = np.empty(shape, dtype=dtype)
        assert 0 <= at and at + a.nbytes <= self.nbytes
        assert ref.hip().hipDeviceSynchronize() == 0
        assert ref.hip().hipMemcpy(a.ctypes.data, self.ptr + at, a.nbytes, 2) == 0
        return a

    def __del__(self):
        if self.p.value:
            ref.hip().hipFree(self.p)
            self.p = C.c_void_p()


def test_quantise_dequantise_and_drop(capi):
    n, d, tail = 280001, 32768, 40  # 9.2e9 values: 18 GB, 4.6 GB of codes
    row = 2 * d
    rng = np.random.default_rng(0)
    x = ref.store(rng.normal(size=(tail, d)), 2)
    v = ref.load(x, 2)
    dx = Big(n * row)
    dx.put((n - tail) * row, x)
    p, q = capi.mxfp_code_pitch(d), capi.mxfp_scale_pitch(d)
    codes, scales = Big(n * p), Big(n * q)
    drop = capi.Dropout(0.3, 5, 1, 1 << 40)
    keep = ref.keep(tail, d, capi.Dropout(0.3, 5, 1, (1 << 40) + n - tail))
    for dr, want in ((None, v), (drop, np.where(keep, v, 0.0))):
        capi.mxfp_quantize(dx.ptr, 2, n, d, d, codes.ptr, p, scales.ptr, q, drop=dr)
        c, s = ref.pack(*ref.quantize(want), p, q)
        assert np.array_equal(codes.get((n - tail) * p, (tail, p), np.uint8), c)
        assert np.array_equal(scales.get((n - tail) * q, (tail, q), np.uint8), s)
        assert not codes.get((n - tail - 9) * p, (9, p), np.uint8).any()
    out = Big(n * d * 4)
    capi.mxfp_dequantize(codes.ptr, p, scales.ptr, q, n, d, out.ptr, 1, d)
    assert np.array_equal(out.get((n - tail) * d * 4, (tail, d), np.float32), ref.rounded(np.where(keep, v, 0.0)))
    del out, codes, scales
    # the transpose: 32768 rows of 280001 columns; the last 41 rows of x end the last 3 blocks
    p, q = capi.mxfp_code_pitch(n), capi.mxfp_scale_pitch(n)
    codes, scales = Big(d * p), Big(d * q)
    first = (n - tail) // 32 * 32
    capi.mxfp_quantize(dx.ptr, 2, n, d, d, codes.ptr, p, scales.ptr, q, transpose=True, drop=drop)
    full = np.zeros((n - first, d))
    full[first - n:][n - tail - first:] = np.where(keep, v, 0.0)
    code, s = ref.quantize(full.T)
    blocks = s.shape[1]
    c, s = ref.pack(code, s, 16 * blocks, blocks)
    for j in (0, 7, d // 2, d - 8, d - 1):
        assert np.array_equal(codes.get(j * p + first // 2, (16 * blocks,), np.uint8), c[j])
        assert np.array_equal(scales.get(j * q + first // 32, (blocks,), np.uint8), s[j])
    del codes, scales
    capi.dropout_apply(dx.ptr, 2, n, d, d, dx.ptr, d, drop)
    got = ref.load(dx.get((n - tail) * row, (tail, d), np.uint16), 2)
    want = v * keep * ref.kept_scale(0.3)
    assert (got[~keep] == 0).all()
    # a float's rounding of the factor and of the product, then to bfloat16
    assert (np.abs(got - want) <= np.abs(want) * (2.0 ** -8 + 2.0 ** -22)).all()


@pytest.mark.parametrize("n", [5, 300])
def test_product_of_rows_far_apart(capi, n):
    m, k, lda, ldsa = 600, 300, 1 << 23, 1 << 23  # 5 GB of codes, 5 GB of scales
    rng = np.random.default_rng(n)
    a, b = ref.quantize(rng.normal(size=(m, k))), ref.quantize(rng.normal(size=(n, k)))
    p, q = capi.mxfp_code_pitch(k), capi.mxfp_scale_pitch(k)
    ca, sa = ref.pack(*a, p, q)
    cb, sb = (ref.Dev(t) for t in ref.pack(*b, p, q))
    da, ds = Big(m * lda), Big(m * ldsa)
    for i in range(m):
        da.put(i * lda, ca[i])
        ds.put(i * ldsa, sa[i])
    va, vb = ref.values(*a)[:, :k], ref.values(*b)[:, :k]
    for swap in (False, True):
        r, t = (n, m) if swap else (m, n)
        out = ref.Dev(np.zeros((r, t), dtype=np.float32))
        one, two = (da.ptr, lda, ds.ptr, ldsa), (cb.ptr, p, sb.ptr, q)
        capi.mxfp_matmul(r, t, k, *(two + one if swap else one + two), out.ptr, 1, t)
        want = (vb @ va.T) if swap else va @ vb.T
        bound = _bound(vb, va, k, want, 1) if swap else _bound(va, vb, k, want, 1)
        assert (np.abs(out.get() - want) <= bound).all()


@pytest.mark.parametrize("m, n", [(70001, 70000), (3, 9000000), (9000000, 3)])
def test_product_large_result(capi, m, n):
    # 4.9e9 results of bfloat16; or one side of 9e6 rows at a pitch of 512 bytes
    k, tail = 100, 30
    long_side = max(m, n) > 1000000
    p, q = 512 if long_side else capi.mxfp_code_pitch(k), capi.mxfp_scale_pitch(k)
    rng = np.random.default_rng(1)
    ops, vals = [], []
    for rows in (m, n):
        last = min(rows, tail)
        code, s = ref.quantize(rng.normal(size=(last, k)))
        c, t = ref.pack(code, s, p, q)
        dc, ds = Big(rows * p), Big(rows * q)
        dc.put((rows - last) * p, c)
        ds.put((rows - last) * q, t)
        ops += [dc, ds]
        vals.append(ref.values(code, s)[:, :k])
    ldc = n if n > 3 else 600  # rows of the result far apart
    out = Big(m * ldc * 2)
    drop = capi.Dropout(0.25, 7, 2, 5)
    for dr in (None, drop):
        capi.mxfp_matmul(m, n, k, ops[0].ptr, p, ops[1].ptr, q, ops[2].ptr, p, ops[3].ptr, q, out.ptr, 2, ldc,
                         1.0, dr)
        rows, cols = vals[0].shape[0], vals[1].shape[0]
        want = vals[0] @ vals[1].T
        f = 1.0
        if dr:
            col0 = n - cols
            first = col0 // 8 * 8
            # the mask of the last columns: eight at a time, so its words start at a multiple of 8
            keep = _keep_columns(rows, first, n, capi.Dropout(0.25, 7, 2, 5 + m - rows))[:, col0 - first:]
            f = ref.kept_scale(0.25)
            want = want * keep * f
        bound = _bound(*vals, k, want, 2, f)
        for i in range(rows):
            at = ((m - rows + i) * ldc + n - cols) * 2
            got = ref.load(out.get(at, (cols,), np.uint16), 2)
            assert (np.abs(got - want[i]) <= bound[i]).all()
            if dr:
                assert (got[~keep[i]] == 0).all()


def _keep_columns(n, c0, c1, drop):
    """Columns c0 .. c1 of the mask, by the generator itself: word j % 8 of counter j / 8."""
    rows = drop.row0 + np.arange(n, dtype=np.uint64)[:, None]
    groups = np.arange(c0 // 8, -(-c1 // 8), dtype=np.uint64)[None, :]
    low = np.uint64(0xFFFFFFFF)
    ctr = [np.broadcast_to(v, (n, groups.shape[1])) for v in
           (groups & low, rows & low, rows >> np.uint64(32), np.full((1, 1), drop.step, np.uint64))]
    words = ref.philox(ctr, (drop.seed & 0xFFFFFFFF, drop.seed >> 32))
    parts = []
    for w in words:
        w = np.asarray(w, dtype=np.uint64)
        parts += [w & np.uint64(0xFFFF), w >> np.uint64(16) & np.uint64(0xFFFF)]
    return np.stack(parts, -1).reshape(n, -1)[:, :c1 - c0] >= ref.threshold(drop.rate)


def test_more_rows_than_a_launch_holds(capi):
    # 300 million rows of two values
    n, d, tail = 300000001, 2, 1000
    rng = np.random.default_rng(4)
    x = rng.normal(size=(tail, d)).astype(np.float32)
    drop = capi.Dropout(0.5, 9, 2, 1 << 33)
    keep = ref.keep(tail, d, capi.Dropout(0.5, 9, 2, (1 << 33) + n - tail))
    dx = Big(n * d * 4)
    dx.put((n - tail) * d * 4, x)
    codes, scales = Big(n * 16), Big(n)
    capi.mxfp_quantize(dx.ptr, 1, n, d, d, codes.ptr, 16, scales.ptr, 1, drop=drop)
    want = np.where(keep, x, 0).astype(np.float64)
    c, s = ref.quantize(want)
    assert np.array_equal(codes.get((n - tail) * 16, (tail, 16), np.uint8), ref.pack(c, s, 16, 1)[0])
    assert np.array_equal(scales.get(n - tail, (tail, 1), np.uint8), s)
    capi.dropout_apply(dx.ptr, 1, n, d, d, dx.ptr, d, drop)
    assert np.array_equal(dx.get((n - tail) * d * 4, (tail, d), np.float32), 2 * want.astype(np.float32))
    capi.mxfp_dequantize(codes.ptr, 16, scales.ptr, 1, n, d, dx.ptr, 1, d)
    assert np.array_equal(dx.get((n - tail) * d * 4, (tail, d), np.float32), ref.rounded(want))


@pytest.mark.parametrize("swap", [False, True])
def test_product_of_more_rows_than_the_few_rows_kernel_takes(capi, swap):
    many, few, k, tail = 140000003, 3, 8, 500
    rng = np.random.default_rng(5)
    a, b = ref.quantize(rng.normal(size=(tail, k))), ref.quantize(rng.normal(size=(few, k)))
    da, ds, out = Big(many * 64), Big(many * 4), Big(many * few * 4)
    for big, part, size in zip((da, ds), ref.pack(*a, 64, 4), (64, 4)):
        big.put((many - tail) * size, part)
    cb, sb = (ref.Dev(t) for t in ref.pack(*b, 64, 4))
    va, vb = ref.values(*a)[:, :k], ref.values(*b)[:, :k]
    one, two = (da.ptr, 64, ds.ptr, 4), (cb.ptr, 64, sb.ptr, 4)
    bound = _bound(va, vb, k, va @ vb.T, 1)
    if swap:
        capi.mxfp_matmul(few, many, k, *two, *one, out.ptr, 1, many)
        got = np.stack([out.get((i * many + many - tail) * 4, (tail,), np.float32) for i in range(few)], 1)
    else:
        capi.mxfp_matmul(many, few, k, *one, *two, out.ptr, 1, few)
        got = out.get((many - tail) * few * 4, (tail, few), np.float32)
    assert (np.abs(got - va @ vb.T) <= bound).all()


def test_shard(plr):
    # 2.2e6 x 4096: 4.8 GB of codes, 72 GB before them; every 20000 rows repeat, so sums are known
    from paracel_amd import Dropout

    piece, times, d = 20000, 110, 4096
    rng = np.random.default_rng(2)
    X, theta = rng.random((piece, d)) - 0.5, rng.normal(size=d) / 8
    y = (rng.random(piece) < 0.5) * 1.0
    plr.set_data(X, y)
    plr.pack_data()
    plr.set_dropout(None)
    base = plr.loss_grad(theta)
    linear = plr.predict_linear(theta)
    drop = Dropout(0.5, 3, 1, (1 << 32) - piece)
    grad, loss = 0, 0
    for i in range(times):
        plr.set_dropout(Dropout(0.5, 3, 1, (1 << 32) - piece + i * piece))
        g, l, _ = plr.loss_grad(theta)
        grad, loss = grad + g, loss + l
    plr.set_dropout(None)
    plr.alloc_data(piece * times, d)
    for i in range(times):
        plr.set_data_chunk(i * piece, X, y)
    plr.pack_data()
    g, l, n = plr.loss_grad(theta)
    assert n == piece * times

    def same(a, b):
        # every sum of up to 2.2e6 terms that change sign is off by at most its terms' magnitudes
        # times 2^-52 times the additions along one chain of partial sums
        assert np.abs(a - b).max() <= 1e-10 * np.abs(b).max()

    same(g, base[0] * times)
    same(np.array([l]), np.array([base[1] * times]))
    same(plr.predict_linear(theta)[-piece:], linear)
    assert np.array_equal(plr.get_data(piece * times - 5, 5)[0], ref.rounded(X[-5:]))
    plr.set_dropout(drop)
    g, l, _ = plr.loss_grad(theta)
    same(g, grad)
    same(np.array([l]), np.array([loss]))


@pytest.mark.parametrize("n, d", [(40000003, 2), (9000001, 40), (3000001, 70)])
def test_narrow_shards(plr, n, d):
    # rows of the narrow layouts are packed in pieces of 256 MB; a pattern of 1000 rows repeats
    rng = np.random.default_rng(d)
    P, theta = rng.normal(size=(1000, d)), rng.normal(size=d)
    y = (rng.random(1000) < 0.5) * 1.0
    plr.alloc_data(n, d)
    step = 3000000
    for r in range(0, n, step):  # (a multiple of the pattern)
        m = min(step, n - r)
        plr.set_data_chunk(r, np.resize(P, (m, d)), np.resize(y, m))
    plr.pack_data()
    Q = ref.rounded(P)
    for at in (0, 16777000, 16777216, 8388000, n - 1000, 838860):
        if at + 1000 <= n:
            assert np.array_equal(plr.get_data(at, 1000)[0], np.roll(Q, -(at % 1000), axis=0))
    times = np.bincount(np.arange(1000), minlength=1000) * (n // 1000) + (np.arange(1000) < n % 1000)
    z = Q @ theta
    h = 1 / (1 + np.exp(-z))
    want = ((h - y) * times) @ Q
    loss = -(np.where(y == 1, np.log(h), np.log(1 - h)) * times).sum()
    g, l, rows = plr.loss_grad(theta)
    assert rows == n and abs(l - loss) <= 1e-10 * abs(loss)
    # the terms of a column's sum change sign: off by at most their magnitudes times 2^-52 times
    # the additions along one chain of partial sums, here counted as 2000
    most = (np.abs((h - y) * times)) @ np.abs(Q)
    assert (np.abs(g - want) <= 2000 * 2.0 ** -52 * most).all()
