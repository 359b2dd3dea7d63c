"""The 4-bit operators and dropout on the GPU against their plain numpy form in 64 bits: codes and
masks bit for bit, products and rounded results within bounds derived beside each check; then a
run of them as a training step uses them, gradients against differences, and graph replays."""
import ctypes as C

import numpy as np
import pytest

import mxfp_ref as ref

pytestmark = pytest.mark.gpu

NAMES = ["f64", "f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def capi():
    from paracel_amd import capi

    capi.load_library()
    return capi


def features(rng, n, d):
    """Rows and columns of different sizes, zeros among them."""
    x = rng.normal(size=(n, d)) * 2.0 ** rng.integers(-6, 7, size=(n, 1))
    return x * (rng.random((n, d)) > 0.1) * 2.0 ** rng.integers(-2, 3, size=(1, d))


def padded(x, ld, fill):
    out = np.full((x.shape[0], ld), fill, dtype=x.dtype)
    out[:, :x.shape[1]] = x
    return out


def device_codes(capi, x, dtype, transpose=False, drop=None, ldx=None, skew=0, ldc=None, lds=None):
    """Quantise on the device; returns (codes, scales) with the pitches asked for, poisoned before."""
    n, d = x.shape
    rows, cols = (d, n) if transpose else (n, d)
    ldx = ldx or d
    ldc = ldc or capi.mxfp_code_pitch(max(cols, 1))
    lds = lds or capi.mxfp_scale_pitch(max(cols, 1))
    dx = ref.Dev(padded(x, ldx, x.dtype.type(1) if dtype != 2 else np.uint16(0x7FC0)), skew)
    codes = ref.Dev(np.full((rows + 1, ldc), 0xEE, dtype=np.uint8))
    scales = ref.Dev(np.full((rows + 1, lds), 0xDD, dtype=np.uint8))
    capi.mxfp_quantize(dx.ptr, dtype, n, d, ldx, codes.ptr, ldc, scales.ptr, lds, transpose, drop)
    return codes.get(), scales.get()


SHAPES = [(1, 1), (1, 2048), (3, 7), (5, 31), (5, 32), (4, 33), (130, 100), (33, 129), (64, 128),
          (257, 520), (1000, 41), (31, 4100), (0, 64)]


@pytest.mark.parametrize("n, d", SHAPES)
@pytest.mark.parametrize("dtype", range(4), ids=NAMES)
@pytest.mark.parametrize("transpose", [False, True], ids=["rows", "columns"])
def test_quantize(capi, n, d, dtype, transpose):
    rng = np.random.default_rng(n * 7919 + d)
    x = ref.store(features(rng, n, d), dtype)
    v = ref.load(x, dtype)
    for drop in (None, capi.Dropout(0.3, 0x123456789ABCDEF, 7, 1 << 33)):
        w = np.where(ref.keep(n, d, drop), v, 0.0)
        code, s = ref.quantize(w.T if transpose else w)
        for ldx, skew in ((d, 0), (d + 3, 0 if dtype == 0 else [8, 4, 2, 2][dtype])):
            got = device_codes(capi, x, dtype, transpose, drop, ldx, skew)
            rows, cols = (d, n) if transpose else (n, d)
            if n == 0:
                assert (got[0] == 0xEE).all()
                continue
            want = ref.pack(code, s, got[0].shape[1], got[1].shape[1])
            # a code of minus zero stands for the value plus zero does
            same = lambda a: np.where((a & 0x0F) == 8, a & 0xF0, a)  # noqa: E731
            same2 = lambda a: np.where((a & 0xF0) == 0x80, a & 0x0F, a)  # noqa: E731
            assert np.array_equal(same2(same(got[0][:rows])), same2(same(want[0])))
            assert np.array_equal(got[1][:rows], want[1])
            # the row behind the last one is left as it was
            assert (got[0][rows:] == 0xEE).all() and (got[1][rows:] == 0xDD).all()


@pytest.mark.parametrize("transpose", [False, True], ids=["rows", "columns"])
def test_quantize_pitches(capi, transpose):
    # the narrowest pitches there are (a shard's), and wide ones whose rest is left alone
    rng = np.random.default_rng(5)
    x = ref.store(features(rng, 70, 70), 1)
    v = ref.load(x, 1)
    code, s = ref.quantize(v.T if transpose else v)
    for ldc, lds in ((48, 3), (64, 4), (64, 5), (192, 11)):
        codes, scales = device_codes(capi, x, 1, transpose, ldc=ldc, lds=lds)
        want = ref.pack(code, s, ldc, lds)
        w, q = min(ldc, 64), min(lds, 4)
        assert np.array_equal(codes[:70, :w], want[0][:, :w]) and (codes[:, w:] == 0xEE).all()
        assert np.array_equal(scales[:70, :q], want[1][:, :q]) and (scales[:, q:] == 0xDD).all()


@pytest.mark.parametrize("dtype", range(4), ids=NAMES)
def test_quantize_edges(capi, dtype):
    # ties in both directions, saturation, zeros, the type's largest and smallest, NaN, infinities
    tiny = [2.0 ** -1074, 2.0 ** -149, 2.0 ** -133, 2.0 ** -24][dtype]
    big = [np.finfo(np.float64).max, np.finfo(np.float32).max, 3.3895313892515355e38, 65504.0][dtype]
    rows = [np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -5.0, 4.0] * 3)[:32],
            np.full(32, tiny), np.r_[big, np.full(31, tiny)], np.r_[-big, np.zeros(31)],
            np.zeros(32), -np.zeros(32), np.r_[np.nan, np.ones(31)], np.r_[np.ones(31), np.inf],
            np.r_[np.ones(31), -np.inf], np.r_[2.0 ** -14, np.full(31, 2.0 ** -16)],
            np.linspace(-8, 8, 32)]
    if dtype == 0:  # a double next to a tie must not round to the tie first
        rows.append(np.r_[6.0, np.full(10, 0.25 * (1 + 2.0 ** -50)), np.full(10, 2.5 * (1 - 2.0 ** -50)),
                          np.full(11, 3.5 * (1 - 2.0 ** -52))])
    x = ref.store(np.array(rows), dtype)
    v = ref.load(x, dtype)
    code, s = ref.quantize(v)
    codes, scales = device_codes(capi, x, dtype)
    assert np.array_equal(scales[:len(rows), :1], s)
    got = np.stack([codes[:len(rows), :16] & 15, codes[:len(rows), :16] >> 4], -1).reshape(len(rows), 32)
    ok = s[:, 0] != 255
    assert np.array_equal(ref.values(got, s)[ok], ref.values(code, s)[ok])
    codes, scales = device_codes(capi, np.ascontiguousarray(x.T), dtype, True)
    assert np.array_equal(scales[:len(rows), :1], s)
    # and back: NaN throughout where the block was not finite
    for out in range(4):
        _check_dequantize(capi, got, s, 32, out)


def _check_dequantize(capi, code, s, d, dtype, ldo=None, skew=0):
    n = code.shape[0]
    ldo = ldo or d
    c, q = ref.pack(code, s, capi.mxfp_code_pitch(d), capi.mxfp_scale_pitch(d))
    dc, dq = ref.Dev(c), ref.Dev(q)
    poison = ref.store(np.full((n + 1, ldo), 77.0), dtype)
    out = ref.Dev(poison, skew)
    capi.mxfp_dequantize(dc.ptr, c.shape[1], dq.ptr, q.shape[1], n, d, out.ptr, dtype, ldo)
    got = out.get()
    # the values are exact in 64 bits: one rounding to the type
    want = ref.store(ref.values(code, s)[:, :d], dtype)
    assert np.array_equal(ref.load(got[:n, :d], dtype), ref.load(want, dtype), equal_nan=True)
    assert np.array_equal(got[n:], poison[n:]) and np.array_equal(got[:n, d:], poison[:n, d:])


@pytest.mark.parametrize("n, d", SHAPES)
@pytest.mark.parametrize("dtype", range(4), ids=NAMES)
def test_dequantize(capi, n, d, dtype):
    rng = np.random.default_rng(d)
    code, s = ref.quantize(features(rng, n, d))
    _check_dequantize(capi, code, s, d, dtype)
    _check_dequantize(capi, code, s, d, dtype, d + 5, [8, 4, 2, 2][dtype])


@pytest.mark.parametrize("n, d", SHAPES)
@pytest.mark.parametrize("dtype", range(4), ids=NAMES)
def test_dropout(capi, n, d, dtype):
    rng = np.random.default_rng(d + 1)
    x = ref.store(rng.normal(size=(n, d)), dtype)
    v = ref.load(x, dtype)
    size = [8, 4, 2, 2][dtype]
    for rate in (0.0, 0.1, 0.5, 65535 / 65536):
        drop = capi.Dropout(rate, 0xFEDCBA9876543210, 0xFFFFFFFF, 5)
        k = ref.keep(n, d, drop)
        for ldx, ldo, skew in ((d, d, 0), (d + 1, d + 6, size)):
            dx = ref.Dev(padded(x, ldx, x.dtype.type(3)), skew)
            poison = ref.store(np.full((n + 1, ldo), 77.0), dtype)
            out = ref.Dev(poison, skew)
            capi.dropout_apply(dx.ptr, dtype, n, d, ldx, out.ptr, ldo, drop)
            got = out.get()
            g, want = ref.load(got[:n, :d], dtype), v * ref.kept_scale(rate)
            assert (g[~k] == 0).all()
            # the factor and the product are rounded to the working type (at most 2^-24 each in
            # 32 bits, 2^-53 in 64), then the result to the element type
            work = 2.0 ** -53 if dtype == 0 else 2.0 ** -24
            tol = (1 + ref.HALF_STEP[dtype]) * (1 + work) ** 2 - 1
            fine = np.abs(want) < (6e4 if dtype == 3 else 1e300)
            assert (np.abs(g - want) <= tol * np.abs(want) + 2.0 ** -25)[k & fine].all()
            assert np.array_equal(got[n:], poison[n:]) and np.array_equal(got[:n, d:], poison[:n, d:])


def test_dropout_in_place_and_of_nan(capi):
    x = np.full((40, 100), np.nan, dtype=np.float32)
    drop = capi.Dropout(0.5, 3)
    dx = ref.Dev(x)
    capi.dropout_apply(dx.ptr, 1, 40, 100, 100, dx.ptr, 100, drop)
    got, k = dx.get(), ref.keep(40, 100, drop)
    assert (got[~k] == 0).all() and np.isnan(got[k]).all()


# -- the product -------------------------------------------------------------------------------
MATMULS = [(1, 1, 1), (1, 1, 128), (1, 300, 1000), (2, 17, 129), (3, 64, 2048), (16, 16, 128),
           (15, 33, 100), (17, 129, 257), (33, 1000, 4100), (64, 64, 512), (65, 63, 130),
           (128, 256, 1000), (255, 257, 384), (300, 520, 777), (512, 512, 1024), (1, 5000, 8192),
           (1000, 1, 300), (7, 9, 16500), (256, 768, 640), (513, 1025, 2100),
           (4100, 2200, 300), (2049, 4097, 129), (5000, 20, 300), (40, 9000, 260),
           (50, 8200, 640), (20000, 50, 513), (64, 64, 128), (17, 4000, 2000),
           (4100, 4100, 200), (4097, 3900, 300), (1100, 2300, 500), (70, 4000, 1000), (500, 500, 4000)]


def _matmul(capi, a, b, k, dtype, alpha=1.0, drop=None, pad=0, ldc=None, poison=77.0, more=0):
    """a, b: (codes, scales) in whole blocks.  `pad`: extra chunks of pitch, filled with NaN scales
    and codes that must not be read."""
    m, n = a[0].shape[0], b[0].shape[0]
    p, q = capi.mxfp_code_pitch(k), capi.mxfp_scale_pitch(k)
    dev = []
    for code, s in (a, b):
        c, t = ref.pack(code, s, p + 64 * pad, q + 4 * pad)
        c[:, p:], t[:, q:] = 0x77, 255
        dev += [ref.Dev(c), ref.Dev(t)]
    ldc = ldc or n
    out = ref.Dev(ref.store(np.full((m + 1, ldc), poison), dtype))
    size = capi.mxfp_matmul_workspace(m, n, k) + more
    space = ref.Dev(np.full(max(size, 1), 0xA5, dtype=np.uint8))
    capi.mxfp_matmul(m, n, k, dev[0].ptr, p + 64 * pad, dev[1].ptr, q + 4 * pad, dev[2].ptr,
                     p + 64 * pad, dev[3].ptr, q + 4 * pad, out.ptr, dtype, ldc, alpha, drop,
                     space.ptr, size)
    got = out.get()
    assert np.array_equal(got[m:], ref.store(np.full((1, ldc), poison), dtype))
    assert np.array_equal(got[:m, n:], ref.store(np.full((m, ldc - n), poison), dtype))
    return ref.load(got[:m, :n], dtype)


def _bound(va, vb, k, want, dtype, factor=1.0):
    """Products of two 4-bit values are exact.  The 128 of an instruction meet in a tree of 7
    levels and join the running sum, one addition per chunk; work split along k joins its parts in
    at most 64 more; each addition is off by at most one step, 2^-23, of the sum of magnitudes.
    Two roundings of 2^-24 for the factors, one half step of the result's type."""
    mag = factor * (np.abs(va) @ np.abs(vb).T)
    adds = (k + 127) // 128 + 8 + 64
    least = [0, 2.0 ** -149, 2.0 ** -133, 2.0 ** -24][dtype]
    return adds * 2.0 ** -23 * mag + (ref.HALF_STEP[dtype] + 2.0 ** -23) * np.abs(want) + least


@pytest.mark.parametrize("m, n, k", MATMULS)
@pytest.mark.parametrize("dtype", [1, 2, 3], ids=NAMES[1:])
def test_matmul(capi, m, n, k, dtype):
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    a, b = ref.quantize(features(rng, m, k) / 16), ref.quantize(rng.normal(size=(n, k)) / 16)
    va, vb = ref.values(*a)[:, :k], ref.values(*b)[:, :k]
    want = 0.5 * (va @ vb.T)
    got = _matmul(capi, a, b, k, dtype, 0.5, pad=1, ldc=n + 3)
    assert (np.abs(got - want) <= _bound(va, vb, k, want, dtype, 0.5)).all()
    # aligned rows of the result
    got2 = _matmul(capi, a, b, k, dtype, 0.5, ldc=-(-n // 8) * 8)
    assert np.array_equal(got, got2)
    # dropout of the result
    drop = capi.Dropout(0.4, 99, 2, 77)
    keep = ref.keep(m, n, drop)
    got = _matmul(capi, a, b, k, dtype, 0.5, drop, ldc=n + 3)
    assert (got[~keep] == 0).all()
    want = want * ref.kept_scale(0.4)
    assert (np.abs(got - want) <= _bound(va, vb, k, want, dtype, 0.5 * ref.kept_scale(0.4)))[keep].all()


@pytest.mark.parametrize("m, n, k", [(1, 40, 300), (20, 70, 1000), (300, 300, 600)])
def test_matmul_extremes(capi, m, n, k):
    # scales far apart within a row, a block of NaN, rows of zeros
    rng = np.random.default_rng(3)
    x, y = rng.normal(size=(m, k)), rng.normal(size=(n, k))
    x *= 2.0 ** rng.integers(-50, 50, size=(m, -(-k // 32))).repeat(32, 1)[:, :k]
    x[m // 2] = 0
    y[n // 3, 40] = np.nan
    a, b = ref.quantize(x), ref.quantize(y)
    va, vb = ref.values(*a)[:, :k], ref.values(*b)[:, :k]
    got = _matmul(capi, a, b, k, 1)
    nan = np.isnan(got)
    assert nan[:, n // 3].all() and nan.sum() == m
    vb[n // 3] = 0
    want = va @ vb.T
    assert (np.abs(got - want) <= _bound(va, vb, k, want, 1))[~nan].all()
    assert (got[m // 2][~nan[m // 2]] == 0).all()


def test_matmul_empty(capi):
    lib = capi.load_library()
    assert lib.plr_last_error(None) is not None
    capi.mxfp_matmul(0, 5, 100, None, 64, None, 4, None, 64, None, 4, None, 1, 5)
    capi.mxfp_matmul(5, 0, 100, None, 64, None, 4, None, 64, None, 4, None, 1, 5)


def test_matmul_is_reproducible(capi):
    rng = np.random.default_rng(8)
    for m, n, k in ((1, 700, 8000), (40, 500, 9000), (600, 600, 1500)):
        a, b = ref.quantize(rng.normal(size=(m, k))), ref.quantize(rng.normal(size=(n, k)))
        first = _matmul(capi, a, b, k, 1)
        assert np.array_equal(first, _matmul(capi, a, b, k, 1, more=4096))


# -- together: a linear layer with dropout, forward and backward --------------------------------
def _layer(capi, x, w, dz, drop):
    """z, dx, dw of z = drop(x) w^T through the operators, f32 in and out, operands quantised."""
    n, d = x.shape
    o = w.shape[0]
    up = drop.scale if drop else 1.0

    def q(v, transpose=False, dr=None):
        rows, cols = v.shape[::-1] if transpose else v.shape
        dv = ref.Dev(v)
        c = ref.Dev(np.empty((rows, capi.mxfp_code_pitch(cols)), dtype=np.uint8))
        s = ref.Dev(np.empty((rows, capi.mxfp_scale_pitch(cols)), dtype=np.uint8))
        capi.mxfp_quantize(dv.ptr, 1, *v.shape, v.shape[1], c.ptr, c.like.shape[1], s.ptr,
                           s.like.shape[1], transpose, dr)
        assert ref.hip().hipDeviceSynchronize() == 0
        return c, s

    def mul(a, b, k, alpha=1.0, dr=None):
        m, n2 = a[0].like.shape[0], b[0].like.shape[0]
        out = ref.Dev(np.empty((m, n2), dtype=np.float32))
        size = capi.mxfp_matmul_workspace(m, n2, k)
        space = ref.Dev(np.empty(max(size, 1), dtype=np.uint8))
        capi.mxfp_matmul(m, n2, k, a[0].ptr, a[0].like.shape[1], a[1].ptr, a[1].like.shape[1], b[0].ptr,
                         b[0].like.shape[1], b[1].ptr, b[1].like.shape[1], out.ptr, 1, n2, alpha, dr,
                         space.ptr, size)
        return out.get().astype(np.float64)

    z = mul(q(x, dr=drop), q(w), d, up)
    dx = mul(q(dz), q(w, True), o, 1.0, drop)
    dw = mul(q(dz, True), q(x, True, drop), n, up)
    return z, dx, dw


@pytest.mark.parametrize("n, d, o", [(40, 70, 33), (300, 257, 130), (129, 1000, 64)])
@pytest.mark.parametrize("rate", [0.0, 0.25])
def test_layer_matches_plain(capi, n, d, o, rate):
    rng = np.random.default_rng(n)
    drop = capi.Dropout(rate, 5, 6, 7) if rate else None
    x, w, dz = (rng.normal(size=s).astype(np.float32) for s in ((n, d), (o, d), (n, o)))
    up, k = (ref.kept_scale(rate), ref.keep(n, d, drop)) if rate else (1.0, np.ones((n, d)))
    z, dx, dw = _layer(capi, x, w, dz, drop)
    for got, a, b, f, mask in ((z, x * k, w, up, 1), (dx, dz, w.T, up, k), (dw, dz.T, (x * k).T, up, 1)):
        va, vb = ref.rounded(a), ref.rounded(b)
        want = f * (va @ vb.T) * mask
        assert (np.abs(got - want) <= _bound(va, vb, a.shape[1], want, 1, f)).all()


def test_layer_gradient_against_differences(capi):
    # values that 4 bits hold exactly in either orientation (so quantisation is the identity):
    # L = sum(dz * z) is bilinear, and a difference over one entry IS the derivative
    rng = np.random.default_rng(12)
    n, d, o = 50, 40, 35
    x, w, dz = (rng.choice([-3.0, -2, -1, 1, 2, 3], size=s).astype(np.float32)
                for s in ((n, d), (o, d), (n, o)))
    for v in (x, w, dz):  # every block's largest is 4: the unit is the same everywhere
        v[::8, :], v[:, ::8] = 4.0, 4.0
    drop = capi.Dropout(0.5, 21)  # factor 2: exact
    z, dx, dw = _layer(capi, x, w, dz, drop)
    loss = lambda xx, ww: float((_layer(capi, xx, ww, dz, drop)[0] * dz).sum())  # noqa: E731
    base = loss(x, w)
    for i, j in [(1, 1), (3, 9), (17, 33), (49, 39)]:
        x2 = x.copy()
        x2[i, j] -= 1 if x2[i, j] > -3 else -1
        assert (loss(x2, w) - base) / (x2[i, j] - x[i, j]) == dx[i, j]
    for i, j in [(1, 1), (9, 3), (34, 39)]:
        w2 = w.copy()
        w2[i, j] -= 1 if w2[i, j] > -3 else -1
        assert (loss(x, w2) - base) / (w2[i, j] - w[i, j]) == dw[i, j]


# -- streams and graphs -------------------------------------------------------------------------
def test_graph_replays(capi):
    """Quantise, multiply and drop on a captured stream of its own; two graphs with workspaces of
    their own, replayed in turn with eager work between them, give the eager bits every time."""
    h = ref.hip()
    rng = np.random.default_rng(4)
    stream = C.c_void_p()
    assert h.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    drop = capi.Dropout(0.2, 8)

    class Case:
        def __init__(self, m, n, k):
            self.m, self.n, self.k = m, n, k
            self.x, self.w = ref.Dev(rng.normal(size=(m, k))), ref.Dev(rng.normal(size=(n, k)))
            p, q = capi.mxfp_code_pitch(k), capi.mxfp_scale_pitch(k)
            self.p, self.q = p, q
            e = lambda *s: ref.Dev(np.zeros(s, dtype=np.uint8))  # noqa: E731
            self.c = [e(m, p), e(m, q), e(n, p), e(n, q)]
            self.out = ref.Dev(np.zeros((m, n), dtype=np.float32))
            self.size = capi.mxfp_matmul_workspace(m, n, k)
            self.space = e(max(self.size, 1))

        def run(self):
            m, n, k, c, st = self.m, self.n, self.k, self.c, stream.value
            capi.mxfp_quantize(self.x.ptr, 0, m, k, k, c[0].ptr, self.p, c[1].ptr, self.q, drop=drop,
                               stream=st)
            capi.mxfp_quantize(self.w.ptr, 0, n, k, k, c[2].ptr, self.p, c[3].ptr, self.q, stream=st)
            capi.mxfp_matmul(m, n, k, c[0].ptr, self.p, c[1].ptr, self.q, c[2].ptr, self.p, c[3].ptr,
                             self.q, self.out.ptr, 1, n, 1.0, drop, self.space.ptr, self.size, stream=st)
            capi.dropout_apply(self.out.ptr, 1, m, n, n, self.out.ptr, n, drop, stream=st)

    cases, graphs = [Case(1, 3000, 8192), Case(300, 500, 700)], []
    for c in cases:
        c.run()
        assert h.hipStreamSynchronize(stream) == 0
        c.want = c.out.get()
        g, x = C.c_void_p(), C.c_void_p()
        assert h.hipStreamBeginCapture(stream, 0) == 0
        try:
            c.run()
        finally:
            rc = h.hipStreamEndCapture(stream, C.byref(g))
        assert rc == 0 and h.hipGraphInstantiate(C.byref(x), g, None, None, 0) == 0
        graphs.append((g, x))
    for replay in range(4):
        for c, (g, x) in zip(cases, graphs):
            c.out.put(np.full((c.m, c.n), np.nan, dtype=np.float32))
        for c, (g, x) in zip(cases, graphs):
            assert h.hipGraphLaunch(x, stream) == 0
        assert h.hipStreamSynchronize(stream) == 0
        for c in cases:
            assert np.array_equal(c.out.get(), c.want), "replay %d" % replay
        cases[replay % 2].run()
        assert h.hipStreamSynchronize(stream) == 0
    for g, x in graphs:
        assert h.hipGraphExecDestroy(x) == 0 and h.hipGraphDestroy(g) == 0
    assert h.hipStreamDestroy(stream) == 0
