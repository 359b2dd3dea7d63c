"""The product's tiles over many steps of k, its strips beside a multiple of the tile, and the
transposed quantiser's own rounding.  PATHS is chosen by which kernels a product of these sizes is
cut into on a device of 256 compute units; test_host_side.py checks without a GPU that every
kernel of the product is reached by it and by test_gpu_mxfp.MATMULS."""
import numpy as np
import pytest

import mxfp_ref as ref
from test_gpu_mxfp import NAMES, _bound, _check_dequantize, _matmul, device_codes, features

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from paracel_amd import capi

    capi.load_library()
    return capi


# m, n, k, type.  Steps of 128 along k: 13 to 17 and more, so that the ring of four stages, the
# groups of four steps with every remainder and the ring of three groups of scales are gone round.
PATHS = [
    (2300, 4090, 1800, 1),  # tiles of 256 x 256, ragged; 15 steps
    (4094, 4138, 1750, 2),  # ... and a strip of 42 columns; 14
    (4120, 4093, 2000, 3),  # ... and of 24 rows; 16
    (4140, 4120, 2100, 2),  # ... and both; 17
    (2000, 4060, 2700, 2),  # tiles of 128 x 256; 22
    (4100, 2048, 2690, 1),  # ... and a strip of 4 rows; 22
    (1063, 1021, 2031, 3),  # tiles of 128 x 128; 16
    (1545, 2546, 1596, 2),  # ... and a strip of 9 rows; 13
    (2995, 1312, 1953, 1),  # ... and of 32 columns; 16
    # few rows on one side, and small products, in the kernels' other forms
    (700, 9, 2100, 2), (30, 9000, 300, 3), (9000, 30, 300, 1), (9000, 40, 260, 2), (600, 500, 1500, 3),
]


@pytest.mark.parametrize("m, n, k, dtype", PATHS)
def test_matmul_paths(capi, m, n, k, dtype):
    rng = np.random.default_rng(m + n + k)
    a, b = ref.quantize(features(rng, m, k) / 16), ref.quantize(rng.normal(size=(n, k)) / 16)
    va, vb = ref.values(*a)[:, :k], ref.values(*b)[:, :k]
    want = 0.75 * (va @ vb.T)
    bound = _bound(va, vb, k, want, dtype, 0.75)
    got = _matmul(capi, a, b, k, dtype, 0.75, pad=1, ldc=n + 3)
    assert (np.abs(got - want) <= bound).all()
    # the mask of the result: rows and columns of the strips are those of the whole
    drop = capi.Dropout(0.5, 0x1234567887654321, 5, (1 << 32) - 1000)  # factor 2: exact
    keep = ref.keep(m, n, drop)
    got = _matmul(capi, a, b, k, dtype, 0.75, drop, ldc=-(-n // 8) * 8)
    assert (got[~keep] == 0).all()
    # twice the value, and twice its bound but for the type's smallest step, which is in it once
    assert (np.abs(got - 2 * want) <= 2 * bound)[keep].all()


@pytest.mark.parametrize("dtype", range(4), ids=NAMES)
def test_quantize_edges_along_columns(capi, dtype):
    # the values of test_quantize_edges as columns of x: every one of them passes through the columns
    # that are taken 16 bytes at a time and through the ones behind the last whole 16 bytes, in a
    # whole block of 32 rows in front of one that ends early
    tiny = [2.0 ** -1074, 2.0 ** -149, 2.0 ** -133, 2.0 ** -24][dtype]
    big = [np.finfo(np.float64).max, np.finfo(np.float32).max, 3.3895313892515355e38, 65504.0][dtype]
    cols = [np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -5.0, 4.0] * 3)[:32],
            np.full(32, tiny), np.r_[big, np.full(31, tiny)], np.r_[-big, np.zeros(31)],
            np.zeros(32), -np.zeros(32), np.r_[np.nan, np.ones(31)], np.r_[np.ones(31), np.inf],
            np.r_[np.ones(31), -np.inf], np.r_[2.0 ** -14, np.full(31, 2.0 ** -16)],
            np.linspace(-8, 8, 32)]
    if dtype == 0:
        cols.append(np.r_[6.0, np.full(10, 0.25 * (1 + 2.0 ** -50)), np.full(10, 2.5 * (1 - 2.0 ** -50)),
                          np.full(11, 3.5 * (1 - 2.0 ** -52))])
    v = 16 // [8, 4, 2, 2][dtype]
    while len(cols) % v != v - 1:
        cols.append(np.full(32, 1.5))
    cols = [np.r_[c, c[:5]] for c in cols]
    for turn in range(len(cols)):
        x = ref.store(np.array(cols[turn:] + cols[:turn]).T, dtype)
        for drop in (None, capi.Dropout(0.5, turn)):
            w = np.where(ref.keep(*x.shape, drop), ref.load(x, dtype), 0.0)
            _same_codes(device_codes(capi, x, dtype, True, drop), *ref.quantize(w.T))


def _same_codes(got, code, s):
    want = ref.pack(code, s, got[0].shape[1], got[1].shape[1])
    n = code.shape[0]

    def plus(a):  # a code of minus zero stands for the value plus zero does
        a = np.where((a & 0x0F) == 8, a & 0xF0, a)
        return np.where((a & 0xF0) == 0x80, a & 0x0F, a)

    assert np.array_equal(got[1][:n], want[1])
    assert np.array_equal(plus(got[0][:n]), plus(want[0]))


def test_factor_of_a_dropped_product(capi):
    # 2^-30 times these sums is below the smallest normal number of 32 bits, times the mask's
    # factor it is not: the two are joined before the sum is rounded.  Everything is exact.
    drop = capi.Dropout(1 - 2.0 ** -8, 3, 1, 9)  # factor 256
    for m, n, k in ((16, 20000, 64), (30, 9000, 64), (500, 600, 64), (1063, 1021, 2031), (2300, 4090, 1800)):
        x, y = np.zeros((m, k)), np.zeros((n, k))
        x[:, 0], y[:, 0] = 2.0 ** -50, 2.0 ** -50
        x[:, 32], y[:, 32] = 2.0 ** -60, 2.0 ** -61
        got = _matmul(capi, ref.quantize(x), ref.quantize(y), k, 1, 2.0 ** -30, drop)
        keep = ref.keep(m, n, drop)
        assert keep.any()
        assert (got == np.where(keep, 2.0 ** -122 + 2.0 ** -143, 0)).all()


@pytest.mark.parametrize("dtype", range(4), ids=NAMES)
@pytest.mark.parametrize("transpose", [False, True], ids=["rows", "columns"])
def test_quantize_far_from_one(capi, dtype, transpose):
    # magnitudes over the type's whole range, its subnormal numbers and scales of 0 and 254 among them
    rng = np.random.default_rng(dtype)
    low, high = [(-140, 135), (-140, 127), (-140, 127), (-24, 15)][dtype]
    e = np.arange(low, high + 1)
    x = rng.integers(1, 256, size=(e.size, 37)) / 256.0 * rng.choice([-1, 1], size=(e.size, 37))
    with np.errstate(over="ignore"):
        x = ref.store(np.ldexp(x, e[:, None] + 1), dtype)
    v = ref.load(x, dtype)
    assert np.isfinite(v).all()
    if transpose:
        x = np.ascontiguousarray(x.T)
    _same_codes(device_codes(capi, x, dtype, transpose), *ref.quantize(v))


@pytest.mark.parametrize("dtype", range(4), ids=NAMES)
def test_every_code_under_every_scale(capi, dtype):
    s = np.arange(256, dtype=np.uint8)[:, None]
    code = np.tile(np.r_[np.arange(16), np.arange(16)[::-1]].astype(np.uint8), (256, 1))
    with np.errstate(over="ignore"):
        _check_dequantize(capi, code, s, 32, dtype)


@pytest.mark.parametrize("m, n, k", [(1, 300, 200), (40, 70, 1000), (300, 300, 600), (1063, 1021, 2031)])
def test_matmul_of_scales_at_both_ends(capi, m, n, k):
    # 2^-127 times 2^127, the smallest scale and the largest: exact sums of small whole numbers
    rng = np.random.default_rng(k)
    x, y = rng.integers(-3, 4, size=(m, k)) * 1.0, rng.integers(-3, 4, size=(n, k)) * 1.0
    a, b = (_codes_of(v) for v in (x, y))
    low = rng.integers(0, 255, size=a[1].shape[1])
    low[:2] = 0, 254
    a = (a[0], np.tile(low.astype(np.uint8), (m, 1)))
    b = (b[0], np.tile((254 - low).astype(np.uint8), (n, 1)))
    got = _matmul(capi, a, b, k, 1)
    assert (got == x @ y.T).all()


def _codes_of(v):
    """Codes of whole numbers from -3 to 3, whatever the scale, in whole blocks."""
    code = np.array([0, 2, 4, 5], dtype=np.uint8)[np.abs(v).astype(int)] | (v < 0).astype(np.uint8) << 3
    out = np.zeros((v.shape[0], -(-v.shape[1] // 32) * 32), dtype=np.uint8)
    out[:, :v.shape[1]] = code
    return out, np.zeros((v.shape[0], out.shape[1] // 32), dtype=np.uint8)
