"""The 4-bit and dropout entry points without a GPU: their plain numpy form against published
values and the format's own table, and every refusal of arguments (made before the device is
looked at)."""
import ctypes as C

import numpy as np
import pytest

import mxfp_ref as ref


def test_philox_known_answers():
    # the generator's published test vectors (Random123's kat_vectors, philox4x32 with 10 rounds)
    for c, k, want in [
        ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
        ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
        ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
         (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
    ]:
        assert tuple(int(v) for v in ref.philox(c, k)) == want


def test_mask_rate_and_independence():
    from paracel_amd import Dropout

    d = Dropout(0.25, seed=11, step=3, row0=1 << 33)
    k = ref.keep(2000, 1000, d)
    # 2e6 draws: three standard deviations of the mean are 0.0009
    assert abs(k.mean() - 0.75) < 1e-3
    assert abs((k[:, 1:] == k[:, :-1]).mean() - (0.75 ** 2 + 0.25 ** 2)) < 2e-3
    assert abs((k == ref.keep(2000, 1000, Dropout(0.25, 11, 4, 1 << 33))).mean() - 0.625) < 2e-3
    # rows keep their mask when a batch starts further down
    assert np.array_equal(k[500:], ref.keep(1500, 1000, Dropout(0.25, 11, 3, (1 << 33) + 500)))
    assert Dropout(0.1, 0).scale == ref.kept_scale(0.1) == 65536 / (65536 - 6554)


def test_reference_rounding():
    x = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.26, 7.9, 0.2, -4.9]])
    got = ref.rounded(x)
    # 7.9 is the block's largest: the unit is 2^0, ties go to the even code, 7.9 saturates
    assert got.tolist() == [[0, 1, 1, 2, 2, 4, 4, 6, -0.5, 6, 0, -4]]
    code, s = ref.quantize(np.array([[np.nan] + [1.0] * 40, [0.0] * 41, [2.0 ** -140] * 41]))
    assert s.tolist() == [[255, 125], [0, 0], [0, 0]]
    assert ref.quantize(np.array([[1e300]]))[1][0, 0] == 254


@pytest.fixture()
def capi():
    from paracel_amd import capi

    capi.load_library()
    return capi


P = 1 << 20  # stands for an aligned device address that no refused call may touch


def refused(what, f, *a, **k):
    from paracel_amd import PlrError

    with pytest.raises(PlrError) as e:
        f(*a, **k)
    assert e.value.code == -1 and what in str(e.value), str(e.value)


def test_pitches(capi):
    assert [capi.mxfp_code_pitch(d) for d in (1, 128, 129, 1000)] == [64, 64, 128, 512]
    assert [capi.mxfp_scale_pitch(d) for d in (1, 128, 129, 1000)] == [4, 4, 8, 32]
    assert capi.mxfp_code_pitch(0) == 0 and capi.mxfp_scale_pitch(-5) == 0


@pytest.mark.parametrize("change, what", [
    (dict(dtype=4), "unknown element type"), (dict(n=-1), "n >= 0"), (dict(d=0), "d >= 1"),
    (dict(ldx=99), "ldx"), (dict(ldc=63), "code pitch"), (dict(ldc=48), "code pitch"),
    (dict(lds=3), "scale pitch"), (dict(dx=None), "NULL"), (dict(dcodes=None), "NULL"),
    (dict(dscales=None), "NULL"), (dict(dx=P + 2), "aligned"), (dict(dcodes=P + 8), "aligned"),
    (dict(n=1 << 60), "too large"), (dict(d=1 << 35, ldx=1 << 35), "2^34"),
    (dict(n=1 << 34, transpose=True, ldc=1 << 33, lds=1 << 29), "one launch"),
    (dict(device=-1), "device_id"), (dict(device=1000), "device_id"),
])
def test_quantize_refusals(capi, change, what):
    a = dict(dx=P, dtype=1, n=5, d=100, ldx=100, dcodes=P, ldc=64, dscales=P, lds=4)
    a.update(change)
    refused(what, capi.mxfp_quantize, **a)


@pytest.mark.parametrize("rate, row0, what", [(-0.1, 0, "rate"), (1.0, 0, "rate"),
                                              (0.999999, 0, "rate"), (float("nan"), 0, "rate"),
                                              (0.5, -1, "row0")])
def test_dropout_refusals(capi, rate, row0, what):
    drop = capi.Dropout(rate, 1, 0, row0)
    refused(what, capi.dropout_apply, P, 1, 5, 100, 100, P, 100, drop)
    refused(what, capi.mxfp_quantize, P, 1, 5, 100, 100, P, 64, P, 4, drop=drop)
    refused(what, capi.mxfp_matmul, 5, 5, 100, P, 64, P, 4, P, 64, P, 4, P, 1, 5, drop=drop)


@pytest.mark.parametrize("change, what", [
    (dict(dtype=7), "unknown element type"), (dict(n=-1), "n >= 0"), (dict(d=0), "d >= 1"),
    (dict(ldo=99), "ldo"), (dict(ldx=99), "ldx"), (dict(dx=None), "NULL"), (dict(dout=None), "NULL"),
    (dict(dx=P + 2), "aligned"), (dict(dout=P + 1), "aligned"), (dict(drop=None), "drop"),
    (dict(n=1 << 60), "too large"),
])
def test_dropout_apply_refusals(capi, change, what):
    a = dict(dx=P, dtype=1, n=5, d=100, ldx=100, dout=P, ldo=100, drop=capi.Dropout(0.5, 1))
    a.update(change)
    refused(what, capi.dropout_apply, **a)


@pytest.mark.parametrize("change, what", [
    (dict(dtype=9), "unknown element type"), (dict(n=-1), "n >= 0"), (dict(d=0), "d >= 1"),
    (dict(ldo=99), "ldo"), (dict(ldc=48), "code pitch"), (dict(ldc=72), "code pitch"),
    (dict(lds=3), "scale pitch"), (dict(dout=None), "NULL"), (dict(dcodes=None), "NULL"),
    (dict(dcodes=P + 4), "aligned"), (dict(dout=P + 2), "aligned"), (dict(n=1 << 60), "too large"),
])
def test_dequantize_refusals(capi, change, what):
    a = dict(dcodes=P, ldc=64, dscales=P, lds=4, n=5, d=100, dout=P, dtype=1, ldo=100)
    a.update(change)
    refused(what, capi.mxfp_dequantize, **a)


@pytest.mark.parametrize("change, what", [
    (dict(dtype=0), "PLR_F32"), (dict(m=-1), "m >= 0"), (dict(n=-1), "n >= 0"), (dict(k=0), "k >= 1"),
    (dict(lda=48), "code pitches"), (dict(ldb=80), "code pitches"), (dict(k=129), "code pitches"),
    (dict(ldsa=6), "scale pitches"), (dict(ldsb=2), "scale pitches"), (dict(ldc=6), "ldc"),
    (dict(da=None), "NULL"), (dict(dsb=None), "NULL"), (dict(dc=None), "NULL"),
    (dict(da=P + 8), "16-byte"), (dict(dsa=P + 2), "4-byte"), (dict(dc=P + 2), "element type"),
    (dict(m=1 << 40), "2^31"), (dict(lda=1 << 62), "2^23"), (dict(k=(1 << 24) + 1), "2^24"),
    (dict(ldsb=1 << 24), "2^23"), (dict(ldc=1 << 62), "too large"),
])
def test_matmul_refusals(capi, change, what):
    a = dict(m=5, n=7, k=100, da=P, lda=64, dsa=P, ldsa=4, db=P, ldb=64, dsb=P, ldsb=4, dc=P, dtype=1,
             ldc=7)
    a.update(change)
    refused(what, capi.mxfp_matmul, **a)


def test_matmul_workspace_is_asked_for(capi):
    assert [capi.mxfp_matmul_workspace(m, n, k) for m, n, k in ((1, 1, 1), (100, 4096, 16384))] == [0, 0]
    refused("workspace", capi.mxfp_matmul, 5, 7, 100, P, 64, P, 4, P, 64, P, 4, P, 1, 7,
            workspace=P, workspace_bytes=-1)


def test_context_calls_refuse_null(capi):
    lib = capi.load_library()
    assert lib.plr_pack_data(None) == -1
    assert lib.plr_set_dropout(None, C.byref(capi.Dropout(0.5, 1))) == -1


@pytest.mark.parametrize("alpha, rate", [(1e300, 0), (-1e39, 0), (1e-40, 0), (1e-320, 0), (-1e-39, 0.5),
                                         (1e34, 65535 / 65536)])
def test_matmul_refuses_factors_that_32_bits_do_not_hold(capi, alpha, rate):
    refused("alpha", capi.mxfp_matmul, 5, 7, 100, P, 64, P, 4, P, 64, P, 4, P, 1, 7, alpha=alpha,
            drop=capi.Dropout(rate, 1))
