"""The 4-bit operators and dropout on streams of their own, from several threads at once, on skewed
pointers, and two contexts with packed shards side by side."""
import ctypes as C
import threading

import numpy as np
import pytest

import mxfp_ref as ref
from test_gpu_mxfp import _bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from paracel_amd import capi as m

    return m


class Chain:
    """x -> dropout -> 4 bits -> product with w -> dropout, on a stream that waits for no other."""

    def __init__(self, capi, m, n, k, seed):
        self.capi, self.m, self.n, self.k = capi, m, n, k
        rng = np.random.default_rng(seed)
        self.stream = C.c_void_p()
        assert ref.hip().hipStreamCreateWithFlags(C.byref(self.stream), 1) == 0
        p, q = capi.mxfp_code_pitch(k), capi.mxfp_scale_pitch(k)
        x, w = rng.normal(size=(m, k)).astype(np.float32), rng.normal(size=(n, k))
        self.p, self.q, self.drop = p, q, capi.Dropout(0.5, seed, 3)  # factor 2: exact
        self.src, self.x = ref.Dev(x), ref.Dev(np.zeros_like(x))
        self.w = [ref.Dev(t) for t in ref.pack(*ref.quantize(w), p, q)]
        self.c = [ref.Dev(np.zeros((m, s), dtype=np.uint8)) for s in (p, q)]
        self.out = ref.Dev(np.zeros((m, n), dtype=np.float32))
        keep = ref.keep(m, k, self.drop)
        va = ref.rounded(np.where(keep, x, 0).astype(np.float64) * 2)
        vb = ref.rounded(w)
        kept = ref.keep(m, n, self.drop)
        self.want = np.where(kept, 2 * (va @ vb.T), 0)
        self.bound = np.where(kept, _bound(va, vb, k, self.want, 1, 2.0), 0)

    def clear(self):
        for b in (self.x, self.out, *self.c):
            b.put(b.like)

    def run(self):
        a, st = self.capi, self.stream.value
        a.dropout_apply(self.src.ptr, 1, self.m, self.k, self.k, self.x.ptr, self.k, self.drop, stream=st)
        a.mxfp_quantize(self.x.ptr, 1, self.m, self.k, self.k, self.c[0].ptr, self.p, self.c[1].ptr, self.q,
                        stream=st)
        a.mxfp_matmul(self.m, self.n, self.k, self.c[0].ptr, self.p, self.c[1].ptr, self.q, self.w[0].ptr,
                      self.p, self.w[1].ptr, self.q, self.out.ptr, 1, self.n, 1.0, self.drop, stream=st)

    def check(self):
        assert ref.hip().hipStreamSynchronize(self.stream) == 0
        assert (np.abs(self.out.get() - self.want) <= self.bound).all()

    def close(self):
        assert ref.hip().hipStreamDestroy(self.stream) == 0


SIZES = [(3000, 260, 4000), (1, 5000, 3000), (700, 90, 9000), (500, 1025, 300)]


def test_each_on_its_own_stream(capi):
    chains = [Chain(capi, *s, i + 1) for i, s in enumerate(SIZES)]
    for _ in range(3):
        for c in chains:
            c.clear()
        for c in chains:
            c.run()
        for c in chains:
            c.check()
    for c in chains:
        c.close()


def test_threads(capi):
    chains = [Chain(capi, *s, i + 11) for i, s in enumerate(SIZES)]
    failed = []

    def work(c):
        try:
            for _ in range(5):
                c.clear()
                c.run()
                c.check()
        except BaseException as e:  # noqa: B902
            failed.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in chains]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for c in chains:
        c.close()


@pytest.mark.parametrize("m, n, k", [(1, 300, 500), (30, 200, 500), (300, 300, 300), (2200, 2300, 200)])
@pytest.mark.parametrize("dtype", [1, 2, 3])
def test_results_at_any_alignment(capi, m, n, k, dtype):
    rng = np.random.default_rng(m)
    a, b = ref.quantize(rng.normal(size=(m, k))), ref.quantize(rng.normal(size=(n, k)))
    p, q = capi.mxfp_code_pitch(k), capi.mxfp_scale_pitch(k)
    ops = [ref.Dev(t) for pair in (a, b) for t in ref.pack(*pair, p, q)]
    va, vb = ref.values(*a)[:, :k], ref.values(*b)[:, :k]
    want = va @ vb.T
    size = 4 if dtype == 1 else 2
    for skew in (size, 3 * size):
        poison = ref.store(np.full((m + 1, n + 5), 77.0), dtype)
        out = ref.Dev(poison, skew)
        capi.mxfp_matmul(m, n, k, ops[0].ptr, p, ops[1].ptr, q, ops[2].ptr, p, ops[3].ptr, q, out.ptr, dtype,
                         n + 5)
        got = out.get()
        assert (np.abs(ref.load(got[:m, :n], dtype) - want) <= _bound(va, vb, k, want, dtype)).all()
        assert np.array_equal(got[:, n:], poison[:, n:]) and np.array_equal(got[m:], poison[m:])


@pytest.mark.parametrize("dtype", range(4))
def test_values_at_any_alignment(capi, dtype):
    n, d = 70, 333
    size = (8, 4, 2, 2)[dtype]
    rng = np.random.default_rng(dtype)
    x = ref.store(rng.normal(size=(n, d)), dtype)
    v = ref.load(x, dtype).astype(np.float64)
    drop = capi.Dropout(0.5, 9)
    keep = ref.keep(n, d, drop)
    for skew in (size, 16 - size):
        dx, out = ref.Dev(x, skew), ref.Dev(np.zeros_like(x), size)
        for tr in (False, True):
            r, c = (d, n) if tr else (n, d)
            p, q = capi.mxfp_code_pitch(c), capi.mxfp_scale_pitch(c) + 1
            codes, scales = ref.Dev(np.zeros((r, p), np.uint8)), ref.Dev(np.zeros((r, q), np.uint8), 1)
            capi.mxfp_quantize(dx.ptr, dtype, n, d, d, codes.ptr, p, scales.ptr, q, transpose=tr)
            code, s = ref.quantize(v.T if tr else v)
            assert np.array_equal(codes.get(), ref.pack(code, s, p, q)[0])
            assert np.array_equal(scales.get()[:, :s.shape[1]], s)
            if not tr:
                capi.mxfp_dequantize(codes.ptr, p, scales.ptr, q, n, d, out.ptr, dtype, d)
                assert np.array_equal(ref.load(out.get(), dtype), ref.load(ref.store(ref.rounded(v), dtype), dtype))
        capi.dropout_apply(dx.ptr, dtype, n, d, d, out.ptr, d, drop)
        assert np.array_equal(ref.load(out.get(), dtype), np.where(keep, 2 * v, 0))


def test_two_contexts_at_once(oracle):
    from paracel_amd import Dropout, Plr

    jobs, failed = [], []
    for i, (n, d) in enumerate([(4000, 300), (300, 17000), (9000, 40)]):
        rng = np.random.default_rng(i)
        X, theta = rng.normal(size=(n, d)) / np.sqrt(d), rng.normal(size=d)
        y = (rng.random(n) < 0.5) * 1.0
        drop = Dropout(0.5, 100 + i, i)
        D = np.where(ref.keep(n, d, drop), 2 * ref.rounded(X), 0)
        jobs.append((X, y, theta, drop, oracle.gsum(D, y, theta), oracle.gsum(ref.rounded(X), y, theta)))

    def work(job):
        X, y, theta, drop, dropped, whole = job
        try:
            with Plr(0) as p:
                p.set_data(X, y)
                p.pack_data()
                for _ in range(10):
                    for dr, want in ((drop, dropped), (None, whole)):
                        p.set_dropout(dr)
                        g = p.loss_grad(theta)[0]
                        assert np.linalg.norm(g - want) <= 1e-11 * np.linalg.norm(want)
        except BaseException as e:  # noqa: B902
            failed.append(e)

    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
