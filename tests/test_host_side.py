"""The library's host side on a runtime without a device (hip_stub.cpp): calls that overlap, calls
that fail half way, and what is launched.  Each check runs in a process of its own, which loads the
stand-in in place of the HIP runtime."""
import os
import subprocess
import sys
import textwrap

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

PRELUDE = """
import ctypes as C, sys, threading
stub = C.CDLL({stub!r}, mode=C.RTLD_GLOBAL)
stub.stub_launch.restype = stub.stub_kernel.restype = C.c_char_p
for f in (stub.stub_calls, stub.stub_live, stub.stub_launches, stub.stub_kernels):
    f.restype = C.c_long
for f in (stub.stub_launch, stub.stub_kernel, stub.stub_fail_at):
    f.argtypes = [C.c_long]
sys.path[:0] = [{root!r}, {here!r}]
import numpy as np
from paracel_amd import Plr, PlrError, capi
capi.load_library()
P = 1 << 20  # stands for an aligned device address

def launches():
    out = [stub.stub_launch(i).decode() for i in range(stub.stub_launches())]
    stub.stub_clear()
    return out
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("stub") / "hip_stub.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                    "-I", os.path.join(ROCM, "include"), "-Wl,-soname,libamdhip64.so.7", "-o", so,
                    os.path.join(HERE, "hip_stub.cpp")], check=True)

    def run(body):
        code = PRELUDE.format(stub=so, root=os.path.dirname(HERE), here=HERE) + textwrap.dedent(body)
        r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=110)
        assert r.returncode == 0, r.stdout + r.stderr
        return r.stdout

    return run


def test_each_thread_reads_its_own_failure(check):
    check("""
        wrong = []

        def work(what, f, *a):
            for _ in range(4000):
                try:
                    f(*a)
                except PlrError as e:
                    if what not in str(e):
                        wrong.append((what, str(e)))

        jobs = [("unknown element type", capi.mxfp_quantize, P, 9, 5, 100, 100, P, 64, P, 4),
                ("drop must not be NULL", capi.dropout_apply, P, 1, 5, 100, 100, P, 100, None),
                ("ldo must be", capi.mxfp_dequantize, P, 64, P, 4, 5, 100, P, 1, 99),
                ("exceeds", capi.loss_grad_noalloc, P, P, 4, 100, 1 << 20, P, P)]
        threads = [threading.Thread(target=work, args=j) for j in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong, (len(wrong), wrong[0])
    """)


def test_a_failure_in_another_thread_is_still_told(check):
    # a thread without a failure of its own reads the process's last one
    check("""
        def fail():
            try:
                Plr(99)
            except PlrError:
                pass

        t = threading.Thread(target=fail)
        t.start()
        t.join()
        assert "device_id out of range" in capi.load_library().plr_last_error(None).decode()
    """)


@pytest.mark.parametrize("n, d, first", [(50, 100, 0), (40, 20, 0), (60, 70, 0), (30, 16400, 0), (20, 20000, 0),
                                         (33, 258, 1), (0, 40, 0)])
def test_packing_that_fails_leaves_the_shard(check, n, d, first):
    check(f"""
        n, d = {n}, {d}
        X, y, theta = np.ones((n, d)), np.zeros(n), np.ones(d)
        k = 0
        while True:
            k += 1
            p = Plr(0)
            p.set_option("first_column_is_one", {first})
            p.set_data(X, y)
            info = p.kernel_info()
            stub.stub_fail_at(k)
            try:
                p.pack_data()
                done = stub.stub_calls() < k
            except PlrError as e:
                done = False
                assert e.code in (-2, -3) and "out of memory" in str(e), (e.code, str(e))
                stub.stub_fail_at(0)
                # the doubles are resident as before, and pack when asked again
                assert p.kernel_info() == info, (k, p.kernel_info())
                rows, cols = C.c_int64(), C.c_int64()
                p._lib.plr_get_shape(p._h, C.byref(rows), C.byref(cols))
                assert (rows.value, cols.value) == (n, d)
                p.loss_grad(theta)
                p.pack_data()
            stub.stub_fail_at(0)
            assert "4-bit" in p.kernel_info()
            p.loss_grad(theta)
            p.close()
            assert stub.stub_live() == 0, (k, stub.stub_live())
            if done:
                break
        assert k > 5
    """)


def test_the_widest_rows(check):
    # the first sweep takes a row in pieces of 128 blocks, a workgroup down the grid to each
    check("""
        most = 65535 * 128 * 32
        p = Plr(0)
        p.alloc_data(1, most + 1)
        info = p.kernel_info()
        try:
            p.pack_data()
            assert False, p.kernel_info()
        except PlrError as e:
            assert e.code == -5 and str(most) in str(e), str(e)
        assert p.kernel_info() == info
        p.close()
        p = Plr(0)
        p.alloc_data(1, most)
        p.pack_data()
        p.calc_loss(np.zeros(most))
        assert any("packed_pass" in l and " 65535 " in l for l in launches())
    """)


def test_an_error_left_behind_is_not_the_calls_own(check):
    # the caller's earlier failure (600: an event that was not ready) is still its thread's last error
    check("""
        drop = capi.Dropout(0.5, 1)
        for call in (lambda: capi.mxfp_quantize(P, 1, 5, 100, 100, P, 64, P, 4),
                     lambda: capi.mxfp_dequantize(P, 64, P, 4, 5, 100, P, 1, 100),
                     lambda: capi.dropout_apply(P, 1, 5, 100, 100, P, 100, drop),
                     lambda: capi.mxfp_matmul(5, 7, 100, P, 64, P, 4, P, 64, P, 4, P, 1, 7)):
            stub.stub_error(600)
            call()
            assert len(launches()) == 1
    """)


def test_the_products_tested_reach_every_kernel(check):
    # the shapes of the GPU tests: every kernel of the product that the library has (in one of its
    # three result types, with and without dropout; a shape is tested both ways), every size of
    # tile over long k with rows or with columns over, and groups of four steps with every remainder
    check("""
        import test_gpu_mxfp, test_gpu_mxfp_paths
        reached, over, steps = set(), set(), {}
        short = lambda k: k.split("matmul_")[1].split(">")[0].replace("<bfloat16, false, ", "<")
        for m, n, k in test_gpu_mxfp.MATMULS + [c[:3] for c in test_gpu_mxfp_paths.PATHS]:
            p, q = capi.mxfp_code_pitch(k), capi.mxfp_scale_pitch(k)
            capi.mxfp_matmul(m, n, k, P, p, P, q, P, p, P, q, P, 2, n)
            got = [short(l) for l in launches()]
            reached.update(got)
            if "tiles" in got[0] and k > 12 * 128:
                over.update((got[0], l.split(", ")[-1]) for l in got[1:])
                steps.setdefault(got[0], set()).add(-(-k // 128) % 4)
        kernels = [stub.stub_kernel(i).decode() for i in range(stub.stub_kernels())]
        kernels = {short(k) for k in kernels if "matmul_" in k and "<bfloat16, false, " in k}
        assert kernels and not kernels - reached, kernels - reached
        assert len(steps) == len([k for k in kernels if "tiles" in k]) == 3
        assert {0, 1, 2, 3} in steps.values()
        assert {t for t, _ in over} == set(steps)  # strips of rows (false) and of columns (true)
        assert {s for _, s in over} == {"false", "true"}
    """)
