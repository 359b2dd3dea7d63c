"""Plain numpy forms of the 4-bit format and the dropout mask, in 64 bits (no code of the
package): what the tests of the device operators compare with."""
import ctypes as C

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


# -- element types: f64, f32, bf16 (held as uint16), f16 ------------------------------------
def to_bf16(x):
    """float32 -> bfloat16 bits, nearest even."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(x)
    return np.where(nan, np.uint16(0x7FC0), r)


def from_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def store(x, dtype):
    """float64 values as an array of element type 0..3 (f64, f32, bf16, f16)."""
    with np.errstate(over="ignore"):
        if dtype == 2:
            return to_bf16(np.asarray(x, dtype=np.float32))
        return np.asarray(x).astype([np.float64, np.float32, None, np.float16][dtype])


def load(a, dtype):
    return from_bf16(a) if dtype == 2 else a.astype(np.float64)


HALF_STEP = [2.0 ** -53, 2.0 ** -24, 2.0 ** -8, 2.0 ** -11]  # relative, at most


# -- the mask --------------------------------------------------------------------------------
def philox(c, key):
    """Philox4x32-10: c four uint64 arrays of 32-bit values, key (low, high)."""
    low = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) for v in c]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), q & low,
             (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def threshold(rate):
    return int(np.rint(rate * 65536))


def kept_scale(rate):
    return 65536.0 / (65536 - threshold(rate))


def keep(n, d, drop):
    """Boolean n x d: the values a Dropout keeps."""
    if drop is None:
        return np.ones((n, d), dtype=bool)
    rows = np.arange(n, dtype=np.uint64) + np.uint64(drop.row0)
    g = np.arange((d + 7) // 8, dtype=np.uint64)
    one = np.ones((n, g.size), dtype=np.uint64)
    c = philox([one * g, one * (rows & np.uint64(0xFFFFFFFF))[:, None],
                one * (rows >> np.uint64(32))[:, None], one * np.uint64(drop.step)],
               (drop.seed & 0xFFFFFFFF, drop.seed >> 32))
    w = np.stack([v for x in c for v in (x & np.uint64(0xFFFF), x >> np.uint64(16))], -1)
    return w.reshape(n, 8 * g.size)[:, :d] >= threshold(drop.rate)


# -- the format ------------------------------------------------------------------------------
def quantize(x):
    """(codes, scales): a 4-bit code per value, rows filled to whole blocks, and a byte per block."""
    x = np.asarray(x, dtype=np.float64)
    n, d = x.shape
    v = np.zeros((n, -(-d // 32) * 32))
    v[:, :d] = x
    v = v.reshape(n, v.shape[1] // 32, 32)
    ok = np.isfinite(v).all(-1)
    top = np.abs(np.where(np.isfinite(v), v, 0)).max(-1) if v.size else np.zeros(v.shape[:2])
    e = np.frexp(top)[1].astype(np.int64) - 3  # floor(log2 top) - 2
    s = np.where(top == 0, 0, np.clip(e + 127, 0, 254))
    a = np.abs(np.where(ok[..., None], v, 0))
    # to the scale's units exactly; far above it the value saturates anyway
    a = np.minimum(np.ldexp(a, (127 - s)[..., None]), 8)
    lo = np.searchsorted(GRID, a, side="right") - 1
    hi = np.minimum(lo + 1, 7)
    below, above = a - GRID[lo], GRID[hi] - a
    up = (above < below) | ((above == below) & (lo % 2 == 1))
    code = np.where((lo < 7) & up, hi, lo) + 8 * (np.signbit(v) & ok[..., None])
    s = np.where(ok, s, 255)
    return code.reshape(n, 32 * s.shape[1]).astype(np.uint8), s.astype(np.uint8)


def values(code, s):
    """float64 values of codes and scales (whole blocks)."""
    n = code.shape[0]
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7]
    p = np.where(s == 255, np.nan, np.ldexp(1.0, s.astype(np.int64) - 127))
    return (v.reshape(n, s.shape[1], 32) * p[..., None]).reshape(code.shape)


def rounded(x):
    """What the 4-bit form of x stands for."""
    return values(*quantize(x))[:, :np.shape(x)[1]]


def pack(code, s, ldc, lds):
    """Bytes as the operators hold them, at the given pitches, zeros behind the blocks."""
    n = code.shape[0]
    c, q = np.zeros((n, ldc), dtype=np.uint8), np.zeros((n, lds), dtype=np.uint8)
    c[:, :code.shape[1] // 2] = code[:, ::2] | code[:, 1::2] << 4
    q[:, :s.shape[1]] = s
    return c, q


# -- device memory, from the HIP runtime as a C caller's would be ------------------------------
_hip = None


def hip():
    global _hip
    if _hip is None:
        h = C.CDLL("libamdhip64.so.7")
        h.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
        h.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
        h.hipFree.argtypes = [C.c_void_p]
        for f, args in (("hipStreamCreateWithFlags", [C.POINTER(C.c_void_p), C.c_uint]),
                        ("hipStreamBeginCapture", [C.c_void_p, C.c_int]),
                        ("hipStreamEndCapture", [C.c_void_p, C.POINTER(C.c_void_p)]),
                        ("hipGraphInstantiate", [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p,
                                                 C.c_char_p, C.c_size_t]),
                        ("hipGraphLaunch", [C.c_void_p, C.c_void_p]),
                        ("hipStreamSynchronize", [C.c_void_p]), ("hipStreamDestroy", [C.c_void_p]),
                        ("hipGraphExecDestroy", [C.c_void_p]), ("hipGraphDestroy", [C.c_void_p])):
            getattr(h, f).argtypes = args
        _hip = h
    return _hip


class Dev:
    """A device copy of a numpy array, `skew` bytes behind an aligned address."""

    def __init__(self, host, skew=0):
        host = np.ascontiguousarray(host)
        self.like, self.p = host, C.c_void_p()
        assert hip().hipMalloc(C.byref(self.p), max(host.nbytes, 1) + skew) == 0
        self.ptr = self.p.value + skew
        self.put(host)

    def put(self, host):
        if host.nbytes:
            assert hip().hipMemcpy(self.ptr, host.ctypes.data, host.nbytes, 1) == 0

    def get(self):
        out = np.empty_like(self.like)
        assert hip().hipDeviceSynchronize() == 0
        if out.nbytes:
            assert hip().hipMemcpy(out.ctypes.data, self.ptr, out.nbytes, 2) == 0
        return out

    def __del__(self):
        if self.p.value:
            hip().hipFree(self.p)
            self.p = C.c_void_p()
