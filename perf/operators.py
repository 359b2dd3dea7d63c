"""The 4-bit and dropout operators as measured workloads.

Four operators: quantisation to microscaled 4-bit floating point (blocks of 32 values that share a
power of two, values of sign, two exponent bits and a mantissa bit), the matrix product of two such
matrices, dropout whose mask is a function of (seed, step, row, column), and the logistic-regression
pass over a shard that is held in 4 bits.  `own` chooses between the plain forms below and the calls
of `paracel_amd`.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one sample of a 2048-column shard, as a server quantises what it is asked to score
        {"name": "quantize one row", "kind": "quantize", "n": 1, "d": 2048, "type": "bf16",
         "out": "bf16", "transpose": False, "rate": 0.0},
        # the shard of the 2 000 000 x 512 configuration's eighth worker, from doubles, at load time
        {"name": "quantize shard f64", "kind": "quantize", "n": 250000, "d": 512, "type": "f64",
         "out": "f32", "transpose": False, "rate": 0.0},
        # activations of a training step, dropped and laid out for the weight gradient, ragged
        {"name": "quantize transposed dropped", "kind": "quantize", "n": 16385, "d": 4100,
         "type": "bf16", "out": "bf16", "transpose": True, "rate": 0.1},
        # one row against a large 4-bit matrix: scoring a single request
        {"name": "product one row", "kind": "product", "m": 1, "n": 16384, "k": 8192, "out": "bf16"},
        # a small batch of requests, odd sizes
        {"name": "product small batch", "kind": "product", "m": 33, "n": 9000, "k": 4100, "out": "f32"},
        # a whole block of samples against many outputs
        {"name": "product large", "kind": "product", "m": 16384, "n": 8192, "k": 4096, "out": "bf16"},
        # forward and backward of a linear layer with dropout on its input, all products in 4 bits
        {"name": "linear training step", "kind": "linear", "n": 4096, "d": 2048, "o": 4100,
         "type": "bf16", "rate": 0.1},
        # dropout of one row
        {"name": "dropout one row", "kind": "dropout", "n": 1, "d": 1000, "type": "f32", "rate": 0.5},
        # dropout of a step's activations (forward; the backward is the same call on the gradient)
        {"name": "dropout activations", "kind": "dropout", "n": 32768, "d": 8192, "type": "bf16",
         "rate": 0.1},
        # the 100 000 x 100 configuration in 4 bits: short passes, where latency counts
        {"name": "pass small", "kind": "pass", "n": 100000, "d": 100, "rate": 0.0},
        # an ordinary shard of 1000 columns, trained with dropout
        {"name": "pass dropped", "kind": "pass", "n": 200000, "d": 1000, "rate": 0.2},
        # wide rows, one column past a power of two
        {"name": "pass wide", "kind": "pass", "n": 12000, "d": 16385, "rate": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "linear", "dropout", "pass"])
    rate = rng.choice([0.0, 0.1, rng.uniform(0.02, 0.9)])
    if kind == "quantize":
        d = _log(rng, 2, 16500)
        n = _log(rng, 1, max(1, min(260000, 120000000 // d)))
        t = rng.choice(["f64", "f32", "bf16", "f16"])
        return {"kind": kind, "n": n, "d": d, "type": t, "out": "bf16" if t == "bf16" else "f32",
                "transpose": rng.random() < 0.5, "rate": rate}
    if kind == "product":
        k, n = _log(rng, 8, 16500), _log(rng, 1, 16500)
        m = _log(rng, 1, max(1, min(16500, 500000000000 // (n * k))))
        return {"kind": kind, "m": m, "n": n, "k": k, "out": rng.choice(["f32", "bf16", "f16"])}
    if kind == "linear":
        d, o = _log(rng, 16, 5000), _log(rng, 16, 5000)
        n = _log(rng, 16, 5000)
        return {"kind": kind, "n": n, "d": d, "o": o, "type": rng.choice(["f32", "bf16", "f16"]),
                "rate": rate}
    if kind == "dropout":
        d = _log(rng, 2, 16500)
        n = _log(rng, 1, max(1, min(300000, 120000000 // d)))
        return {"kind": kind, "n": n, "d": d, "type": rng.choice(["f64", "f32", "bf16", "f16"]),
                "rate": rate}
    d = _log(rng, 2, 20000)
    n = _log(rng, 1, max(1, min(300000, 150000000 // d)))
    return {"kind": kind, "n": n, "d": d, "rate": rate}


def work(case):
    k = case["kind"]
    if k == "quantize":
        v = case["n"] * case["d"]  # the values once, their 4.25 bits written and read back, the result
        return {"bytes": int(v * (SIZE[case["type"]] + 2 * 17 / 32 + SIZE[case["out"]])), "flops": 4 * v}
    if k == "product":
        m, n, c = case["m"], case["n"], case["k"]
        return {"bytes": int((m + n) * c * 17 / 32 + m * n * SIZE[case["out"]]), "flops": 2 * m * n * c}
    if k == "linear":
        n, d, o = case["n"], case["d"], case["o"]
        return {"bytes": 2 * (n * d + d * o + n * o) * SIZE[case["type"]], "flops": 6 * n * d * o}
    v = case["n"] * case["d"]
    if k == "dropout":
        return {"bytes": 2 * v * SIZE[case["type"]], "flops": 2 * v}
    return {"bytes": int(v * 17 / 32) + 8 * case["n"] + 16 * case["d"], "flops": 4 * v}


# ------------------------------------------------------------ the plain forms
def _threshold(rate):
    return int(round(rate * 65536))


def _keep(n, d, drop):
    """The kept positions of an n x d matrix: Philox4x32-10 of (column // 8, row, step) under the
    seed gives eight 16-bit words, one per column; a value stays where its word reaches the rate."""
    low = 0xFFFFFFFF
    row = drop["row0"] + torch.arange(n, device="cuda", dtype=torch.int64)[:, None]
    col = torch.arange((d + 7) // 8, device="cuda", dtype=torch.int64)[None, :]
    a, b = col.expand(n, -1), (row & low).expand(-1, col.shape[1])
    c, e = (row >> 32).expand(-1, col.shape[1]), torch.full_like(a, drop["step"])
    k0, k1 = drop["seed"] & low, drop["seed"] >> 32
    for _ in range(10):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, e = ((q >> 32) & low) ^ b ^ k0, q & low, ((p >> 32) & low) ^ e ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16, c & 0xFFFF, c >> 16,
                         e & 0xFFFF, e >> 16], -1)
    return words.reshape(n, -1)[:, :d] >= _threshold(drop["rate"])


def _kept_scale(rate):
    return 65536.0 / (65536 - _threshold(rate))


def _blocks(x):
    """Rows cut into blocks of 32, the last one filled up with zeros."""
    n, d = x.shape
    return torch.nn.functional.pad(x, (0, -d % 32)).reshape(n, -1, 32)


def _power(e, dtype):
    """2^e, exactly (a device's pow need not be), for the exponents of scale bytes."""
    return ((e.long() + 1023) << 52).view(torch.float64).to(dtype)


def _e2m1(x):
    """(values on the 4-bit grid, exponents) of the blocks of every row of x."""
    v = _blocks(x)
    e = (torch.frexp(v.abs().amax(-1, keepdim=True)).exponent - 3).clamp(-127, 127)
    v = v * _power(-e, v.dtype)
    a = v.abs()
    q = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2))
    q = torch.copysign(q.clamp(max=6.0), v)
    return q, torch.where(v.abs().amax(-1, keepdim=True) > 0, e, torch.full_like(e, -127))


def _rounded(x):
    """What the 4-bit codes of x stand for."""
    n, d = x.shape
    q, e = _e2m1(x)
    return (q * _power(e, q.dtype)).reshape(n, -1)[:, :d]


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _packed(x):
    """Codes (two per byte, the even column in the low half, rows of whole 128-column chunks) and
    scale bytes of x, as the operators take them."""
    q, e = _e2m1(torch.nn.functional.pad(x, (0, -x.shape[1] % 128)))
    a = q.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code + 8 * torch.signbit(q).to(torch.uint8)).reshape(x.shape[0], -1)
    return code[:, ::2] + 16 * code[:, 1::2], (e + 127).to(torch.uint8).reshape(x.shape[0], -1)


def _unpacked(codes, scales, d):
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    v = grid[torch.stack([codes & 15, codes >> 4], -1).long()].reshape(codes.shape[0], -1, 32)
    return (v * _power(scales.int() - 127, v.dtype)[:, :, None]).reshape(codes.shape[0], -1)[:, :d]


# ------------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _features(g, n, d):
    """Values of a block of samples: normal, rows and columns of different sizes, some exact zeros."""
    x = _randn(g, n, d)
    x *= torch.exp2(torch.randint(-6, 7, (n, 1), device="cuda", generator=g).float())
    x *= torch.exp2(torch.randint(-2, 3, (1, d), device="cuda", generator=g).float())
    return x * (torch.rand(n, d, device="cuda", generator=g) > 0.05)


def _drop(case, seed):
    """Rate, seed and position of a step; a worker's first row can lie far out."""
    return {"rate": case.get("rate", 0.0), "seed": (seed * 0x9E3779B97F4A7C15 + 1) & (2**63 - 1),
            "step": seed % 1000, "row0": (seed % 3) << 33}


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = case["kind"]
    if k == "product":
        a = _packed(_features(g, case["m"], case["k"]))
        b = _packed(_randn(g, case["n"], case["k"]) * 0.05)
        return {"a": a, "b": b, "alpha": 0.5}
    if k == "linear":
        t = TYPES[case["type"]]
        return {"x": _randn(g, case["n"], case["d"]).to(t),
                "w": (_randn(g, case["o"], case["d"]) / math.sqrt(case["d"])).to(t),
                "dz": (_randn(g, case["n"], case["o"]) * 0.01).to(t)}
    if k == "pass":
        x = _randn(g, case["n"], case["d"]).double() / math.sqrt(case["d"])
        theta = _randn(g, case["d"]).double()
        y = (torch.rand(case["n"], device="cuda", generator=g) < torch.sigmoid(x @ theta)).double()
        return {"x": x, "y": y, "theta": 0.3 * theta}
    x = _features(g, case["n"], case["d"])
    if case["type"] == "f64":
        x = x.double() * (1 + 1e-9 * _randn(g, case["n"], 1))
    return {"x": x.to(TYPES[case["type"]])}


def prepare(case, seed):
    state = {"case": case, "drop": _drop(case, seed), **_inputs(case, seed)}
    if case["kind"] == "pass":
        state["theta"] = state["theta"].cpu().numpy()
        if own:
            # the resident shard: uploaded once, then held in 4 bits
            from paracel_amd import Plr

            state["plr"] = Plr(torch.cuda.current_device())
            state["plr"].set_data(state.pop("x").cpu().numpy(), state.pop("y").cpu().numpy())
            state["plr"].pack_data()
            state["plr"].set_timing(False)
        else:
            state["x"] = _rounded(state["x"]).float()
        torch.cuda.empty_cache()
    elif own:
        state["buffers"] = {}
    return state


# ------------------------------------------------------------ the own calls
def _buffer(state, name, shape, dtype):
    """A tensor the program keeps from call to call."""
    if name not in state["buffers"]:
        state["buffers"][name] = torch.empty(shape, dtype=dtype, device="cuda")
    return state["buffers"][name]


def _own_codes(state, name, n, d):
    from paracel_amd import capi

    return (_buffer(state, name + " codes", (n, capi.mxfp_code_pitch(d)), torch.uint8),
            _buffer(state, name + " scales", (n, capi.mxfp_scale_pitch(d)), torch.uint8))


def _own_quantize(state, name, x, transpose=False, drop=None):
    from paracel_amd import capi

    n, d = x.shape
    q = _own_codes(state, name, d if transpose else n, n if transpose else d)
    capi.mxfp_quantize(x.data_ptr(), _own_type(x.dtype), n, d, x.stride(0), q[0].data_ptr(),
                       q[0].stride(0), q[1].data_ptr(), q[1].stride(0), transpose=transpose, drop=drop,
                       device=x.device.index, stream=torch.cuda.current_stream().cuda_stream)
    return q


def _own_type(dtype):
    from paracel_amd import capi

    return {torch.float64: capi.PLR_F64, torch.float32: capi.PLR_F32, torch.bfloat16: capi.PLR_BF16,
            torch.float16: capi.PLR_F16}[dtype]


def _own_matmul(state, name, a, b, k, dtype, alpha, drop=None):
    from paracel_amd import capi

    m, n = a[0].shape[0], b[0].shape[0]
    c = _buffer(state, name, (m, n), dtype)
    size = capi.mxfp_matmul_workspace(m, n, k)
    space = _buffer(state, name + " workspace", (max(size, 1),), torch.uint8)
    capi.mxfp_matmul(m, n, k, a[0].data_ptr(), a[0].stride(0), a[1].data_ptr(), a[1].stride(0),
                     b[0].data_ptr(), b[0].stride(0), b[1].data_ptr(), b[1].stride(0), c.data_ptr(),
                     _own_type(dtype), c.stride(0), alpha=alpha, drop=drop, workspace=space.data_ptr(),
                     workspace_bytes=size, device=c.device.index,
                     stream=torch.cuda.current_stream().cuda_stream)
    return c


def _own_run(state):
    from paracel_amd import capi

    case, k, q = state["case"], state["case"]["kind"], state["drop"]
    drop = capi.Dropout(q["rate"], q["seed"], q["step"], q["row0"]) if q["rate"] else None
    if k == "quantize":
        codes, scales = _own_quantize(state, "x", state["x"], case["transpose"], drop)
        n, d = (case["d"], case["n"]) if case["transpose"] else (case["n"], case["d"])
        out = _buffer(state, "out", (n, d), TYPES[case["out"]])
        capi.mxfp_dequantize(codes.data_ptr(), codes.stride(0), scales.data_ptr(), scales.stride(0), n, d,
                             out.data_ptr(), _own_type(out.dtype), out.stride(0), device=out.device.index,
                             stream=torch.cuda.current_stream().cuda_stream)
        return out
    if k == "product":
        return _own_matmul(state, "c", state["a"], state["b"], case["k"], TYPES[case["out"]], state["alpha"])
    if k == "linear":
        x, w, dz, t = state["x"], state["w"], state["dz"], TYPES[case["type"]]
        up = drop.scale if drop else 1.0
        z = _own_matmul(state, "z", _own_quantize(state, "x", x, drop=drop), _own_quantize(state, "w", w),
                        case["d"], t, up)
        dx = _own_matmul(state, "dx", _own_quantize(state, "dz", dz), _own_quantize(state, "wt", w, True),
                         case["o"], t, 1.0, drop)
        dw = _own_matmul(state, "dw", _own_quantize(state, "dzt", dz, True),
                         _own_quantize(state, "xt", x, True, drop), case["n"], t, up)
        return {"z": z, "dx": dx, "dw": dw}
    if k == "dropout":
        x = state["x"]
        out = _buffer(state, "out", x.shape, x.dtype)
        capi.dropout_apply(x.data_ptr(), _own_type(x.dtype), *x.shape, x.stride(0), out.data_ptr(),
                           out.stride(0), capi.Dropout(q["rate"], q["seed"], q["step"], q["row0"]),
                           device=out.device.index, stream=torch.cuda.current_stream().cuda_stream)
        return out
    state["plr"].set_dropout(drop)
    grad, loss, _ = state["plr"].loss_grad(state["theta"])
    return {"grad": grad, "loss": loss}


def run(state):
    if own:
        return _own_run(state)
    case, k, drop = state["case"], state["case"]["kind"], state["drop"]
    if k == "product":
        a, b = _unpacked(*state["a"], case["k"]), _unpacked(*state["b"], case["k"])
        return (state["alpha"] * (a @ b.T)).to(TYPES[case["out"]])
    if k == "quantize":
        x = _wide(state["x"])
        if drop["rate"]:
            x = x * _keep(case["n"], case["d"], drop)
        return _rounded(x.T if case["transpose"] else x).to(TYPES[case["out"]])
    if k == "linear":
        x, w, dz, t = state["x"].float(), state["w"].float(), state["dz"].float(), TYPES[case["type"]]
        up, keep = 1.0, 1.0
        if drop["rate"]:
            up, keep = _kept_scale(drop["rate"]), _keep(case["n"], case["d"], drop)
        z = up * (_rounded(x * keep) @ _rounded(w).T)
        dx = (_rounded(dz) @ _rounded(w.T).T) * keep * up
        dw = up * (_rounded(dz.T) @ _rounded((x * keep).T).T)
        return {"z": z.to(t), "dx": dx.to(t), "dw": dw.to(t)}
    if k == "dropout":
        x = _wide(state["x"])
        return (x * _keep(case["n"], case["d"], drop) * _kept_scale(drop["rate"])).to(state["x"].dtype)
    # the pass: 64 bits, as the framework's passes are
    x, theta = state["x"].double(), torch.from_numpy(state["theta"]).cuda()
    if drop["rate"]:
        x = x * _keep(case["n"], case["d"], drop) * _kept_scale(drop["rate"])
    h = 1 / (1 + torch.exp(-(x @ theta)))
    loss = -torch.where(state["y"] == 1, torch.log(h), torch.log(1 - h)).sum()
    grad = (h - state["y"]) @ x
    return {"grad": grad.cpu().numpy(), "loss": float(loss)}


# ------------------------------------------- the definitions, once more, in 64 bits
def _exact_keep(n, d, drop):
    """The mask by 16-bit limbs: every product and carry below 2^49."""
    def mul(x, m):
        lo = (x & 0xFFFF) * m
        hi = (x >> 16) * m + (lo >> 16)
        return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)

    groups = torch.arange(n * ((d + 7) // 8), device="cuda")
    per = (d + 7) // 8
    row = groups // per + drop["row0"]
    c = [groups % per, row % 2**32, row // 2**32, torch.zeros_like(row) + drop["step"]]
    for r in range(10):
        k0 = (drop["seed"] + r * 0x9E3779B9) % 2**32
        k1 = (drop["seed"] // 2**32 + r * 0xBB67AE85) % 2**32
        h0, l0 = mul(c[0], 0xD2511F53)
        h1, l1 = mul(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
    col = torch.arange(d, device="cuda")
    word = torch.stack(c).reshape(4, n, per)[(col % 8) // 2, :, col // 8].T
    word = torch.where(col % 2 == 1, word // 65536, word % 65536)
    return word.double() / 65536 >= round(drop["rate"] * 65536) / 65536


def _exact_power(i):
    """2^i for whole i from -127 to 127, from a table."""
    return torch.tensor([math.ldexp(1.0, k) for k in range(-127, 128)], dtype=torch.float64,
                        device="cuda")[i.long() + 127]


def _exact_rounded(x):
    """Nearest of the grid's values, ties to the even code, under the block's power of two."""
    n, d = x.shape
    out = torch.zeros(n, -(-d // 32) * 32, dtype=torch.float64, device="cuda")
    out[:, :d] = x
    v = out.view(n, -1, 32)
    top = v.abs().max(-1, keepdim=True).values
    power = ((top.view(torch.int64) >> 52) - 1023 - 2).clamp(-127, 127)
    a = v.abs() * _exact_power(-power)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    middle = (grid[1:] + grid[:-1]) / 2
    code = torch.bucketize(a, middle)
    tie = (middle[code.clamp(max=6)] == a) & (code % 2 == 1) & (code < 7)
    return (torch.sign(v) * grid[code + tie.long()] * _exact_power(power)).reshape(n, -1)[:, :d]


def _exact_values(codes, scales, k):
    nibble = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.int64, device="cuda")
    nibble[:, 0::2], nibble[:, 1::2] = codes % 16, codes // 16
    e, m = (nibble // 2) % 4, nibble % 2
    v = torch.where(e == 0, 0.5 * m, (1 << e) * (0.5 + 0.25 * m)).double()
    v = torch.where(nibble >= 8, -v, v)
    return (v * _exact_power(scales.long() - 127).repeat_interleave(32, 1))[:, :k]


def exact(case, seed):
    k, drop = case["kind"], _drop(case, seed)
    data = _inputs(case, seed)
    up = 65536 / (65536 - round(drop["rate"] * 65536))
    if k == "product":
        return data["alpha"] * (_exact_values(*data["a"], case["k"]) @ _exact_values(*data["b"], case["k"]).T)
    if k == "quantize":
        x = data["x"].double()
        if drop["rate"]:
            x = torch.where(_exact_keep(case["n"], case["d"], drop), x, 0.0)
        return _exact_rounded(x.T if case["transpose"] else x)
    if k == "linear":
        keep = _exact_keep(case["n"], case["d"], drop).double()
        x, w, dz = data["x"].double() * keep, data["w"].double(), data["dz"].double()
        return {"z": up * (_exact_rounded(x) @ _exact_rounded(w).T),
                "dx": up * keep * (_exact_rounded(dz) @ _exact_rounded(w.T).T),
                "dw": up * (_exact_rounded(dz.T) @ _exact_rounded(x.T).T)}
    if k == "dropout":
        return torch.where(_exact_keep(case["n"], case["d"], drop), up * data["x"].double(), 0.0)
    x, theta, y = _exact_rounded(data["x"]), data["theta"], data["y"]
    if drop["rate"]:
        x = torch.where(_exact_keep(case["n"], case["d"], drop), up * x, 0.0)
    z = (x * theta).sum(1)
    residual = torch.sigmoid(z) - y
    loss = torch.nn.functional.softplus(torch.where(y == 1, -z, z)).sum()
    return {"grad": (x * residual[:, None]).sum(0).cpu().numpy(), "loss": float(loss)}
