"""Cases of the microscaled (MX) operators, their plain forms and their definition in 64 bits.

An MX matrix holds its numbers in blocks of 32 along the contracted axis: 4-bit (e2m1) or 8-bit (e4m3) floating point
codes and one power-of-two scale 2^(s - 127) a block.  Five operators work on such matrices: the quantisation, the
product, the product grouped by expert, the root-mean-square norm that gives an MX operand, and the linear layer with
its backward pass whose three products are MX products.

``own`` False: the operators in elementary torch operations.  ``own`` True: this repository's package.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 32
EMAX = {"e2m1": 2, "e4m3": 8}                 # exponent of the largest number of the element type
EMIN = {"e2m1": 0, "e4m3": -6}                # exponent of its smallest normal number
MANTISSA = {"e2m1": 1, "e4m3": 3}
LARGEST = {"e2m1": 6.0, "e4m3": 448.0}
EPS = 1e-6


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # activations of a decode batch before a 4-bit product
        {"name": "quantise 16x4096 e2m1", "op": "quantise", "rows": 16, "cols": 4096, "axis": 1, "fmt": "e2m1",
         "dtype": "bf16"},
        # activations of a long prefill
        {"name": "quantise 16384x8192 e4m3", "op": "quantise", "rows": 16384, "cols": 8192, "axis": 1, "fmt": "e4m3",
         "dtype": "bf16"},
        # a weight kept as k x n in 32 bits, packed once per update, at sizes that divide nothing
        {"name": "quantise 5001x4095 down e2m1", "op": "quantise", "rows": 5001, "cols": 4095, "axis": 0,
         "fmt": "e2m1", "dtype": "fp32"},
        # one token through a projection with 4-bit weights
        {"name": "product 1x4096x4096 e4m3 e2m1", "op": "product", "m": 1, "n": 4096, "k": 4096, "a": "e4m3",
         "b": "e2m1", "dtype": "bf16"},
        # a ragged batch in 8 bits, sizes that fill no tile
        {"name": "product 333x1000x2080 e4m3", "op": "product", "m": 333, "n": 1000, "k": 2080, "a": "e4m3",
         "b": "e4m3", "dtype": "fp16"},
        # a long prefill through a wide layer, both operands in 4 bits
        {"name": "product 16384x8192x8192 e2m1", "op": "product", "m": 16384, "n": 8192, "k": 8192, "a": "e2m1",
         "b": "e2m1", "dtype": "bf16"},
        # a decode batch over many experts: a few rows each, some experts without any
        {"name": "grouped 256 rows 32 experts", "op": "grouped", "rows": 256, "spare": 3, "experts": 32, "n": 2048,
         "k": 4096, "a": "e4m3", "b": "e2m1", "dtype": "bf16"},
        # prefill over experts that are used very unevenly
        {"name": "grouped 16384 rows 16 experts", "op": "grouped", "rows": 16384, "spare": 0, "experts": 16,
         "n": 4096, "k": 2048, "a": "e4m3", "b": "e2m1", "dtype": "bf16"},
        # the norm before a projection, one token
        {"name": "norm 1x4096", "op": "norm", "rows": 1, "cols": 4096, "fmt": "e4m3", "dtype": "bf16",
         "residual": True},
        # the same over a long prefill
        {"name": "norm 16384x8192", "op": "norm", "rows": 16384, "cols": 8192, "fmt": "e4m3", "dtype": "bf16",
         "residual": True},
        # a training step's linear layer on a small ragged batch: y, dx and dw
        {"name": "linear 200x1000x520", "op": "linear", "m": 200, "n": 1000, "k": 520, "fmt": "e4m3",
         "dtype": "bf16"},
        # the same at the size of a layer
        {"name": "linear 8192x4096x4096", "op": "linear", "m": 8192, "n": 4096, "k": 4096, "fmt": "e4m3",
         "dtype": "bf16"},
    ]


def _size(rng, low, high):
    """A size between low and high, even over the logarithm; every third one a multiple of 64."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.34:
        v = (v + 63) // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["quantise", "product", "grouped", "norm", "linear"])
    fmts = ["e2m1", "e4m3"]
    if op == "quantise":
        return {"op": op, "rows": _size(rng, 1, 16384), "cols": _size(rng, 32, 8192), "axis": rng.choice([0, 1]),
                "fmt": rng.choice(fmts), "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "product":
        return {"op": op, "m": _size(rng, 1, 16384), "n": _size(rng, 64, 8192), "k": _size(rng, 32, 8192),
                "a": rng.choice(fmts), "b": rng.choice(fmts), "dtype": rng.choice(["bf16", "fp16"])}
    if op == "grouped":
        return {"op": op, "rows": _size(rng, 1, 16384), "spare": rng.choice([0, 0, 7]),
                "experts": rng.choice([1, 3, 8, 16]), "n": _size(rng, 64, 4096), "k": _size(rng, 32, 4096),
                "a": rng.choice(fmts), "b": rng.choice(fmts), "dtype": rng.choice(["bf16", "fp16"])}
    if op == "norm":
        return {"op": op, "rows": _size(rng, 1, 16384), "cols": _size(rng, 32, 8192), "fmt": rng.choice(fmts),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "residual": rng.random() < 0.7}
    return {"op": op, "m": _size(rng, 1, 8192), "n": _size(rng, 64, 4096), "k": _size(rng, 32, 4096),
            "fmt": "e4m3" if rng.random() < 0.7 else "e2m1", "dtype": rng.choice(["bf16", "fp16"])}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _activations(g, rows, cols, dtype):
    """Normal values, rows of uneven size, a few large channels, and now and then a token of zeros (padding)."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g))
    x *= torch.where(torch.rand(1, cols, device="cuda", generator=g) < 0.01, 20.0, 1.0)
    if rows > 4:
        x *= (torch.rand(rows, 1, device="cuda", generator=g) > 0.01).float()
    return x.to(dtype)


def _weights(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g) * (shape[-1] ** -0.5)


def _handle(codes, scales, fmt, k):
    """An operand as a program holds it: the codes and scales as a checkpoint stores them, or the package's matrix."""
    if own:
        return _package().MXMatrix.from_codes(codes, scales, fmt, k)
    return codes, scales, fmt, k


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    s = {"case": case}
    dt = DTYPES[case["dtype"]]
    if op == "quantise":
        s["x"] = _activations(g, case["rows"], case["cols"], dt)
    elif op == "norm":
        s["x"] = _activations(g, case["rows"], case["cols"], dt)
        s["residual"] = _activations(g, case["rows"], case["cols"], dt) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * torch.randn(case["cols"], device="cuda", generator=g)).to(dt)
    elif op == "product":
        a = _activations(g, case["m"], case["k"], torch.float32)
        s["a"] = _handle(*_pack(a, case["a"]))
        s["b"] = _handle(*_pack(_weights(g, case["n"], case["k"]), case["b"]))
    elif op == "grouped":
        T, E = case["rows"], case["experts"]
        share = -torch.log(torch.rand(E, device="cuda", generator=g).clamp_min(1e-7))
        place = torch.rand(T, device="cuda", generator=g)
        edges = torch.cumsum(share / share.sum(), 0)
        ends = (place[:, None] < edges[None, :-1]).sum(0) if E > 1 else torch.zeros(0, device="cuda")
        ends = torch.cat([ends.to(torch.int32), torch.tensor([T], dtype=torch.int32, device="cuda")])
        s["ends"] = ends
        s["longest"] = int(torch.diff(ends, prepend=ends.new_zeros(1)).max())
        a = _activations(g, T + case["spare"], case["k"], torch.float32)
        s["a"] = _handle(*_pack(a, case["a"]))
        s["b"] = _handle(*_pack(_weights(g, E, case["n"], case["k"]), case["b"]))
    else:
        s["x"] = _activations(g, case["m"], case["k"], dt).requires_grad_()
        s["w"] = _weights(g, case["n"], case["k"]).to(dt).requires_grad_()
        s["dy"] = (torch.randn(case["m"], case["n"], device="cuda", generator=g) * 0.01).to(dt)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _blocks(x):
    """x in 32 bits, its last axis filled with zeros to whole blocks, as (..., blocks, 32)."""
    x = x.float()
    k = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -k % BLOCK))
    return x.reshape(*x.shape[:-1], -1, BLOCK)


def _power(e):
    """2^e for whole e from -126 to 127, from the bits (a power function may be off in the last place)."""
    return (e.int() + 127 << 23).view(torch.float32)


def _scaled(x, e):
    """x 2^e in two steps, each of them a power in range."""
    h = e // 2
    return x * _power(h) * _power(e - h)


def _quantise(x, fmt):
    """(element values, scale exponents) of x in blocks along its last axis."""
    b = _blocks(x)
    top = b.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(top)                                      # top = f 2^e with f in [1/2, 1)
    e = torch.where(top > 0, e - 1 - EMAX[fmt], -127).clamp_min(-127)
    v = _scaled(b, -e)
    _, f = torch.frexp(v)
    step = _power(torch.clamp_min(f - 1, EMIN[fmt]) - MANTISSA[fmt])
    q = (torch.round(v / step) * step).clamp(-LARGEST[fmt], LARGEST[fmt])
    return q, e


def _round(x, fmt):
    """x on the grid of its blocks, in 32 bits."""
    q, e = _quantise(x, fmt)
    v = _scaled(q, e)
    return v.reshape(*v.shape[:-2], -1)[..., :x.shape[-1]]


def _pack(x, fmt):
    """The codes (two 4-bit codes a byte, the lower half first) and scales of x as a checkpoint stores them."""
    q, e = _quantise(x, fmt)
    q = q.reshape(*q.shape[:-2], -1)
    if fmt == "e4m3":
        codes = q.to(torch.float8_e4m3fn).view(torch.uint8)[..., :x.shape[-1]].contiguous()
    else:
        table = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=q.device)
        c = torch.bucketize(q.abs(), table, out_int32=True).to(torch.uint8) + torch.signbit(q).to(torch.uint8) * 8
        codes = (c[..., 0::2] + c[..., 1::2] * 16)[..., :(x.shape[-1] + 1) // 2].contiguous()
    return codes, (e.squeeze(-1) + 127).to(torch.uint8), fmt, x.shape[-1]


def _values(codes, scales, fmt, k):
    """What codes and scales stand for, in 32 bits."""
    if fmt == "e4m3":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        table = torch.cat([table, -table])
        v = table[torch.stack([codes & 15, codes >> 4], -1).int()].reshape(*codes.shape[:-1], -1)[..., :k]
    e = (scales.int() - 127).repeat_interleave(BLOCK, -1)[..., :k]
    return _scaled(v, e)


def _matmul(a, b):
    """a b^T in full 32 bits."""
    return torch.matmul(a, b.transpose(-1, -2))


def _plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "quantise":
        x = s["x"] if case["axis"] == 1 else s["x"].T
        return _round(x, case["fmt"]).to(torch.bfloat16)
    if case["op"] == "norm":
        t = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
        y = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * s["weight"].float()
        return {"values": _round(y, case["fmt"]).to(torch.bfloat16),
                "sum": None if s["residual"] is None else t.to(dt)}
    if case["op"] == "product":
        return _matmul(_values(*s["a"]), _values(*s["b"])).to(dt)
    if case["op"] == "grouped":
        a, b, ends = _values(*s["a"]), _values(*s["b"]), s["ends"].long()
        starts = torch.nn.functional.pad(ends[:-1], (1, 0))
        row = torch.arange(a.shape[0], device=a.device)
        take = (starts[:, None] + row[None, :s["longest"]]).clamp_max(a.shape[0] - 1)
        c = _matmul(a[take], b)
        e = torch.searchsorted(ends, row, right=True)
        f = e.clamp_max(ends.numel() - 1)
        c = c[f, (row - starts[f]).clamp_max(s["longest"] - 1)]
        return torch.where((e < ends.numel())[:, None], c, 0.0).to(dt)
    x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
    f = case["fmt"]
    y = _matmul(_round(x, f), _round(w, f))
    dx = _matmul(_round(dy, f), _round(w.T, f))
    dw = _matmul(_round(dy.T, f), _round(x.T, f))
    return {"y": y.to(dt), "dx": dx.to(dt), "dw": dw.to(dt)}


# ---- the framework's operators -------------------------------------------------------------------------------------
def _framework(s):
    ozk = _package()
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "quantise":
        return ozk.mx_quantize(s["x"], case["fmt"], axis=case["axis"]).dequantize(torch.bfloat16)
    if case["op"] == "norm":
        q, t = ozk.mx_rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, fmt=case["fmt"])
        return {"values": q.dequantize(torch.bfloat16), "sum": t}
    if case["op"] == "product":
        return ozk.mx_matmul(s["a"], s["b"], dtype=dt)
    if case["op"] == "grouped":
        return ozk.mx_grouped_matmul(s["a"], s["b"], s["ends"], dtype=dt)
    y = ozk.mx_linear(s["x"], s["w"], fmt=case["fmt"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def run(state):
    torch.backends.cuda.matmul.allow_tf32 = False
    return _framework(state) if own else _plain(state)


# ---- the least work of a pass --------------------------------------------------------------------------------------
def _held(count, k, fmt):
    """Bytes of `count` rows of k numbers as codes and scales."""
    return count * ((k + 1) // 2 if fmt == "e2m1" else k) + count * ((k + BLOCK - 1) // BLOCK)


def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "quantise":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size + 2), "flops": 4 * n}
    if op == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 2) + case["cols"] * size, "flops": 9 * n}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _held(m, k, case["a"]) + _held(n, k, case["b"]) + m * n * size, "flops": 2 * m * n * k}
    if op == "grouped":
        m, n, k, E = case["rows"], case["n"], case["k"], case["experts"]
        used = min(E, m)                                         # experts that have a row: at most these are read
        return {"bytes": _held(m, k, case["a"]) + _held(used * n, k, case["b"]) + (m + case["spare"]) * n * size,
                "flops": 2 * m * n * k}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": 2 * (m * k + n * k + m * n) * size, "flops": 6 * m * n * k}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def _power64(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _grid64(fmt):
    """The magnitudes of the element type by code, from its bits."""
    bits = MANTISSA[fmt]
    codes = torch.arange(8 if fmt == "e2m1" else 127, dtype=torch.float64, device="cuda")
    exponent, mantissa = torch.div(codes, 2 ** bits, rounding_mode="floor"), codes % 2 ** bits
    bias = 1 - EMIN[fmt]
    normal = (1 + mantissa / 2 ** bits) * _power64(exponent - bias)
    return torch.where(exponent > 0, normal, mantissa / 2 ** bits * 2.0 ** EMIN[fmt])


def _round64(x, fmt):
    """The nearest number of the block's grid for each value of x (ties to the even code), block by block."""
    x = x.double()
    k = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = b.abs().max(-1, keepdim=True).values
    power = torch.floor(torch.log2(top.clamp_min(2.0 ** -200)))
    power = torch.where(_power64(power) > top, power - 1, power)   # where the logarithm was rounded to the next
    power = torch.where(_power64(power + 1) <= top, power + 1, power)
    scale = _power64((power - EMAX[fmt]).clamp_min(-127.0))
    grid = _grid64(fmt)
    middle = (grid[1:] + grid[:-1]) / 2
    mag = b.abs() / scale
    low, high = torch.bucketize(mag, middle), torch.bucketize(mag, middle, right=True)
    code = torch.where(low % 2 == 0, low, high)
    return (torch.sign(b) * grid[code] * scale).flatten(-2)[..., :k]


def _values64(codes, scales, fmt, k):
    if fmt == "e2m1":
        low = codes % 16
        c = torch.stack((low, (codes - low) // 16), -1).flatten(-2)[..., :k].long()
        v = torch.where(c > 7, -1.0, 1.0).double() * _grid64(fmt)[c % 8]
    else:
        c = codes.long()
        v = torch.where(c > 127, -1.0, 1.0).double() * _grid64(fmt)[c % 128]
    return v * _power64(scales.long() - 127).repeat_interleave(BLOCK, -1)[..., :k]


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op == "quantise":
        return _round64(s["x"] if case["axis"] == 1 else s["x"].T, case["fmt"])
    if op == "norm":
        t = s["x"].double()
        if s["residual"] is not None:
            t = t + s["residual"].double()
        y = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * s["weight"].double()
        return {"values": _round64(y, case["fmt"]), "sum": None if s["residual"] is None else t}
    if op == "product":
        return _values64(*s["a"]) @ _values64(*s["b"]).T
    if op == "grouped":
        a, ends = _values64(*s["a"]), [0] + s["ends"].tolist()
        c = torch.zeros(a.shape[0], case["n"], dtype=torch.float64, device="cuda")
        codes, scales, fmt, k = s["b"]
        for e in range(case["experts"]):
            c[ends[e]:ends[e + 1]] = a[ends[e]:ends[e + 1]] @ _values64(codes[e], scales[e], fmt, k).T
        return c
    x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
    f = case["fmt"]
    return {"y": _round64(x, f) @ _round64(w, f).T, "dx": _round64(dy, f) @ _round64(w.T, f).T,
            "dw": _round64(dy.T, f) @ _round64(x.T, f).T}
