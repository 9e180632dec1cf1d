"""The microscaled (MX) operators (matrix_numbers_b200.mx, csrc/mx.cu, csrc/mx_gemm.cu) against their definitions in
64 bits (tests/mx_reference.py): quantisation code for code, products of values whose FP32 sums are exact bit for bit,
products of ordinary values within the error of an FP32 sum and one rounding, the grouped product with empty, tiny and
uneven groups, the norm, the linear layer and its gradients; refusals, streams, graphs and strided operands."""
import ctypes

import numpy as np
import pytest

import mx_reference as R

FMTS = ["e2m1", "e4m3"]
PAIRS = [(a, b) for a in FMTS for b in FMTS]
NAMES = ["float32", "float16", "bfloat16"]


# ------------------------------------------------------------------------------------------------------------ CPU
def test_grids():
    assert R.grid("e2m1").tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    g = R.grid("e4m3")
    assert g[1] == 2.0 ** -9 and g[8] == 2.0 ** -6 and g[-1] == 448 and np.all(np.diff(g) > 0)


def test_operand_sizes(pkg):
    L = pkg._lib.lib()
    for fmt, per in ((0, 64), (1, 128)):                         # bytes of 128 elements
        for g, rows, k in [(1, 1, 1), (1, 128, 128), (1, 129, 129), (5, 300, 1000), (2, 2 ** 20, 4096)]:
            kt = -(-k // 128)
            assert L.ozk_mx_code_bytes(fmt, g, rows, k) == g * rows * kt * per
            assert L.ozk_mx_scale_bytes(g, rows, k) == g * -(-rows // 128) * kt * 512
    for bad in [(2, 1, 1, 1), (0, 0, 1, 1), (0, 1, 0, 1), (0, 1, 1, 0), (0, 1, 1, 2 ** 28 + 1)]:
        assert L.ozk_mx_code_bytes(*bad) == 0
    assert L.ozk_mx_scale_bytes(1, 1, 0) == 0


def test_c_abi_refusals(pkg):
    """Every invalid argument is answered with OZK_ERR_ARG before any device work."""
    L = pkg._lib.lib()
    p = 4096                                                     # an aligned address that nothing reads
    quant = [p, 0, 1, 4, 64, 0, 64, 1, 0, 0, p, p, None]
    for at, v in [(0, None), (0, p + 2), (1, 3), (1, -1), (2, 0), (3, 0), (4, 0), (4, 2 ** 28 + 1), (5, -1), (6, -1), (7, -1),
                  (8, 2), (10, None), (10, p + 8), (11, None), (11, p + 4)]:
        a = list(quant)
        a[at] = v
        assert L.ozk_mx_quantize(*a) == -1, (at, v)
    for f, a, at in ((L.ozk_mx_quantize, quant, 3), (L.ozk_mx_dequantize, [p, p, 0, 1, 4, 64, p, 0, None], 4),
                     (L.ozk_mx_gemm, [p, p, 0, p, p, 1, 4, 8, 64, p, 8, 2, p, None], 6),
                     (L.ozk_mx_rms_norm, [p, None, p, 2, 0, 4, 64, 64, 0, 1e-6, 1, 0, None, p, p, None], 5)):
        a = list(a)
        a[at] = 2 ** 31 - 1                                      # rows whose tiles would not count in 32 bits
        assert f(*a) == -1
    both = [p, 0, 4, 64, 64, 1, 0, 0, p, p, None]
    for at, v in [(0, None), (1, 3), (2, 0), (2, 2 ** 28 + 1), (3, 0), (4, -1), (5, -1), (6, 2), (8, None), (8, p + 16),
                  (9, None)]:
        a = list(both)
        a[at] = v
        assert L.ozk_mx_quantize_both(*a) == -1, (at, v)
    fwd = [p, 2, 64, 1, p, 2, 64, 1, 4, 8, 64, 1, 0, p, p, None, None, p, p, None]
    for at, v in [(0, None), (1, 4), (2, -1), (4, None), (5, -1), (7, -1), (8, 0), (9, 0), (10, 0), (11, 3), (13, None),
                  (14, p + 8), (15, p + 8), (16, p + 4), (17, None), (18, None)]:
        a = list(fwd)
        a[at] = v
        assert L.ozk_mx_linear_forward(*a) == -1, (at, v)
    bwd = [p, 2, 8, 1, p, p, 4, 8, 64, 1, 0, p, p, p, 2, p, 2, p, None]
    for at, v in [(0, None), (0, p + 1), (1, 3), (2, -1), (4, None), (5, None), (6, 0), (7, 0), (8, 0), (9, 2), (11, None),
                  (12, None), (13, p + 1), (14, 3), (15, p + 1), (16, -1), (17, None)]:
        a = list(bwd)
        a[at] = v
        assert L.ozk_mx_linear_backward(*a) == -1, (at, v)
    a = list(bwd)
    a[13] = a[15] = None
    assert L.ozk_mx_linear_backward(*a) == -1                    # no gradient wanted
    assert L.ozk_mx_quantize(p, 0, 2 ** 16, 2 ** 30, 2 ** 20, 0, 64, 1, 0, 0, p, p, None) == -1   # more tiles than a grid
    deq = [p, p, 0, 1, 4, 64, p, 0, None]
    for at, v in [(0, None), (0, p + 8), (1, None), (2, 5), (3, 0), (4, 0), (5, 0), (6, None), (6, p + 2), (7, 3)]:
        a = list(deq)
        a[at] = v
        assert L.ozk_mx_dequantize(*a) == -1, (at, v)
    gemm = [p, p, 0, p, p, 1, 4, 8, 64, p, 8, 2, p, None]
    for at, v in [(0, None), (0, p + 16), (1, None), (1, p + 8), (2, 2), (3, None), (3, p + 16), (4, None), (5, -1),
                  (6, 0), (7, 0), (8, 0), (9, None), (9, p + 1), (10, 7), (11, 3), (12, None)]:
        a = list(gemm)
        a[at] = v
        assert L.ozk_mx_gemm(*a) == -1, (at, v)
    group = [p, p, 0, p, p, 1, 4, 8, 64, 3, p, 1, p, 8, 2, p, None]
    for at, v in [(0, None), (6, 0), (9, 0), (9, 1025), (10, None), (10, p + 2), (12, None), (13, 7), (14, 4), (15, None)]:
        a = list(group)
        a[at] = v
        assert L.ozk_mx_grouped_gemm(*a) == -1, (at, v)
    norm = [p, None, p, 2, 0, 4, 64, 64, 0, 1e-6, 1, 0, None, p, p, None]
    for at, v in [(0, None), (0, p + 1), (1, p + 1), (2, None), (2, p + 1), (12, p + 1), (3, 7), (5, 0), (6, 0), (7, -1), (8, -1), (9, 0.0), (9, float("nan")),
                  (9, float("inf")), (10, 2), (13, None), (13, p + 8), (14, None)]:
        a = list(norm)
        a[at] = v
        assert L.ozk_mx_rms_norm(*a) == -1, (at, v)
    assert isinstance(ctypes.sizeof(ctypes.c_size_t), int)


def test_python_refusals_without_a_device(pkg):
    import torch
    x = torch.zeros(4, 64)
    for call in [lambda: pkg.mx_quantize(x), lambda: pkg.mx_quantize([1.0]), lambda: pkg.mx_matmul(x, x),
                 lambda: pkg.mx_grouped_matmul(x, x, x), lambda: pkg.mx_rms_norm(x, x[0]), lambda: pkg.mx_linear(x, x),
                 lambda: pkg.MXMatrix("e3m2", None, 4, 64, 0), lambda: pkg.MXMatrix("e2m1", None, 4, 0, 0),
                 lambda: pkg.MXMatrix("e2m1", None, 4, 2 ** 28 + 1, 0), lambda: pkg.MXMatrix("e2m1", None, 2 ** 31, 1, 0),
                 lambda: pkg.MXMatrix.from_codes(x, x, "e2m1")]:
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------------------------------------ GPU
def _f64(t):
    return t.detach().double().cpu().numpy()


def _values(rng, shape):
    """Normal values over a wide range of block magnitudes, with zeros, ties, whole blocks of zeros."""
    x = rng.standard_normal(shape) * np.exp2(rng.integers(-12, 12, size=shape[:-1] + (1,)))
    x[rng.random(shape) < 0.1] = 0.0
    ties = rng.random(shape) < 0.2                               # quarters and eighths: halfway between many grid numbers
    x[ties] = rng.integers(-64, 65, size=int(ties.sum())) / 8.0
    if shape[-1] > 64:
        x[..., 32:64] = 0.0
    return x


def _put(x, name):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(getattr(torch, name)).cuda()


def _same(q, x, fmt, rule):
    """q holds the codes and scales that the definition gives for the float64 values x (contracted axis last)."""
    codes, scales = R.quantize(x, fmt, rule)
    np.testing.assert_array_equal(q.scales().cpu().numpy(), scales)
    np.testing.assert_array_equal(q.codes().cpu().numpy(), R.pack(codes, fmt))


SHAPES = [(1, 1), (1, 32), (3, 31), (2, 33), (16, 128), (128, 256), (129, 257), (37, 1000), (300, 96), (5, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("fmt", FMTS)
def test_quantize(pkg, name, fmt):
    rng = np.random.default_rng(1)
    for shape in SHAPES:
        for rule in ("floor", "ceil"):
            x = _put(_values(rng, shape), name)
            q = pkg.mx_quantize(x, fmt, rule=rule)
            assert q.shape == shape
            _same(q, _f64(x), fmt, rule)
            q = pkg.mx_quantize(x, fmt, axis=0, rule=rule)       # blocks down the columns
            assert q.shape == shape[::-1]
            _same(q, _f64(x).T, fmt, rule)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_quantize_strides(pkg, name):
    """Views of every kind: padded rows, offsets off a 16-byte boundary, transposed, steps, expanded, groups."""
    import torch
    rng = np.random.default_rng(2)
    base = _put(_values(rng, (150, 300)), name)
    views = [base[:, :200], base[:, 1:], base[3:, 5:262], base.T, base.T[1:, 3:], base[::2, ::3], base[:, ::2].T,
             base[:1].expand(40, 300), base[:, :1].expand(150, 70), base[5, 7].expand(33, 65), base[:, 8:136], base[:1]]
    for i, v in enumerate(views):
        for axis in (0, 1):
            want = _f64(v) if axis == 1 else _f64(v).T
            _same(pkg.mx_quantize(v, FMTS[i % 2], axis=axis), want, FMTS[i % 2], "floor")
    g = _put(_values(rng, (3, 140, 70)), name)
    for v in (g, g.transpose(0, 1), g.transpose(1, 2), g[:, 1:, 1:], g[:1].expand(4, 140, 70)):
        _same(pkg.mx_quantize(v, "e2m1"), _f64(v), "e2m1", "floor")
        _same(pkg.mx_quantize(v, "e4m3", axis=1), _f64(v).transpose(0, 2, 1), "e4m3", "floor")
    assert pkg.mx_quantize(torch.empty(0, 64, device="cuda")).dequantize().shape == (0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_both(pkg, name, fmt):
    """Both operands from one read equal the two quantisations, aligned or not."""
    rng = np.random.default_rng(22)
    base = _put(_values(rng, (300, 264)), name)
    for v in (base, base[:, :200], base[:1], base[:, :1], base[:129, 8:137], base[:, 1:], base.T, base[5, 7].expand(33, 65)):
        a, b = pkg.mx_quantize_both(v, fmt, rule="ceil")
        _same(a, _f64(v), fmt, "ceil")
        _same(b, _f64(v).T, fmt, "ceil")


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_special_values(pkg, fmt):
    """NaN, infinities, the largest and smallest numbers of each type, negative zero, exact ties, saturation."""
    import torch
    rows = []
    for v in [np.nan, np.inf, -np.inf, 3.4e38, -3.4e38, 1e-45, 1e-38, 1.1754944e-38, 0.0, -0.0, 6.0, 6.5, 7.0, 7.99,
              448.0, 464.0, 480.0, 511.0, 2.0 ** -126, 2.0 ** -130, 1.0, 2.0 ** 127]:
        r = np.linspace(-1.0, 1.0, 96).astype(np.float32)
        r[40] = v
        rows.append(r)
        r = np.zeros(96, np.float32)
        r[33] = v
        r[95] = v
        rows.append(r)
    g = R.grid(fmt)
    for s in (1.0, -1.0, 2.0 ** -100):                           # all halfway points of the grid, block by block
        mids = np.concatenate([(g[1:] + g[:-1]) / 2, g]) * s
        for i in range(0, mids.size, 31):
            r = np.zeros(96, np.float32)
            part = mids[i:i + 31]
            r[32:32 + part.size] = part
            r[63] = g[-1] * s                                    # fixes the block's scale
            rows.append(r)
    x = np.stack(rows)
    for rule in ("floor", "ceil"):
        for axis in (1, 0):
            t = torch.from_numpy(x if axis == 1 else np.ascontiguousarray(x.T)).cuda()
            q = pkg.mx_quantize(t, fmt, axis=axis, rule=rule)
            _same(q, x.astype(np.float64), fmt, rule)
            got = _f64(q.dequantize(torch.float32))
            want = R.rounded(x, fmt, rule)
            np.testing.assert_array_equal(got, want.astype(np.float32).astype(np.float64))
    for name in ("float16", "bfloat16"):
        t = torch.from_numpy(x).cuda().to(getattr(torch, name))
        _same(pkg.mx_quantize(t, fmt), _f64(t), fmt, "floor")
        _same(pkg.mx_quantize(t.T.contiguous(), fmt, axis=0), _f64(t), fmt, "floor")


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("name", NAMES)
def test_dequantize_and_from_codes(pkg, fmt, name):
    """Codes and scales of every value to numbers (one rounding to the type) and back, plain and in groups."""
    import torch
    rng = np.random.default_rng(3)
    dt = getattr(torch, name)
    for shape in [(1, 1), (5, 31), (130, 257), (3, 40, 100), (2, 200, 64)]:
        codes = rng.integers(0, 16 if fmt == "e2m1" else 256, size=shape, dtype=np.uint8)
        scales = rng.integers(100, 140, size=shape[:-1] + (-(-shape[-1] // 32),), dtype=np.uint8)
        scales.flat[0] = 255
        c, s = torch.from_numpy(R.pack(codes, fmt)).cuda(), torch.from_numpy(scales).cuda()
        q = pkg.MXMatrix.from_codes(c, s, fmt, shape[-1])
        assert q.shape == shape and torch.equal(q.codes(), c) and torch.equal(q.scales(), s)
        want = torch.from_numpy(R.decode(codes, scales, fmt)).to(dt).double().numpy()
        np.testing.assert_array_equal(_f64(q.dequantize(dt)), want)


# ---- products -------------------------------------------------------------------------------------------------------
def _exact_operand(pkg, rng, fmt, rows, k, groups=None):
    """Random codes with scales of 1/2, 1 and 2, and the numbers: multiples of 1/4 up to 12.  A sum of up to 4096 products
    is a multiple of 1/16 below 2^20, exact in FP32 in any order."""
    import torch
    shape = (rows, k) if groups is None else (groups, rows, k)
    if fmt == "e2m1":
        codes = rng.integers(0, 16, size=shape, dtype=np.uint8)
    else:                                                        # 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives
        codes = np.array([0, 0x30, 0x38, 0x3c, 0x40, 0x44, 0x48, 0x4c], np.uint8)[rng.integers(0, 8, size=shape)]
        codes |= rng.integers(0, 2, size=shape, dtype=np.uint8) << 7
    scales = rng.integers(126, 129, size=shape[:-1] + (-(-k // 32),), dtype=np.uint8)
    q = pkg.MXMatrix.from_codes(torch.from_numpy(R.pack(codes, fmt)).cuda(), torch.from_numpy(scales).cuda(), fmt, k)
    return q, R.decode(codes, scales, fmt)


PRODUCT_SHAPES = [(1, 1, 1), (1, 128, 128), (2, 40, 31), (31, 129, 256), (33, 100, 160), (64, 257, 384), (65, 64, 640),
                  (127, 130, 33), (128, 256, 512), (129, 255, 1000), (300, 700, 300), (1, 4096, 4096), (20, 300, 2080),
                  (513, 770, 1100), (1500, 2400, 300), (2300, 2310, 300), (4100, 3000, 700)]


@pytest.mark.gpu
def test_product_exact_small_first(pkg):
    """One tile of each kind of instruction, all sums exact: equal to the definition bit for bit."""
    import torch
    rng = np.random.default_rng(4)
    for a, b in PAIRS:
        A, av = _exact_operand(pkg, rng, a, 128, 256)
        B, bv = _exact_operand(pkg, rng, b, 128, 256)
        C = pkg.mx_matmul(A, B, dtype=torch.float32)
        torch.cuda.synchronize()
        pkg.mx_check_errors()
        np.testing.assert_array_equal(_f64(C), av @ bv.T, err_msg=f"{a} {b}")


@pytest.mark.gpu
@pytest.mark.parametrize("a,b", PAIRS)
def test_product_exact(pkg, a, b):
    """Every shape (tile edges, single rows and columns, the split over K) and output type, bit for bit."""
    import torch
    rng = np.random.default_rng(5)
    for m, n, k in PRODUCT_SHAPES:
        A, av = _exact_operand(pkg, rng, a, m, k)
        B, bv = _exact_operand(pkg, rng, b, n, k)
        want = torch.from_numpy(av @ bv.T).float()
        for name in NAMES:
            dt = getattr(torch, name)
            C = pkg.mx_matmul(A, B, dtype=dt)
            assert torch.equal(C.cpu(), want.to(dt)), (m, n, k, name)
    pkg.mx_check_errors()


def _close_product(C, av, bv, k, half_step, what=""):
    """|C - A B^T| within an FP32 sum's error and one rounding.  The sum of k products: the tensor cores add at most 32
    products and the running sum at a time, each such step exact but for a truncation of at most 2^-22 of the largest
    magnitude that takes part, which is at most the sum of the products' magnitudes: k / 32 + 1 steps of 2^-22; the split
    over a cluster adds at most 8 roundings of 2^-24."""
    mag = np.abs(av) @ np.abs(bv).T
    want = av @ bv.T
    tol = (k / 32 + 4) * 2.0 ** -22 * mag
    tol = tol + half_step * (np.abs(want) + tol)
    bad = np.abs(C - want) > tol
    assert not bad.any(), (what, int(bad.sum()), np.abs(C - want).max(), tol.min())


@pytest.mark.gpu
@pytest.mark.parametrize("a,b", PAIRS)
def test_product_ordinary_values(pkg, a, b):
    import torch
    rng = np.random.default_rng(6)
    for m, n, k in [(1, 300, 1000), (50, 129, 2048), (200, 300, 4096), (130, 260, 95)]:
        x, w = rng.standard_normal((m, k)), rng.standard_normal((n, k)) * np.exp2(rng.integers(-9, 9, size=(n, 1)))
        A, B = pkg.mx_quantize(_put(x, "float32"), a), pkg.mx_quantize(_put(w, "float32"), b)
        av, bv = R.rounded(x.astype(np.float32), a), R.rounded(w.astype(np.float32), b)
        for name, half in (("float32", 0.0), ("float16", 2.0 ** -11), ("bfloat16", 2.0 ** -8)):
            if name == "float16" and np.abs(av @ bv.T).max() > 60000:
                continue
            C = _f64(pkg.mx_matmul(A, B, dtype=getattr(torch, name)))
            mag_floor = 2.0 ** -25 if name == "float16" else 0.0    # half a step of FP16's subnormal numbers
            _close_product(np.where(np.abs(C - av @ bv.T) <= mag_floor, av @ bv.T, C), av, bv, k, half, (m, n, k, name))
    pkg.mx_check_errors()


@pytest.mark.gpu
def test_product_scales_far_apart(pkg):
    """Scales over e8m0's range: the product of two scales stays in FP32's range, each factor alone need not be near it;
    a NaN scale makes its row (and no other) NaN."""
    import torch
    for a, b in PAIRS:
        m, n, k = 40, 50, 64
        A, av = _exact_operand(pkg, np.random.default_rng(7), a, m, k)
        B, bv = _exact_operand(pkg, np.random.default_rng(8), b, n, k)
        for up in (100, -100):
            sa, sb = A.scales().int() + up, B.scales().int() - up
            A2 = pkg.MXMatrix.from_codes(A.codes(), sa.to(torch.uint8), a, k)
            B2 = pkg.MXMatrix.from_codes(B.codes(), sb.to(torch.uint8), b, k)
            np.testing.assert_array_equal(_f64(pkg.mx_matmul(A2, B2, dtype=torch.float32)), av @ bv.T)
        s = A.scales()
        s[3, 1] = 255
        C = _f64(pkg.mx_matmul(pkg.MXMatrix.from_codes(A.codes(), s, a, k), B, dtype=torch.float32))
        want = av @ bv.T
        want[3] = np.nan
        np.testing.assert_array_equal(C, want)


@pytest.mark.gpu
def test_product_into_given_rows(pkg):
    """C given: strided rows, an offset off a 16-byte boundary, and nothing around them touched."""
    import torch
    rng = np.random.default_rng(9)
    for m, n, k in [(5, 72, 64), (70, 72, 200), (140, 300, 96), (1, 1, 40)]:
        A, av = _exact_operand(pkg, rng, "e2m1", m, k)
        B, bv = _exact_operand(pkg, rng, "e2m1", n, k)
        for name in NAMES:
            for off, extra in ((0, 8), (8, 8), (1, 5), (0, 0)):
                buf = torch.full((m + 2, n + off + extra), 7.0, dtype=getattr(torch, name), device="cuda")
                C = buf[1:m + 1, off:off + n]
                assert pkg.mx_matmul(A, B, C=C) is C
                want = torch.full_like(buf, 7.0)
                want[1:m + 1, off:off + n] = torch.from_numpy(av @ bv.T).float().to(buf.dtype).cuda()
                assert torch.equal(buf, want), (m, n, k, name, off)


# ---- grouped --------------------------------------------------------------------------------------------------------
def _grouped_want(av, bv, ends):
    want = np.zeros((av.shape[0], bv.shape[1]))
    before = 0
    for g, e in enumerate(ends):
        e = min(max(e, before), av.shape[0])
        want[before:e] = av[before:e] @ bv[g].T
        before = e
    return want, before


GROUPS = [(1, 1, [1]), (5, 3, [0, 5, 5]), (40, 4, [0, 0, 0, 0]), (200, 5, [1, 2, 130, 131, 200]), (300, 3, [128, 256, 300]),
          (290, 2, [31, 33]), (64, 33, list(range(1, 65, 2)) + [64]), (1000, 2, [3, 1000]), (500, 3, [499, 499, 500]),
          (260, 1, [259]), (90, 40, [0] * 39 + [90]),
          (2100, 3, [700, 701, 2090]), (1300, 1, [1299]), (5000, 2, [3333, 5000])]


@pytest.mark.gpu
@pytest.mark.parametrize("a,b", PAIRS)
def test_grouped(pkg, a, b):
    import torch
    rng = np.random.default_rng(10)
    for rows, experts, ends in GROUPS:
        n, k = int(rng.integers(1, 300)), int(rng.integers(1, 300))
        A, av = _exact_operand(pkg, rng, a, rows, k)
        B, bv = _exact_operand(pkg, rng, b, n, k, experts)
        e = torch.tensor(ends, dtype=torch.int32, device="cuda")
        want, last = _grouped_want(av, bv, ends)
        C = _f64(pkg.mx_grouped_matmul(A, B, e, dtype=torch.float32))
        np.testing.assert_array_equal(C, want, err_msg=str((rows, n, k, ends)))
        given = torch.full((rows, n + 3), 5.0, device="cuda")
        pkg.mx_grouped_matmul(A, B, e, C=given[:, :n])
        got = _f64(given)
        assert (got[last:] == 5.0).all() and (got[:, n:] == 5.0).all()
        np.testing.assert_array_equal(got[:last, :n], C[:last])
    pkg.mx_check_errors()


@pytest.mark.gpu
def test_grouped_ends_out_of_order(pkg):
    """Ends that descend or lie outside the rows count as the nearest in order: no access outside the operands."""
    import torch
    rng = np.random.default_rng(11)
    A, av = _exact_operand(pkg, rng, "e2m1", 150, 64)
    B, bv = _exact_operand(pkg, rng, "e2m1", 40, 64, 4)
    for ends in ([-5, 70, 20, 150], [10, 2 ** 31 - 1, 3, -2 ** 31], [200, 0, 0, 0], [0, 0, 0, -1]):
        want, _ = _grouped_want(av, bv, ends)
        e = torch.tensor(ends, dtype=torch.int32, device="cuda")
        np.testing.assert_array_equal(_f64(pkg.mx_grouped_matmul(A, B, e, dtype=torch.float32)), want)


@pytest.mark.gpu
def test_grouped_most_groups(pkg):
    import torch
    rng = np.random.default_rng(12)
    A, av = _exact_operand(pkg, rng, "e2m1", 1500, 32)
    B, bv = _exact_operand(pkg, rng, "e2m1", 8, 32, 1024)
    ends = np.sort(rng.integers(0, 1501, size=1024)).astype(np.int32)
    want, _ = _grouped_want(av, bv, ends.tolist())
    C = pkg.mx_grouped_matmul(A, B, torch.from_numpy(ends).cuda(), dtype=torch.float32)
    np.testing.assert_array_equal(_f64(C), want)
    with pytest.raises(ValueError):
        B2, _ = _exact_operand(pkg, rng, "e2m1", 1, 32, 1025)
        pkg.mx_grouped_matmul(A, B2, torch.zeros(1025, dtype=torch.int32, device="cuda"))


# ---- norm -----------------------------------------------------------------------------------------------------------
def _norm_want(x, w, r, eps):
    t = x if r is None else x + r
    return t, t / np.sqrt((t * t).mean(-1, keepdims=True) + eps) * w


def _near_codes(q, y, fmt, rule):
    """The operand's numbers against the 64-bit norm y.  The kernel's y is off by a few FP32 roundings (a sum of d squares
    in FP32 over a tree, a division, a square root, two products: below 2^-19 of the value for the sizes here), so a code
    is the right one or, where y is within that of a rounding border, its neighbour: one step of 2^(1 - mantissa bits) of
    the value or, below the smallest normal, of the block; where the block's largest value is within it of a power of two,
    the scale may be the neighbouring one."""
    got = _f64(q.dequantize(__import__("torch").float32))
    codes, scales = R.quantize(y, fmt, rule)
    s = q.scales().cpu().numpy().astype(int)
    off = s != scales
    top = np.abs(R.blocks(y)).max(-1)
    frac = np.frexp(np.where(top == 0, 1.0, top))[0] * 2
    border = np.minimum(np.abs(frac - 1), np.abs(frac - 2)) < 2.0 ** -18
    cut = 1.5 if fmt == "e2m1" else 1.75
    border |= np.abs(frac - cut) < 2.0 ** -18
    assert not (off & ~border).any()
    lo, hi = R.rounded(y * (1 - 2.0 ** -18), fmt, rule), R.rounded(y * (1 + 2.0 ** -18), fmt, rule)
    ok = (got == lo) | (got == hi) | (got == R.rounded(y, fmt, rule))
    ok |= np.repeat(off, 32, -1)[..., :y.shape[-1]]
    assert ok.all(), (int((~ok).sum()), got[~ok][:4], y[~ok][:4])


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("fmt", FMTS)
def test_rms_norm(pkg, name, fmt):
    import torch
    rng = np.random.default_rng(13)
    for rows, d in [(1, 1), (1, 32), (7, 33), (3, 128), (130, 100), (5, 1024), (2, 1025), (9, 4096), (3, 5000), (2, 8192),
                    (2, 8200), (1, 33000), (2, 40960)]:
        for with_res in (False, True):
            x, w = _put(rng.standard_normal((rows, d)) * 3, name), _put(1 + 0.1 * rng.standard_normal(d), name)
            r = _put(rng.standard_normal((rows, d)), name) if with_res else None
            if rows > 4:
                x[2] = 0.0
                if with_res:
                    r[2] = 0.0
            wt = w.float() if d % 3 == 0 else w
            rule = "ceil" if d % 2 else "floor"
            q, s = pkg.mx_rms_norm(x, wt, residual=r, eps=1e-5, fmt=fmt, rule=rule)
            t, y = _norm_want(_f64(x), _f64(wt), None if r is None else _f64(r), 1e-5)
            if r is None:
                assert s is None
            else:
                assert torch.equal(s, (x.float() + r.float()).to(x.dtype))
            assert q.shape == (rows, d)
            _near_codes(q, y, fmt, rule)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [264, 777, 1032, 1999, 2056, 3001, 4104, 4098, 8191, 8200, 8201])
def test_rms_norm_many_rows(pkg, d):
    """Rows enough for the kernel that streams them: the last ones against the definition, a row of NaN, one of squares
    beyond FP32, and all of them against the same rows in small batches (another kernel, other orders of the sum)."""
    import torch
    rng = np.random.default_rng(23)
    rows = 600 + d % 7
    for name, fmt, with_res in (("bfloat16", "e4m3", True), ("float32", "e2m1", False)):
        x, w = _put(rng.standard_normal((rows, d)), name), _put(1 + 0.1 * rng.standard_normal(d), name)
        x[rows - 2] = 1e30
        x[rows - 3, 9] = float("nan")
        r = _put(rng.standard_normal((rows, d)), name) if with_res else None
        q, s = pkg.mx_rms_norm(x, w, residual=r, fmt=fmt)
        got = q.dequantize(torch.float32)
        assert np.isnan(_f64(got[rows - 3])).all()
        if r is not None:
            assert torch.equal(s.nan_to_num(), (x.float() + r.float()).to(x.dtype).nan_to_num())
        off, base = 3, _put(rng.standard_normal((rows, d + 7)), name)   # strided rows that start anywhere
        v = base[:, off:off + d]
        a, b = pkg.mx_rms_norm(v, w, residual=v, fmt=fmt), pkg.mx_rms_norm(v.contiguous(), w, residual=v.contiguous(), fmt=fmt)
        assert torch.equal(a[1], (2 * v.float()).to(x.dtype)) and torch.equal(a[1], b[1])
        assert (a[0].dequantize() != b[0].dequantize()).sum() <= 64 + rows * d * 2.0 ** -16
        keep = [0, 1, rows // 2, rows - 2, rows - 1]
        _, y = _norm_want(_f64(x[keep]), _f64(w), None if r is None else _f64(r[keep]), 1e-6)
        sub = pkg.MXMatrix.from_codes(q.codes()[keep].contiguous(), q.scales()[keep].contiguous(), fmt, d)
        _near_codes(sub, y, fmt, "floor")
        few = torch.cat([pkg.mx_rms_norm(x[i:i + 100], w, residual=None if r is None else r[i:i + 100], fmt=fmt)[0]
                         .dequantize(torch.float32) for i in range(0, rows, 100)])
        same = (few == got) | (few.isnan() & got.isnan())
        # a sum in another order moves a value across a border between codes about once in 2^20 values
        assert (~same).sum() <= 64 + rows * d * 2.0 ** -16


@pytest.mark.gpu
def test_rms_norm_views(pkg):
    """Leading axes, strided rows, rows off a 16-byte boundary, a row of NaN, an empty batch."""
    import torch
    rng = np.random.default_rng(14)
    base = _put(rng.standard_normal((6, 4, 200)), "bfloat16")
    w = _put(1 + rng.standard_normal(96) * 0.1, "float32")
    for v in (base[:, :, :96], base[:, :, 3:99], base[:, :, ::2][..., :96], base[::2, 1:3, 8:104]):
        r = _put(rng.standard_normal(v.shape), "bfloat16")
        q, s = pkg.mx_rms_norm(v, w, residual=r)
        assert s.shape == v.shape and torch.equal(s, (v.float() + r.float()).bfloat16())
        _, y = _norm_want(_f64(v).reshape(-1, 96), _f64(w), _f64(r).reshape(-1, 96), 1e-6)
        _near_codes(q, y, "e4m3", "floor")
    x = base[:, 0, :96].clone()
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    q, _ = pkg.mx_rms_norm(x, w)
    got = _f64(q.dequantize())
    assert np.isnan(got[2]).all() and np.isfinite(got[[0, 1, 4, 5]]).all() and np.isnan(got[3, :32]).all()
    big = torch.full((2, 96), 1e30, device="cuda")             # squares beyond FP32
    big[0, :48] = -3e25
    q, _ = pkg.mx_rms_norm(big, w)
    _near_codes(q, _norm_want(_f64(big), _f64(w), None, 1e-6)[1], "e4m3", "floor")
    q, s = pkg.mx_rms_norm(torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda"),
                           residual=torch.empty(0, 64, device="cuda"))
    assert q.shape == (0, 64) and s.shape == (0, 64)


# ---- linear layer ---------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("name", NAMES)
def test_linear_and_gradients(pkg, fmt, name):
    """y, dx and dw against the formulas with the rounded operands."""
    import torch
    rng = np.random.default_rng(15)
    half = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[name]
    for lead, n, k in [((1,), 40, 33), ((3, 50), 130, 300), ((70,), 257, 64)]:
        x = _put(rng.standard_normal((*lead, k)), name).requires_grad_()
        w = _put(rng.standard_normal((n, k)) * k ** -0.5, name).requires_grad_()
        dy = _put(rng.standard_normal((*lead, n)), name)
        y = pkg.mx_linear(x, w, fmt=fmt)
        assert y.shape == (*lead, n) and y.dtype == x.dtype
        y.backward(dy)
        xv, wv, gv = _f64(x).reshape(-1, k), _f64(w), _f64(dy).reshape(-1, n)
        m = xv.shape[0]
        for got, a, b, kk in ((y, R.rounded(xv, fmt), R.rounded(wv, fmt), k),
                              (x.grad, R.rounded(gv, fmt), R.rounded(wv.T, fmt), n),
                              (w.grad, R.rounded(gv.T, fmt), R.rounded(xv.T, fmt), m)):
            got = _f64(got).reshape(a.shape[0], b.shape[0])
            tiny = np.abs(got - a @ b.T) <= (2.0 ** -25 if name == "float16" else 0.0)
            _close_product(np.where(tiny, a @ b.T, got), a, b, kk, half, (name, fmt, kk))


@pytest.mark.gpu
def test_linear_gradient_against_differences(pkg):
    """On values that the blocks hold exactly (small whole numbers) the layer is the bilinear form itself: its differences
    along whole-number steps are its gradients, exactly."""
    import torch
    rng = np.random.default_rng(16)
    m, n, k = 9, 40, 70
    def whole(shape):
        v = rng.integers(-2, 3, size=shape).astype(np.float32)
        return torch.from_numpy(v).cuda()
    x, w, dy = whole((m, k)).requires_grad_(), whole((n, k)).requires_grad_(), whole((m, n))
    with torch.no_grad():                                        # every block along every axis reaches 2: one scale
        x[:, ::8], w[:, ::8], x[::8], w[::8], dy[:, ::8], dy[::8] = 2.0, 2.0, 2.0, 2.0, 2.0, 2.0
    loss = (pkg.mx_linear(x, w) * dy).sum()
    dx, dw = torch.autograd.grad(loss, (x, w))
    def value(xx, ww):
        return float((pkg.mx_linear(xx, ww).detach().double() * dy.double()).sum())
    base = value(x, w)
    for _ in range(6):
        sx, sw = whole((m, k)).sign(), whole((n, k)).sign()
        assert value(x + sx, w) - base == float((dx.double() * sx.double()).sum())
        assert value(x, w + sw) - base == float((dw.double() * sw.double()).sum())


@pytest.mark.gpu
def test_linear_shared_and_partial(pkg):
    """A leaf used twice adds its gradients; only the wanted gradients are computed; an expanded dy; an empty batch; no
    second derivative."""
    import torch
    rng = np.random.default_rng(17)
    x, w = _put(rng.standard_normal((20, 64)), "float32"), _put(rng.standard_normal((64, 64)), "float32")
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    (pkg.mx_linear(xg, wg) + pkg.mx_linear(2 * xg, wg)).sum().backward()
    one = R.rounded(np.ones((20, 64)), "e4m3") @ R.rounded(_f64(w).T, "e4m3").T
    tol = 64 * 2.0 ** -22 * np.abs(_f64(w)).sum() / 64
    assert np.abs(_f64(xg.grad) - 3 * one).max() <= 4 * tol
    xg, wg = x.clone().requires_grad_(), w.clone()
    pkg.mx_linear(xg, wg).sum().backward()
    assert wg.grad is None and xg.grad is not None
    xg, wg = x[:0].clone().requires_grad_(), w.clone().requires_grad_()
    y = pkg.mx_linear(xg, wg)
    y.sum().backward()
    assert y.shape == (0, 64) and xg.grad.shape == (0, 64) and (wg.grad == 0).all()
    xg = x.clone().requires_grad_()
    g, = torch.autograd.grad(pkg.mx_linear(xg, w).square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
def test_linear_other_forms(pkg):
    """A vector, a transposed and a wider weight, an input that needs no gradient: equal to the plain call or its parts."""
    import torch
    rng = np.random.default_rng(24)
    x, w = _put(rng.standard_normal((30, 72)), "bfloat16"), _put(rng.standard_normal((40, 72)), "bfloat16")
    y = pkg.mx_linear(x, w)
    assert torch.equal(pkg.mx_linear(x[3], w), pkg.mx_linear(x[3:4], w)[0])
    assert torch.equal(pkg.mx_linear(x, w.t().contiguous().t()), y) and torch.equal(pkg.mx_linear(x, w.float()), y)
    assert torch.equal(pkg.mx_linear(x.t().contiguous().t(), w), y)
    assert torch.equal(y, pkg.mx_matmul(pkg.mx_quantize(x, "e4m3"), pkg.mx_quantize(w, "e4m3")))
    dy = _put(rng.standard_normal((30, 40)), "bfloat16")
    grads = []
    for need_x, need_w, weight in ((True, True, w), (True, False, w), (False, True, w), (True, True, w.float())):
        xx, ww = x.clone().requires_grad_(need_x), weight.clone().requires_grad_(need_w)
        pkg.mx_linear(xx, ww).backward(dy)
        grads.append((xx.grad, ww.grad))
    (dx, dw), (dx1, none), (none2, dw1), (dx2, dw2) = grads
    assert none is None and none2 is None and torch.equal(dx, dx1) and torch.equal(dw, dw1) and torch.equal(dx, dx2)
    assert dw2.dtype == torch.float32 and torch.equal(dw2.bfloat16(), dw)
    with torch.no_grad():
        assert not pkg.mx_linear(x.clone().requires_grad_(), w).requires_grad


# ---- as they are used together --------------------------------------------------------------------------------------
def _block(pkg, x, h, gain, W1, experts, ends):
    import torch
    q, h = pkg.mx_rms_norm(x, gain, residual=h)
    y = pkg.mx_matmul(q, W1, dtype=torch.bfloat16)
    z = pkg.mx_grouped_matmul(pkg.mx_quantize(y, "e2m1"), experts, ends)
    return z, h


def _block_inputs(pkg, rows, seed):
    import torch
    rng = np.random.default_rng(seed)
    x, h = _put(rng.standard_normal((rows, 256)), "bfloat16"), _put(rng.standard_normal((rows, 256)), "bfloat16")
    gain = _put(1 + 0.1 * rng.standard_normal(256), "bfloat16")
    W1 = pkg.mx_quantize(_put(rng.standard_normal((320, 256)) / 16, "bfloat16"), "e2m1")
    E = pkg.mx_quantize(_put(rng.standard_normal((4, 192, 320)) / 16, "bfloat16"), "e2m1")
    ends = torch.tensor([rows // 5, rows // 5, rows - 1, rows], dtype=torch.int32, device="cuda")
    return x, h, gain, W1, E, ends


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 333])
def test_block(pkg, rows):
    """Norm, projection, quantisation and experts in a row: equal to the steps' definitions applied one after another to
    the values that the step before gave."""
    import torch
    x, h, gain, W1, E, ends = _block_inputs(pkg, rows, 18)
    z, h2 = _block(pkg, x, h, gain, W1, E, ends)
    q, h3 = pkg.mx_rms_norm(x, gain, residual=h)
    assert torch.equal(h2, h3)
    y = pkg.mx_matmul(q, W1)
    _close_product(_f64(y), _f64(q.dequantize(torch.float32)), _f64(W1.dequantize(torch.float32)), 256, 2.0 ** -8)
    av = R.rounded(_f64(y), "e2m1")
    want, _ = _grouped_want(av, _f64(E.dequantize(torch.float32)), ends.tolist())
    tol = 2.0 ** -8 * np.abs(want) + (320 / 32 + 4) * 2.0 ** -21 * np.abs(av).max() * 320
    assert (np.abs(_f64(z) - want) <= tol).all()
    pkg.mx_check_errors()


@pytest.mark.gpu
def test_graphs_and_streams(pkg):
    """Captured on a side stream and replayed with new inputs, two graphs at once, and eager calls on two streams: the
    same results as one call after another."""
    import torch
    x, h, gain, W1, E, ends = _block_inputs(pkg, 100, 19)
    want = [t.clone() for t in _block(pkg, x, h, gain, W1, E, ends)]
    x2, h2 = x * 0.5 + 1, h - x
    want2 = [t.clone() for t in _block(pkg, x2, h2, gain, W1, E, ends)]
    graphs, outs, ins = [], [], []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            xs, hs = torch.zeros_like(x), torch.zeros_like(h)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(_block(pkg, xs, hs, gain, W1, E, ends))
            graphs.append(g)
            ins.append((xs, hs))
    torch.cuda.synchronize()
    for a, b in (((x, h), (x2, h2)), ((x2, h2), (x, h))):
        for (xs, hs), (xx, hh) in zip(ins, (a, b)):
            xs.copy_(xx)
            hs.copy_(hh)
        torch.cuda.synchronize()
        t = [torch.cuda.Stream(), torch.cuda.Stream()]
        for g, st in zip(graphs, t):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, xx in zip(outs, (a, b)):
            w = want if xx[0] is x else want2
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])
    t = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st in t:
        with torch.cuda.stream(st):
            got.append(_block(pkg, x, h, gain, W1, E, ends))
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    pkg.mx_check_errors()


@pytest.mark.gpu
def test_linear_captured(pkg):
    """Forward and backward captured together and replayed with new values, after an eager pass over the same leaves whose
    graph is gone (as torch wants of any captured backward pass)."""
    import torch
    rng = np.random.default_rng(20)
    x, w = _put(rng.standard_normal((40, 96)), "bfloat16").requires_grad_(), _put(rng.standard_normal((64, 96)), "bfloat16").requires_grad_()
    dy = _put(rng.standard_normal((40, 64)), "bfloat16")
    def eager():
        y = pkg.mx_linear(x, w)
        return [y.detach()] + list(torch.autograd.grad(y, (x, w), dy))
    eager()
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        y = pkg.mx_linear(x, w)
        got = torch.autograd.grad(y, (x, w), dy)
    got = [y.detach()] + list(got)
    del y
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager()))
        with torch.no_grad():
            x.mul_(-1.5)
            dy.add_(0.25)


@pytest.mark.gpu
def test_threads(pkg):
    """Calls from several host threads at once, each on its own stream."""
    import threading
    import torch
    x, h, gain, W1, E, ends = _block_inputs(pkg, 70, 25)
    want = _block(pkg, x, h, gain, W1, E, ends)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = _block(pkg, x, h, gain, W1, E, ends)
                s.synchronize()
                if not (torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    pkg.mx_check_errors()


@pytest.mark.gpu
def test_stream_recorded(pkg):
    """An operand used on another stream keeps its memory until that stream is done with it."""
    import torch
    A = pkg.mx_quantize(torch.ones(256, 256, device="cuda"))
    want = pkg.mx_matmul(A, A)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)                            # about 10 ms
        got = pkg.mx_matmul(A, A)
    A.record_stream(s)
    del A
    junk = [pkg.mx_quantize(torch.full((256, 256), 3.0, device="cuda")) for _ in range(8)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(junk) == 8


def test_operand_from_a_pickle_is_checked(pkg):
    import torch
    for args in [("e2m1", None, 4, 64, torch.zeros(768, dtype=torch.uint8)), ("e2m1", None, 4, 64, None),
                 ("e2m1", None, -4, 64, None), ("e2m1", -1, -4, 64, None)]:
        with pytest.raises(ValueError):
            pkg.mx._from_buffer(*args)
    for groups, rows in ((None, -4), (-1, 4), (-1, -4)):
        with pytest.raises(ValueError):
            pkg.MXMatrix("e2m1", groups, rows, 64, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_copies_stand_alone(pkg, fmt):
    """A deep copy, a shallow one and a pickle outlive the operand they were taken from, and a deep one is another memory."""
    import copy
    import io
    import torch
    rng = np.random.default_rng(31)
    x = _put(rng.standard_normal((3, 37, 100)), "float32")
    for of in (x, x[1]):
        q = pkg.mx_quantize(of, fmt)
        want = q.dequantize(torch.float32)
        stored = io.BytesIO()
        torch.save(q, stored)
        stored.seek(0)
        copies = [copy.deepcopy(q), copy.copy(q), torch.load(stored, weights_only=False)]
        assert copies[1]._code_ptr == q._code_ptr
        assert len({c._code_ptr for c in (*copies, q)}) == 3
        for c in copies:
            assert (c._code_ptr, c._scale_ptr - c._code_ptr) == (c._buffer.data_ptr(), q._scale_ptr - q._code_ptr)
        q._buffer.fill_(1)                                       # reaches the shallow copy alone
        for c, same in zip(copies, (True, False, True)):
            assert c.shape == q.shape and c.fmt == fmt and torch.equal(c.dequantize(torch.float32), want) == same
        del q
        for c in (copies[0], copies[2]):
            if c.groups is None:
                assert torch.equal(pkg.mx_matmul(c, copies[0]), pkg.mx_matmul(pkg.mx_quantize(of, fmt), copies[0]))


@pytest.mark.gpu
def test_negated_views(pkg):
    """A view whose elements are stored with the other sign is refused as an operand, and followed as a gradient."""
    import torch
    z = torch.randn(64, 64, dtype=torch.complex64, device="cuda")
    neg, plain = z.conj().imag, -z.imag
    assert neg.is_neg() and torch.equal(neg, plain)
    w = torch.ones(64, device="cuda")
    q = pkg.mx_quantize(plain)
    for call in [lambda: pkg.mx_quantize(neg), lambda: pkg.mx_quantize_both(neg), lambda: pkg.mx_matmul(q, q, C=neg),
                 lambda: pkg.mx_rms_norm(neg, w), lambda: pkg.mx_linear(neg, plain),
                 lambda: pkg.mx_rms_norm(plain, torch._neg_view(w)), lambda: pkg.mx_rms_norm(plain, w, residual=neg),
                 lambda: pkg.mx_linear(plain, neg)]:
        with pytest.raises(ValueError):
            call()
    x = plain.clone().requires_grad_()
    y = pkg.mx_linear(x, plain)
    want, = torch.autograd.grad(y, x, plain, retain_graph=True)
    got, = torch.autograd.grad(y, x, neg)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_given_output_and_autograd(pkg):
    """A C that a backward pass kept counts as changed, one that requires a gradient is refused; so is a dual number."""
    import torch
    q = pkg.mx_quantize(torch.ones(8, 64, device="cuda"))
    q3 = pkg.mx_quantize(torch.ones(1, 8, 64, device="cuda"))
    ends = torch.tensor([8], dtype=torch.int32, device="cuda")
    for run in (lambda C: pkg.mx_matmul(q, q, C=C), lambda C: pkg.mx_grouped_matmul(q, q3, ends, C=C)):
        C = torch.zeros(8, 8, device="cuda")
        w = torch.ones(8, 8, device="cuda", requires_grad=True)
        y = (w * C).sum()
        assert run(C) is C and (C == 64).all()
        with pytest.raises(RuntimeError):
            y.backward()
        with pytest.raises(ValueError):
            run(w)
        with torch.no_grad():
            assert (run(w) == 64).all()
        with torch.inference_mode():
            C = torch.zeros(8, 8, device="cuda")
        assert (run(C) == 64).all()
    x = torch.ones(8, 64, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        for args in ((dual, x), (x, dual)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                pkg.mx_linear(*args)
        assert (pkg.mx_linear(x, x) == 64).all()


@pytest.mark.gpu
def test_error_word(pkg):
    """A flag in the device's error word is raised once, under every name of the device."""
    import torch
    q = pkg.mx_quantize(torch.ones(8, 64, device="cuda"))
    pkg.mx_matmul(q, q)
    pkg.mx_check_errors()
    at = torch.cuda.current_device()
    for name in (None, "cuda", at, f"cuda:{at}", torch.device("cuda"), torch.device("cuda", at)):
        pkg.mx._error_words[at].fill_(5)
        with pytest.raises(pkg._lib.OzkError):
            pkg.mx_check_errors(name)
        pkg.mx_check_errors(name)
    with pytest.raises(ValueError):
        pkg.mx_check_errors("cpu")


@pytest.mark.gpu
def test_empty_operands(pkg):
    import torch
    for shape in ((0, 64), (3, 0, 64), (0, 5, 64)):
        q = pkg.mx_quantize(torch.empty(shape, device="cuda"), "e2m1")
        assert q.codes().shape == (*shape[:-1], 32) and q.scales().shape == (*shape[:-1], 2)
        assert q.dequantize().shape == shape
        r = pkg.MXMatrix.from_codes(q.codes(), q.scales(), "e2m1")
        assert r.shape == shape
    a, b = pkg.mx_quantize(torch.empty(0, 64, device="cuda")), pkg.mx_quantize(torch.ones(5, 64, device="cuda"))
    assert pkg.mx_matmul(a, b).shape == (0, 5) and pkg.mx_matmul(b, a).shape == (5, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("axis", [0, 1])
def test_quantize_beyond_32_bit_offsets(pkg, axis):
    """More than 2^32 bytes and 2^31 elements: the last vectors, whose offsets pass 32 bits, against the definition."""
    import torch
    rows, k = 2 ** 15 + 3, 2 ** 16 + 64                          # 2.15e9 values
    x = torch.zeros((rows, k) if axis == 1 else (k, rows), dtype=torch.bfloat16, device="cuda")
    last = x[-3:] if axis == 1 else x[:, -3:]
    rng = np.random.default_rng(26)
    last.copy_(_put(rng.standard_normal(tuple(last.shape)), "bfloat16"))
    q = pkg.mx_quantize(x, "e4m3", axis=axis)
    want = _f64(last) if axis == 1 else _f64(last).T
    del x
    codes, scales = R.quantize(want, "e4m3")
    pitch = -(-k // 128) * 128
    got = q._buffer[:rows * pitch].view(rows, pitch)[-3:, :k]
    np.testing.assert_array_equal(got.cpu().numpy(), codes)
    np.testing.assert_array_equal(q.scales()[-3:].cpu().numpy(), scales)
    del got, q
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_product_beyond_32_bit_offsets(pkg):
    """A C of more than 2^32 bytes: its corners, and a grouped one's last rows."""
    import torch
    rng = np.random.default_rng(27)
    m, n, k = 66000, 33000, 32
    A, av = _exact_operand(pkg, rng, "e2m1", m, k)
    B, bv = _exact_operand(pkg, rng, "e2m1", n, k)
    C = pkg.mx_matmul(A, B)
    for r, c in ((slice(0, 50), slice(0, 50)), (slice(m - 50, m), slice(n - 50, n)), (slice(m - 50, m), slice(0, 50)),
                 (slice(m // 2, m // 2 + 50), slice(n // 2, n // 2 + 50))):
        want = torch.from_numpy(av[r] @ bv[c].T).float().bfloat16()
        assert torch.equal(C[r, c].cpu(), want)
    B1 = pkg.MXMatrix.from_codes(B.codes()[None], B.scales()[None], "e2m1")
    D = pkg.mx_grouped_matmul(A, B1, torch.tensor([m - 5], dtype=torch.int32, device="cuda"))
    assert torch.equal(D[:m - 5], C[:m - 5]) and (D[m - 5:] == 0).all()
    del C, D
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_product_nan_codes(pkg):
    """The NaN code of e4m3 makes its row or column NaN, and no other."""
    import torch
    rng = np.random.default_rng(28)
    A, av = _exact_operand(pkg, rng, "e4m3", 40, 96)
    B, bv = _exact_operand(pkg, rng, "e2m1", 50, 96)
    c = A.codes()
    c[7, 33] = 0x7f
    c[9, 95] = 0xff
    C = _f64(pkg.mx_matmul(pkg.MXMatrix.from_codes(c, A.scales(), "e4m3"), B, dtype=torch.float32))
    want = av @ bv.T
    want[[7, 9]] = np.nan
    np.testing.assert_array_equal(C, want)


@pytest.mark.gpu
def test_repeatable(pkg):
    """The same call gives the same bits, split over a cluster or not."""
    import torch
    rng = np.random.default_rng(21)
    for m, n, k in [(1, 4096, 4096), (40, 512, 2048), (300, 300, 4096)]:
        A, B = pkg.mx_quantize(_put(rng.standard_normal((m, k)), "float32"), "e4m3"), pkg.mx_quantize(_put(rng.standard_normal((n, k)), "float32"), "e2m1")
        first = pkg.mx_matmul(A, B, dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(first, pkg.mx_matmul(A, B, dtype=torch.float32))


@pytest.mark.gpu
def test_python_refusals(pkg):
    import torch
    x = torch.zeros(8, 64, device="cuda")
    q, q3 = pkg.mx_quantize(x), pkg.mx_quantize(x.expand(3, 8, 64))
    other = pkg.mx_quantize(torch.zeros(8, 96, device="cuda"))
    ends = torch.zeros(3, dtype=torch.int32, device="cuda")
    w = torch.ones(64, device="cuda")
    codes, scales = q.codes(), q.scales()
    bad = [lambda: pkg.mx_quantize(x, "e5m2"), lambda: pkg.mx_quantize(x, rule="up"), lambda: pkg.mx_quantize(x, axis=2),
           lambda: pkg.mx_quantize(x, axis=-3), lambda: pkg.mx_quantize(x.expand(2, 8, 64), axis=0),
           lambda: pkg.mx_quantize(x[0]), lambda: pkg.mx_quantize(x.double()), lambda: pkg.mx_quantize(x[:, :0]),
           lambda: pkg.mx_quantize(x.expand(2, 2, 8, 64)), lambda: q.dequantize(torch.float64),
           lambda: pkg.mx_matmul(q, other), lambda: pkg.mx_matmul(q, q3), lambda: pkg.mx_matmul(q3, q),
           lambda: pkg.mx_matmul(q, x), lambda: pkg.mx_matmul(q, q, dtype=torch.int32),
           lambda: pkg.mx_matmul(q, q, C=torch.empty(8, 9, device="cuda")),
           lambda: pkg.mx_matmul(q, q, C=torch.empty(8, 8)), lambda: pkg.mx_matmul(q, q, C=torch.empty(8, 8, device="cuda").T),
           lambda: pkg.mx_matmul(q, q, C=torch.empty(1, 8, device="cuda").expand(8, 8)),
           lambda: pkg.mx_matmul(q, q, C=torch.empty(8, 8, dtype=torch.float64, device="cuda")),
           lambda: pkg.mx_grouped_matmul(q, q, ends), lambda: pkg.mx_grouped_matmul(q3, q3, ends),
           lambda: pkg.mx_grouped_matmul(q, q3, ends[:2]), lambda: pkg.mx_grouped_matmul(q, q3, ends.long()),
           lambda: pkg.mx_grouped_matmul(q, q3, ends.cpu()), lambda: pkg.mx_grouped_matmul(q, q3, [0, 0, 8]),
           lambda: pkg.mx_grouped_matmul(q, q3, torch.zeros(6, dtype=torch.int32, device="cuda")[::2]),
           lambda: pkg.mx_rms_norm(x, w[:63]), lambda: pkg.mx_rms_norm(x, w.half()), lambda: pkg.mx_rms_norm(x, w, eps=0.0),
           lambda: pkg.mx_rms_norm(x, w, eps=float("nan")), lambda: pkg.mx_rms_norm(x, w, residual=x[:4]),
           lambda: pkg.mx_rms_norm(x, w, residual=x.half()), lambda: pkg.mx_rms_norm(x, w, fmt="fp8"),
           lambda: pkg.mx_rms_norm(x.double(), w), lambda: pkg.mx_linear(x, w), lambda: pkg.mx_linear(x, x[:, :32]),
           lambda: pkg.mx_linear(x, x.double()), lambda: pkg.mx_linear(x[:, :0], x[:, :0]),
           lambda: pkg.mx_quantize_both(x[:0]), lambda: pkg.mx_quantize_both(x[0]), lambda: pkg.mx_quantize_both(x, "int4"), lambda: pkg.mx_linear(x, x, fmt="int8"),
           lambda: pkg.MXMatrix.from_codes(codes, scales[:, :1], "e2m1"), lambda: pkg.MXMatrix.from_codes(codes, scales, "e4m3"),
           lambda: pkg.MXMatrix.from_codes(codes, scales, "e2m1", 62), lambda: pkg.MXMatrix.from_codes(codes.int(), scales, "e2m1"),
           lambda: pkg.MXMatrix.from_codes(codes.cpu(), scales, "e2m1")]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert (pkg.mx_matmul(q, q) == 0).all()                      # and the operators still work
