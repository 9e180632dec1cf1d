"""The microscaled (MX) operators at the ends of their ranges: values near FP32's largest, long rows, blocks that end inside
their 32 with a NaN in them, modes of torch in which a call is the first one, waits that run out, and the products' tiles
over sizes that only one rule reaches.  Definitions in 64 bits: tests/mx_reference.py."""
import numpy as np
import pytest

import mx_reference as R
from test_mx import FMTS, PAIRS, _exact_operand, _f64, _norm_want, _put, _same


def _near(q, y, fmt):
    """The operand's numbers against the 64-bit norm y: the code of y or, where y is within the kernel's error of a rounding
    border, its neighbour; any scale where the block's largest value is that near to a border between scales.  The error: a
    thread adds at most max(32, d / 1024) squares one after another, and ten levels join the threads' sums, each step off
    by half a step of FP32 (2^-24 of the sum); a root halves that; then the root itself (one step at most), its product with
    the value and the one with the weight, half a step each: 4 half steps in all, and one to spare.  Below FP32's normal numbers
    y is off by 2^-149, which no grid here sees: the finest has steps of 2^-136."""
    band = ((max(32, y.shape[-1] / 1024) + 10) / 2 + 5) * 2.0 ** -24
    got = q.dequantize(__import__("torch").float32).double().cpu().numpy()
    codes, scales = R.quantize(y, fmt)
    off = q.scales().cpu().numpy().astype(int) != scales
    top = np.abs(R.blocks(y)).max(-1)
    frac = np.frexp(np.where(top == 0, 1.0, top))[0] * 2
    assert not (off & ~(np.minimum(np.abs(frac - 1), np.abs(frac - 2)) < 2 * band)).any()
    ok = (got == R.rounded(y, fmt)) | (got == R.rounded(y * (1 - band), fmt)) | (got == R.rounded(y * (1 + band), fmt))
    ok |= np.repeat(off, 32, -1)[..., :y.shape[-1]]
    assert ok.all(), (int((~ok).sum()), got[~ok][:4], y[~ok][:4])


# ---- norm: the whole range of FP32 ---------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 600])
@pytest.mark.parametrize("name", ["float32", "bfloat16"])
def test_norm_of_the_largest_values(pkg, rows, name):
    """t weight is beyond FP32 and y is not: rows of the largest values, uneven ones, ones with small values beside them,
    in the kernels for few and for many rows."""
    rng = np.random.default_rng(41)
    for d in (96, 777, 1024, 4096):
        x = rng.standard_normal((rows, d))
        x[0] = 3e38
        x[1] *= 6e37
        x[2] = 1e-6
        x[2, :8] = 3e38
        x[3] *= 1e20
        x, w = _put(x, name), _put(1.5 + 0.1 * rng.standard_normal(d), "float32")
        keep = [0, 1, 2, 3, 4, rows - 1]
        _, y = _norm_want(_f64(x[keep]), _f64(w), None, 1e-6)
        for fmt in FMTS:
            q, _ = pkg.mx_rms_norm(x, w, fmt=fmt)
            _near(pkg.MXMatrix.from_codes(q.codes()[keep].contiguous(), q.scales()[keep].contiguous(), fmt, d), y, fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 600])
def test_norm_of_a_large_gain(pkg, rows):
    """The gain may be as large as its product with a normed value allows."""
    rng = np.random.default_rng(42)
    x, w = _put(rng.standard_normal((rows, 300)) * 1e18, "float32"), _put(rng.uniform(1e24, 1e25, 300), "float32")
    q, _ = pkg.mx_rms_norm(x, w)
    y = _norm_want(_f64(x), _f64(w), None, 1e-6)[1]
    _near(q, y, "e4m3")


@pytest.mark.gpu
@pytest.mark.parametrize("d", [2 ** 17, 2 ** 18 + 5, 2 ** 21])
def test_norm_of_long_rows_of_the_largest_values(pkg, d):
    """However many squares beyond FP32 a row adds."""
    import torch
    rng = np.random.default_rng(43)
    x = torch.full((2, d), 3.3e38, device="cuda")
    x[1, ::3] = -1e37
    w = _put(1.3 + 0.1 * rng.standard_normal(d), "float32")
    q, _ = pkg.mx_rms_norm(x, w)
    _near(q, _norm_want(_f64(x), _f64(w), None, 1e-6)[1], "e4m3")


# ---- blocks that end inside their 32 -------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("name", ["float32", "float16", "bfloat16"])
def test_codes_of_bad_blocks_end_with_the_vector(pkg, fmt, name):
    """A NaN or an infinite value in the last block: the stored codes are the definition's, with nothing in the half of a
    byte behind an odd length, and the same after a round trip; rows, columns and both, aligned or not, in groups."""
    import torch
    rng = np.random.default_rng(44)
    for k in (1, 31, 33, 97, 200):
        for bad in (np.nan, np.inf):
            x = rng.standard_normal((5, k + 3))
            x[1, k - 1] = bad
            x[3, 0] = -bad
            t = _put(x, name)[:, :k]
            down = _put(x.T, name)[:k]
            for q in (pkg.mx_quantize(t, fmt), pkg.mx_quantize(down, fmt, axis=0), pkg.mx_quantize(t.contiguous(), fmt),
                      pkg.mx_quantize(down.T.contiguous().T, fmt, axis=0), pkg.mx_quantize_both(t, fmt)[0],
                      pkg.mx_quantize_both(down, fmt)[1], pkg.mx_quantize_both(down.T.contiguous().T, fmt)[1]):
                _same(q, _f64(t), fmt, "floor")
                back = pkg.MXMatrix.from_codes(q.codes(), q.scales(), fmt, k)
                assert torch.equal(back.codes(), q.codes())
                one, w = pkg.mx_quantize(torch.ones(2, k, device="cuda"), fmt), q.dequantize(torch.float32)
                assert torch.equal(pkg.mx_matmul(q, one)[:, 0].isnan(), w.isnan().any(1))
            _same(pkg.mx_quantize(t.expand(2, 5, k), fmt), np.stack([_f64(t)] * 2), fmt, "floor")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 700])
def test_codes_of_a_bad_row_of_the_norm(pkg, rows):
    import torch
    for d in (33, 777):
        x = torch.ones(rows, d, device="cuda")
        x[1, 3] = float("nan")
        q, _ = pkg.mx_rms_norm(x, torch.ones(d, device="cuda"), fmt="e2m1")
        assert (q.scales()[1] == 255).all() and (q.codes()[1, :-1] == 0x77).all() and (q.codes()[1, -1] == 7).all()
        assert torch.equal(pkg.MXMatrix.from_codes(q.codes(), q.scales(), "e2m1", d).codes(), q.codes())
        w = pkg.mx_quantize(torch.ones(3, d, device="cuda"))
        assert pkg.mx_matmul(q, w).isnan().all(1).nonzero().flatten().tolist() == [1]


# ---- the first product on a device ---------------------------------------------------------------------------------------
@pytest.fixture
def no_word(pkg):
    """The state before the first product on the device."""
    import torch
    torch.cuda.synchronize()
    at = torch.cuda.current_device()
    kept = pkg.mx._error_words.pop(at, None)
    yield at
    torch.cuda.synchronize()
    if kept is not None:
        pkg.mx._error_words[at] = kept


def _word_works(pkg, at, q):
    import torch
    assert (pkg.mx_matmul(q, q, dtype=torch.float32) == 64).all()
    for mode in (torch.no_grad, torch.inference_mode, torch.enable_grad):
        with mode():
            pkg.mx._error_words[at].add_(4)
        with pytest.raises(pkg._lib.OzkError):
            pkg.mx_check_errors()
        pkg.mx_check_errors()


@pytest.mark.gpu
def test_first_product_in_inference_mode(pkg, no_word):
    """The error word that it allocates can be read and cleared in any mode."""
    import torch
    q = pkg.mx_quantize(torch.ones(8, 64, device="cuda"))
    with torch.inference_mode():
        assert (pkg.mx_matmul(q, q) == 64).all()
    pkg.mx._error_words[no_word].add_(4)
    with pytest.raises(pkg._lib.OzkError):
        pkg.mx_check_errors()
    _word_works(pkg, no_word, q)


@pytest.mark.gpu
def test_first_product_under_a_tracer(pkg, no_word):
    """Tensors without memory are refused, and nothing of them is kept."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode
    q = pkg.mx_quantize(torch.ones(8, 64, device="cuda"))
    with FakeTensorMode(allow_non_fake_inputs=True):
        C = torch.empty(8, 8, device="cuda")
        for call in (lambda: pkg.mx_matmul(q, q), lambda: pkg.mx_matmul(q, q, C=C)):
            with pytest.raises((pkg._lib.OzkError, RuntimeError)):
                call()
    _word_works(pkg, no_word, q)


@pytest.mark.gpu
@pytest.mark.parametrize("transform", ["grad", "vmap", "device"])
def test_first_product_under_a_transform(pkg, no_word, transform):
    import torch
    q = pkg.mx_quantize(torch.ones(8, 64, device="cuda"))
    def f(x):
        return x + pkg.mx_matmul(q, q, C=C).sum()
    C = torch.empty(8, 8, device="cuda")
    try:
        if transform == "device":
            with torch.device("cpu"):
                f(torch.ones(3, device="cuda"))
        else:
            getattr(torch.func, transform)(lambda x: f(x).sum())(torch.ones(3, device="cuda"))
    except (RuntimeError, ValueError, pkg._lib.OzkError):
        pass                                                     # refused is fine; what counts is what is left behind
    _word_works(pkg, no_word, q)


# ---- gradients that there are not ----------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_norm_refuses_what_would_lose_a_gradient(pkg):
    """An input that requires a gradient is refused while gradients are recorded, and so is a dual number; without them the
    call is the plain one."""
    import torch
    x, r, w = (torch.randn(8, 64, device="cuda"), torch.randn(8, 64, device="cuda"), torch.ones(64, device="cuda"))
    q, t = pkg.mx_rms_norm(x, w, residual=r)
    for at in range(3):
        args = [a.clone().requires_grad_(i == at) for i, a in enumerate((x, w, r))]
        with pytest.raises(ValueError, match="gradient"):
            pkg.mx_rms_norm(args[0], args[1], residual=args[2])
        if at < 2:
            with pytest.raises(ValueError, match="gradient"):
                pkg.mx_rms_norm(args[0], args[1])
        for mode in (torch.no_grad, torch.inference_mode):
            with mode():
                q1, t1 = pkg.mx_rms_norm(args[0], args[1], residual=args[2])
            assert torch.equal(t1, t) and torch.equal(q1.codes(), q.codes()) and torch.equal(q1.scales(), q.scales())
            assert not t1.requires_grad
    with torch.autograd.forward_ad.dual_level():
        for at in range(3):
            args = [torch.autograd.forward_ad.make_dual(a, a) if i == at else a for i, a in enumerate((x, w, r))]
            with pytest.raises(ValueError, match="tangent"):
                pkg.mx_rms_norm(args[0], args[1], residual=args[2])
        assert torch.equal(pkg.mx_rms_norm(x, w, residual=r)[1], t)


# ---- waits that run out --------------------------------------------------------------------------------------------------
def test_wait_selftest_refusals(pkg):
    L = pkg._lib.lib()
    p = 4096                                                     # an aligned address that nothing reads
    good = [p, p, 0, p, p, 1, 4, 8, 64, p, 8, 2, 10 ** 6, 0, p, None]
    for at, v in [(0, None), (3, p + 16), (6, 0), (10, 7), (11, 3), (12, 99), (12, 4 * 10 ** 9 + 1), (14, None)]:
        a = list(good)
        a[at] = v
        assert L.ozk_mx_wait_selftest(*a) == -1, (at, v)


def _selftest(pkg, A, B, limit_ns, hold):
    """(C, error flags, milliseconds on the device) of a product whose waits end after limit_ns."""
    import torch
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    C = torch.full((A.rows, B.rows), float("nan"), device="cuda")
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    pkg._lib.check(pkg._lib.lib().ozk_mx_wait_selftest(
        A._code_ptr, A._scale_ptr, A._fmt, B._code_ptr, B._scale_ptr, B._fmt, A.rows, B.rows, A.k, C.data_ptr(), B.rows, 0,
        limit_ns, hold, err.data_ptr(), torch.cuda.current_stream().cuda_stream), "ozk_mx_wait_selftest")
    b.record()
    torch.cuda.synchronize()
    return C, int(err.item()), a.elapsed_time(b)


# rows, columns, k, formats, loads of the CTA with the most: one shape for each tile
TILES = [(20, 300, 1024, "e4m3", "e2m1", 2), (50, 300, 1024, "e2m1", "e4m3", 2), (100, 300, 100, "e2m1", "e2m1", 1),
         (100, 384 * 148 + 8, 128, "e4m3", "e4m3", 2), (1700, 1700, 100, "e2m1", "e2m1", 1), (1700, 1700, 100, "e4m3", "e2m1", 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,a,b,loads", TILES)
def test_timeout_waits_for_the_loads_in_flight(pkg, m, n, k, a, b, loads):
    """No stage is ever full, so the issuing warp and the epilogue give up after 20 ms, when the producer has long issued its
    last load and left.  The kernel must not end before it has waited for those loads, which shows in its time: their
    barriers, of which more is expected than comes, take the limit of 1 s each."""
    rng = np.random.default_rng(51)
    (A, av), (B, bv) = _exact_operand(pkg, rng, a, m, k), _exact_operand(pkg, rng, b, n, k)
    _, err, ms = _selftest(pkg, A, B, 20_000_000, 1)
    assert err in (2, 4, 6)                                      # the issuing warp's flag, the epilogue's, or both
    assert 1000 * loads < ms < 1000 * loads + 900
    C, err, _ = _selftest(pkg, A, B, 4 * 10 ** 9, 0)             # and the device is as it was
    assert err == 0
    np.testing.assert_array_equal(C[:64].double().cpu().numpy(), av[:64] @ bv.T)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,a,b", [(20, 200, 2 ** 25, "e2m1", "e2m1"), (50, 200, 2 ** 24, "e4m3", "e2m1"),
                                       (300, 300, 2 ** 22, "e2m1", "e4m3"), (100, 384 * 148 + 8, 2 ** 15, "e4m3", "e2m1"),
                                       (1700, 1700, 2 ** 22, "e2m1", "e2m1"), (1700, 1700, 2 ** 20, "e4m3", "e4m3")])
def test_timeout_in_the_middle(pkg, m, n, k, a, b):
    """Limits that end the waits of an ordinary long product wherever they happen to be, its loads and MMAs in flight: flags,
    or the right product; and the right product from the call that follows, whose CTAs take over the same shared memory and
    TMEM.  (A wait looks at the clock after some hundred polls, so how many end is up to the device.)"""
    import torch
    torch.manual_seed(52)

    def operand(rows, fmt):
        codes = torch.randint(0, 256 if fmt == "e2m1" else 120, (rows, k // (2 if fmt == "e2m1" else 1)), dtype=torch.uint8, device="cuda")
        return pkg.MXMatrix.from_codes(codes, torch.full((rows, k // 32), 120, dtype=torch.uint8, device="cuda"), fmt)

    A, B = operand(m, a), operand(n, b)
    want = pkg.mx_matmul(A, B, dtype=torch.float32)
    flags = []
    for limit in (100, 10_000, 100_000, 300_000, 4 * 10 ** 9):
        for _ in range(3):
            C, err, _ = _selftest(pkg, A, B, limit, 0)
            assert 0 <= err < 8 and (err or torch.equal(C, want))
            flags.append(err)
            assert torch.equal(pkg.mx_matmul(A, B, dtype=torch.float32), want)
    assert flags[-3:] == [0, 0, 0]                               # the last limit is the ordinary one
    pkg.mx_check_errors()
    assert any(flags) or n > 50000                               # whose tiles are too short for it


# ---- every tile of the products, over sizes where its rings and accumulators wrap ----------------------------------------
def _exact_on_device(pkg, fmt, rows, k, groups=None):
    """As test_mx._exact_operand, made on the device: the operand and its numbers in FP32 (multiples of 1/4 up to 12)."""
    import torch
    shape = (rows, k) if groups is None else (groups, rows, k)
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    c = torch.randint(0, 16, shape, dtype=torch.uint8, device="cuda")
    v = table[(c & 7).int()] * torch.where(c > 7, -1.0, 1.0)
    scales = torch.randint(126, 129, (*shape[:-1], -(-k // 32)), dtype=torch.uint8, device="cuda")
    v *= torch.exp2(scales.float() - 127).repeat_interleave(32, -1)[..., :k]
    if fmt == "e4m3":
        of = torch.tensor([0, 0x30, 0x38, 0x3c, 0x40, 0x44, 0x48, 0x4c], dtype=torch.uint8, device="cuda")
        codes = of[(c & 7).int()] | (c >> 3 << 7)
    else:
        c = torch.nn.functional.pad(c, (0, k % 2))
        codes = c[..., 0::2] | (c[..., 1::2] << 4)
    return pkg.MXMatrix.from_codes(codes.contiguous(), scales, fmt, k), v


@pytest.mark.gpu
@pytest.mark.parametrize("a,b", PAIRS)
@pytest.mark.parametrize("k", [32, 1100])
def test_product_of_some_rows_and_many_columns(pkg, a, b, k):
    """33 to 128 rows and columns enough for the 128 x 256 tile, two of which a CTA takes in turn, bit for bit."""
    import torch
    torch.manual_seed(61)
    n = 384 * torch.cuda.get_device_properties(0).multi_processor_count + 8
    B, bv = _exact_on_device(pkg, b, n, k)
    for m in (33, 128):
        A, av = _exact_on_device(pkg, a, m, k)
        want = av.double() @ bv.double().T
        for dt in (torch.float32, torch.bfloat16):
            assert torch.equal(pkg.mx_matmul(A, B, dtype=dt), want.to(dt)), (m, dt)
    pkg.mx_check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("a,b", PAIRS)
@pytest.mark.parametrize("k", [1100, 4096])
@pytest.mark.parametrize("rows,experts", [(1500, 32), (4000, 12)])
def test_grouped_of_long_rows(pkg, rows, experts, k, a, b):
    """Groups of fewer and of more rows than the rule's border (64 on average), long K and several tiles a CTA, with empty
    groups, groups that start and end inside a tile, and rows behind the last: bit for bit in FP32, and in bf16 with rows
    that leave as boxes."""
    import torch
    torch.manual_seed(62)
    rng = np.random.default_rng(63)
    ends = np.sort(rng.integers(0, rows - 6, size=experts))
    ends[3], ends[4], ends[experts // 2] = ends[5], ends[5], ends[experts // 2 + 1]
    ends = ends.tolist()
    e = torch.tensor(ends, dtype=torch.int32, device="cuda")
    for n, dt in ((2100, torch.float32), (2104, torch.bfloat16)):
        A, av = _exact_on_device(pkg, a, rows, k)
        B, bv = _exact_on_device(pkg, b, n, k, experts)
        want = torch.zeros(rows, n, dtype=torch.float64, device="cuda")
        for g, (first, last) in enumerate(zip([0] + ends, ends)):
            want[first:last] = av[first:last].double() @ bv[g].double().T
        assert torch.equal(pkg.mx_grouped_matmul(A, B, e, dtype=dt), want.to(dt))
        given = torch.full((rows, n + 8), 5.0, dtype=dt, device="cuda")
        pkg.mx_grouped_matmul(A, B, e, C=given[:, :n])
        assert torch.equal(given[:ends[-1], :n], want[:ends[-1]].to(dt))
        assert (given[ends[-1]:] == 5.0).all() and (given[:, n:] == 5.0).all()
    pkg.mx_check_errors()
