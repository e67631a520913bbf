"""The scoring head's operators on the GPU against their definitions in 64 bits
(oracle/scoring_oracle.py).

Tolerances.  u = 2^-24 is half a step of fp32, a sum of N terms in fp32 in any
order is off by at most N u sum|terms| (first order), a rounding to bf16 / fp16 by
2^-8 / 2^-11 of the value."""
import numpy as np
import pytest

from oracle import scoring_oracle as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {"float32": U, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
DTYPES = ["float32", "bfloat16", "float16"]


@pytest.fixture(scope="module")
def sc():
    import torch
    assert torch.cuda.is_available()
    from medical_rag_amd import scoring
    return scoring


def rows(n, d, dtype, seed=0, spread=1.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))
    return x.to(getattr(torch, dtype)).cuda()


def f64(t):
    return t.double().cpu().numpy()


def check_quantized(got, x64, fmt):
    codes, scales = orc.mx_quantize(x64, fmt)
    assert np.array_equal(got.scales.cpu().numpy(), scales)
    assert np.array_equal(got.values.cpu().numpy(), orc.pack(codes, fmt))


# ---- rows to microscaled floating point and back ---------------------------------

SHAPES = [(1, 1), (1, 32), (2, 31), (3, 33), (5, 127), (4, 128), (7, 129), (34, 1000), (17, 1024), (3, 4100), (1000, 8), (66001, 9), (8200, 1032)]


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_is_the_oracle_bit_for_bit(sc, dtype, fmt):
    for i, (n, d) in enumerate(SHAPES):
        x = rows(n, d, dtype, seed=i)
        got = sc.mx_quantize(x, fmt)
        check_quantized(got, f64(x), fmt)
        assert len(got) == n and got.d == d and got.nbytes == got.values.numel() + got.scales.numel()


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_quantize_extremes(sc, fmt):
    """Zeros, the smallest and largest numbers, ties of elements and of the scale, NaN
    and infinity in single blocks."""
    import torch
    big = torch.finfo(torch.float32).max
    x = torch.zeros(16, 64)
    x[1] = -0.0
    x[2, 3] = 1e-45                                  # below every element of the lowest scale
    x[3, :32] = torch.linspace(-2, 2, 32) * 2.0 ** -126
    x[4] = big
    x[5, 7], x[5, 40] = -big, 2.0 ** -100
    x[6, :] = torch.arange(64) * 0.25                # ties between elements in many blocks
    x[7, 0], x[7, 1], x[7, 32], x[7, 33] = 7.0, 3.5, 6.9999995, 5.0
    x[8, 0], x[8, 1], x[8, 32], x[8, 33] = 464.0, 456.0, 464.00003, 17.0
    x[9, 5] = float("nan")
    x[10, 37] = float("inf")
    x[11, 0], x[11, 63] = -float("inf"), 3.0
    x[12] = torch.randn(64, generator=torch.Generator().manual_seed(1)) * 2.0 ** 100
    x[13] = -torch.arange(64) * 0.0625
    x[14] = torch.randn(64, generator=torch.Generator().manual_seed(2)) * 2.0 ** -130
    x[15] = 2.0 ** torch.arange(-32, 32).float()
    got = sc.mx_quantize(x.cuda(), fmt)
    check_quantized(got, x.double().numpy(), fmt)
    back = sc.mx_dequantize(got, torch.float32).cpu()
    assert torch.isnan(back[9, :32]).all() and torch.isfinite(back[9, 32:]).all()
    assert torch.isnan(back[10, 32:]).all() and (back[10, :32] == 0).all()
    assert torch.isnan(back[11, :32]).all() and back[11, 63] == 3


def test_more_rows_than_one_launch_counts(sc):
    """2^32 threads and more: every row is written, the last ones too (all rows are one row)."""
    import torch
    for n, d in ((150_000_000, 200), (300_000_000, 2)):     # 2 and 1 groups of 128 a row, 16 threads each
        x = torch.linspace(-3, 5, d, device="cuda")[None]
        got, one = sc.mx_quantize(x.expand(n, d)), sc.mx_quantize(x)
        words, want = got.values.view(torch.int64), one.values.view(torch.int64)
        step = 1 << 24
        assert all((words[lo:lo + step] == want).all() for lo in range(0, n, step))
        assert all((got.scales[lo:lo + step] == one.scales).all() for lo in range(0, n, step))
        if d == 2:
            out = torch.full((n, d), 7.0, dtype=torch.bfloat16, device="cuda")
            sc.mx_dequantize(got, out=out)
            back = sc.mx_dequantize(one)
            assert all((out[lo:lo + step] == back).all() for lo in range(0, n, step))
        del got, words


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_dequantize_rounds_once(sc, dtype, fmt):
    import torch
    for i, (n, d) in enumerate(SHAPES):
        codes, scales = orc.mx_quantize(f64(rows(n, d, "float32", seed=50 + i, spread=3.0)), fmt)
        packed = sc.MxRows(torch.from_numpy(orc.pack(codes, fmt)).cuda(), torch.from_numpy(scales).cuda(), d, fmt)
        got = sc.mx_dequantize(packed, getattr(torch, dtype))
        want = torch.from_numpy(orc.mx_values(codes, scales, fmt, d)).to(getattr(torch, dtype))
        assert got.dtype == want.dtype and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_dequantize_at_every_width_and_address(sc, dtype, fmt):
    """Into rows that start anywhere, with what lies between and behind them left alone; blocks of very different scales."""
    import torch
    dt = getattr(torch, dtype)
    for d in list(range(1, 18)) + [31, 33, 63, 65, 95, 97, 120, 121, 125, 126, 127, 128, 129, 135, 136, 250, 255, 257]:
        x = rows(5, d, "float32", seed=d) * torch.exp2(torch.randint(-6, 6, (1, d), generator=torch.Generator().manual_seed(d)).float()).cuda()
        q = sc.mx_quantize(x, fmt)
        want = sc.mx_dequantize(q, torch.float32).to(dt)
        for start in range(9):
            for gap in (0, 1, 8):
                flat = torch.full((5 * (d + gap) + 32,), 7.0, dtype=dt, device="cuda")
                out = flat[start:start + 5 * (d + gap)].view(5, d + gap)[:, :d]
                sc.mx_dequantize(q, out=out)
                assert torch.equal(out, want), (d, start, gap)
                out.fill_(7.0)
                assert bool((flat == 7.0).all()), (d, start, gap)


def test_every_code_and_scale_reads_back(sc):
    """All 256 bytes under all 256 scale bytes, e4m3's own NaNs included."""
    import torch
    for fmt in ("mxfp4", "mxfp8"):
        byte = torch.arange(256, dtype=torch.uint8)
        width = 64 if fmt == "mxfp4" else 128
        values = torch.stack([byte.roll(i)[:width] for i in range(256)])
        scales = byte[:, None].expand(256, 4).contiguous()
        got = sc.mx_dequantize(sc.MxRows(values.cuda(), scales.cuda(), 128, fmt), torch.float32)
        want = torch.from_numpy(orc.mx_values(orc.unpack(values.numpy(), fmt), scales.numpy(), fmt, 128)).float()
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=7.5), torch.nan_to_num(want, nan=7.5))


def test_rows_strided_misaligned_and_far_apart(sc):
    import torch
    whole = rows(9, 300, "bfloat16", seed=3)
    for view in (whole[:, 1:], whole[::2, :200], whole[:, 3:67], whole.t(), whole[:, ::3], whole[2:3].expand(4, 300), whole[:0]):
        got = sc.mx_quantize(view, "mxfp4")
        check_quantized(got, f64(view), "mxfp4")
    out = torch.full((9, 500), 7.0, dtype=torch.bfloat16, device="cuda")
    q = sc.mx_quantize(whole, "mxfp8")
    sc.mx_dequantize(q, out=out[:, 101:401])
    assert torch.equal(out[:, 101:401], sc.mx_dequantize(q)) and (out[:, :101] == 7).all() and (out[:, 401:] == 7).all()
    # rows whose offsets pass 32 bits
    far = torch.empty(3 * (2 ** 31 + 8), dtype=torch.bfloat16, device="cuda").as_strided((3, 70), (2 ** 31 + 8, 1))
    far.copy_(whole[:3, :70])
    check_quantized(sc.mx_quantize(far, "mxfp8"), f64(far), "mxfp8")
    sc.mx_dequantize(sc.mx_quantize(whole[3:6, :70].contiguous()), out=far)
    assert torch.equal(far, sc.mx_dequantize(sc.mx_quantize(whole[3:6, :70].contiguous())))


# ---- norm --------------------------------------------------------------------------

def check_norm(sc, x, w, eps, res, fmt):
    """Each value within half a step of its block's scale of the exact one, and the
    scale the exact one's unless its largest value is within the error of a border.
    The error before rounding: the mean of squares is a sum of at most 64 squares a
    thread and a tree of 16 (80 u), halved by the root; root, division and three
    products add 6 u: 46 u, taken as 2^-18."""
    import torch
    got, h = sc.rms_norm_mx(x, w, eps, res, fmt)
    if res is None:
        assert h is None
        h = x
    else:
        want_h = (x.float() + res.float()).to(x.dtype)
        assert torch.equal(h, want_h)
    y = orc.rms_norm(f64(h), f64(w), eps)
    n, d = y.shape
    codes, scales = orc.unpack(got.values.cpu().numpy(), fmt), got.scales.cpu().numpy()
    back = orc.mx_values(codes, scales, fmt, orc.padded(d))
    full = np.zeros((n, orc.padded(d)))
    full[:, :d] = y
    s = scales.astype(int) - 127
    unit = np.repeat(np.ldexp(1.0, s), 32, axis=1)
    bits, low = (1, 0) if fmt == "mxfp4" else (3, -6)
    err = 2.0 ** -18 * np.abs(full)
    step = np.ldexp(1.0, np.maximum(np.frexp((np.abs(full) + err) / unit)[1] - 1, low) - bits) * unit
    assert (np.abs(back - full) <= step / 2 + err).all()
    amax = np.abs(full).reshape(n, -1, 32).max(2)
    lo, hi = orc.mx_scale(amax * (1 - 2.0 ** -18), fmt), orc.mx_scale(amax * (1 + 2.0 ** -18), fmt)
    assert ((s >= lo) & (s <= hi)).all()
    assert (back[:, d:] == 0).all()


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rms_norm(sc, dtype, fmt):
    import torch
    for i, (n, d) in enumerate([(1, 1), (3, 7), (2, 33), (1, 64), (5, 512), (4, 513), (6, 1000), (3, 1024), (2, 2049), (1, 4096), (3, 5000), (2, 8192)]):
        x, res = rows(n, d, dtype, seed=i), rows(n, d, dtype, seed=100 + i)
        w = (1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(i))).cuda()
        check_norm(sc, x, w.to(x.dtype), 1e-6, res, fmt)
        check_norm(sc, x, w, 1e-5, None, fmt)


def test_rms_norm_wide_rows(sc):
    for d in (8193, 16384, 65536):
        check_norm(sc, rows(2, d, "bfloat16", seed=d), rows(1, d, "bfloat16", seed=d + 1)[0], 1e-6, rows(2, d, "bfloat16", seed=d + 2), "mxfp8")


def test_rms_norm_rows_without_a_norm(sc):
    """A zero row gives zeros whatever eps; a row with a NaN or an infinity gives NaN
    and leaves its neighbours alone."""
    import torch
    x = rows(5, 200, "bfloat16", seed=4)
    x[1], x[2, 5], x[3, 7] = 0, float("nan"), float("inf")
    w = torch.ones(200, dtype=torch.bfloat16, device="cuda")
    for eps in (1e-6, 0.0):
        y = sc.mx_dequantize(sc.rms_norm_mx(x, w, eps)[0], torch.float32)
        if eps:
            assert (y[1] == 0).all()
        assert torch.isnan(y[2]).all()
        # inf / inf in its own block; the row's other values are x / inf = 0
        assert torch.isnan(y[3, :32]).all() and (y[3, 32:] == 0).all()
        alone = sc.mx_dequantize(sc.rms_norm_mx(x[4:], w, eps)[0], torch.float32)
        assert torch.equal(y[4:], alone)


def test_rms_norm_strides(sc):
    import torch
    big, res = rows(6, 400, "float16", seed=8), rows(6, 400, "float16", seed=9)
    w = rows(1, 400, "float16", seed=10)[0]
    for cols in (slice(0, 256), slice(1, 257), slice(8, 264)):
        check_norm(sc, big[::2, cols], w[cols], 1e-6, res[1::2, cols], "mxfp8")
    check_norm(sc, big[:, ::2], w[::2], 1e-6, res[:, 1::2], "mxfp8")
    check_norm(sc, big, w, 1e-6, res[:1].expand(6, 400), "mxfp8")
    assert len(sc.rms_norm_mx(big[:0], w, 1e-6, res[:0])[0]) == 0


# ---- product -----------------------------------------------------------------------

def stored(sc, n, d, fmt, seed, exact=False):
    """MxRows of random values and what they stand for.  exact: small whole elements
    under scale 1, whose products' sums fit 24 bits and so have no rounding at all."""
    import torch
    rng = np.random.default_rng(seed)
    if exact:
        grid = orc.GRID[fmt]
        few = [i for i, v in enumerate(grid) if v in (0, 1, 2, 3, 4, 6)]
        codes = rng.choice(few, size=(n, orc.padded(d))) + rng.integers(0, 2, size=(n, orc.padded(d))) * (8 if fmt == "mxfp4" else 128)
        codes = codes.astype(np.uint8)
        codes[:, d:] = 0
        scales = np.full((n, orc.padded(d) // 32), 127, np.uint8)
    else:
        codes, scales = orc.mx_quantize(rng.standard_normal((n, d)) * np.exp(rng.standard_normal((n, 1)) + 0.5 * rng.standard_normal((1, d))), fmt)
    packed = sc.MxRows(torch.from_numpy(orc.pack(codes, fmt)).cuda(), torch.from_numpy(scales).cuda(), d, fmt)
    return packed, orc.mx_values(codes, scales, fmt, d)


MATMULS = [(1, 1, 1), (1, 16, 32), (1, 1000, 4096), (2, 17, 100), (3, 129, 128), (15, 64, 300), (16, 255, 256), (17, 300, 384), (33, 257, 1000),
           (64, 1, 512), (65, 511, 129), (100, 640, 768), (128, 128, 128), (255, 257, 513), (256, 256, 1024), (257, 520, 640), (700, 300, 200)]


# results large enough for tiles (more than three million): every tile shape, one K step to many, partial tiles
TILES = [(64, 50001, 100), (50, 70000, 200), (65, 47003, 384), (128, 24001, 1500), (129, 24000, 256), (513, 6001, 513), (300, 10111, 1030),
         (700, 24100, 1100), (2100, 1500, 130)]


def product(va, vb):
    """The float64 products, a (m, n) tensor on the GPU."""
    import torch
    return torch.from_numpy(va).cuda() @ torch.from_numpy(vb).cuda().t()


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_matmul_of_whole_numbers_is_exact(sc, fmt, out):
    import torch
    for i, (m, n, d) in enumerate(MATMULS + TILES):
        a, va = stored(sc, m, d, fmt, seed=i, exact=True)
        b, vb = stored(sc, n, d, "mxfp4", seed=100 + i, exact=True)
        got = sc.mx_matmul(a, b, getattr(torch, out))
        assert torch.equal(got, product(va, vb).to(getattr(torch, out))), (m, n, d)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_matmul_through_several_chunks_of_b(sc, fmt):
    """Rows so long that B's tiles are taken in chunks, the last one narrower; whole numbers, exact."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)

    def whole(n, d, fmt):
        # a random element, its sign in the type's highest bit: 0, 1, 2, 3, 4, 6 in either type
        few = torch.tensor([0, 2, 4, 5, 6, 7] if fmt == "mxfp4" else [0x00, 0x38, 0x40, 0x44, 0x48, 0x4C], dtype=torch.uint8, device="cuda")
        codes = few[torch.randint(0, 6, (n, d), device="cuda", generator=g)]
        codes |= torch.randint(0, 2, (n, d), device="cuda", generator=g, dtype=torch.uint8) << (3 if fmt == "mxfp4" else 7)
        if fmt == "mxfp4":
            codes = codes[:, ::2] | codes[:, 1::2] << 4
        return sc.MxRows(codes.contiguous(), torch.full((n, d // 32), 127, dtype=torch.uint8, device="cuda"), d, fmt)

    for m, n, d in ((300, 10500, 16384), (130, 24000, 8192)):
        a, b = whole(m, d, fmt), whole(n, d, "mxfp4")
        want = sc.mx_dequantize(a, torch.float32).double() @ sc.mx_dequantize(b, torch.float32).double().t()
        assert float(want.abs().max()) > 0
        for out in (torch.float32, torch.bfloat16):
            assert torch.equal(sc.mx_matmul(a, b, out), want.to(out)), (m, n, d, out)


def check_matmul(got, va, vb, fmt):
    """Sums of d products in fp32: d u sum |a b|.  (Products of an 8-bit element with a
    4-bit one have at most 6 bits, so they are exact.)  bf16 results of 8-bit rows may
    come from the matrix instruction that keeps 2^-16 of its largest product: 128
    of them per step then add 2^-9 of the largest |a b| at most; and every result
    is rounded once."""
    import torch
    want, size = product(va, vb), product(np.abs(va), np.abs(vb))
    err = va.shape[1] * U * size
    name = str(got.dtype).replace("torch.", "")
    if name == "bfloat16" and fmt == "mxfp8":
        err = err + 2.0 ** -13 * size
    off = got.double() - want
    assert bool((off.abs() <= err + HALF_STEP[name] * want.abs() * (1 + 2.0 ** -7)).all())
    # and far better than that over all: roundings do not add up in one direction
    rel = float(torch.linalg.norm(off) / torch.linalg.norm(want).clamp(min=1e-30))
    assert rel <= (2e-6 if name == "float32" else 2.0 ** -8), rel


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_matmul(sc, fmt, out):
    import torch
    for i, (m, n, d) in enumerate(MATMULS + [(9, 100, 8192), (300, 700, 4096)] + TILES):
        a, va = stored(sc, m, d, fmt, seed=200 + i)
        b, vb = stored(sc, n, d, "mxfp4", seed=300 + i)
        check_matmul(sc.mx_matmul(a, b, getattr(torch, out)), va, vb, fmt)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_matmul_into_strided_rows_and_nothing_else(sc, fmt):
    import torch
    for m, n, d in ((5, 70, 200), (300, 333, 256), (40, 260, 300), (60, 50003, 128), (100, 31001, 200), (300, 10501, 130)):
        a, va = stored(sc, m, d, fmt, seed=1, exact=True)
        b, vb = stored(sc, n, d, "mxfp4", seed=2, exact=True)
        for dtype in (torch.float32, torch.bfloat16):
            want = product(va, vb).to(dtype)
            for off in (0, 1, 3, 8):
                for more in (37, 44):
                    whole = torch.full((m + 2, n + more), -5.0, dtype=dtype, device="cuda")
                    out = whole[1:m + 1, off:off + n]
                    assert sc.mx_matmul(a, b, out=out) is out
                    assert torch.equal(out, want)
                    out.fill_(-5.0)
                    assert (whole == -5).all()
    a, va = stored(sc, 2, 64, fmt, seed=3, exact=True)
    b, vb = stored(sc, 50, 64, "mxfp4", seed=4, exact=True)
    far = torch.empty(2 ** 31 + 200, dtype=torch.float32, device="cuda").as_strided((2, 50), (2 ** 31 + 40, 1))
    assert torch.equal(sc.mx_matmul(a, b, out=far), product(va, vb).float())
    a, va = stored(sc, 70, 64, fmt, seed=3, exact=True)
    b, vb = stored(sc, 50000, 64, "mxfp4", seed=4, exact=True)
    far = torch.empty(69 * (2 ** 26) + 50000, dtype=torch.bfloat16, device="cuda").as_strided((70, 50000), (2 ** 26, 1))
    assert torch.equal(sc.mx_matmul(a, b, out=far), product(va, vb).bfloat16())


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_matmul_nan_blocks_stay_in_their_rows_and_columns(sc, fmt):
    import torch
    for m, n, d in ((3, 40, 256), (290, 300, 256), (50, 61000, 256), (290, 11000, 256)):
        a, va = stored(sc, m, d, fmt, seed=5)
        b, vb = stored(sc, n, d, "mxfp4", seed=6)
        a.scales[1, 2] = 255
        b.scales[7, 0] = 255
        for dtype in (torch.float32, torch.bfloat16):
            got = torch.isnan(sc.mx_matmul(a, b, dtype))
            want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
            want[1], want[:, 7] = True, True
            assert torch.equal(got, want)


def test_matmul_far_scales(sc):
    """Blocks whose scales are at the ends of their range."""
    import torch
    for m, n in ((2, 270), (280, 270), (280, 11000)):
        for fmt in ("mxfp8", "mxfp4"):
            a, va = stored(sc, m, 128, fmt, seed=7, exact=True)
            b, vb = stored(sc, n, 128, "mxfp4", seed=8, exact=True)
            want = product(va, vb)
            a.scales.fill_(127 + 100)
            b.scales.fill_(127 - 110)
            assert torch.equal(sc.mx_matmul(a, b), (want * 2.0 ** -10).float())
            a.scales.fill_(20)
            b.scales.fill_(250)
            assert torch.equal(sc.mx_matmul(a, b), (want * 2.0 ** 16).float())


# few rows, and every tile shape
UNEVEN = [(3, 300, 256), (290, 333, 1000), (64, 50001, 256), (128, 24001, 520), (300, 10111, 4096), (700, 24100, 300)]


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_matmul_keeps_small_products_beside_large_ones_that_cancel(sc, fmt, out):
    """Two pairs of large elements in each row of A whose products cancel exactly, the
    smallest elements beside them.  All products are whole multiples of one unit whose sums in
    any order stay below 2^24 of it: nothing may be rounded but the result."""
    import torch
    for i, (m, n, d) in enumerate(UNEVEN):
        rng = np.random.default_rng(40 + i)
        signed = lambda codes, f: codes + rng.integers(0, 2, size=codes.shape) * (8 if f == "mxfp4" else 128)  # noqa: E731
        b = signed(rng.integers(1, 8, size=(n, orc.padded(d))), "mxfp4")
        b_scales = np.full((n, orc.padded(d) // 32), 127, np.uint8)
        a_scales = np.full((m, orc.padded(d) // 32), 127, np.uint8)
        if fmt == "mxfp8":      # 1 .. 7 times 2^-9 beside 256 .. 448; the unit is 2^-10, 4 * 448 * 6 + 4096 * 7 * 2^-9 * 6 < 2^14
            a = signed(rng.integers(1, 8, size=(m, orc.padded(d))), fmt)
            a[:, [2, 40]] = signed(rng.integers(0x78, 0x7F, size=(m, 2)), fmt)
        else:                   # 0.5 .. 6 beside 2^12 times that in two blocks; the unit is 1/4, 4 * 36 * 2^12 + 4096 * 36 < 2^20
            a = signed(rng.integers(1, 8, size=(m, orc.padded(d))), fmt)
            a[:, :128] = 0
            a_scales[:, :4] = 127 + 12
            a[:, [2, 40]] = signed(rng.integers(1, 8, size=(m, 2)), fmt)
        a[:, [70, 101]] = a[:, [2, 40]]
        b[:, [70, 101]] = b[:, [2, 40]] ^ 8
        a[:, d:], b[:, d:] = 0, 0
        a, b = a.astype(np.uint8), b.astype(np.uint8)
        pa = sc.MxRows(torch.from_numpy(orc.pack(a, fmt)).cuda(), torch.from_numpy(a_scales).cuda(), d, fmt)
        pb = sc.MxRows(torch.from_numpy(orc.pack(b, "mxfp4")).cuda(), torch.from_numpy(b_scales).cuda(), d, "mxfp4")
        want = product(orc.mx_values(a, a_scales, fmt, d), orc.mx_values(b, b_scales, "mxfp4", d))
        assert torch.equal(sc.mx_matmul(pa, pb, getattr(torch, out)), want.to(getattr(torch, out))), (m, n, d)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_matmul_of_columns_of_far_magnitudes(sc, fmt, out):
    """As a model's hidden states are, a few columns far above the others.  An instruction
    adds 32 products or 128 to the running sum; d / 32 + 128 additions in a row at most, each off
    by one step of 32 bits (2 u) at most, and the result is rounded once."""
    import torch
    for i, (m, n, d) in enumerate(UNEVEN):
        g = torch.Generator(device="cuda").manual_seed(i)
        x = torch.randn(m, d, generator=g, device="cuda") * torch.exp(3 * torch.randn(1, d, generator=g, device="cuda"))
        a, b = sc.mx_quantize(x, fmt), sc.mx_quantize(torch.randn(n, d, generator=g, device="cuda"))
        va, vb = sc.mx_dequantize(a, torch.float32).double(), sc.mx_dequantize(b, torch.float32).double()
        want, size = va @ vb.t(), va.abs() @ vb.abs().t()
        got = sc.mx_matmul(a, b, getattr(torch, out)).double()
        assert bool(((got - want).abs() <= 2 * (d / 32 + 128) * U * size + HALF_STEP[out] * want.abs() * (1 + 2.0 ** -7)).all()), (m, n, d)


# around the sizes at which tiles take over from waves on their own, of 8- and of 4-bit rows: the last rows before
# and the first ones behind, and few rows against very many
CROSSINGS = [(1, 4_000_003, 100), (16, 400_001, 130), (17, 117_001, 130), (17, 118_001, 130), (64, 23_400, 200), (64, 23_500, 200),
             (64, 31_300, 200), (65, 30_700, 130), (128, 17_500, 100), (128, 17_700, 300), (129, 34_800, 100), (129, 35_003, 200), (1100, 4100, 300),
             (4_194_240, 1, 33), (4_194_241, 1, 33)]


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_matmul_where_waves_and_tiles_meet(sc, fmt):
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)

    def whole(n, d, fmt):       # 0, 1, 2, 3, 4, 6 of both signs
        few = torch.tensor([0, 2, 4, 5, 6, 7] if fmt == "mxfp4" else [0x00, 0x38, 0x40, 0x44, 0x48, 0x4C], dtype=torch.uint8, device="cuda")
        codes = few[torch.randint(0, 6, (n, orc.padded(d)), device="cuda", generator=g)]
        codes |= torch.randint(0, 2, codes.shape, device="cuda", generator=g, dtype=torch.uint8) << (3 if fmt == "mxfp4" else 7)
        codes[:, d:] = 0
        if fmt == "mxfp4":
            codes = codes[:, ::2] | codes[:, 1::2] << 4
        return sc.MxRows(codes.contiguous(), torch.full((n, orc.padded(d) // 32), 127, dtype=torch.uint8, device="cuda"), d, fmt)

    for m, n, d in CROSSINGS:
        a, b = whole(m, d, fmt), whole(n, d, "mxfp4")
        want = sc.mx_dequantize(a, torch.float32).double() @ sc.mx_dequantize(b, torch.float32).double().t()
        assert float(want.abs().max()) > 0
        for dtype in (torch.float32, torch.bfloat16):
            assert torch.equal(sc.mx_matmul(a, b, dtype), want.to(dtype)), (m, n, d)


def test_matmul_result_rows_start_on_128_bytes(sc):
    import torch
    a, _ = stored(sc, 3, 64, "mxfp8", seed=1)
    for n, dtype, stride in ((1023, torch.float32, 1023), (1024, torch.float32, 1024), (1025, torch.float32, 1056), (1025, torch.bfloat16, 1088)):
        got = sc.mx_matmul(a, stored(sc, n, 64, "mxfp4", seed=2)[0], dtype)
        assert got.shape == (3, n) and got.stride() == (stride, 1)


def test_matmul_rows_of_a_view_and_empty_operands(sc):
    import torch
    a, va = stored(sc, 40, 300, "mxfp8", seed=9, exact=True)
    b, vb = stored(sc, 90, 300, "mxfp4", seed=10, exact=True)
    got = sc.mx_matmul(a.rows(3, 9), b.rows(11, 88))
    assert torch.equal(got.cpu(), torch.from_numpy(va[3:9] @ vb[11:88].T).float())
    assert sc.mx_matmul(a.rows(0, 0), b).shape == (0, 90) and sc.mx_matmul(a, b.rows(5, 5)).shape == (40, 0)


# ---- log probabilities ---------------------------------------------------------------

def check_logprobs(sc, logits, tokens, top_k):
    """The sum of exponentials is a chain of at most v / 256 + 64 additions in fp32, each
    exponential good to 2 u and |z| 1.5 u (its rounded argument), z itself to u |z|.
    With r the largest |z| that counts (exp(-100) does not): the log of the sum is off
    by c = (v / 256 + 72 + 3 min(r, 100)) u, a log probability by that and 2 u of
    its value and of its parts, the entropy by c (1 + entropy + 1)."""
    got = sc.token_logprobs(logits, tokens, top_k)
    x = f64(logits)
    t = tokens.cpu().numpy() if tokens is not None else np.zeros((len(x), 0), np.int64)
    t = t[:, None] if t.ndim == 1 else t
    lp, entropy, ids, tlp = orc.token_logprobs(x, t, top_k)
    assert got.logprobs.shape == lp.shape and got.entropy.shape == entropy.shape and got.top_ids.shape == ids.shape
    assert np.array_equal(got.top_ids.cpu().numpy(), ids)
    finite = np.where(np.isfinite(x), x, np.nan)
    with np.errstate(all="ignore"):
        import warnings
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            reach = np.nan_to_num(np.nanmax(finite, 1) - np.nanmin(finite, 1))
    c = (x.shape[1] / 256 + 72 + 3 * np.minimum(reach, 100)) * U

    def near(a, b, tol):
        a = f64(a)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isneginf(a), np.isneginf(b))
        ok = np.isfinite(b)
        assert (np.abs(a[ok] - b[ok]) <= tol[ok]).all(), (np.abs(a[ok] - b[ok]).max(), tol[ok].max())
    near(got.logprobs, lp, np.broadcast_to(c[:, None], lp.shape) + 4 * U * np.abs(np.nan_to_num(lp, posinf=0, neginf=0)))
    near(got.top_logprobs, tlp, np.broadcast_to(c[:, None], tlp.shape) + 4 * U * np.abs(np.nan_to_num(tlp, posinf=0, neginf=0)))
    near(got.entropy, entropy, c * (2 + np.nan_to_num(entropy)))
    return got


def logits_of(n, v, dtype, seed, spread=3.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, v, generator=g) * spread).to(getattr(torch, dtype)).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs(sc, dtype):
    import torch
    for i, (n, v, g, k) in enumerate([(1, 1, 1, 1), (1, 2, 1, 64), (3, 7, 2, 3), (5, 64, 1, 5), (2, 65, 3, 64), (4, 1000, 1, 0), (9, 4097, 2, 1),
                                      (1, 8192, 2, 20), (2, 50257, 1, 20), (40, 3001, 7, 64), (1, 131072, 2, 20), (1, 262143, 1, 64), (300, 515, 1, 2)]):
        x = logits_of(n, v, dtype, seed=i)
        t = torch.randint(0, v, (n, g), generator=torch.Generator().manual_seed(i)).cuda()
        check_logprobs(sc, x, t, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [100, 9000, 40000])
def test_masked_rows_and_rows_without_a_distribution(sc, dtype, v):
    import torch
    x = logits_of(12, v, dtype, seed=5)
    low = torch.finfo(x.dtype).min
    inf = float("inf")
    x[1] = -inf                                     # nothing left
    x[2] = -inf
    x[2, v - 1] = 3.0                               # one token left
    x[3, torch.rand(v, generator=torch.Generator().manual_seed(1)).cuda() < 0.9] = -inf
    x[4] = low                                      # uniform at the lowest value
    x[5, : v // 2] = low
    x[6, v // 3] = float("nan")
    x[7, v // 2] = inf
    x[8] = float("nan")
    x[9, 1:] = -inf
    x[9, 0] = low
    x[10, v // 2:] = -inf
    x[11] = torch.finfo(x.dtype).max
    t = torch.tensor([[0, v - 1, v // 3, -1, -100, v, 2 ** 40]]).expand(12, 7).contiguous().cuda()
    got = check_logprobs(sc, x, t, 64)
    assert (got.logprobs[1, :3] == -inf).all() and got.entropy[1] == 0 and (got.top_ids[1] == -1).all()
    assert got.logprobs[2, 1] == 0 and got.entropy[2] == 0 and got.top_ids[2, 0] == v - 1 and (got.top_ids[2, 1:] == -1).all()
    check_logprobs(sc, x, t[:, :2], 0)


def test_ties_go_to_the_lower_id(sc):
    import torch
    for v in (50, 700, 20000, 100000):
        for levels in (1, 2, 5):
            x = torch.randint(0, levels, (4, v), generator=torch.Generator().manual_seed(levels)).float()
            x[1] *= -0.0                            # zeros of both signs are equal
            check_logprobs(sc, x.cuda(), None, 64)
            check_logprobs(sc, x.to(torch.bfloat16).cuda(), None, 7)
    rising = torch.arange(30000, dtype=torch.float32).expand(2, 30000).contiguous().cuda()     # every logit enters the list
    check_logprobs(sc, rising, None, 64)
    check_logprobs(sc, rising.flip(1).contiguous(), None, 64)


@pytest.mark.parametrize("top_k", [11, 12, 13, 20, 48, 49])
def test_alternatives_sorted_at_once_or_one_by_one(sc, top_k):
    """Few and many candidates in the first and in later parts of a row, in orders that bring all or none of them late."""
    import torch
    for n, v in ((3, 20), (2, 300), (2, 5000), (5, 30000), (2, 140000)):
        x = logits_of(n, v, "float32", seed=v)
        check_logprobs(sc, x, None, top_k)
        check_logprobs(sc, x.sort(dim=1).values.contiguous(), None, top_k)
        check_logprobs(sc, x.sort(dim=1, descending=True).values.to(torch.bfloat16), None, top_k)
        check_logprobs(sc, x.round().to(torch.float16), None, top_k)            # ties by the hundred
        few = torch.full_like(x, -float("inf"))
        few[:, ::max(1, v // 13)] = x[:, ::max(1, v // 13)]
        check_logprobs(sc, few, None, top_k)


def test_logits_strided_misaligned_and_far_apart(sc):
    import torch
    for dtype in DTYPES:
        whole = logits_of(7, 9001, dtype, seed=2)
        for view in (whole[:, 1:], whole[:, :9000], whole[1::2, 3:8195], whole.t()[:50], whole[:, ::2], whole[2:3].expand(4, 9001)):
            check_logprobs(sc, view, torch.zeros(len(view), dtype=torch.int64, device="cuda"), 5)
    far = torch.empty(2 * (2 ** 32 + 3) + 6000, dtype=torch.bfloat16, device="cuda").as_strided((3, 5000), (2 ** 32 + 3, 1))
    far.copy_(logits_of(3, 5000, "bfloat16", seed=3))
    check_logprobs(sc, far, torch.tensor([4999, 0, 17], device="cuda"), 3)
    assert sc.token_logprobs(far[:0], far[:0, 0].long(), 3).top_ids.shape == (0, 3)


def test_rms_norm_more_rows_than_one_launch_counts(sc):
    import torch
    n, d = 17_000_000, 513
    x, res, w = rows(1, d, "bfloat16", seed=1), rows(1, d, "bfloat16", seed=2), rows(1, d, "bfloat16", seed=3)[0]
    got, h = sc.rms_norm_mx(x.expand(n, d), w, residual=res.expand(n, d), format="mxfp4")
    one, h1 = sc.rms_norm_mx(x, w, residual=res, format="mxfp4")
    words, want, step = got.values.view(torch.int64), one.values.view(torch.int64), 1 << 22
    for lo in range(0, n, step):
        assert (words[lo:lo + step] == want).all() and (got.scales[lo:lo + step] == one.scales).all() and (h[lo:lo + step] == h1).all()


# ---- how they are called ---------------------------------------------------------------

def test_refusals(sc):
    import torch
    x = torch.zeros(4, 64, device="cuda")
    q4, q8 = sc.mx_quantize(x), sc.mx_quantize(x, "mxfp8")
    for error, call in (
            (TypeError, lambda: sc.mx_quantize(x.double())), (TypeError, lambda: sc.mx_quantize(x.int())), (ValueError, lambda: sc.mx_quantize(x[0])),
            (ValueError, lambda: sc.mx_quantize(x, "mxfp6")), (ValueError, lambda: sc.mx_quantize(x.clone().requires_grad_())),
            (ValueError, lambda: sc.mx_quantize(x[:, :0])),
            (TypeError, lambda: sc.mx_dequantize(q4, torch.float64)), (ValueError, lambda: sc.mx_dequantize(q4, out=torch.zeros(4, 65, device="cuda"))),
            (ValueError, lambda: sc.mx_dequantize(q4, out=torch.zeros(64, 4, device="cuda").t())),
            (ValueError, lambda: sc.mx_dequantize(q4, out=torch.zeros(1, 64, device="cuda").expand(4, 64))),
            (ValueError, lambda: sc.MxRows(q4.values, q4.scales, 200)), (ValueError, lambda: sc.MxRows(q4.values, q4.scales, 64, "mxfp8")),
            (ValueError, lambda: sc.MxRows(q4.values[:2], q4.scales, 64)), (ValueError, lambda: sc.MxRows(q4.values.t(), q4.scales, 64)),
            (ValueError, lambda: sc.rms_norm_mx(x, x[0, :32])), (ValueError, lambda: sc.rms_norm_mx(x, x[0].half())),
            (ValueError, lambda: sc.rms_norm_mx(x, x[0], residual=x[:2])), (ValueError, lambda: sc.rms_norm_mx(x, x[0], residual=x.half())),
            (ValueError, lambda: sc.rms_norm_mx(x, x[0], -1.0)), (ValueError, lambda: sc.rms_norm_mx(x, x[0].clone().requires_grad_())),
            (ValueError, lambda: sc.rms_norm_mx(torch.zeros(1, 65537, device="cuda"), torch.zeros(65537, device="cuda"))),
            (ValueError, lambda: sc.mx_matmul(q4, q8)), (ValueError, lambda: sc.mx_matmul(q8, sc.mx_quantize(x[:, :32]))),
            (TypeError, lambda: sc.mx_matmul(q8, q4, torch.float16)), (ValueError, lambda: sc.mx_matmul(q8, q4, out=torch.zeros(4, 5, device="cuda"))),
            (ValueError, lambda: sc.mx_matmul(q8, q4, out=torch.zeros(1, 4, device="cuda").expand(4, 4))),
            (ValueError, lambda: sc.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda"))),
            (ValueError, lambda: sc.token_logprobs(x, torch.zeros(4, dtype=torch.int32, device="cuda"))),
            (ValueError, lambda: sc.token_logprobs(x, torch.zeros(4, dtype=torch.int64))), (ValueError, lambda: sc.token_logprobs(x, None, 65)),
            (ValueError, lambda: sc.token_logprobs(x[:, :0])), (TypeError, lambda: sc.token_logprobs(x.double()))):
        with pytest.raises(error):
            call()
    with torch.no_grad():
        sc.mx_quantize(x.clone().requires_grad_())


def test_copies_have_their_own_memory(sc):
    """deepcopy and pickle of rows made in one allocation, of given tensors and of a view."""
    import copy
    import pickle

    import torch
    made = sc.mx_quantize(rows(5, 200, "float32"), "mxfp8")
    given = sc.MxRows(made.values.clone(), made.scales.clone(), 200, "mxfp8")
    for r in (made, given, made.rows(1, 4)):
        want = sc.mx_dequantize(r, torch.float32)
        copies = [copy.deepcopy(r), pickle.loads(pickle.dumps(r))]
        kept = r.values.clone()
        r.values.zero_()
        for c in copies:
            assert torch.equal(sc.mx_dequantize(c, torch.float32), want) and (len(c), c.d, c.format) == (len(r), 200, "mxfp8")
        r.values.copy_(kept)


def test_out_is_seen_by_autograd(sc):
    """A tensor that a recorded operation needs is overwritten: its backward pass says so; one that records is refused."""
    import torch
    x = torch.ones(4, 64, device="cuda")
    q4, q8 = sc.mx_quantize(x), sc.mx_quantize(x, "mxfp8")
    for call, shape in ((lambda o: sc.mx_dequantize(q4, out=o), (4, 64)), (lambda o: sc.mx_matmul(q8, q4, out=o), (4, 4))):
        out, w = torch.zeros(shape, device="cuda"), torch.ones(shape, device="cuda", requires_grad=True)
        y = (out * w).sum()
        assert call(out) is out and bool((out != 0).all())
        with pytest.raises(RuntimeError):
            y.backward()
        with pytest.raises(ValueError):
            call(w)
        with pytest.raises(ValueError):
            call(out.cpu())


def head(sc, x, res, w, vocab, tokens):
    y, h = sc.rms_norm_mx(x, w, 1e-6, res)
    return (h,) + tuple(sc.token_logprobs(sc.mx_matmul(y, vocab), tokens, 5))


def test_the_head_as_a_run(sc):
    """Residual, norm, vocabulary product, log probabilities, one behind the other:
    against the same steps in 64 bits on the 8-bit rows the norm gave."""
    import torch
    for n, d, v in ((1, 256, 1000), (34, 1024, 5003), (300, 512, 2000)):
        x, res = rows(n, d, "bfloat16", seed=1), rows(n, d, "bfloat16", seed=2)
        w = rows(1, d, "bfloat16", seed=3)[0]
        vocab = sc.mx_quantize(rows(v, d, "bfloat16", seed=4, spread=0.1), "mxfp4")
        tokens = torch.randint(0, v, (n, 2), generator=torch.Generator().manual_seed(5)).cuda()
        h, lp, entropy, ids, tlp = head(sc, x, res, w, vocab, tokens)
        y, _ = sc.rms_norm_mx(x, w, 1e-6, res)
        a, b = f64(sc.mx_dequantize(y, torch.float32)), f64(sc.mx_dequantize(vocab, torch.float32))
        want = a @ b.T
        slack = d * U * (np.abs(a) @ np.abs(b).T).max(axis=1)       # of a logit
        wlp, went, _, _ = orc.token_logprobs(want, tokens.cpu().numpy(), 0)
        tol = (2 * slack + (v / 256 + 400) * U)[:, None]
        assert (np.abs(f64(lp) - wlp) <= tol + 4 * U * np.abs(wlp)).all()
        # the alternatives are the best logits, to within what two logits may be off
        best = -np.sort(-want, axis=1)[:, :5]
        assert (np.abs(np.take_along_axis(want, ids.cpu().numpy(), 1) - best) <= 2 * slack[:, None]).all()


@pytest.mark.parametrize("n", [3, 300])
def test_captured_and_replayed(sc, n):
    """The head in a HIP graph, replayed on new inputs with eager work in between."""
    import torch
    d, v = 300, 20000
    x, res, w = rows(n, d, "bfloat16", seed=1), rows(n, d, "bfloat16", seed=2), rows(1, d, "bfloat16", seed=3)[0]
    vocab = sc.mx_quantize(rows(v, d, "bfloat16", seed=4, spread=0.1), "mxfp4")
    tokens = torch.arange(n, device="cuda")[:, None].contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        head(sc, x, res, w, vocab, tokens)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = head(sc, x, res, w, vocab, tokens)
    with torch.cuda.graph(other):
        got2 = head(sc, res, x, w, vocab, tokens)
    for i in range(4):
        x.copy_(rows(n, d, "bfloat16", seed=10 + i))
        res.copy_(rows(n, d, "bfloat16", seed=20 + i))
        tokens.copy_(torch.randint(0, v, (n, 1), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        for g, want in ((got, head(sc, x, res, w, vocab, tokens)), (got2, head(sc, res, x, w, vocab, tokens))):
            for a, b in zip(g, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("n", [1, 64, 130])
def test_on_two_streams_at_once_and_twice_the_same(sc, n):
    import torch
    x, res, w = rows(n, 1024, "bfloat16", seed=1), rows(n, 1024, "bfloat16", seed=2), rows(1, 1024, "bfloat16", seed=3)[0]
    vocab = sc.mx_quantize(rows(30000, 1024, "bfloat16", seed=4, spread=0.1), "mxfp4")
    tokens = torch.randint(0, 30000, (n, 1), generator=torch.Generator().manual_seed(5)).cuda()
    want = head(sc, x, res, w, vocab, tokens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for s, out in zip(streams, got):
            with torch.cuda.stream(s):
                out.append(head(sc, x, res, w, vocab, tokens))
    torch.cuda.synchronize()
    for out in got:
        for run in out:
            for a, b in zip(run, want):
                assert torch.equal(a, b)


def test_dual_tensors_are_refused(sc):
    """The kernels would drop a forward-mode tangent without a word."""
    import torch
    from torch.autograd import forward_ad
    x, w = rows(3, 64, "float32"), torch.ones(64, device="cuda")
    packed = sc.mx_quantize(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: sc.mx_quantize(dual), lambda: sc.rms_norm_mx(dual, w), lambda: sc.rms_norm_mx(x, w, 1e-6, dual),
                     lambda: sc.rms_norm_mx(x, forward_ad.make_dual(w, torch.ones_like(w))), lambda: sc.token_logprobs(dual),
                     lambda: sc.mx_dequantize(packed, out=dual), lambda: sc.mx_matmul(packed, packed, out=dual[:, :3])):
            with pytest.raises(ValueError):
                call()
        check_quantized(sc.mx_quantize(forward_ad.unpack_dual(dual).primal), f64(x), "mxfp4")


def test_a_refused_out_counts_as_untouched(sc):
    """A call refused for its out's shape, type or strides leaves a backward pass that saved it fine."""
    import torch
    packed = sc.mx_quantize(rows(3, 64, "float32"))
    w = torch.ones(3, 65, device="cuda", requires_grad=True)
    out = torch.ones(3, 65, device="cuda")
    loss = (w * out).sum()
    version = out._version
    for call in (lambda: sc.mx_dequantize(packed, out=out), lambda: sc.mx_matmul(packed, packed, out=out), lambda: sc.mx_matmul(packed, packed, out=out[:, ::2]),
                 lambda: sc.mx_dequantize(packed, torch.bfloat16, out=out[:, :64]), lambda: sc.mx_matmul(packed, packed, out=out[:1].expand(3, 65)[:, :3]),
                 lambda: sc.mx_dequantize(packed, out=out[:1].expand(3, 65)[:, :64])):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            call()
    half = torch.ones(3, 3, dtype=torch.float16, device="cuda")
    with pytest.raises(TypeError):
        sc.mx_matmul(packed, packed, out=half)
    assert out._version == version and half._version == 0
    loss.backward()
    assert torch.equal(w.grad, out)
    sc.mx_dequantize(packed, out=out[:, :64])
    assert out._version > version


def test_lazily_negated_tensors(sc):
    """The imaginary part of a conjugate holds the other sign in memory; one column of it needs no copy for its strides."""
    import torch
    z = torch.complex(rows(5, 40, "float32", seed=1), rows(5, 40, "float32", seed=2)).conj()
    for cols in (slice(0, 1), slice(0, 40)):
        x = z[:, cols].imag
        assert x.is_neg()
        plain = x.resolve_neg().contiguous()
        assert not plain.is_neg() and torch.equal(plain, x + 0)
        check_quantized(sc.mx_quantize(x), f64(plain), "mxfp4")
        for w, res in ((torch.ones(x.shape[1], device="cuda"), x), (z[0, cols].imag, plain)):
            got, want = sc.rms_norm_mx(x, w, 1e-6, res), sc.rms_norm_mx(plain, w.resolve_neg().contiguous(), 1e-6, plain)
            assert torch.equal(got[1], want[1]) and torch.equal(got[0].values, want[0].values) and torch.equal(got[0].scales, want[0].scales)
        assert torch.equal(sc.token_logprobs(x, top_k=1).top_ids, sc.token_logprobs(plain, top_k=1).top_ids)
        packed = sc.mx_quantize(plain)
        with pytest.raises(ValueError):
            sc.mx_dequantize(packed, out=z[:, cols].imag)


@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-33, 1e-6])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rms_norm_of_rows_whose_squares_underflow(sc, dtype, eps):
    """Squares below what 32 bits hold, down to the smallest numbers, with an eps above, among or below them; a zero
    row gives zeros without an eps too.  Every width of a workgroup."""
    import torch
    for d in (1, 33, 512, 1000, 2049, 5000, 9000):
        x = rows(8, d, "float32", seed=d, spread=0.0)
        for i, scale in enumerate((1.0, 1e-14, 1e-16, 1e-19, 1e-22, 1e-30, 1e-38, 1e-42)):
            x[i] *= scale
        x = x.to(getattr(torch, dtype))
        w = rows(1, d, "float32", seed=d + 1)[0]
        x = x[(x != 0).any(dim=1)]      # one element may have rounded to zero
        check_norm(sc, x, w, float(torch.tensor(eps)), None, "mxfp8")
        check_norm(sc, x, w, float(torch.tensor(eps)), 0 * x, "mxfp4")
        zero = torch.zeros(3, d, dtype=x.dtype, device="cuda")
        zero[1] = x[0]
        y = sc.mx_dequantize(sc.rms_norm_mx(zero, w, eps)[0], torch.float32)
        assert (y[0] == 0).all() and (y[2] == 0).all() and torch.equal(y[1:2], sc.mx_dequantize(sc.rms_norm_mx(x[:1], w, eps)[0], torch.float32))
