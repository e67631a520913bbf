"""CPU-side checks of the scoring head: its oracle against independent conversions,
and every refusal that needs no GPU."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import scoring_oracle as orc


def test_oracle_elements_are_the_formats():
    """The e4m3 list against torch's type, the e2m1 list against its definition."""
    codes = torch.arange(127, dtype=torch.uint8)
    assert np.array_equal(orc.GRID["mxfp8"], codes.view(torch.float8_e4m3fn).double().numpy())
    e2m1 = [(m / 2 if e == 0 else (1 + m / 2) * 2 ** (e - 1)) for e in range(4) for m in range(2)]
    assert orc.GRID["mxfp4"].tolist() == e2m1


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_oracle_rounds_to_nearest_even_within_half_a_step(fmt):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 200)) * np.exp(rng.standard_normal((40, 200)))
    codes, scales = orc.mx_quantize(x, fmt)
    assert codes.shape == (40, 256) and scales.shape == (40, 8)
    assert np.array_equal(orc.unpack(orc.pack(codes, fmt), fmt), codes)
    back = orc.mx_values(codes, scales, fmt, 200)
    unit = np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, axis=1)[:, :200]
    bits, low = (1, 0) if fmt == "mxfp4" else (3, -6)
    step = np.ldexp(1.0, np.maximum(np.frexp(np.abs(x) / unit)[1] - 1, low) - bits) * unit
    assert (np.abs(back - x) <= step / 2).all()
    if fmt == "mxfp8":      # the same elements as torch's conversion of the scaled values
        want = torch.from_numpy(np.pad(x / unit, ((0, 0), (0, 56)))).clamp(-448, 448).to(torch.float8_e4m3fn)
        assert np.array_equal(want.view(torch.uint8).numpy(), codes)
    # no smaller scale would do
    amax = np.abs(np.pad(x, ((0, 0), (0, 56)))).reshape(40, -1, 32).max(2)
    with np.errstate(divide="ignore"):
        r = amax / np.ldexp(1.0, scales.astype(int) - 127 - 1)
    assert ((r >= 7) if fmt == "mxfp4" else (r > 464))[amax > 0].all()


def test_oracle_scale_borders():
    for fmt, below, above in (("mxfp4", 6.999, 7.0), ("mxfp8", 464.0, 464.001)):
        for e in (-20, 0, 90):
            assert orc.mx_scale(np.float64(below * 2.0 ** e), fmt) == e
            assert orc.mx_scale(np.float64(above * 2.0 ** e), fmt) == e + 1
        assert orc.mx_scale(np.float64(2.0 ** -140), fmt) == -127 and orc.mx_scale(np.float64(0), fmt) == -127


def test_oracle_log_probabilities_against_torch():
    torch.manual_seed(0)
    x = torch.randn(7, 50, dtype=torch.float64) * 4
    lp, entropy, ids, tlp = orc.token_logprobs(x.numpy(), np.arange(14).reshape(7, 2), 5)
    want = torch.log_softmax(x, 1)
    np.testing.assert_allclose(lp, want.gather(1, torch.arange(14).reshape(7, 2)).numpy(), rtol=1e-12)
    np.testing.assert_allclose(entropy, torch.distributions.Categorical(logits=x).entropy().numpy(), rtol=1e-12)
    assert np.array_equal(ids, x.topk(5).indices.numpy())
    np.testing.assert_allclose(tlp, want.topk(5).values.numpy(), rtol=1e-12)


def refuses(rc, *words):
    from medical_rag_amd import _native
    assert rc == _native.MTR_ERR_INVALID
    for w in words:
        assert w in _native.last_error(), _native.last_error()


def test_c_refusals_come_before_any_hip_call():
    """No GPU here: a call that got past its checks would fail with another code."""
    from medical_rag_amd import _native
    lib = _native.lib()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 63) // 64 * 64
    vp = ctypes.c_void_p
    q = lambda x=at, dt=0, n=2, d=8, ld=8, f=0, v=at, s=at: lib.mtr_mx_quantize(vp(x), dt, n, d, ld, f, vp(v), vp(s), 0, None)  # noqa: E731
    refuses(q(dt=1), "dtype")
    refuses(q(f=2), "format")
    refuses(q(n=-1), "shape")
    refuses(q(d=0), "shape")
    refuses(q(d=2 ** 31 - 1), "shape")
    refuses(q(n=2 ** 31, d=8), "shape")
    refuses(q(n=2 ** 24, d=2 ** 20), "shape")
    refuses(q(n=2 ** 62, d=512), "shape")
    refuses(q(x=None), "NULL")
    refuses(q(v=None), "NULL")
    refuses(q(s=None), "NULL")
    refuses(q(v=at + 8), "16 bytes")
    refuses(q(s=at + 2), "on 4")
    refuses(q(x=at + 2), "address")
    refuses(q(ld=-1), "stride")
    assert q(n=0, x=None, v=None, s=None) == _native.MTR_OK
    dq = lambda o=at, dt=0, n=2, d=8, ld=8, f=0: lib.mtr_mx_dequantize(vp(at), vp(at), f, n, d, vp(o), dt, ld, 0, None)  # noqa: E731
    refuses(dq(dt=9), "dtype")
    refuses(dq(f=-1), "format")
    refuses(dq(o=None), "NULL")
    refuses(dq(ld=7), "stride")
    refuses(dq(o=at + 1, dt=2), "address")
    assert dq(n=0) == _native.MTR_OK

    def norm(x=at, r=None, w=at, dt=2, wdt=2, n=2, d=8, ldx=8, ldr=8, eps=1e-6, f=1, ro=None):
        return lib.mtr_rms_norm_mx(vp(x), vp(r), vp(w), dt, wdt, n, d, ldx, ldr, eps, f, vp(ro), vp(at), vp(at), 0, None)
    refuses(norm(wdt=3), "weight")
    refuses(norm(d=65537), "65536")
    refuses(norm(eps=-1.0), "eps")
    refuses(norm(eps=float("nan")), "eps")
    refuses(norm(r=at), "together")
    refuses(norm(ro=at), "together")
    refuses(norm(r=at, ro=at + 1024, x=at + 1024), "of its own")
    refuses(norm(r=at, ro=at, x=at + 1024), "of its own")
    refuses(norm(w=None), "NULL")
    refuses(norm(x=at + 1), "address")
    refuses(norm(ldx=-8), "stride")
    assert norm(n=0) == _native.MTR_OK

    def mm(av=at, af=1, m=2, bv=at, n=2, d=8, o=at, dt=0, ld=2, w=None, wb=0):
        return lib.mtr_mx_matmul(vp(av), vp(at), af, m, vp(bv), vp(at), n, d, vp(o), dt, ld, vp(w), wb, 0, None)
    refuses(mm(dt=3), "output dtype")
    refuses(mm(af=5), "format")
    refuses(mm(av=at + 4), "16 bytes")
    refuses(mm(bv=None), "NULL")
    refuses(mm(o=None), "NULL")
    refuses(mm(ld=1), "stride")
    refuses(mm(m=-1), "shape")
    refuses(mm(n=2 ** 29 + 1, ld=2 ** 30), "shape")
    refuses(mm(m=2 ** 29 + 1), "shape")
    assert lib.mtr_mx_matmul_workspace(4, 2 ** 29 + 1, 8) == 0
    assert lib.mtr_mx_matmul_workspace(3000, 5000, 1000) > 0 and lib.mtr_mx_matmul_workspace(0, 5, 5) == 0
    refuses(mm(m=3000, n=5000, d=1000, ld=5000), "workspace")
    refuses(mm(m=3000, n=5000, d=1000, ld=5000, w=at, wb=64), "workspace")
    refuses(mm(m=3000, n=5000, d=1000, ld=5000, w=at + 2, wb=1 << 30), "workspace")
    assert mm(m=0, o=None) == _native.MTR_OK and mm(n=0, o=None) == _native.MTR_OK

    def lp(x=at, dt=0, n=2, v=100, ld=100, t=at, g=1, k=0, l=at, e=at, ti=at, tl=at, w=at, wb=1 << 20):
        return lib.mtr_token_logprobs(vp(x), dt, n, v, ld, vp(t), g, k, vp(l), vp(e), vp(ti), vp(tl), vp(w), wb, 0, None)
    refuses(lp(dt=1), "dtype")
    refuses(lp(v=0), "shape")
    refuses(lp(v=2 ** 31), "shape")
    refuses(lp(n=-1), "shape")
    refuses(lp(n=2 ** 30), "shape")
    refuses(lp(k=65), "top_k")
    refuses(lp(k=-1), "top_k")
    refuses(lp(g=-1), "n_tokens")
    refuses(lp(t=None), "NULL")
    refuses(lp(e=None), "NULL")
    refuses(lp(k=1, ti=None), "NULL")
    refuses(lp(t=at + 4), "address")
    assert lib.mtr_token_logprobs_workspace(1, 131072, 20) > 0
    refuses(lp(n=1, v=131072, ld=131072, k=20, wb=16), "workspace")
    refuses(lp(n=1, v=131072, ld=131072, k=20, w=None), "workspace")
    assert lp(n=0, x=None, e=None) == _native.MTR_OK
    assert lib.mtr_token_logprobs_workspace(-1, 5, 1) == 0 and lib.mtr_token_logprobs_workspace(4, 0, 1) == 0


def test_python_refuses_what_is_not_on_a_gpu():
    from medical_rag_amd import scoring
    x = torch.zeros(4, 64)
    for call in (lambda: scoring.mx_quantize(x), lambda: scoring.mx_quantize(np.zeros((2, 3))), lambda: scoring.rms_norm_mx(x, torch.ones(64)),
                 lambda: scoring.token_logprobs(x), lambda: scoring.MxRows(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 64)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        scoring.MxRows(None, None, 8, "int4")
    with pytest.raises(ValueError):
        scoring.MxRows(None, None, 0)
    for d in (2 ** 31, 2 ** 32 + 5):        # would reach the library as another width
        with pytest.raises(ValueError):
            scoring.MxRows.empty(1, d, "mxfp4", "cpu")


def test_constants_match_the_header():
    import re

    from medical_rag_amd import _native
    from test_abi_cpu import HEADER
    text = open(HEADER).read()
    for name in ("MTR_MX_BLOCK", "MTR_MX_PAD", "MTR_RMS_NORM_MAX_WIDTH", "MTR_MAX_ALTERNATIVES"):
        assert int(re.search(rf"#define {name} (\d+)", text).group(1)) == getattr(_native, name)
    for name in ("MTR_MX_FP4", "MTR_MX_FP8"):
        assert int(re.search(rf"{name} = (\d+)", text).group(1)) == getattr(_native, name)


def test_products_of_few_rows_want_no_workspace():
    """One to 16 rows take the kernel that reads B once, however many rows it has; a workspace for all
    of B's scales would belong to the other one."""
    from medical_rag_amd import _native
    need = _native.lib().mtr_mx_matmul_workspace
    for m, n, d in ((1, 4_000_000, 768), (1, 2 ** 29, 64), (12, 262144, 4096), (16, 262144, 2048), (16, 10_000_000, 1024)):
        assert need(m, n, d) == 0, (m, n, d)
    for m, n, d in ((17, 262144, 2048), (64, 131072, 4096), (2048, 131072, 4096), (2 ** 29, 1, 32), (5_000_000, 1, 32)):
        assert need(m, n, d) > 0, (m, n, d)


def test_tensors_with_derivatives_are_refused():
    from torch.autograd import forward_ad

    from medical_rag_amd import scoring
    x = torch.zeros(4, 64)
    scoring._no_derivative(x, "it")
    recorded = x.clone().requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        scoring._no_derivative(recorded, "it")
    with torch.no_grad():
        scoring._no_derivative(recorded, "it")
    with forward_ad.dual_level():
        scoring._no_derivative(x, "it")
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for t in (dual, dual[1:], dual.t(), dual * 2):
            with pytest.raises(ValueError, match="forward"):
                scoring._no_derivative(t, "it")
        scoring._no_derivative(forward_ad.unpack_dual(dual).primal, "it")
