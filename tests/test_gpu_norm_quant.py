"""Residual addition + RMS norm + 8-bit output against 64-bit arithmetic.

Tolerances. h is one rounding of an f32 sum: equal. y is computed in double
and rounded twice to f32 (after the scaled product, after the weight): within
2^-23 of the exact value, relatively. An int8 code is the nearest one, so
|code * scale - y| <= scale / 2, plus y's own error (below 2^-22 |y|) and the
2^-24 of the scale; an e4m3 code is within 2^-4 of the value (half a step of 3
fraction bits), or half the smallest step, 2^-10, of the block's scale."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["f32", "bf16", "f16"]


def _dt(t):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[t]


def _run(rb, x, r, w, fmt, eps=1e-5, h=None):
    import torch
    rows, cols = x.shape
    h = torch.empty_like(x) if r is not None and h is None else h
    codes = torch.empty(rows, cols, dtype=torch.int8 if fmt == 0 else torch.uint8, device=x.device)
    scales = (torch.full((rows,), np.nan, device=x.device) if fmt == 0 else
              torch.zeros(rows, cols // 32, dtype=torch.uint8, device=x.device))
    rb.add_rmsnorm_quant(x, r, w, eps, fmt, codes, scales, h)
    rb.sync_status()
    return h, codes, scales


def _check(x, r, w, fmt, h, codes, scales, eps=1e-5):
    import torch
    want_h = x if r is None else (x.float() + r.float()).to(x.dtype)
    if r is not None:
        assert torch.equal(h, want_h)
    hd = want_h.double()
    y = hd / torch.sqrt(hd.square().mean(1, keepdim=True) + eps) * w.double()
    if fmt == 0:
        amax = y.abs().amax(1)
        s = torch.where(amax > 0, amax / 127, 1.0)
        assert ((scales.double() - s).abs() <= s * 2.0 ** -21).all()
        d = (codes.double() * scales.double()[:, None] - y).abs()
        assert (d <= s[:, None] * (0.5 + 2.0 ** -15) + y.abs() * 2.0 ** -21).all()
    else:
        b = y.unflatten(1, (-1, 32))
        step = torch.pow(2.0, scales.double() - 127)[..., None]
        amax = b.abs().amax(-1, keepdim=True)
        assert (scales >= 128).all()
        assert (amax <= 224 * step * (1 + 2.0 ** -20)).all()
        assert ((step == 2) | (amax > 112 * step * (1 - 2.0 ** -20))).all()
        v = codes.view(torch.float8_e4m3fn).double().unflatten(1, (-1, 32)) * step
        assert ((v - b).abs() <= b.abs() * (2.0 ** -4 + 2.0 ** -20) + step * 2.0 ** -10).all()


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (7, 512), (5, 544), (9, 1024), (2, 2016), (33, 4096),
                                       (17, 5120), (3, 8192), (4, 12288), (2, 16384), (3, 16416), (2, 40000)])
def test_shapes(rb, cuda, rows, cols, t, fmt):
    import torch
    g = torch.Generator("cuda").manual_seed(rows * cols)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, r, w = (20 * rn(rows, cols)).to(_dt(t)), rn(rows, cols).to(_dt(t)), rn(cols)
    _check(x, r, w, fmt, *_run(rb, x, r, w, fmt))
    _check(x, None, w, fmt, *_run(rb, x, None, w, fmt))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", [4, 12, 36, 100, 516, 1028])
def test_int8_columns_of_four(rb, cuda, t, cols):
    import torch
    g = torch.Generator("cuda").manual_seed(cols)
    x, r = ((torch.randn(6, cols, generator=g, device="cuda")).to(_dt(t)) for _ in range(2))
    w = torch.ones(cols, device="cuda")
    _check(x, r, w, 0, *_run(rb, x, r, w, 0))


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_strides_and_in_place(rb, cuda, t, fmt):
    import torch
    g = torch.Generator("cuda").manual_seed(5)
    big = torch.randn(11, 352, generator=g, device="cuda").to(_dt(t))
    x, r = big[:, 16:272], torch.randn(11, 264, generator=g, device="cuda").to(_dt(t))[:, 4:260]  # (8-byte rows)
    r = r if t == "bf16" else big[:, 64:320]
    w = torch.randn(256, generator=g, device="cuda")
    _check(x, r, w, fmt, *_run(rb, x, r, w, fmt))
    for target in (0, 1):  # the sum replaces x or the residual
        xs, rs = x.contiguous(), r.contiguous()
        args = (xs.clone(), rs.clone())
        h, codes, scales = _run(rb, args[0], args[1], w, fmt, h=args[target])
        _check(xs, rs, w, fmt, h, codes, scales)


def test_equals_the_separate_steps(rb, cuda):
    """The codes and scales of rouge_rmsnorm followed by the quantizers, bit for bit."""
    import ctypes as C

    import torch
    L = rb.lib()
    L.rouge_rmsnorm.argtypes, L.rouge_rmsnorm.restype = [C.c_void_p, C.c_int, C.c_void_p, C.c_float, C.c_void_p], None
    rng = np.random.default_rng(3)
    for cols in (256, 4096):
        x = (rng.standard_normal((5, cols)) * np.exp(rng.uniform(-30, 30, (5, 1)))).astype(np.float32)
        x[3] = 0
        w = rng.uniform(0.5, 1.5, cols).astype(np.float32)
        y = np.empty_like(x)
        p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
        for i in range(5):
            L.rouge_rmsnorm(p(x[i]), cols, p(w), 1e-5, p(y[i]))
        yd = torch.from_numpy(y).cuda()
        q, s = torch.empty(5, cols, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
        rb.quantize_i8_rows(yd, s, q)
        m, e = torch.empty(5, cols, dtype=torch.uint8, device="cuda"), torch.empty(5, cols // 32, dtype=torch.uint8,
                                                                                   device="cuda")
        rb.mx_quantize(yd, rb.FMT_E4M3, m, e)
        xd, wd = torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda()
        _, c0, s0 = _run(rb, xd, None, wd, 0)
        _, c1, s1 = _run(rb, xd, None, wd, 1)
        assert torch.equal(c0, q) and torch.equal(s0, s) and torch.equal(c1, m) and torch.equal(s1, e)


@pytest.mark.parametrize("fmt", [0, 1])
def test_special_rows(rb, cuda, fmt):
    """Zeros, huge, tiny, infinite and NaN rows leave the other rows alone, and a zero row codes zeros."""
    import torch
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(8, 640, generator=g, device="cuda")
    w = torch.ones(640, device="cuda")
    _, good, gs = _run(rb, x, None, w, fmt)
    y = x.clone()
    y[1] = 0
    y[2] *= 1e30
    y[3] *= 1e-30
    y[4, 7] = float("inf")
    y[5, 9] = float("nan")
    _, codes, scales = _run(rb, y, None, w, fmt)
    for i in (0, 6, 7):
        assert torch.equal(codes[i], good[i]) and torch.equal(scales[i], gs[i])
    assert (codes[1] == 0).all()
    fine = torch.tensor([0, 1, 2, 6, 7])
    _check(y[fine], None, w, fmt, None, codes[fine.cuda()], scales[fine.cuda()])


def test_no_rows_and_rows_behind(rb, cuda):
    import torch
    x = torch.randn(4, 64, device="cuda")
    codes, scales = torch.full((6, 64), 77, dtype=torch.int8, device="cuda"), torch.full((6,), 7.0, device="cuda")
    rb.add_rmsnorm_quant(x[:0], None, torch.ones(64, device="cuda"), 1e-5, 0, codes, scales)
    assert (codes == 77).all() and (scales == 7).all()
    rb.add_rmsnorm_quant(x, None, torch.ones(64, device="cuda"), 1e-5, 0, codes, scales)
    rb.sync_status()
    assert (codes[4:] == 77).all() and (scales[4:] == 7).all() and (scales[:4] != 7).all()


def _separate_steps(rb, h, w, eps):
    """int8 codes and scales, MXFP8 codes and scales of rouge_rmsnorm followed by the quantizers."""
    import ctypes as C

    import torch
    L = rb.lib()
    L.rouge_rmsnorm.argtypes, L.rouge_rmsnorm.restype = [C.c_void_p, C.c_int, C.c_void_p, C.c_float, C.c_void_p], None
    x, wn = np.ascontiguousarray(h.float().cpu().numpy()), w.cpu().numpy()
    y = np.empty_like(x)
    p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    for i in range(x.shape[0]):
        L.rouge_rmsnorm(p(x[i]), x.shape[1], p(wn), eps, p(y[i]))
    yd = torch.from_numpy(y).cuda()
    rows, cols = y.shape
    q, s = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    rb.quantize_i8_rows(yd, s, q)
    m, e = torch.empty(rows, cols, dtype=torch.uint8, device="cuda"), torch.empty(rows, cols // 32, dtype=torch.uint8,
                                                                                  device="cuda")
    rb.mx_quantize(yd, rb.FMT_E4M3, m, e)
    return q, s, m, e


@pytest.mark.parametrize("scale", [1e30, 1e33, 1e36, 2e38, 1e-30, 1e-37, 1e-40, 1e-43])
@pytest.mark.parametrize("eps", [1e-5, 0.0])
def test_rows_at_the_ends_of_f32(rb, cuda, scale, eps):
    """Rows whose inverse root leaves f32's normal range, or whose outputs do: still the separate steps' codes."""
    import torch
    g = torch.Generator("cuda").manual_seed(9)
    x = (0.4 + 1.2 * torch.rand(300, 512, generator=g, device="cuda")) * scale
    x = torch.where(torch.rand(x.shape, generator=g, device="cuda") < 0.5, x, -x)
    w = 0.5 + torch.rand(512, generator=g, device="cuda")
    q, s, m, e = _separate_steps(rb, x, w, eps)
    _, c0, s0 = _run(rb, x, None, w, 0, eps)
    _, c1, s1 = _run(rb, x, None, w, 1, eps)
    assert torch.equal(s0, s) and torch.equal(c0, q) and torch.equal(c1, m) and torch.equal(s1, e)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", [96, 5120, 16416])
def test_equals_the_separate_steps_with_residual(rb, cuda, t, cols):
    import torch
    g = torch.Generator("cuda").manual_seed(cols)
    x, r = ((3 * torch.randn(9, cols, generator=g, device="cuda")).to(_dt(t)) for _ in range(2))
    w = 0.5 + torch.rand(cols, generator=g, device="cuda")
    q, s, m, e = _separate_steps(rb, (x.float() + r.float()).to(x.dtype), w, 1e-5)
    _, c0, s0 = _run(rb, x, r, w, 0)
    _, c1, s1 = _run(rb, x, r, w, 1)
    assert torch.equal(s0, s) and torch.equal(c0, q) and torch.equal(c1, m) and torch.equal(s1, e)
