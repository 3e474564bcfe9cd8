"""GEMMs with bias, activation and residual in the epilogue against 64 bits.

Operands are multiples of 2^-3 (or whole numbers) small enough that every
sum is exact in f32 in any order, so only the epilogue rounds. With v the
value before it: the bias adds a rounding of 2^-24 (|v| + |bias|); gelu's
derivative is below 1.13 and erf is within 2 ulp (CUDA's bound), which 1 + erf
turns into at most 2^-22 of |v|; silu's fast exponential and divide are within
2 + 1.173 |v| and 2 ulp, so within (5 + 1.2 |v|) 2^-23 of |v|; the residual adds
2^-24 of the sum, the output half a step of its type. Scales (two products)
add 2 * 2^-24 |v| before all that."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _dt(t):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[t]


def _operands(kind, M, N, K, layout, seed):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    ri = lambda n, *s: torch.randint(-n, n + 1, s, generator=g, device="cuda")  # noqa: E731
    if kind == "i8":
        A, B = ri(127, M, K).to(torch.int8), ri(127, N, K).to(torch.int8)
        sa = (0.5 + torch.rand(M, generator=g, device="cuda")) / 64
        sb = (0.5 + torch.rand(N, generator=g, device="cuda")) / (64 * math.sqrt(K))
        v = (A.double() @ B.double().T) * sa.double()[:, None] * sb.double()
    elif kind == "e4m3":
        A, B = ri(8, M, K).float().to(torch.float8_e4m3fn), ri(8, N, K).float().to(torch.float8_e4m3fn)
        sa, sb = torch.full((1,), 0.21, device="cuda"), torch.full((1,), 0.3 / math.sqrt(K), device="cuda")
        v = (A.double() @ B.double().T) * float(sa) * float(sb)
    else:
        A, B = (ri(8, M, K) / 8).to(_dt(kind)), (ri(8, N, K) / 8).to(_dt(kind))
        sa = sb = None
        v = A.double() @ B.double().T
    return A, (B if layout == 1 else B.T.contiguous()), sa, sb, v, g


def _call(rb, kind, A, B, layout, out, sa, sb, ep):
    import torch
    ot = rb.OUT_F32 if out.dtype == torch.float32 else rb.OUT_BF16
    if kind == "i8":
        rb.gemm_i8(A, B, layout, out, ot, sa, 1, sb, 1, epilogue=ep)
    elif kind == "e4m3":
        rb.gemm_e4m3(A, B, layout, out, ot, sa, sb, epilogue=ep)
    else:
        rb.gemm_f16(A, B, layout, out, ot, kind == "bf16", epilogue=ep)
    rb.sync_status()


def _check(v, out, act, bias, res):
    import torch
    e = 2.0 ** -24
    z = v + (bias.double() if bias is not None else 0)
    err = 2 * e * v.abs() + e * (z.abs() + e)
    a = z.abs()
    if act == 1:
        y = z.clamp(min=0)
    elif act == 2:
        y, err = z * torch.special.ndtr(z), 1.13 * err + 2.0 ** -22 * a
    elif act == 3:
        y, err = z * torch.sigmoid(z), 1.1 * err + (5 + 1.2 * a) * 2.0 ** -23 * a
    else:
        y = z
    if res is not None:
        y = y + res.double()
        err = err + e * y.abs()
    half = torch.finfo(out.dtype).eps / 2
    err = err + (y.abs() + err) * half + 1e-30
    d = (out.double() - y).abs()
    assert (d <= err).all(), ((d - err).max().item(), (d / err).max().item())


KINDS = ["i8", "bf16", "f16", "e4m3"]


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("res,out", [("", "f32"), ("f32", "f32"), ("f16", "bf16"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("kind", KINDS)
def test_epilogue(rb, cuda, kind, act, res, out):
    import torch
    M, N, K = 137, 264, 272
    A, B, sa, sb, v, g = _operands(kind, M, N, K, 1, 7)
    bias = torch.randn(N, generator=g, device="cuda")
    r = torch.randn(M, N, generator=g, device="cuda").to(_dt(res)) if res else None
    c = torch.empty(M, N, dtype=_dt(out), device="cuda")
    _call(rb, kind, A, B, 1, c, sa, sb, rb.Epilogue(bias, act, r))
    _check(v, c, act, bias, r)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (1, 4096, 512), (24, 1040, 4160), (32, 2048, 1008), (33, 2048, 1024),
                                   (16, 8208, 640), (16, 1040, 4096), (129, 48, 64), (2500, 4112, 128),
                                   (4096, 2576, 256), (300, 8208, 144)])
@pytest.mark.parametrize("kind", KINDS)
def test_shapes(rb, cuda, kind, M, N, K, layout):
    import torch
    A, B, sa, sb, v, g = _operands(kind, M, N, K, layout, M + N)
    bias = torch.randn(N, generator=g, device="cuda")
    r = torch.randn(M, N, generator=g, device="cuda").bfloat16()
    c = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    _call(rb, kind, A, B, layout, c, sa, sb, rb.Epilogue(bias, 3, r))
    _check(v, c, 3, bias, r)


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_tile_modes(rb, cuda, mode):
    import torch
    A, B, sa, sb, v, g = _operands("i8", 700, 1072, 384, 1, 3)
    r = torch.randn(700, 1072, generator=g, device="cuda")
    c = torch.empty(700, 1072, device="cuda")
    with rb.tile_mode(mode):
        _call(rb, "i8", A, B, 1, c, sa, sb, rb.Epilogue(None, 0, r))
    _check(v, c, 0, None, r)


@pytest.mark.parametrize("N", [1, 5, 31, 33, 100])
def test_odd_columns_strides_and_alignment(rb, cuda, N):
    """Rows that no 16-byte vector divides: bias, residual and output one element off, wide pitches."""
    import torch
    M, K = 70, 64
    A, B, _, _, v, g = _operands("bf16", M, N, K, 1, N)
    bias = torch.randn(N + 1, generator=g, device="cuda")[1:]
    for t in ("f32", "bf16", "f16"):
        r = torch.randn(M, N + 9, generator=g, device="cuda").to(_dt(t))[:, 3:3 + N]
        big = torch.full((M, N + 7), 5.0, device="cuda")
        c = big[:, 2:2 + N]
        _call(rb, "bf16", A, B, 1, c, None, None, rb.Epilogue(bias, 2, r))
        _check(v, c, 2, bias, r)
        assert (big[:, :2] == 5).all() and (big[:, 2 + N:] == 5).all()


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(16, 1024, 512), (3000, 2080, 256)])
def test_residual_in_place(rb, cuda, out, M, N, K):
    import torch
    A, B, sa, sb, v, g = _operands("i8", M, N, K, 1, 11)
    c = torch.randn(M, N, generator=g, device="cuda").to(_dt(out))
    r = c.clone()
    _call(rb, "i8", A, B, 1, c, sa, sb, rb.Epilogue(None, 0, c))
    _check(v, c, 0, None, r)


def test_empty_epilogue_equals_the_plain_gemm(rb, cuda):
    import torch
    A, B, sa, sb, _, _ = _operands("i8", 513, 1040, 512, 1, 2)
    c, d = (torch.empty(513, 1040, device="cuda") for _ in range(2))
    _call(rb, "i8", A, B, 1, c, sa, sb, rb.Epilogue())
    rb.gemm_i8(A, B, 1, d, rb.OUT_F32, sa, 1, sb, 1)
    assert torch.equal(c, d)


def test_specials(rb, cuda):
    """Infinities and NaN go through: relu keeps NaN, silu(-inf) is NaN as -inf / inf, a NaN bias fills its column."""
    import torch
    A = torch.zeros(40, 64, dtype=torch.bfloat16, device="cuda")
    B = torch.zeros(48, 64, dtype=torch.bfloat16, device="cuda")
    bias = torch.zeros(48, device="cuda")
    bias[1], bias[2], bias[3], bias[4], bias[5] = float("nan"), float("inf"), -float("inf"), 200.0, -200.0
    for act in range(4):
        c = torch.empty(40, 48, dtype=torch.bfloat16, device="cuda")
        _call(rb, "bf16", A, B, 1, c, None, None, rb.Epilogue(bias, act))
        assert c[:, 1].isnan().all() and not c[:, [0] + list(range(4, 48))].isnan().any()
        assert (c[:, 2] == float("inf")).all()
        assert (c[:, 4] == 200).all()
        if act:
            assert (c[:, 5].abs() < 1e-30).all()


def test_captured_and_replayed(rb, cuda):
    import torch
    A, B, sa, sb, v, g = _operands("i8", 64, 512, 256, 1, 9)
    r = torch.randn(64, 512, generator=g, device="cuda")
    c = torch.empty(64, 512, device="cuda")
    ep = rb.Epilogue(None, 1, r)
    _call(rb, "i8", A, B, 1, c, sa, sb, ep)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rb.gemm_i8(A, B, 1, c, rb.OUT_F32, sa, 1, sb, 1, epilogue=ep)
    r.mul_(-2)
    c.zero_()
    graph.replay()
    torch.cuda.synchronize()
    _check(v, c, 1, None, r)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("M,N,K", [(1, 1024, 4096), (32, 8192, 1040), (33, 528, 512), (513, 1040, 512), (1000, 4128, 2064)])
@pytest.mark.parametrize("kind", KINDS)
def test_empty_epilogue_gives_the_plain_entrys_bits(rb, cuda, kind, M, N, K, layout):
    """Also where the fused entry takes another tile: sums of random products, in the same order."""
    import torch
    A, B, sa, sb, _, g = _operands(kind, M, N, K, layout, M)
    if kind in ("bf16", "f16"):
        A, B = (torch.randn(t.shape, generator=g, device="cuda").to(t.dtype) for t in (A, B))
    c, d = (torch.empty(M, N, device="cuda") for _ in range(2))
    _call(rb, kind, A, B, layout, c, sa, sb, rb.Epilogue())
    if kind == "i8":
        rb.gemm_i8(A, B, layout, d, rb.OUT_F32, sa, 1, sb, 1)
    elif kind == "e4m3":
        rb.gemm_e4m3(A, B, layout, d, rb.OUT_F32, sa, sb)
    else:
        rb.gemm_f16(A, B, layout, d, rb.OUT_F32, kind == "bf16")
    assert torch.equal(c, d)
