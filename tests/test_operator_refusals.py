"""Argument checks of the quantized decoder step's entries, without a GPU:
every call is refused (or found to lack a device) before any pointer is used."""
import ctypes as C

import pytest

A = 1 << 20  # an aligned address that is never dereferenced


@pytest.fixture()
def call(rb):
    L = rb.lib()

    def run(name, *args):
        st = getattr(L, name)(*args)
        assert L.rouge_b200_last_error() == st or st == rb.OK
        L.rouge_b200_clear_error()
        return st
    return run


def _norm_args(**kw):
    a = dict(x=A, ldx=64, r=A, ldr=64, w=A, eps=1e-5, rows=4, cols=64, type=0, h=A, ldh=64, fmt=0, codes=A,
             scales=A, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw", [dict(x=None), dict(w=None), dict(codes=None), dict(scales=None), dict(rows=-1),
                                dict(cols=0), dict(ldx=60), dict(ldr=60), dict(ldh=60), dict(r=None),
                                dict(h=None), dict(type=3), dict(type=-1), dict(fmt=2)])
def test_norm_invalid(rb, call, kw):
    assert call("rouge_b200_add_rmsnorm_quant", *_norm_args(**kw)) == rb.EINVAL


@pytest.mark.parametrize("kw", [dict(cols=62), dict(cols=48, fmt=1), dict(x=A + 4), dict(r=A + 8), dict(h=A + 8),
                                dict(w=A + 8), dict(ldx=65), dict(type=1, ldx=66), dict(rows=(1 << 30) + 1), dict(codes=A + 2),
                                dict(scales=A + 1)])
def test_norm_unsupported(rb, call, kw):
    assert call("rouge_b200_add_rmsnorm_quant", *_norm_args(**kw)) == rb.EUNSUPPORTED


def _kv(rb, **kw):
    a = dict(k_codes=A, k_scales=A, v_codes=A, v_scales=A, gs_k=None, gs_v=None, pages=4, page=16, Hkv=2, Dh=64)
    a.update(kw)
    return rb._KV4C(*a.values())


CACHE_BAD = [(dict(k_codes=None), "EINVAL"), (dict(v_scales=None), "EINVAL"), (dict(pages=0), "EINVAL"),
             (dict(page=0), "EINVAL"), (dict(Hkv=0), "EINVAL"), (dict(Dh=0), "EINVAL"),
             (dict(page=24), "EUNSUPPORTED"), (dict(Dh=72), "EUNSUPPORTED"), (dict(Dh=272), "EUNSUPPORTED"),
             (dict(k_codes=A + 8), "EUNSUPPORTED"), (dict(v_scales=A + 1), "EUNSUPPORTED"),
             (dict(gs_k=A + 2), "EUNSUPPORTED"), (dict(pages=1 << 20, page=2048), "EUNSUPPORTED")]


@pytest.mark.parametrize("kw,status", CACHE_BAD)
@pytest.mark.parametrize("name", ["rouge_b200_kv4_write", "rouge_b200_kv4_read"])
def test_cache_refused(rb, call, name, kw, status):
    assert call(name, _kv(rb, **kw), A, 128, A, 128, 0, 3, A, None) == getattr(rb, status)


@pytest.mark.parametrize("name", ["rouge_b200_kv4_write", "rouge_b200_kv4_read"])
def test_tokens_refused(rb, call, name):
    c = _kv(rb)
    ok = [A, 128, A, 128, 0, 3, A, None]
    for i, v, st in ((0, None, rb.EINVAL), (2, None, rb.EINVAL), (6, None, rb.EINVAL), (1, 120, rb.EINVAL),
                     (3, 64, rb.EINVAL), (4, 4, rb.EINVAL), (5, -1, rb.EINVAL), (0, A + 4, rb.EUNSUPPORTED),
                     (1, 130, rb.EUNSUPPORTED), (6, A + 2, rb.EUNSUPPORTED)):
        args = list(ok)
        args[i] = v
        assert call(name, c, *args) == st, (i, v)
    assert call(name, None, *ok) == rb.EINVAL


def _attn(rb, cache=None, **kw):
    a = dict(Q=A, type=2, B=2, Hq=4, cu_q=A, max_q=3, kv_len=A, table=A, max_pages=5, O=A, scale=0.0, causal=1,
             window=0, ws=A, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return [cache if cache is not None else _kv(rb)] + list(a.values())


@pytest.mark.parametrize("kw,status", CACHE_BAD)
def test_attention_cache_refused(rb, call, kw, status):
    assert call("rouge_b200_attention_kv4", *_attn(rb, _kv(rb, **kw))) == getattr(rb, status)


@pytest.mark.parametrize("kw,status", [
    (dict(Q=None), "EINVAL"), (dict(O=None), "EINVAL"), (dict(kv_len=None), "EINVAL"), (dict(table=None), "EINVAL"),
    (dict(B=0), "EINVAL"), (dict(Hq=3), "EINVAL"), (dict(Hq=0), "EINVAL"), (dict(max_q=0), "EINVAL"),
    (dict(max_pages=0), "EINVAL"), (dict(window=-1), "EINVAL"), (dict(cu_q=None), "EINVAL"),
    (dict(type=4), "EINVAL"), (dict(Q=A + 8), "EUNSUPPORTED"), (dict(O=A + 2), "EUNSUPPORTED"),
    (dict(ws=A + 16), "EUNSUPPORTED"), (dict(max_pages=1 << 28), "EUNSUPPORTED"),
    (dict(max_q=1 << 30, Hq=8), "EUNSUPPORTED")])
def test_attention_refused(rb, call, kw, status):
    assert call("rouge_b200_attention_kv4", *_attn(rb, **kw)) == getattr(rb, status)


def _ep(rb, **kw):
    a = dict(bias=A, residual=A, ldr=64, residual_type=0, act=0)
    a.update(kw)
    return rb._EpilogueC(*a.values())


@pytest.mark.parametrize("kw", [dict(act=-1), dict(act=4), dict(ldr=60), dict(residual_type=3),
                                dict(residual_type=-1), dict(residual=A + 2), dict(bias=A + 1),
                                dict(residual=A + 1, residual_type=2)])
def test_epilogue_refused(rb, call, kw):
    ep = _ep(rb, **kw)
    assert call("rouge_b200_gemm_i8_fused", 32, 64, 64, A, A, 1, A, 1, A, 1, ep, A, 64, 0, None) == rb.EINVAL
    assert call("rouge_b200_gemm_e4m3_fused", 32, 64, 64, A, A, 1, A, A, ep, A, 64, 0, None) == rb.EINVAL
    assert call("rouge_b200_gemm_f16_fused", 32, 64, 64, A, A, 1, 0, ep, A, 64, 0, None) == rb.EINVAL


def test_fused_gemm_refused(rb, call):
    ep = _ep(rb)
    i8 = [32, 64, 64, A, A, 1, A, 1, A, 1, ep, A, 64, 0, None]
    for i, v, st in ((0, 0, rb.EINVAL), (3, None, rb.EINVAL), (6, None, rb.EINVAL), (8, None, rb.EINVAL),
                     (10, None, rb.EINVAL), (11, None, rb.EINVAL), (12, 60, rb.EINVAL), (13, rb.OUT_I32, rb.EINVAL),
                     (5, 2, rb.EINVAL), (3, A + 8, rb.EUNSUPPORTED), (2, 60, rb.EUNSUPPORTED)):
        args = list(i8)
        args[i] = v
        assert call("rouge_b200_gemm_i8_fused", *args) == st, (i, v)
    assert call("rouge_b200_gemm_e4m3_fused", 32, 64, 64, A, A, 1, A, None, ep, A, 64, 0, None) == rb.EINVAL


def test_no_device(rb, call):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert call("rouge_b200_add_rmsnorm_quant", *_norm_args()) == rb.ENODEV
    assert call("rouge_b200_kv4_write", _kv(rb), A, 128, A, 128, 0, 3, A, None) == rb.ENODEV
    assert call("rouge_b200_attention_kv4", *_attn(rb)) == rb.ENODEV
    assert call("rouge_b200_gemm_f16_fused", 32, 64, 64, A, A, 1, 0, _ep(rb), A, 64, 0, None) == rb.ENODEV


def test_workspace_of_nothing_is_zero(rb):
    L = rb.lib()
    for args in ((0, 4, 2, 64, 1, 64, 0), (1, 3, 2, 64, 1, 64, 0), (1, 4, 2, 300, 1, 64, 0), (1, 4, 2, 64, 0, 64, 0),
                 (1, 4, 2, 64, 1, 0, 0), (1, 4, 2, 64, 1, 64, 7)):
        assert L.rouge_b200_attention_kv4_workspace(*args) == 0
    L.rouge_b200_clear_error()


def test_python_checks(rb):
    import torch
    z = torch.zeros
    with pytest.raises(ValueError):
        rb.KV4Cache(z(2, 1, 16, 32, dtype=torch.uint8), z(2, 1, 16, 3, dtype=torch.uint8),
                    z(2, 1, 16, 32, dtype=torch.uint8), z(2, 1, 16, 4, dtype=torch.uint8))
    c = rb.KV4Cache.empty(2, 1, 16, 64, device="cpu")
    assert (c.page, c.Hkv, c.Dh, c.pages) == (16, 1, 64, 2)
    with pytest.raises(ValueError):
        rb.kv4_write(c, z(3, 1, 64), z(3, 1, 32), z(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        rb.kv4_write(c, z(3, 1, 64), z(3, 1, 64), z(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        rb.Epilogue(residual=z(4, 4, dtype=torch.int8))
    with pytest.raises(ValueError):
        rb.Epilogue(bias=z(5)).check(4, 4)
    with pytest.raises(ValueError):
        rb.Epilogue(residual=z(4, 5)).check(4, 4)
    with pytest.raises(ValueError):
        rb.attention_kv4(z(2, 4, 32), c, z(2, dtype=torch.int32), z(2, 1, dtype=torch.int32))
    for bad in (dict(w=z(32)), dict(codes=z(3, 64, dtype=torch.int8)), dict(scales=z(4, dtype=torch.int8))):
        a = dict(w=z(64), codes=z(4, 64, dtype=torch.int8), scales=z(4)) | bad
        with pytest.raises(ValueError):
            rb.add_rmsnorm_quant(z(4, 64), None, a["w"], 1e-5, 0, a["codes"], a["scales"])
    with pytest.raises(ValueError):
        rb.add_rmsnorm_quant(z(4, 64), z(4, 32), z(64), 1e-5, 0, z(4, 64, dtype=torch.int8), z(4), z(4, 64))


def test_ragged_queries_need_max_q(rb):
    import torch
    z, i32 = torch.zeros, torch.int32
    c = rb.KV4Cache.empty(2, 1, 16, 64, device="cpu")
    with pytest.raises(ValueError, match="max_q"):
        rb.attention_kv4(z(4, 4, 64), c, z(2, dtype=i32), z(2, 1, dtype=i32), cu_q=z(3, dtype=i32))
    with pytest.raises(ValueError, match="one query"):
        rb.attention_kv4(z(2, 4, 64), c, z(2, dtype=i32), z(2, 1, dtype=i32), max_q=2)


@pytest.mark.parametrize("kind", ["i8", "e4m3", "f16", "bf16"])
@pytest.mark.parametrize("layout", [0, 1])
def test_fused_gemm_tensors_are_checked(rb, kind, layout):
    """Anything the kernel would read or write past a tensor's end, or take for another type."""
    import torch
    M, N, K = 8, 48, 32
    dt = dict(i8=torch.int8, e4m3=torch.float8_e4m3fn, f16=torch.float16, bf16=torch.bfloat16)[kind]
    z = torch.zeros
    B = (K, N) if layout == 0 else (N, K)
    good = dict(A=z(M, K, dtype=dt), B=z(B, dtype=dt), C=z(M, N), out=rb.OUT_F32, sa=z(M), sb=z(N), rows=1, cols=1,
                ep=rb.Epilogue(z(N), 0, z(M, N)))

    def call(**kw):
        a = good | kw
        if kind == "i8":
            rb.gemm_i8(a["A"], a["B"], layout, a["C"], a["out"], a["sa"], a["rows"], a["sb"], a["cols"],
                       epilogue=a["ep"])
        elif kind == "e4m3":
            rb.gemm_e4m3(a["A"], a["B"], layout, a["C"], a["out"], a["sa"], a["sb"], epilogue=a["ep"])
        else:
            rb.gemm_f16(a["A"], a["B"], layout, a["C"], a["out"], kind == "bf16", epilogue=a["ep"])

    bad = [dict(C=z(M, N, dtype=torch.bfloat16)), dict(out=rb.OUT_BF16), dict(C=z(M, N, dtype=torch.float64)),
           dict(C=z(M - 1, N)), dict(C=z(M, N - 1)), dict(C=z(M, 2 * N)[:, ::2]), dict(C=z(N, M).T),
           dict(A=z(M, 2 * K, dtype=dt)[:, :K]), dict(A=z(M, K + 16, dtype=dt)), dict(A=z(M, K)),
           dict(B=z(B)), dict(B=z(B[::-1], dtype=dt).T), dict(B=z(B[0] + (layout == 0), B[1] + layout, dtype=dt)),
           dict(ep=rb.Epilogue(z(N + 1))), dict(ep=rb.Epilogue(residual=z(M, N + 1)))]
    if kind == "i8":
        bad += [dict(sa=z(M - 1)), dict(sb=z(N - 1)), dict(sa=z(2 * M)[::2]), dict(sb=z(N, dtype=torch.float64)),
                dict(sa=z(0), rows=0), dict(sb=z(0), cols=0)]
    if kind == "e4m3":
        bad += [dict(sa=z(0)), dict(sb=z(1, dtype=torch.float16))]
    for kw in bad:
        with pytest.raises(ValueError):
            call(**kw)


def test_pitch_of_one_row(rb):
    import torch
    row = torch.zeros(64, 1).T  # [1, 64] whose row stride is 1
    assert row.stride(0) == 1 and rb.Epilogue(residual=row).c.ldr == 64
    assert rb.Epilogue(residual=torch.zeros(3, 80)[:, :64]).c.ldr == 80


@pytest.mark.parametrize("name", ["cu_q", "kv_len", "table"])
def test_attention_misaligned_indices_refused(rb, call, name):
    assert call("rouge_b200_attention_kv4", *_attn(rb, **{name: A + 2})) == rb.EUNSUPPORTED
