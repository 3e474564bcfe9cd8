"""Python binding of librouge_b200.so (the C ABI in include/rouge/numerics_b200.h).

A thin ctypes layer: every function here calls one exported C entry point.
Device-pointer entries take torch CUDA tensors and the current torch stream;
host-pointer (drop-in) entries take numpy arrays, exactly as a C caller of
the reference rouge-numerics API passes host buffers. There is no CPU
fallback: if the shared library is missing or the GPU path fails, calls
raise.
"""
from __future__ import annotations

import ctypes as C
import os
import re
import subprocess

import numpy as np

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_DIR = os.path.join(os.path.dirname(PKG_DIR), "lib")
LIB_PATH = os.path.join(LIB_DIR, "librouge_b200.so")
REPO_ROOT = os.path.dirname(os.path.dirname(PKG_DIR))
HEADER = os.path.join(REPO_ROOT, "include", "rouge", "numerics_b200.h")

OK = 0
EINVAL = -1
ENODEV = -2
ECUDA = -3
EUNSUPPORTED = -4
ETIMEOUT = -5
ENOMEM = -6
ETOOBIG = -7

B_KN = 0
B_NK = 1
OUT_F32 = 0
OUT_BF16 = 1
OUT_I32 = 2
TILES_AUTO = 0
TILES_SINGLE = 1
TILES_PAIR = 2


class RougeB200Error(RuntimeError):
    def __init__(self, fn: str, status: int, msg: str):
        super().__init__(f"{fn} failed: {status} ({msg})")
        self.status = status


def build() -> None:
    """Compile librouge_b200.so in-tree (nvcc cross-compiles without a GPU)."""
    subprocess.run(["make", "-s", "-C", os.path.dirname(PKG_DIR), "-j8"], check=True)


_P = C.c_void_p
_I = C.c_int
_F = C.c_float
_SZ = C.c_size_t
_U64 = C.c_uint64


class GemmConfig(C.Structure):
    """RougeGemmConfig (numerics.h:35-41)."""
    _fields_ = [("tile_m", _I), ("tile_n", _I), ("tile_k", _I), ("unroll", _I), ("split_k", _I)]

    def astuple(self):
        return (self.tile_m, self.tile_n, self.tile_k, self.unroll, self.split_k)


class GemmProfile(C.Structure):
    """RougeGemmProfile (numerics.h:44-48)."""
    _fields_ = [("cfg", GemmConfig), ("gflops", C.c_double), ("iters", C.c_longlong)]


class _EpilogueC(C.Structure):
    """RougeB200Epilogue."""
    _fields_ = [("bias", _P), ("residual", _P), ("ldr", C.c_longlong), ("residual_type", _I), ("act", _I)]


class _KV4C(C.Structure):
    """RougeB200KV4."""
    _fields_ = [("k_codes", _P), ("k_scales", _P), ("v_codes", _P), ("v_scales", _P), ("gs_k", _P),
                ("gs_v", _P), ("pages", _I), ("page", _I), ("Hkv", _I), ("Dh", _I)]


_LL = C.c_longlong
_SIGS = {
    "rouge_b200_last_error": (_I, []),
    "rouge_b200_clear_error": (None, []),
    "rouge_b200_status_string": (C.c_char_p, [_I]),
    "rouge_gemm_isa_variant": (C.c_char_p, []),
    "rouge_b200_device_ok": (_I, []),
    "rouge_b200_sync_status": (_I, [_P]),
    "rouge_b200_check_wait_limit": (_I, [C.c_ulonglong, _P]),
    "rouge_b200_w8a8_workspace_bytes": (_SZ, [_I]),
    "rouge_b200_w8a8_linear": (_I, [_I, _I, _I, _P, _P, _P, _P, _P, _P, _I, _I, _P, _P]),
    "rouge_b200_set_sm_budget": (_I, [_I]),
    "rouge_b200_set_tile_mode": (_I, [_I]),
    "rouge_b200_set_clock_probe": (_I, [_P, _I]),
    "rouge_quantize_e4m3": (C.c_uint8, [_F]),
    "rouge_dequantize_e4m3": (_F, [C.c_uint8]),
    "rouge_quantize_f16": (C.c_uint16, [_F]),
    "rouge_dequantize_f16": (_F, [C.c_uint16]),
    "rouge_quantize_bf16": (C.c_uint16, [_F]),
    "rouge_dequantize_bf16": (_F, [C.c_uint16]),
    "rouge_quantize_i8_tensor": (_I, [_P, _I, _P, _P]),
    "rouge_quantize_i8_channel": (_I, [_P, _I, _I, _P, _P]),
    "rouge_dequantize_i8_tensor": (None, [_P, _I, _F, _P]),
    "rouge_dequantize_i8_channel": (None, [_P, _I, _I, _P, _P]),
    "rouge_quantize_i8_group": (_I, [_P, _I, _I, _I, _P, _P, _P]),
    "rouge_dequantize_i8_group": (None, [_P, _I, _I, _I, _P, _P, _P]),
    "rouge_b200_quantize_i8_group": (_I, [_P, _I, _I, _I, _P, _P, _P, _P]),
    "rouge_b200_dequantize_i8_group": (_I, [_P, _I, _I, _I, _P, _P, _P, _P]),
    "rouge_gemm_i8": (None, [_I, _I, _I, _P, _P, _P, _I, _P, _I, _P]),
    "rouge_gemm_i8_noalloc": (_I, [_I, _I, _I, _P, _P, _P, _I, _P, _I, _P]),
    "rouge_gemm_e4m3": (None, [_I, _I, _I, _P, _P, _P, _P]),
    "rouge_gemm_f32": (None, [_I, _I, _I, _P, _P, _P, _P]),
    "rouge_gemm_default_config": (GemmConfig, []),
    "rouge_gemm_candidate_count": (_I, []),
    "rouge_gemm_candidate": (GemmConfig, [_I]),
    "rouge_gemm_flops_per_sec": (C.c_double, [_I, _I, _I, _P, _P, _P, _P]),
    "rouge_gemm_tuned": (GemmProfile, [_I, _I, _I, _P, _P, _P]),
    "rouge_gemm_f16": (None, [_I, _I, _I, _P, _P, _P, _P]),
    "rouge_gemm_bf16": (None, [_I, _I, _I, _P, _P, _P, _P]),
    "rouge_conv2d_f32": (None, [_I] * 9 + [_P, _P, _P, _P, _P]),
    "rouge_conv_implicit_f32": (None, [_I] * 9 + [_P, _P, _P, _P, _P]),
    "rouge_b200_quantize_i8_rows": (_I, [_P, _I, _I, _P, _P, _P]),
    "rouge_b200_dequantize_i8_rows": (_I, [_P, _I, _I, _P, _F, _P, _P]),
    "rouge_b200_absmax_f32": (_I, [_P, _SZ, _P, _P]),
    "rouge_b200_quantize_e4m3_scaled": (_I, [_P, _SZ, _P, _P, _P, _P]),
    "rouge_b200_quantize_e4m3_tensor": (_I, [_P, _SZ, _P, _P, _P, _P]),
    "rouge_b200_mx_quantize": (_I, [_P, _SZ, _I, _P, _P, _P]),
    "rouge_b200_nvfp4_quantize": (_I, [_P, _SZ, C.c_float, _P, _P, _P]),
    "rouge_b200_mx_dequantize": (_I, [_P, _P, _SZ, _I, _P, _P]),
    "rouge_b200_mx_scale_atoms_bytes": (_SZ, [_I, _I]),
    "rouge_b200_mx_scale_atoms": (_I, [_P, _I, _I, _P, _P]),
    "rouge_b200_gemm_mx": (_I, [_I, _I, _I, _P, _I, _P, _P, _I, _P, _P, _I, _I, _P]),
    "rouge_b200_nvfp4_scale_atoms_bytes": (_SZ, [_I, _I]),
    "rouge_b200_nvfp4_scale_atoms": (_I, [_P, _I, _I, _P, _P]),
    "rouge_b200_fp4_pack": (_I, [_P, _SZ, _P, _P]),
    "rouge_b200_nvfp4_quantize_packed": (_I, [_P, _SZ, C.c_float, _P, _P, _P]),
    "rouge_b200_gemm_nvfp4": (_I, [_I, _I, _I, _P, _P, _P, _P, _P, _P, _P, _I, _I, _P]),
    "rouge_b200_attention_workspace": (_SZ, [_I, _I, _I, _I, _I, _I]),
    "rouge_b200_attention_gqa": (_I, [_I, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P, _P,
                                      C.c_float, _I, _I, _I, _P, _SZ, _P]),
    "rouge_b200_transformer_block_workspace": (_SZ, [_I, _I, _I, _I, _I, _I]),
    "rouge_b200_transformer_block": (_I, [_I] * 6 + [_P] * 10 + [_I, C.c_float, C.c_float, _P, _P,
                                                                  _SZ, _P]),
    "rouge_b200_add_rmsnorm_quant": (_I, [_P, _LL, _P, _LL, _P, _F, _I, _I, _I, _P, _LL, _I, _P, _P, _P]),
    "rouge_b200_kv4_write": (_I, [C.POINTER(_KV4C), _P, _LL, _P, _LL, _I, _I, _P, _P]),
    "rouge_b200_kv4_read": (_I, [C.POINTER(_KV4C), _P, _LL, _P, _LL, _I, _I, _P, _P]),
    "rouge_b200_attention_kv4_workspace": (_SZ, [_I] * 7),
    "rouge_b200_attention_kv4": (_I, [C.POINTER(_KV4C), _P, _I, _I, _I, _P, _I, _P, _P, _I, _P, _F, _I, _I,
                                      _P, _SZ, _P]),
    "rouge_b200_mxfp4_scale_atoms_bytes": (_SZ, [_I, _I]),
    "rouge_b200_mxfp4_scale_atoms": (_I, [_P, _I, _I, _P, _P]),
    "rouge_b200_gemm_mxfp4": (_I, [_I, _I, _I, _P, _P, _P, _P, _P, _I, _I, _P]),
    "rouge_quantize_e5m2": (C.c_uint8, [C.c_float]), "rouge_dequantize_e5m2": (C.c_float, [C.c_uint8]),
    "rouge_quantize_e3m2": (C.c_uint8, [C.c_float]), "rouge_dequantize_e3m2": (C.c_float, [C.c_uint8]),
    "rouge_quantize_e2m3": (C.c_uint8, [C.c_float]), "rouge_dequantize_e2m3": (C.c_float, [C.c_uint8]),
    "rouge_quantize_e2m1": (C.c_uint8, [C.c_float]), "rouge_dequantize_e2m1": (C.c_float, [C.c_uint8]),
    "rouge_mx_quantize_f32": (_I, [_P, _I, _I, _P, _P]),
    "rouge_mx_quantize_f32_e2m1": (_I, [_P, _I, _P, _P]),
    "rouge_nvfp4_quantize_f32": (_I, [_P, _I, C.c_float, _P, _P]),
    "rouge_mx_dequantize_f32": (None, [_P, _P, _I, _I, _P]),
    "rouge_mx_dequantize_f32_e2m1": (None, [_P, _P, _I, _P]),
    "rouge_b200_convert_f32_to_f16": (_I, [_P, _SZ, _P, _P]),
    "rouge_b200_convert_f32_to_bf16": (_I, [_P, _SZ, _P, _P]),
    "rouge_b200_convert_e4m3_to_f32": (_I, [_P, _SZ, _P, _P]),
    "rouge_b200_gemm_i8": (_I, [_I, _I, _I, _P, _P, _I, _P, _I, _P, _I, _P, _I, _I, _P]),
    "rouge_b200_gemm_i8_bcast": (_I, [_I, _I, _I, _P, _P, _I, _P, _I, _P, _I, _P, _P, _I,
                                      C.c_longlong, _I, _I, _P]),
    "rouge_b200_gemm_e4m3": (_I, [_I, _I, _I, _P, _P, _I, _P, _P, _P, _I, _I, _P]),
    "rouge_b200_gemm_f16": (_I, [_I, _I, _I, _P, _P, _I, _I, _P, _I, _I, _P]),
    "rouge_b200_gemm_i8_fused": (_I, [_I, _I, _I, _P, _P, _I, _P, _I, _P, _I, C.POINTER(_EpilogueC),
                                      _P, _I, _I, _P]),
    "rouge_b200_gemm_e4m3_fused": (_I, [_I, _I, _I, _P, _P, _I, _P, _P, C.POINTER(_EpilogueC), _P, _I,
                                        _I, _P]),
    "rouge_b200_gemm_f16_fused": (_I, [_I, _I, _I, _P, _P, _I, _I, C.POINTER(_EpilogueC), _P, _I, _I,
                                       _P]),
    "rouge_b200_conv2d_nhwc_f16": (_I, [_I] * 9 + [_P, _P, _P, _P, _I, _P]),
    "rouge_b200_synth_uniform": (_I, [_U64, _SZ, _F, _F, _P]),
    "rouge_b200_synth_normal": (_I, [_U64, _SZ, _F, _F, _P]),
    "rouge_b200_synth_outliers": (C.c_longlong, [_U64, _SZ, _F, _F, _P]),
    "rouge_b200_synth_normal_at": (_I, [_U64, _SZ, _SZ, _F, _F, _P]),
    "rouge_b200_synth_outliers_at": (C.c_longlong, [_U64, _SZ, _SZ, _F, _F, _P]),
    "rouge_b200_unshard_columns": (_I, [_P, _P, _I, _I, _I, _I, _I, _I, _I, _P]),
}

_lib = None


def lib() -> C.CDLL:
    """The loaded shared library (raises if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: run __graft_entry__.build() or "
                               f"make -C rouge-v_b200")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in _SIGS.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def declared_symbols() -> list[str]:
    """Names of every function declared in include/rouge/numerics_b200.h."""
    text = open(HEADER).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(rouge_\w+)\s*\(", text)))


def _check(fn: str, status: int) -> None:
    if status != OK:
        msg = lib().rouge_b200_status_string(status).decode()
        raise RougeB200Error(fn, status, msg)


def _stream():
    """The current CUDA stream of the current device, as a handle. torch's
    raw-handle accessor costs ~0.1 us against ~3 us for building a Stream
    object; the public call is the fallback where the accessor is absent."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if raw is not None:
        return C.c_void_p(raw(torch.cuda.current_device()))
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dp(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _hp(a):
    return a.ctypes.data_as(_P)


# ----------------------------------------------------------------- device API

def quantize_i8_rows(x, scales, out):
    _check("rouge_b200_quantize_i8_rows", lib().rouge_b200_quantize_i8_rows(
        _dp(x), x.shape[0], x.shape[1], _dp(scales), _dp(out), _stream()))


def dequantize_i8_rows(q, scales, out, scale=0.0):
    _check("rouge_b200_dequantize_i8_rows", lib().rouge_b200_dequantize_i8_rows(
        _dp(q), q.shape[0], q.shape[1], _dp(scales), scale, _dp(out), _stream()))


def quantize_i8_group(x, groups, scales, zeros, out):
    _check("rouge_b200_quantize_i8_group", lib().rouge_b200_quantize_i8_group(
        _dp(x), x.shape[0], x.shape[1], groups, _dp(scales), _dp(zeros), _dp(out), _stream()))


def dequantize_i8_group(q, groups, scales, zeros, out):
    _check("rouge_b200_dequantize_i8_group", lib().rouge_b200_dequantize_i8_group(
        _dp(q), q.shape[0], q.shape[1], groups, _dp(scales), _dp(zeros), _dp(out), _stream()))


def absmax(x, amax):
    _check("rouge_b200_absmax_f32", lib().rouge_b200_absmax_f32(_dp(x), x.numel(), _dp(amax), _stream()))


def quantize_e4m3_scaled(x, amax, scale_out, out):
    _check("rouge_b200_quantize_e4m3_scaled", lib().rouge_b200_quantize_e4m3_scaled(
        _dp(x), x.numel(), _dp(amax), _dp(scale_out), _dp(out), _stream()))


def quantize_e4m3_tensor(x, amax_out, scale_out, out):
    _check("rouge_b200_quantize_e4m3_tensor", lib().rouge_b200_quantize_e4m3_tensor(
        _dp(x), x.numel(), _dp(amax_out), _dp(scale_out), _dp(out), _stream()))


FMT_E4M3, FMT_E5M2, FMT_E2M1 = 0, 1, 4


def mx_quantize(x, fmt, codes, scales):
    """MXFP8 / MXFP4 block quantization of a flat f32 tensor (blocks of 32)."""
    _check("rouge_b200_mx_quantize", lib().rouge_b200_mx_quantize(
        _dp(x), x.numel(), fmt, _dp(codes), _dp(scales), _stream()))


def nvfp4_quantize(x, global_scale, codes, scales):
    _check("rouge_b200_nvfp4_quantize", lib().rouge_b200_nvfp4_quantize(
        _dp(x), x.numel(), global_scale, _dp(codes), _dp(scales), _stream()))


def mx_dequantize(codes, scales, fmt, out):
    _check("rouge_b200_mx_dequantize", lib().rouge_b200_mx_dequantize(
        _dp(codes), _dp(scales), codes.numel(), fmt, _dp(out), _stream()))


def mx_scale_atoms(scales, rows, K, atoms):
    """[rows][K/32] E8M0 scales -> the tensor-core atom layout of gemm_mx."""
    _check("rouge_b200_mx_scale_atoms", lib().rouge_b200_mx_scale_atoms(
        _dp(scales), rows, K, _dp(atoms), _stream()))


def mx_scale_atoms_bytes(rows, K):
    return lib().rouge_b200_mx_scale_atoms_bytes(rows, K)


def gemm_mx(A, fmt_a, sfa, B, fmt_b, sfb, C, out_type):
    """C[M][N] = (A x 2^sfa) . (B x 2^sfb)^T, A [M][K], B [N][K] e4m3/e5m2 codes."""
    M, K = A.shape
    N = B.shape[0]
    _check("rouge_b200_gemm_mx", lib().rouge_b200_gemm_mx(
        M, N, K, _dp(A), fmt_a, _dp(sfa), _dp(B), fmt_b, _dp(sfb), _dp(C), C.shape[1], out_type,
        _stream()))


def nvfp4_scale_atoms_bytes(rows, K):
    return lib().rouge_b200_nvfp4_scale_atoms_bytes(rows, K)


def nvfp4_scale_atoms(scales, rows, K, atoms):
    """[rows][K/16] UE4M3 scales -> the tensor-core atom layout of gemm_nvfp4."""
    _check("rouge_b200_nvfp4_scale_atoms", lib().rouge_b200_nvfp4_scale_atoms(
        _dp(scales), rows, K, _dp(atoms), _stream()))


def nvfp4_quantize_packed(x, global_scale, packed, scales):
    _check("rouge_b200_nvfp4_quantize_packed", lib().rouge_b200_nvfp4_quantize_packed(
        _dp(x), x.numel(), global_scale, _dp(packed), _dp(scales), _stream()))


def fp4_pack(codes, packed):
    """e2m1 codes (one per byte) -> two per byte, lower index in the low nibble."""
    _check("rouge_b200_fp4_pack", lib().rouge_b200_fp4_pack(
        _dp(codes), codes.numel(), _dp(packed), _stream()))


def gemm_nvfp4(A, sfa, gs_a, B, sfb, gs_b, C, out_type):
    """C[M][N] = gs_a gs_b (A x sfa) . (B x sfb)^T, A [M][K/2], B [N][K/2] packed e2m1."""
    M, K = A.shape[0], 2 * A.shape[1]
    N = B.shape[0]
    _check("rouge_b200_gemm_nvfp4", lib().rouge_b200_gemm_nvfp4(
        M, N, K, _dp(A), _dp(sfa), None if gs_a is None else _dp(gs_a), _dp(B), _dp(sfb),
        None if gs_b is None else _dp(gs_b), _dp(C), C.shape[1], out_type, _stream()))


def mxfp4_scale_atoms_bytes(rows, K):
    return lib().rouge_b200_mxfp4_scale_atoms_bytes(rows, K)


def mxfp4_scale_atoms(scales, rows, K, atoms):
    _check("rouge_b200_mxfp4_scale_atoms", lib().rouge_b200_mxfp4_scale_atoms(
        _dp(scales), rows, K, _dp(atoms), _stream()))


def gemm_mxfp4(A, sfa, B, sfb, C, out_type):
    """C[M][N] = (A x 2^sfa) . (B x 2^sfb)^T, A [M][K/2], B [N][K/2] packed e2m1."""
    M, K = A.shape[0], 2 * A.shape[1]
    N = B.shape[0]
    _check("rouge_b200_gemm_mxfp4", lib().rouge_b200_gemm_mxfp4(
        M, N, K, _dp(A), _dp(sfa), _dp(B), _dp(sfb), _dp(C), C.shape[1], out_type, _stream()))


def attention_gqa(Q, K, V, O, scale=0.0, causal=1, window=0, kv_off=0, Kq=None, Vq=None,
                  scales_k=None, scales_v=None, workspace=None):
    """O[Hq][S][Dh] from Q[Hq][S][Dh] and K/V[Hkv][Skv][Dh] (f32, or e4m3 Kq/Vq with
    per-head scales); workspace: a uint8 tensor of attention_workspace() bytes."""
    Hq, S, Dh = Q.shape
    src = K if Kq is None else Kq
    Hkv, Skv = src.shape[0], src.shape[1]
    if workspace is None:
        import torch
        workspace = torch.empty(attention_workspace(S, Skv, Dh, Hq, Hkv, Kq is not None),
                                dtype=torch.uint8, device=Q.device)
    d = lambda t: None if t is None else _dp(t)  # noqa: E731
    _check("rouge_b200_attention_gqa", lib().rouge_b200_attention_gqa(
        S, Skv, Dh, Hq, Hkv, _dp(Q), d(K), d(V), d(Kq), d(Vq), d(scales_k), d(scales_v), _dp(O),
        scale, causal, window, kv_off, _dp(workspace), workspace.numel(), _stream()))


def attention_workspace(S, Skv, Dh, Hq, Hkv, fp8_kv=False):
    return lib().rouge_b200_attention_workspace(S, Skv, Dh, Hq, Hkv, int(bool(fp8_kv)))


def transformer_block_workspace(S, D, Hq, Hkv, Dq, Dff):
    return lib().rouge_b200_transformer_block_workspace(S, D, Hq, Hkv, Dq, Dff)


def transformer_block(x, wrms1, wq, wk, wv, wo, wrms2, wgate, wup, wdown, Hq, Hkv, Dq, out,
                      rope_theta=10000.0, rms_eps=1e-5, workspace=None):
    S, D = x.shape
    Dff = wgate.shape[1]
    if workspace is None:
        import torch
        workspace = torch.empty(transformer_block_workspace(S, D, Hq, Hkv, Dq, Dff),
                                dtype=torch.uint8, device=x.device)
    _check("rouge_b200_transformer_block", lib().rouge_b200_transformer_block(
        S, D, Hq, Hkv, Dq, Dq, _dp(x), _dp(wrms1), _dp(wq), _dp(wk), _dp(wv), _dp(wo), _dp(wrms2),
        _dp(wgate), _dp(wup), _dp(wdown), Dff, rope_theta, rms_eps, _dp(out), _dp(workspace),
        workspace.numel(), _stream()))


Q_I8_ROWS, Q_MX_E4M3 = 0, 1


def add_rmsnorm_quant(x, residual, w, eps, out_fmt, codes, scales, h_out=None):
    """h_out = x + residual (both None: h = x), then the 8-bit codes and scales of
    RMSNorm(h) * w: out_fmt Q_I8_ROWS (int8 [rows][cols], f32 [rows]) or Q_MX_E4M3
    (uint8 [rows][cols], uint8 [rows][cols / 32]). Rows of x, residual and h_out
    may be strided; codes and scales are contiguous."""
    import torch
    rows, cols = x.shape
    for t in (residual, h_out):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError("residual and h_out: shape and type of x expected")
    for t in (x, residual, h_out):
        if t is not None and cols > 1 and t.stride(1) != 1:
            raise ValueError("contiguous rows expected")
    if w.dtype != torch.float32 or w.shape != (cols,) or not w.is_contiguous():
        raise ValueError(f"w: contiguous float32 [{cols}] expected")
    size, n = (4, rows) if out_fmt == Q_I8_ROWS else (1, rows * (cols // 32))
    if (codes.element_size() != 1 or codes.numel() < rows * cols or scales.element_size() != size or
            scales.numel() < n or not (codes.is_contiguous() and scales.is_contiguous())):
        raise ValueError(f"codes: {rows * cols} contiguous bytes, scales: {n} contiguous elements of {size} bytes "
                         "expected")
    _check_device(x, residual, w, codes, scales, h_out)
    ld = lambda t: 0 if t is None else t.stride(0) if rows > 1 else max(cols, t.stride(0))  # noqa: E731
    _check("rouge_b200_add_rmsnorm_quant", lib().rouge_b200_add_rmsnorm_quant(
        _ptr(x), ld(x), _ptr(residual), ld(residual), _ptr(w), eps, rows, cols, _type_of(x), _ptr(h_out),
        ld(h_out), out_fmt, _ptr(codes), _ptr(scales), _stream()))


class KV4Cache:
    """A paged 4-bit key / value cache (RougeB200KV4): uint8 tensors
    k_codes, v_codes [pages][Hkv][page][Dh / 2], k_scales, v_scales
    [pages][Hkv][page][Dh / 16] (contiguous), gs_k, gs_v f32 [Hkv] or None."""

    def __init__(self, k_codes, k_scales, v_codes, v_scales, gs_k=None, gs_v=None):
        import torch
        pages, Hkv, page, half = k_codes.shape
        codes, scales = k_codes.shape, (pages, Hkv, page, half // 8)
        if (v_codes.shape != codes or k_scales.shape != scales or v_scales.shape != scales or
                not (k_codes.is_contiguous() and k_scales.is_contiguous() and v_codes.is_contiguous() and
                     v_scales.is_contiguous()) or k_codes.element_size() != 1 or k_scales.element_size() != 1 or
                v_codes.element_size() != 1 or v_scales.element_size() != 1):
            raise ValueError(f"codes: contiguous bytes {tuple(codes)}, scales: {scales} expected")
        for t in (gs_k, gs_v):
            if t is not None and (t.shape != (Hkv,) or t.dtype != torch.float32 or not t.is_contiguous()):
                raise ValueError(f"contiguous float32 [{Hkv}] expected")
        self.tensors = (k_codes, k_scales, v_codes, v_scales, gs_k, gs_v)
        self.pages, self.Hkv, self.page, self.Dh = pages, Hkv, page, 2 * half
        self.c = _KV4C(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
                       _ptr(gs_k), _ptr(gs_v), pages, page, Hkv, 2 * half)
        self.ref = C.byref(self.c)

    @classmethod
    def empty(cls, pages, Hkv, page, Dh, gs_k=None, gs_v=None, device="cuda"):
        """A cache of zeros."""
        import torch
        z = lambda n: torch.zeros(pages, Hkv, page, n, dtype=torch.uint8, device=device)  # noqa: E731
        return cls(z(Dh // 2), z(Dh // 16), z(Dh // 2), z(Dh // 16), gs_k, gs_v)


def _kv4_tokens(cache, K, V, slots):
    import torch
    T = K.shape[0]
    for t in (K, V):
        if t.shape != (T, cache.Hkv, cache.Dh) or t.dtype != K.dtype or (T and (
                t.stride(2) != 1 or t.stride(1) != cache.Dh)):
            raise ValueError(f"[{T}, {cache.Hkv}, {cache.Dh}] with contiguous tokens expected")
    if slots.shape != (T,) or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError(f"slots: contiguous int32 [{T}] expected")
    _check_device(K, V, slots, *cache.tensors)
    ld = lambda t: max(t.stride(0), cache.Hkv * cache.Dh) if T < 2 else t.stride(0)  # noqa: E731
    return (K.data_ptr(), ld(K), V.data_ptr(), ld(V), _type_of(K), T, slots.data_ptr(), _stream())


def kv4_write(cache, K, V, slots):
    """K, V [T][Hkv][Dh] (f32, f16 or bf16; tokens may be strided) into the
    slots [T] (int32; negative: skipped) of a KV4Cache."""
    _check("rouge_b200_kv4_write",
           lib().rouge_b200_kv4_write(cache.ref, *_kv4_tokens(cache, K, V, slots)))


def kv4_read(cache, slots, K, V):
    """The values of slots [T] into K, V [T][Hkv][Dh]."""
    _check("rouge_b200_kv4_read",
           lib().rouge_b200_kv4_read(cache.ref, *_kv4_tokens(cache, K, V, slots)))


def attention_kv4_workspace(B, Hq, Hkv, Dh, max_q, max_kv, type):
    return lib().rouge_b200_attention_kv4_workspace(B, Hq, Hkv, Dh, max_q, max_kv, type)


def attention_kv4(Q, cache, kv_len, page_table, cu_q=None, max_q=None, O=None, scale=0.0, causal=1,
                  window=0, workspace=None):
    """O[T][Hq][Dh] of Q[T][Hq][Dh] over a KV4Cache: sequence b has kv_len[b] keys
    on the pages page_table[b] and the queries cu_q[b] .. cu_q[b + 1] (None: one
    each), at most max_q of them, which is required with cu_q: rows past the max_q-th
    of a sequence are not computed, and sync_status() raises. workspace: uint8, attention_kv4_workspace() bytes."""
    import torch
    B, max_pages = page_table.shape
    T, Hq, Dh = Q.shape
    if O is None:
        O = torch.empty_like(Q)
    if O.shape != Q.shape or O.dtype != Q.dtype or not O.is_contiguous() or not Q.is_contiguous():
        raise ValueError("Q, O: contiguous, of one shape and type")
    if Dh != cache.Dh:
        raise ValueError(f"head size {Dh}, and {cache.Dh} in the cache")
    i32 = torch.int32
    if (kv_len.dtype != i32 or kv_len.shape != (B,) or page_table.dtype != i32 or
            not (kv_len.is_contiguous() and page_table.is_contiguous())):
        raise ValueError(f"contiguous int32 kv_len [{B}] and page_table [{B}, {max_pages}] expected")
    if cu_q is None:
        if T < B or max_q not in (None, 1):
            raise ValueError("without cu_q: one query per sequence")
        max_q = 1
    elif cu_q.dtype != i32 or cu_q.shape != (B + 1,) or not cu_q.is_contiguous():
        raise ValueError(f"cu_q: contiguous int32 [{B + 1}] expected")
    elif max_q is None and T > 0:
        raise ValueError("max_q: the most queries of one sequence expected with cu_q")
    _check_device(Q, O, kv_len, page_table, cu_q, workspace, *cache.tensors)
    ty = _type_of(Q)
    if T == 0:  # (an empty tensor has no address)
        return O
    if workspace is None:
        workspace = torch.empty(attention_kv4_workspace(B, Hq, cache.Hkv, Dh, max_q,
                                                        max_pages * cache.page, ty),
                                dtype=torch.uint8, device=Q.device)
    _check("rouge_b200_attention_kv4", lib().rouge_b200_attention_kv4(
        cache.ref, Q.data_ptr(), ty, B, Hq, _ptr(cu_q), max_q, kv_len.data_ptr(), page_table.data_ptr(),
        max_pages, O.data_ptr(), scale, causal, window, workspace.data_ptr(), workspace.numel(), _stream()))
    return O


def convert_f32_to_f16(x, out):
    _check("rouge_b200_convert_f32_to_f16", lib().rouge_b200_convert_f32_to_f16(
        _dp(x), x.numel(), _dp(out), _stream()))


def convert_f32_to_bf16(x, out):
    _check("rouge_b200_convert_f32_to_bf16", lib().rouge_b200_convert_f32_to_bf16(
        _dp(x), x.numel(), _dp(out), _stream()))


def convert_e4m3_to_f32(x, out):
    _check("rouge_b200_convert_e4m3_to_f32", lib().rouge_b200_convert_e4m3_to_f32(
        _dp(x), x.numel(), _dp(out), _stream()))


T_F32, T_F16, T_BF16 = 0, 1, 2
ACT_NONE, ACT_RELU, ACT_GELU, ACT_SILU = 0, 1, 2, 3


_types = {}


def _type_of(t):
    """ROUGE_B200_T_* of a floating tensor."""
    if not _types:
        import torch
        _types.update({torch.float32: T_F32, torch.float16: T_F16, torch.bfloat16: T_BF16})
    ty = _types.get(t.dtype)
    if ty is None:
        raise TypeError(f"float32, float16 or bfloat16 tensor expected, got {t.dtype}")
    return ty


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check_device(*tensors):
    """Raises for a tensor that is not on the current CUDA device, where the launch goes."""
    import torch
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensor on {t.device}, current device cuda:{dev}")


def _pitch(t):
    """Row pitch of a matrix with contiguous rows (a single row's stride can be any)."""
    return max(t.stride(0), t.shape[-1]) if t.shape[0] < 2 else t.stride(0)


class Epilogue:
    """Epilogue of gemm_i8 / gemm_e4m3 / gemm_f16: act(. + bias[n]) + residual[m][n],
    each optional. bias: f32 [N]; residual: f32, f16 or bf16 [M][N], rows
    contiguous (it may be the output tensor itself); act: ACT_*."""

    def __init__(self, bias=None, act=ACT_NONE, residual=None):
        self.tensors = (bias, residual)  # (kept alive)
        self.c = _EpilogueC(None if bias is None else bias.data_ptr(),
                            None if residual is None else residual.data_ptr(),
                            0 if residual is None else _pitch(residual),
                            T_F32 if residual is None else _type_of(residual), act)
        self.ref = C.byref(self.c)

    def check(self, M, N, *others):
        """Raises unless the tensors fit an M x N output and lie, as the others, on the current device."""
        import torch
        bias, residual = self.tensors
        if bias is not None and (bias.dtype != torch.float32 or bias.shape != (N,) or
                                 not bias.is_contiguous()):
            raise ValueError(f"bias: contiguous float32 [{N}] expected")
        if residual is not None and (residual.shape != (M, N) or (N > 1 and residual.stride(1) != 1)):
            raise ValueError(f"residual: [{M}, {N}] with contiguous rows expected")
        _check_device(bias, residual, *others)


_out_types = {}


def _fused_sizes(epilogue, A, B, b_layout, C_, out_type, esize, scale_a, na, scale_b, nb):
    """Raises unless the tensors of a product with an epilogue have the sizes, element sizes and layouts
    that the kernel reads and writes; na, nb: elements of the scales, None for M and N."""
    import torch
    if not _out_types:
        _out_types.update({OUT_F32: torch.float32, OUT_BF16: torch.bfloat16})
    M, K = A.shape
    N = B.shape[1 if b_layout == B_KN else 0]
    if B.shape[0 if b_layout == B_KN else 1] != K or not (A.is_contiguous() and B.is_contiguous()):
        raise ValueError(f"contiguous A [M, K] and B {'[K, N]' if b_layout == B_KN else '[N, K]'} expected")
    if A.element_size() != esize or B.element_size() != esize:
        raise ValueError(f"A, B: elements of {esize} bytes expected")
    if C_.shape != (M, N) or (N > 1 and C_.stride(1) != 1) or C_.dtype != _out_types.get(out_type, C_.dtype):
        raise ValueError(f"output: [{M}, {N}] of out_type with contiguous rows expected")
    for t, n in ((scale_a, M if na is None else na), (scale_b, N if nb is None else nb)):
        if t is not None and (t.dtype != torch.float32 or t.numel() < n or not t.is_contiguous()):
            raise ValueError(f"scales: {n} contiguous float32 expected")
    epilogue.check(M, N, A, B, C_, scale_a, scale_b)


def gemm_i8(A, B, b_layout, C_, out_type, scales_a=None, a_rows=1, scales_b=None, b_cols=1,
            epilogue=None):
    M, K = A.shape
    N = B.shape[1] if b_layout == B_KN else B.shape[0]
    if epilogue is not None:
        _fused_sizes(epilogue, A, B, b_layout, C_, out_type, 1, scales_a, None if a_rows else 1, scales_b,
                     None if b_cols else 1)
        _check("rouge_b200_gemm_i8_fused", lib().rouge_b200_gemm_i8_fused(
            M, N, K, _ptr(A), _ptr(B), b_layout, _ptr(scales_a), a_rows, _ptr(scales_b), b_cols,
            epilogue.ref, _ptr(C_), _pitch(C_), out_type, _stream()))
        return
    _check("rouge_b200_gemm_i8", lib().rouge_b200_gemm_i8(
        M, N, K, _dp(A), _dp(B), b_layout, _dp(scales_a), a_rows, _dp(scales_b), b_cols,
        _dp(C_), C_.stride(0), out_type, _stream()))


def gemm_i8_bcast(A, B, b_layout, out_type, scales_a, a_rows, scales_b, b_cols, mc_ptr=0,
                  peer_ptrs=(), ldc=0, col_off=0):
    """rouge_b200_gemm_i8_bcast: this rank's M x N block written to column
    col_off of every rank's [M][ldc] output, through the multicast address
    mc_ptr (an int) or the list of peer pointers peer_ptrs (ints)."""
    M, K = A.shape
    N = B.shape[0] if b_layout == B_NK else B.shape[1]
    peers = (C.c_void_p * 8)(*[C.c_void_p(p) for p in peer_ptrs]) if not mc_ptr else None
    _check("rouge_b200_gemm_i8_bcast", lib().rouge_b200_gemm_i8_bcast(
        M, N, K, _dp(A), _dp(B), b_layout, _dp(scales_a), a_rows, _dp(scales_b), b_cols,
        C.c_void_p(mc_ptr) if mc_ptr else None, peers, 0 if mc_ptr else len(peer_ptrs), ldc,
        col_off, out_type, _stream()))


def w8a8_workspace(M, device):
    """Zeroed workspace of rouge_b200_w8a8_linear for M rows (every call
    leaves it zeroed)."""
    import torch
    n = lib().rouge_b200_w8a8_workspace_bytes(M)
    return torch.zeros((n + 3) // 4, dtype=torch.int32, device=device)


def w8a8_linear(X, Wq, sw, Aq, sa, C_, out_type, ws):
    """Aq, sa = per-row int8 quantization of X[M][K]; C = dequant(Aq . Wq^T)
    with Wq[N][K] codes and sw[N] scales (one fused launch when it applies)."""
    M, K = X.shape
    N = Wq.shape[0]
    _check("rouge_b200_w8a8_linear", lib().rouge_b200_w8a8_linear(
        M, N, K, _dp(X), _dp(Wq), _dp(sw), _dp(Aq), _dp(sa), _dp(C_), C_.stride(0), out_type,
        _dp(ws), _stream()))


def gemm_e4m3(A, B, b_layout, C_, out_type, scale_a=None, scale_b=None, epilogue=None):
    M, K = A.shape
    N = B.shape[1] if b_layout == B_KN else B.shape[0]
    if epilogue is not None:
        _fused_sizes(epilogue, A, B, b_layout, C_, out_type, 1, scale_a, 1, scale_b, 1)
        _check("rouge_b200_gemm_e4m3_fused", lib().rouge_b200_gemm_e4m3_fused(
            M, N, K, _ptr(A), _ptr(B), b_layout, _ptr(scale_a), _ptr(scale_b), epilogue.ref,
            _ptr(C_), _pitch(C_), out_type, _stream()))
        return
    _check("rouge_b200_gemm_e4m3", lib().rouge_b200_gemm_e4m3(
        M, N, K, _dp(A), _dp(B), b_layout, _dp(scale_a), _dp(scale_b), _dp(C_), C_.stride(0),
        out_type, _stream()))


def gemm_f16(A, B, b_layout, C_, out_type, is_bf16=False, epilogue=None):
    M, K = A.shape
    N = B.shape[1] if b_layout == B_KN else B.shape[0]
    if epilogue is not None:
        _fused_sizes(epilogue, A, B, b_layout, C_, out_type, 2, None, 1, None, 1)
        _check("rouge_b200_gemm_f16_fused", lib().rouge_b200_gemm_f16_fused(
            M, N, K, _ptr(A), _ptr(B), b_layout, int(is_bf16), epilogue.ref, _ptr(C_),
            _pitch(C_), out_type, _stream()))
        return
    _check("rouge_b200_gemm_f16", lib().rouge_b200_gemm_f16(
        M, N, K, _dp(A), _dp(B), b_layout, int(is_bf16), _dp(C_), C_.stride(0), out_type,
        _stream()))


def conv2d_nhwc_f16(X, Wt, bias, Y, stride, pad, is_bf16=False):
    """X[N][H][W][Cin], Wt[Cout][KH][KW][Cin] (16-bit codes), Y[N][OH][OW][Cout] f32."""
    N, H, W, Cin = X.shape
    Cout, KH, KW, _ = Wt.shape
    _check("rouge_b200_conv2d_nhwc_f16", lib().rouge_b200_conv2d_nhwc_f16(
        N, H, W, Cin, Cout, KH, KW, stride, pad, _dp(X), _dp(Wt), _dp(bias), _dp(Y),
        int(is_bf16), _stream()))


def sync_status():
    _check("rouge_b200_sync_status", lib().rouge_b200_sync_status(_stream()))


def check_wait_limit(limit_ns):
    """Launches the never-completing bounded wait (limit_ns) on the current
    stream and returns the status rouge_b200_sync_status then reports
    (ROUGE_B200_ETIMEOUT when the limit works)."""
    L = lib()
    _check("rouge_b200_check_wait_limit", L.rouge_b200_check_wait_limit(int(limit_ns), _stream()))
    return L.rouge_b200_sync_status(_stream())


class tile_mode:
    """Context manager selecting the GEMM / convolution tile shapes
    (TILES_AUTO, TILES_SINGLE or TILES_PAIR) and restoring the previous mode."""

    def __init__(self, mode: int):
        self.mode = mode

    def __enter__(self):
        prev = lib().rouge_b200_set_tile_mode(self.mode)
        if prev < 0:
            raise RougeB200Error("rouge_b200_set_tile_mode", prev, "unknown mode")
        self.prev = prev
        return self

    def __exit__(self, *exc):
        lib().rouge_b200_set_tile_mode(self.prev)
        return False


class clock_probe:
    """Context manager recording, for every GEMM / convolution launch on the
    current device while it is active, each of the first `ctas` CTAs'
    %clock64 and %globaltimer at its start and end
    (rouge_b200_set_clock_probe). After the launch of interest,
    `sm_mhz()` gives the SM clock each CTA ran at, from those stamps."""

    def __init__(self, ctas: int, device=None):
        import torch
        self.ctas = int(ctas)
        self.stamps = torch.zeros(4 * self.ctas, dtype=torch.int64, device=device or "cuda")

    def __enter__(self):
        _check("rouge_b200_set_clock_probe",
               lib().rouge_b200_set_clock_probe(_dp(self.stamps), self.ctas))
        return self

    def __exit__(self, *exc):
        lib().rouge_b200_set_clock_probe(None, 0)
        return False

    def sm_mhz(self):
        """Per-CTA SM clock in MHz of the last launch (CTAs that wrote no
        stamps are left out)."""
        import numpy as np
        w = self.stamps.view(-1, 4).cpu().numpy().astype(np.float64)
        ok = (w[:, 3] > w[:, 1]) & (w[:, 2] > w[:, 0])
        return (w[ok, 2] - w[ok, 0]) / (w[ok, 3] - w[ok, 1]) * 1000.0


# ------------------------------------------------------------- host drop-in API

def _last_error(fn):
    st = lib().rouge_b200_last_error()
    lib().rouge_b200_clear_error()
    if st != OK:
        raise RougeB200Error(fn, st, lib().rouge_b200_status_string(st).decode())


def host_quantize_i8_channel(x: np.ndarray):
    x = np.ascontiguousarray(x, np.float32)
    rows, cols = x.shape
    s = np.empty(rows, np.float32)
    q = np.empty((rows, cols), np.int8)
    lib().rouge_b200_clear_error()
    if lib().rouge_quantize_i8_channel(_hp(x), rows, cols, _hp(s), _hp(q)) != 1:
        _last_error("rouge_quantize_i8_channel")
        raise RougeB200Error("rouge_quantize_i8_channel", EINVAL, "returned 0")
    return q, s


def host_quantize_i8_tensor(x: np.ndarray):
    x = np.ascontiguousarray(x, np.float32).ravel()
    s = np.zeros(1, np.float32)
    q = np.empty(x.size, np.int8)
    lib().rouge_b200_clear_error()
    if lib().rouge_quantize_i8_tensor(_hp(x), x.size, _hp(s), _hp(q)) != 1:
        _last_error("rouge_quantize_i8_tensor")
        raise RougeB200Error("rouge_quantize_i8_tensor", EINVAL, "returned 0")
    return q, float(s[0])


def host_quantize_i8_group(x: np.ndarray, groups: int):
    x = np.ascontiguousarray(x, np.float32)
    rows, cols = x.shape
    s = np.empty(rows * groups, np.float32)
    z = np.empty(rows * groups, np.uint8)
    q = np.empty((rows, cols), np.uint8)
    lib().rouge_b200_clear_error()
    if lib().rouge_quantize_i8_group(_hp(x), rows, cols, groups, _hp(s), _hp(z), _hp(q)) != 1:
        _last_error("rouge_quantize_i8_group")
        raise RougeB200Error("rouge_quantize_i8_group", EINVAL, "returned 0")
    return q, s, z


def host_dequantize_i8_group(q: np.ndarray, groups: int, s: np.ndarray, z: np.ndarray):
    q = np.ascontiguousarray(q, np.uint8)
    s = np.ascontiguousarray(s, np.float32)
    z = np.ascontiguousarray(z, np.uint8)
    out = np.empty(q.shape, np.float32)
    lib().rouge_b200_clear_error()
    lib().rouge_dequantize_i8_group(_hp(q), q.shape[0], q.shape[1], groups, _hp(s), _hp(z), _hp(out))
    _last_error("rouge_dequantize_i8_group")
    return out


def host_dequantize_i8_channel(q: np.ndarray, scales: np.ndarray):
    q = np.ascontiguousarray(q, np.int8)
    scales = np.ascontiguousarray(scales, np.float32)
    out = np.empty(q.shape, np.float32)
    lib().rouge_b200_clear_error()
    lib().rouge_dequantize_i8_channel(_hp(q), q.shape[0], q.shape[1], _hp(scales), _hp(out))
    _last_error("rouge_dequantize_i8_channel")
    return out


def host_dequantize_i8_tensor(q: np.ndarray, scale: float):
    q = np.ascontiguousarray(q, np.int8).ravel()
    out = np.empty(q.size, np.float32)
    lib().rouge_b200_clear_error()
    lib().rouge_dequantize_i8_tensor(_hp(q), q.size, scale, _hp(out))
    _last_error("rouge_dequantize_i8_tensor")
    return out


def host_gemm_i8(A, B_kn, sa, a_rows, sb, b_cols, out=None):
    A = np.ascontiguousarray(A, np.int8)
    B_kn = np.ascontiguousarray(B_kn, np.int8)
    sa = np.ascontiguousarray(np.atleast_1d(sa), np.float32)
    sb = np.ascontiguousarray(np.atleast_1d(sb), np.float32)
    M, K = A.shape
    N = B_kn.shape[1]
    out = np.empty((M, N), np.float32) if out is None else out
    lib().rouge_b200_clear_error()
    lib().rouge_gemm_i8(M, N, K, _hp(A), _hp(B_kn), _hp(sa), a_rows, _hp(sb), b_cols, _hp(out))
    _last_error("rouge_gemm_i8")
    return out


def _host_gemm_codes(name, A, B_kn, dtype):
    A = np.ascontiguousarray(A, dtype)
    B_kn = np.ascontiguousarray(B_kn, dtype)
    M, K = A.shape
    N = B_kn.shape[1]
    out = np.empty((M, N), np.float32)
    lib().rouge_b200_clear_error()
    getattr(lib(), name)(M, N, K, _hp(A), _hp(B_kn), _hp(out), None)
    _last_error(name)
    return out


def host_gemm_e4m3(A, B_kn):
    return _host_gemm_codes("rouge_gemm_e4m3", A, B_kn, np.uint8)


def host_gemm_f32(A, B_kn, cfg=None, out=None):
    """rouge_gemm_f32: A[M][K] . B[K][N] (f32, host arrays); cfg a
    GemmConfig or None."""
    A = np.ascontiguousarray(A, np.float32)
    B_kn = np.ascontiguousarray(B_kn, np.float32)
    M, K = A.shape
    N = B_kn.shape[1]
    out = np.empty((M, N), np.float32) if out is None else out
    lib().rouge_b200_clear_error()
    lib().rouge_gemm_f32(M, N, K, _hp(A), _hp(B_kn), _hp(out),
                         None if cfg is None else C.cast(C.pointer(cfg), _P))
    _last_error("rouge_gemm_f32")
    return out


def gemm_candidates():
    """The tuner's candidate configurations (rouge_gemm_candidate)."""
    return [lib().rouge_gemm_candidate(i) for i in range(lib().rouge_gemm_candidate_count())]


def gemm_tuned(A, B_kn, out):
    """rouge_gemm_tuned on host arrays; returns the GemmProfile."""
    M, K = A.shape
    N = B_kn.shape[1]
    return lib().rouge_gemm_tuned(M, N, K, _hp(A), _hp(B_kn), _hp(out))


def gemm_flops_per_sec(A, B_kn, out, cfg=None):
    M, K = A.shape
    N = B_kn.shape[1]
    return lib().rouge_gemm_flops_per_sec(M, N, K, _hp(A), _hp(B_kn), _hp(out),
                                          None if cfg is None else C.cast(C.pointer(cfg), _P))


def host_conv2d_f32(x, w, bias, stride, pad, implicit=False):
    """rouge_conv2d_f32 / rouge_conv_implicit_f32: x[N][Cin][H][W],
    w[Cout][Cin][KH][KW], bias[Cout] or None; returns y[N][Cout][OH][OW]."""
    x = np.ascontiguousarray(x, np.float32)
    w = np.ascontiguousarray(w, np.float32)
    N, Cin, H, W = x.shape
    Cout, _, KH, KW = w.shape
    OH = (H + 2 * pad - KH) // stride + 1
    OW = (W + 2 * pad - KW) // stride + 1
    y = np.full((N, Cout, OH, OW), np.nan, np.float32)
    b = None if bias is None else np.ascontiguousarray(bias, np.float32)
    fn = lib().rouge_conv_implicit_f32 if implicit else lib().rouge_conv2d_f32
    lib().rouge_b200_clear_error()
    fn(N, Cin, H, W, Cout, KH, KW, stride, pad, _hp(x), _hp(w), None if b is None else _hp(b),
       _hp(y), None)
    _last_error("rouge_conv_implicit_f32" if implicit else "rouge_conv2d_f32")
    return y


def host_gemm_f16(A, B_kn):
    return _host_gemm_codes("rouge_gemm_f16", A, B_kn, np.uint16)


def host_gemm_bf16(A, B_kn):
    return _host_gemm_codes("rouge_gemm_bf16", A, B_kn, np.uint16)


# ------------------------------------------------------------------ synthetic data

def synth_uniform(seed: int, shape, lo: float, hi: float, out=None) -> np.ndarray:
    out = np.empty(shape, np.float32) if out is None else out
    assert lib().rouge_b200_synth_uniform(seed, out.size, lo, hi, _hp(out)) == 0
    return out


def synth_normal(seed: int, shape, mean: float, std: float, out=None) -> np.ndarray:
    out = np.empty(shape, np.float32) if out is None else out
    assert lib().rouge_b200_synth_normal(seed, out.size, mean, std, _hp(out)) == 0
    return out


def synth_outliers(seed: int, x: np.ndarray, frac: float, mult: float, offset: int = 0) -> int:
    return int(lib().rouge_b200_synth_outliers_at(seed, offset, x.size, frac, mult, _hp(x)))


def synth_normal_at(seed: int, offset: int, shape, mean: float, std: float) -> np.ndarray:
    out = np.empty(shape, np.float32)
    assert lib().rouge_b200_synth_normal_at(seed, offset, out.size, mean, std, _hp(out)) == 0
    return out


def unshard_columns(src, dst, M, N, g, ns, R):
    """src[M/R][g][R][ns] (all-gathered bands) -> dst[M][ldd] row-major."""
    _check("rouge_b200_unshard_columns", lib().rouge_b200_unshard_columns(
        _dp(src), _dp(dst), M, N, g, ns, R, dst.stride(0), src.element_size(), _stream()))
