"""Python binding of libqwq4.so (include/qw/q4ops.h) over ctypes.

Device memory and streams come from PyTorch; every call goes through the C ABI
to the HIP kernels. There is no fallback: if the library is missing or a call
fails, a RuntimeError is raised.
"""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(os.path.dirname(_HERE), "libqwq4.so")
_lib = None

# every symbol include/qw/q4ops.h declares (checked by the CPU tests)
SYMBOLS = (
    "qw_q4_abi_version", "qw_q4_last_error", "qw_q4_gemv", "qw_q4_gemm_workspace_size", "qw_q4_gemm",
    "qw_moe_route", "qw_moe_experts_gemv", "qw_moe_experts_grouped", "qw_moe_grouped_workspace_size", "qw_moe_grouped_tile_m",
    "qw_moe_combine", "qw_q4_unpack", "qw_q4_dequant", "qw_q4_from_engine_order",
    "qw_q4_tiled_size", "qw_q4_tile", "qw_q4_untile", "qw_bf16_to_f16", "qw_read_probe",
    "qw_st_open", "qw_st_close", "qw_st_count", "qw_st_name", "qw_st_tensor",
    "qw_q4_load_staging_size", "qw_q4_load", "qw_q4_tiled_offset",
    "qw_moe_decode_workspace_size", "qw_moe_decode", "qw_moe_decode_static_max_bytes", "qw_moe_decode_static",
    "qw_moe_decode_static_reset", "qw_moe_decode_with_shared_workspace_size", "qw_moe_decode_with_shared",
    "qw_w16_gemv", "qw_w16_tiled_size", "qw_w16_tile", "qw_w16_gemv_tiled", "qw_w16_swiglu_gemv_tiled", "qw_i8_gemv", "qw_i8_tiled_size", "qw_i8_tile",
    "qw_moe_w4a8_tile_m", "qw_moe_w4a8_workspace_size", "qw_moe_experts_w4a8", "qw_quant_rows_i8", "qw_swiglu_gate",
    "qw_quant_tokens_i8", "qw_w8a8_gemm", "qw_w8a8_workspace_size", "qw_w8a8_linear", "qw_moe_w8a8_tile_m",
    "qw_moe_w8a8_workspace_size", "qw_moe_experts_w8a8", "qw_moe_sort", "qw_moe_permute",
    "qw_moe_permute_backward", "qw_moe_unpermute", "qw_moe_unpermute_backward",
    "qw_rms_norm", "qw_rms_norm_i8", "qw_rms_norm_backward_workspace_size", "qw_rms_norm_backward", "qw_lora",
    "qw_lora_backward_workspace_size", "qw_lora_backward", "qw_logprobs_workspace_size", "qw_logprobs",
    "qw_logprobs_backward",
    "qw_wcache_open", "qw_wcache_put", "qw_wcache_get", "qw_wcache_finish", "qw_wcache_close",
)

_P = ctypes.c_void_p
_I = ctypes.c_int
_I64 = ctypes.c_int64
_SZ = ctypes.c_size_t
_F = ctypes.c_float

_SIGS = {
    "qw_q4_abi_version": ([], _I),
    "qw_q4_last_error": ([], ctypes.c_char_p),
    "qw_q4_gemv": ([_P, _P, _P, _P, _I, _I, _P, _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "qw_q4_gemm_workspace_size": ([_I, _I], _SZ),
    "qw_q4_gemm": ([_P, _P, _P, _P, _I, _I, _I, _P, _I, _I, _I, _I, _P, _SZ, _P], _I),
    "qw_moe_route": ([_P, _I, _I, _I, _I] + [_P] * 11 + [_P], _I),
    "qw_moe_experts_gemv": ([_P] * 9 + [_I, _I, _I] + [_P] * 5 + [_I, _I, _I, _P, _P, _I, _P], _I),
    "qw_moe_grouped_workspace_size": ([_I, _I, _I, _I, _I], _SZ),
    "qw_moe_experts_grouped": ([_P] * 9 + [_I, _I, _I] + [_P] * 6 + [_I, _I, _I, _P, _P, _I, _P, _SZ, _P], _I),
    "qw_moe_grouped_tile_m": ([], _I),
    "qw_moe_combine": ([_P, _I, _P, _P, _P, _I, _I, _I, _I, _P, _I, _P], _I),
    "qw_q4_tiled_size": ([_I64, _I64, _P, _P, _P], None),
    "qw_q4_tile": ([_P, _P, _P, _I64, _I64, _P, _P, _P, _P], _I),
    "qw_q4_untile": ([_P, _P, _P, _I64, _I64, _P, _P, _P, _P], _I),
    "qw_q4_unpack": ([_P, _I64, _I64, _P, _P], _I),
    "qw_q4_dequant": ([_P, _P, _P, _I64, _I64, _P, _P], _I),
    "qw_q4_from_engine_order": ([_P, _P, _I64, _P], _I),
    "qw_bf16_to_f16": ([_P, _P, _I64, _P], _I),
    "qw_read_probe": ([_P, _I64, _P], _I),
    "qw_moe_decode_workspace_size": ([_I, _I, _I, _I, _I], _SZ),
    "qw_moe_decode": ([_P, _I, _P, _I, _I, _I, _I] + [_P] * 9 + [_I, _I, _P, _P, _I] + [_P] * 6 + [_I, _P, _SZ, _P], _I),
    "qw_moe_decode_static_max_bytes": ([], _SZ),
    "qw_w16_gemv": ([_P, _I, _P, _I, _I, _P, _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "qw_w16_tiled_size": ([_I, _I], _SZ),
    "qw_w16_tile": ([_P, _I, _I, _I, _P, _P], _I),
    "qw_w16_gemv_tiled": ([_P, _P, _I, _I, _P, _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "qw_w16_swiglu_gemv_tiled": ([_P, _P, _I, _I, _P, _I, _I, _I, _I, _I, _P], _I),
    "qw_i8_gemv": ([_P, _P, _I, _P, _I, _P, _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "qw_i8_tiled_size": ([_I, _I, _I, _P, _P], None),
    "qw_i8_tile": ([_P, _P, _I, _I, _I, _P, _P, _P], _I),
    "qw_moe_w4a8_tile_m": ([], _I),
    "qw_moe_w4a8_workspace_size": ([_I, _I, _I, _I], _SZ),
    "qw_moe_experts_w4a8": ([_P] * 9 + [_I, _I, _I] + [_P] * 6 + [_I, _I, _I, _P, _P, _P, _SZ, _P], _I),
    "qw_quant_rows_i8": ([_P, _I, _I, _I, _I, _P, _P, _P], _I),
    "qw_swiglu_gate": ([_P, _I, _I, _I, _P, _P], _I),
    "qw_quant_tokens_i8": ([_P, _I, _I, _I, _I, _P, _I, _P, _P], _I),
    "qw_w8a8_gemm": ([_P, _I, _P, _P, _I, _P, _I, _P, _I, _I, _I, _I, _P], _I),
    "qw_w8a8_workspace_size": ([_I, _I], _SZ),
    "qw_w8a8_linear": ([_P, _I, _P, _P, _I, _I, _I, _P, _I, _I, _I, _I, _P, _SZ, _P], _I),
    "qw_moe_w8a8_tile_m": ([], _I),
    "qw_moe_w8a8_workspace_size": ([_I, _I, _I, _I], _SZ),
    "qw_moe_experts_w8a8": ([_P] * 6 + [_I, _I, _I] + [_P] * 6 + [_I, _I, _I, _P, _P, _I, _P, _SZ, _P], _I),
    "qw_moe_sort": ([_P, _I, _I, _I, _I] + [_P] * 10, _I),
    "qw_moe_permute": ([_P, _I, _I, _I, _I, _I, _P, _P, _I, _P], _I),
    "qw_moe_permute_backward": ([_P, _I, _I, _P, _I, _I, _I, _P, _I, _I, _P], _I),
    "qw_moe_unpermute": ([_P, _I, _I, _P, _P, _I, _I, _I, _P, _I, _I, _P], _I),
    "qw_moe_unpermute_backward": ([_P, _I, _I, _P, _I, _I, _P, _P, _I, _I, _I, _P, _I, _P, _P], _I),
    "qw_rms_norm": ([_P, _I, _I, _P, _I, _I, _P, _I, _P, _I, _F, _I, _I, _P, _I, _I, _P], _I),
    "qw_rms_norm_i8": ([_P, _I, _I, _P, _I, _I, _P, _I, _P, _I, _F, _I, _I, _P, _I, _P, _P], _I),
    "qw_rms_norm_backward_workspace_size": ([_I, _I], _SZ),
    "qw_rms_norm_backward": ([_P, _I, _I, _P, _I, _I, _P, _I, _F, _P, _I, _I, _I, _P, _I, _P, _P, _SZ, _P], _I),
    "qw_lora": ([_P, _I, _I, _P, _P, _P, _P] + [_I] * 5 + [_P, _P, _I, _P, _I, _I, _P], _I),
    "qw_lora_backward_workspace_size": ([_I] * 5, _SZ),
    "qw_lora_backward": ([_P, _I, _P, _I, _I] + [_P] * 5 + [_I] * 5 + [_P, _I, _P, _I, _P, _P, _P, _SZ, _P], _I),
    "qw_logprobs_workspace_size": ([_I, _I, _I], _SZ),
    "qw_logprobs": ([_P, _I, _I, _P, _I, _I, _I] + [_P] * 6 + [_SZ, _P], _I),
    "qw_logprobs_backward": ([_P, _I, _I] + [_P] * 5 + [_I, _I, _P, _I, _P], _I),
    "qw_moe_decode_static": ([_P, _I, _P, _I, _I, _I, _I] + [_P] * 9 + [_I, _I, _P, _P, _I] + [_P] * 6 + [_I, _P], _I),
    "qw_moe_decode_with_shared_workspace_size": ([_I, _I, _I, _I, _I, _I], _SZ),
    "qw_moe_decode_with_shared": ([_P, _I, _P, _I, _I, _I, _I] + [_P] * 9 + [_I, _I, _P, _P, _I, _P, _P, _P, _I]
                                  + [_P] * 6 + [_I, _P, _SZ, _P], _I),
    "qw_moe_decode_static_reset": ([_P], _I),
    "qw_st_open": ([ctypes.c_char_p, _P], _I),
    "qw_st_close": ([_P], None),
    "qw_wcache_open": ([ctypes.c_char_p, ctypes.c_uint64, _P, _P], _I),
    "qw_wcache_put": ([_P, _P, ctypes.c_size_t, _I, _P], _I),
    "qw_wcache_get": ([_P, _P, ctypes.c_size_t, _I, _P], _I),
    "qw_wcache_finish": ([_P], _I),
    "qw_wcache_close": ([_P], None),
    "qw_st_count": ([_P], _I),
    "qw_st_name": ([_P, _I], ctypes.c_char_p),
    "qw_st_tensor": ([_P, ctypes.c_char_p, _P, _P, _P, _P, _P], _I),
    "qw_q4_load_staging_size": ([_I64, _I64], _SZ),
    "qw_q4_load": ([_P, ctypes.c_char_p, _I64, _I64, _P, _P, _P, _SZ, _P], _I),
    "qw_q4_tiled_offset": ([_I64, _I64, _P, _P, _P], None),
}


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with v620-inference-engine_amd/build.py")
        # torch first: its HIP runtime (same soname as the one the library
        # links) is then the only one in the process, so streams and device
        # pointers from torch are the library's own
        import torch  # noqa: F401
        L = ctypes.CDLL(LIB_PATH)
        for name, (args, res) in _SIGS.items():
            f = getattr(L, name)
            f.argtypes = args
            f.restype = res
        _lib = L
    return _lib


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream():
    """The raw handle of torch's current stream. (torch.cuda.current_stream() builds a Stream object
    around it: 2.7 us of a decode GEMV call's 13.9, this 0.2. It serves where torch has no raw one.)"""
    import torch
    device = torch.cuda.current_device()  # (initialises the device, as the calls below expect)
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream


def _check(rc, fn):
    if rc != 0:
        raise RuntimeError(f"{fn} failed ({rc}): {lib().qw_q4_last_error().decode()}")


def _dev(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("qwq4: all tensors must be on the GPU")


# ------------------------------------------------------------ weight format
def tiled_size(N, K):
    a, b, c = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    lib().qw_q4_tiled_size(N, K, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c))
    return a.value, b.value, c.value


def tile(W, S, Z, N, K):
    """Checkpoint-order (W, S, Z) device tensors -> tiled (Wt, St, Zt or None)."""
    import torch
    wb, sb, zb = tiled_size(N, K)
    Wt = torch.empty(wb // 4, dtype=torch.int32, device=W.device)
    St = torch.empty(sb // 2, dtype=torch.int16, device=W.device)
    Zt = torch.empty(zb // 2, dtype=torch.int16, device=W.device) if Z is not None else None
    _dev(W, S, Z)
    _check(lib().qw_q4_tile(_ptr(W), _ptr(S), _ptr(Z), N, K, _ptr(Wt), _ptr(St), _ptr(Zt), _stream()), "qw_q4_tile")
    return Wt, St, Zt


def untile(Wt, St, Zt, N, K):
    import torch
    G = K // 128
    W = torch.empty((N, K // 8), dtype=torch.int32, device=Wt.device)
    S = torch.empty((N, G), dtype=torch.int16, device=Wt.device)
    Z = torch.empty((N, (G + 7) // 8), dtype=torch.int32, device=Wt.device) if Zt is not None else None
    _check(lib().qw_q4_untile(_ptr(Wt), _ptr(St), _ptr(Zt), N, K, _ptr(W), _ptr(S), _ptr(Z), _stream()),
           "qw_q4_untile")
    return W, S, Z


def tile_experts(W, S, Z, rows, K):
    """[E][rows][...] checkpoint-order expert stacks -> one tiled [E*rows][K] matrix."""
    E = W.shape[0]
    return tile(W.reshape(E * rows, -1), S.reshape(E * rows, -1), None if Z is None else Z.reshape(E * rows, -1),
                E * rows, K)


# ---------------------------------------------------------------- operators
# element-type codes of the *_type arguments (QW_T_F32, QW_T_BF16, QW_T_F16)
T_F32, T_BF16, T_F16 = 0, 1, 2


_codes = {}  # (filled by the first _tcode: this file loads without torch)


def _tcode(t):
    """QW_T_* code of a tensor's dtype (float32, bfloat16, float16)."""
    code = _codes.get(t.dtype)
    if code is None:
        import torch
        _codes.update({torch.float32: T_F32, torch.bfloat16: T_BF16, torch.float16: T_F16})
        code = _codes.get(t.dtype)
        if code is None:
            raise TypeError(f"unsupported element type {t.dtype}")
    return code


def _tdtype(code):
    import torch
    return {T_F32: torch.float32, T_BF16: torch.bfloat16, T_F16: torch.float16}[code]


def _is_f16(x, x_f16):
    """x_f16 given, else from the tensor: float16 -> fp16 rows, anything else
    (bfloat16, or int16 bit patterns) -> bf16 rows."""
    import torch
    return bool(x_f16) if x_f16 is not None else x.dtype == torch.float16


def _rows_out(M, N, y_bf16, accumulate, device):
    """A GEMV's output rows: cleared only where the call adds to them (it writes every element
    otherwise; the clearing launch took 3.8 us)."""
    import torch
    make = torch.zeros if accumulate else torch.empty
    return make((M, N), dtype=torch.bfloat16 if y_bf16 else torch.float32, device=device)


def gemv(W, S, Z, x, N, K, M=None, y=None, y_bf16=False, accumulate=False, xs=None, ys=None, x_f16=None, rpg=0):
    """y[m][n] (+)= sum_k deq(W)[n][k] x[m][off(n) + k], off(n) = (n // rpg) * K when rpg (row
    slices, gpu::gemv_rows). x: bf16 rows (bfloat16, or int16 bit patterns) or fp16 rows (float16,
    or x_f16=True with int16 bit patterns)."""
    import torch
    M = M if M is not None else x.shape[0]
    xs = xs if xs is not None else x.stride(0) if x.dim() == 2 else K
    if y is None:
        y = _rows_out(M, N, y_bf16, accumulate, x.device)
    ys = ys if ys is not None else (y.stride(0) if y.dim() == 2 else N)
    _dev(W, S, Z, x, y)
    rc = lib().qw_q4_gemv(_ptr(W), _ptr(S), _ptr(Z), _ptr(x), int(_is_f16(x, x_f16)), xs, _ptr(y), ys, int(y_bf16),
                          N, K, M, rpg, int(accumulate), _stream())
    _check(rc, "qw_q4_gemv")
    return y


def gemv_w16(W, x, M=None, y=None, y_bf16=False, accumulate=False, f16=None, xs=None, ys=None, rpg=0):
    """y[m][n] (+)= sum_k W[n][k] x[m][k] for 16-bit W [N][K] (row-major, stride W.stride(0)):
    fp16 W with fp16 x (f16 True, the default for float16 tensors) or bf16 with bf16."""
    import torch
    N, K = W.shape
    M = M if M is not None else x.shape[0]
    f16 = _is_f16(x, f16)
    xs = xs if xs is not None else x.stride(0) if x.dim() == 2 else K
    if y is None:
        y = _rows_out(M, N, y_bf16, accumulate, x.device)
    ys = ys if ys is not None else (y.stride(0) if y.dim() == 2 else N)
    _dev(W, x, y)
    rc = lib().qw_w16_gemv(_ptr(W), W.stride(0), _ptr(x), xs, int(f16), _ptr(y), ys, int(y_bf16), N, K, M, rpg,
                           int(accumulate), _stream())
    _check(rc, "qw_w16_gemv")
    return y


def w16_tile(W):
    """16-bit W [N][K] (row-major, stride W.stride(0)) -> the tiled layout qw_w16_gemv_tiled
    reads (a flat tensor of W's dtype, rows padded to a multiple of 16)."""
    import torch
    N, K = W.shape
    Wt = torch.empty(lib().qw_w16_tiled_size(N, K) // 2, dtype=W.dtype, device=W.device)
    _dev(W)
    _check(lib().qw_w16_tile(_ptr(W), W.stride(0), N, K, _ptr(Wt), _stream()), "qw_w16_tile")
    return Wt


def gemv_w16_tiled(Wt, N, K, x, M=None, y=None, y_bf16=False, accumulate=False, f16=None, xs=None, ys=None, rpg=0):
    """gemv_w16 on the tiled layout (w16_tile) of a 16-bit [N][K] matrix."""
    import torch
    M = M if M is not None else x.shape[0]
    f16 = _is_f16(x, f16)
    xs = xs if xs is not None else x.stride(0) if x.dim() == 2 else K
    if y is None:
        y = _rows_out(M, N, y_bf16, accumulate, x.device)
    ys = ys if ys is not None else (y.stride(0) if y.dim() == 2 else N)
    _dev(Wt, x, y)
    rc = lib().qw_w16_gemv_tiled(_ptr(Wt), _ptr(x), xs, int(f16), _ptr(y), ys, int(y_bf16), N, K, M, rpg,
                                 int(accumulate), _stream())
    _check(rc, "qw_w16_gemv_tiled")
    return y


def swiglu_gemv_w16_tiled(Wt, N, v, n, M=None, y=None, y_bf16=False, accumulate=False, ldv=None, ys=None):
    """y = W h with h = fp16(silu(v[:, :n]) v[:, n:2n] sigmoid(v[:, 2n])) (swiglu_gate followed by
    gemv_w16_tiled, in one launch); Wt: fp16 [N][n] tiled by w16_tile, v fp32 [M][>= 2n + 1]."""
    import torch
    M = M if M is not None else v.shape[0]
    ldv = ldv if ldv is not None else v.stride(0) if v.dim() == 2 else 2 * n + 1
    if y is None:
        y = _rows_out(M, N, y_bf16, accumulate, v.device)
    ys = ys if ys is not None else (y.stride(0) if y.dim() == 2 else N)
    _dev(Wt, v, y)
    rc = lib().qw_w16_swiglu_gemv_tiled(_ptr(Wt), _ptr(v), ldv, n, _ptr(y), ys, int(y_bf16), N, M, int(accumulate),
                                        _stream())
    _check(rc, "qw_w16_swiglu_gemv_tiled")
    return y


def i8_tile(W8, scale, group=32):
    """int8 W8 [N][K] and fp32 scale [N][K/group] (row-major, as quantize_rows_i8 writes
    them) -> the kernel format (Wt uint8 bytes, St fp32) qw_i8_gemv reads."""
    import torch
    N, K = W8.shape
    wb, sb = ctypes.c_size_t(), ctypes.c_size_t()
    lib().qw_i8_tiled_size(N, K, group, ctypes.byref(wb), ctypes.byref(sb))
    Wt = torch.empty(wb.value, dtype=torch.uint8, device=W8.device)
    St = torch.empty(sb.value // 4, dtype=torch.float32, device=W8.device)
    _dev(W8, scale)
    _check(lib().qw_i8_tile(_ptr(W8), _ptr(scale), N, K, group, _ptr(Wt), _ptr(St), _stream()), "qw_i8_tile")
    return Wt, St


def gemv_i8(Wt, St, N, K, x, M=None, group=32, rpg=0, y=None, y_bf16=False, accumulate=False, xs=None, ys=None):
    """y[m][n] (+)= sum_g scale[n][g] sum_{k in g} W8[n][k] x[m][off(n) + k] (gpu::gemv_rows_i8) on
    the kernel format (i8_tile) of an int8 [N][K] matrix; fp16 rows x (row n reads slice
    n // rpg when rpg)."""
    import torch
    M = M if M is not None else x.shape[0]
    xs = xs if xs is not None else x.stride(0) if x.dim() == 2 else K
    if y is None:
        y = _rows_out(M, N, y_bf16, accumulate, x.device)
    ys = ys if ys is not None else (y.stride(0) if y.dim() == 2 else N)
    _dev(Wt, St, x, y)
    rc = lib().qw_i8_gemv(_ptr(Wt), _ptr(St), group, _ptr(x), xs, _ptr(y), ys, int(y_bf16), N, K, M, rpg,
                          int(accumulate), _stream())
    _check(rc, "qw_i8_gemv")
    return y


def swiglu_gate(v, n, h=None):
    """h[t][j] = fp16(silu(v[t][j]) * v[t][n + j] * sigmoid(v[t][2n])); v fp32 [T][>= 2n + 1]."""
    import torch
    T = v.shape[0]
    if h is None:
        h = torch.empty((T, n), dtype=torch.float16, device=v.device)
    _dev(v, h)
    _check(lib().qw_swiglu_gate(_ptr(v), v.stride(0), n, T, _ptr(h), _stream()), "qw_swiglu_gate")
    return h


def gemm_workspace_size(T, K):
    return lib().qw_q4_gemm_workspace_size(T, K)


def gemm(W, S, Z, X, N, K, Y=None, y_bf16=False, workspace=None, x_f16=None, y_dtype=None):
    """Y[t][n] = sum_k X[t][k] deq(W)[n][k]; Y fp32, bf16 (y_bf16) or any of float32 / bfloat16 /
    float16 (y_dtype, or the dtype of a given Y; float16 is the reference's f16_out)."""
    import torch
    T = X.shape[0]
    f16 = _is_f16(X, x_f16)
    if Y is None:
        dt = y_dtype if y_dtype is not None else torch.bfloat16 if y_bf16 else torch.float32
        Y = torch.empty((T, N), dtype=dt, device=X.device)
    if workspace is None and not f16:
        workspace = torch.empty(gemm_workspace_size(T, K), dtype=torch.uint8, device=X.device)
    _dev(W, S, Z, X, Y, workspace)
    rc = lib().qw_q4_gemm(_ptr(W), _ptr(S), _ptr(Z), _ptr(X), int(f16), X.stride(0), T, _ptr(Y), Y.stride(0),
                          _tcode(Y), N, K, _ptr(workspace), 0 if workspace is None else workspace.numel(), _stream())
    _check(rc, "qw_q4_gemm")
    return Y


class Route:
    """Device outputs of qw_moe_route."""

    def __init__(self, T, E, topk, device, tile_m=0):
        import torch
        i32 = dict(dtype=torch.int32, device=device)
        self.T, self.E, self.topk, self.tile_m = T, E, topk, tile_m
        self.top_e = torch.empty((T, topk), **i32)
        self.top_w = torch.empty((T, topk), dtype=torch.float32, device=device)
        self.counts = torch.empty(E, **i32)
        self.offsets = torch.empty(E + 1, **i32)
        self.tok_slot = torch.empty((T, topk), **i32)
        self.pair_tok = torch.empty(T * topk, **i32)
        self.active = torch.empty(E, **i32)
        self.n_active = torch.empty(1, **i32)
        nt = (T * topk) // abs(tile_m) + E if tile_m else 0
        self.tile_e = torch.empty(max(nt, 1), **i32) if tile_m else None
        self.tile_m0 = torch.empty(max(nt, 1), **i32) if tile_m else None
        self.n_tiles = torch.empty(1, **i32) if tile_m else None


def moe_route(logits, topk, tile_m=0, out=None):
    T, E = logits.shape
    r = out if out is not None else Route(T, E, topk, logits.device, tile_m)
    kept = getattr(r, "_router", None)
    if kept is not None:  # (moe_sort's choices are shown in their place)
        if kept[1] is None:
            raise ValueError("moe_route: out was made by moe_sort and has no buffers for choices and weights")
        r.top_e, r.top_w = kept
        r._router = None
    _dev(logits)
    rc = lib().qw_moe_route(_ptr(logits), T, E, topk, tile_m, _ptr(r.top_e), _ptr(r.top_w), _ptr(r.counts),
                            _ptr(r.offsets), _ptr(r.tok_slot), _ptr(r.pair_tok), _ptr(r.active), _ptr(r.n_active),
                            _ptr(r.tile_e), _ptr(r.tile_m0), _ptr(r.n_tiles), _stream())
    _check(rc, "qw_moe_route")
    return r


def moe_experts_gemv(gate, up, down, route, x, E, F, h=None, yp=None, x_f16=None, yp_f16=False):
    """gate/up/down: tiled (Wt, St, Zt) of the stacked experts; returns (h fp16, yp fp32, or fp16
    with yp_f16 or an fp16 yp tensor)."""
    import torch
    H = x.shape[1]
    T, topk = route.T, route.topk
    if h is None:
        h = torch.empty((T * topk, F), dtype=torch.float16, device=x.device)
    if yp is None:
        yp = torch.empty((T * topk, H), dtype=torch.float16 if yp_f16 else torch.float32, device=x.device)
    _dev(x, h, yp, *gate, *up, *down)
    rc = lib().qw_moe_experts_gemv(*[_ptr(t) for t in (*gate, *up, *down)], E, H, F, _ptr(route.offsets),
                                   _ptr(route.active), _ptr(route.n_active), _ptr(route.pair_tok), _ptr(x),
                                   int(_is_f16(x, x_f16)), T, topk, _ptr(h), _ptr(yp),
                                   int(yp.dtype == torch.float16), _stream())
    _check(rc, "qw_moe_experts_gemv")
    return h, yp


def moe_grouped_tile_m():
    return lib().qw_moe_grouped_tile_m()


def moe_grouped_workspace_size(T, topk, E, H, F):
    return lib().qw_moe_grouped_workspace_size(T, topk, E, H, F)


def moe_experts_grouped(gate, up, down, route, x, E, F, h=None, yp=None, workspace=None, x_f16=None, yp_f16=False):
    """Grouped expert GEMMs; yp fp32, or fp16 (yp_f16, or an fp16 yp tensor)."""
    import torch
    T, H = x.shape
    topk = route.topk
    if h is None:
        h = torch.empty((T * topk, F), dtype=torch.float16, device=x.device)
    if yp is None:
        yp = torch.empty((T * topk, H), dtype=torch.float16 if yp_f16 else torch.float32, device=x.device)
    f16 = _is_f16(x, x_f16)
    if workspace is None and not f16:
        workspace = torch.empty(max(moe_grouped_workspace_size(T, topk, E, H, F), 1), dtype=torch.uint8,
                                device=x.device)
    _dev(x, h, yp, workspace, *gate, *up, *down)
    rc = lib().qw_moe_experts_grouped(*[_ptr(t) for t in (*gate, *up, *down)], E, H, F, _ptr(route.offsets),
                                      _ptr(route.pair_tok), _ptr(route.tile_e), _ptr(route.tile_m0),
                                      _ptr(route.n_tiles), _ptr(x), int(f16), T, topk, _ptr(h), _ptr(yp),
                                      int(yp.dtype == torch.float16), _ptr(workspace),
                                      0 if workspace is None else workspace.numel(), _stream())
    _check(rc, "qw_moe_experts_grouped")
    return h, yp


def moe_w4a8_tile_m():
    return lib().qw_moe_w4a8_tile_m()


def quant_rows_i8(x, x_f16=None):
    """16-bit rows [R][K] -> (int8 [R][K], fp32 scales [R][K/128]) (the W4A8 quantiser)."""
    import torch
    R, K = x.shape
    q = torch.empty((R, K), dtype=torch.int8, device=x.device)
    sc = torch.empty((R, K // 128), dtype=torch.float32, device=x.device)
    _dev(x)
    _check(lib().qw_quant_rows_i8(_ptr(x), int(_is_f16(x, x_f16)), R, K, x.stride(0), _ptr(q), _ptr(sc), _stream()),
           "qw_quant_rows_i8")
    return q, sc


def moe_experts_w4a8(gate, up, down, route, x, E, F, h=None, yp=None, workspace=None, x_f16=None):
    """The W4A8 grouped expert GEMMs (route made with tile_m = moe_w4a8_tile_m());
    returns (h fp16 [T*k][F], yp fp16 [T*k][H])."""
    import torch
    T, H = x.shape
    topk = route.topk
    if h is None:
        h = torch.empty((T * topk, F), dtype=torch.float16, device=x.device)
    if yp is None:
        yp = torch.empty((T * topk, H), dtype=torch.float16, device=x.device)
    if workspace is None:
        workspace = torch.empty(lib().qw_moe_w4a8_workspace_size(T, topk, H, F), dtype=torch.uint8, device=x.device)
    _dev(x, h, yp, workspace, *gate, *up, *down)
    rc = lib().qw_moe_experts_w4a8(*[_ptr(t) for t in (*gate, *up, *down)], E, H, F, _ptr(route.offsets),
                                   _ptr(route.pair_tok), _ptr(route.tile_e), _ptr(route.tile_m0), _ptr(route.n_tiles),
                                   _ptr(x), int(_is_f16(x, x_f16)), T, topk, _ptr(h), _ptr(yp), _ptr(workspace),
                                   workspace.numel(), _stream())
    _check(rc, "qw_moe_experts_w4a8")
    return h, yp


def moe_combine(yp, route, H, shared=None, out=None, out_bf16=True, out_dtype=None, tok_w=None):
    """out = shared + sum_i w_i yp[slot_i], w the route's top_w or tok_w (float32 [T][k]; a route of moe_sort has no
    weights of its own, and choices without a slot add nothing); yp and shared fp32 or float16 (by dtype), out bf16
    (out_bf16), fp32, or the dtype given (out_dtype, or that of a given out). Other rows (the bfloat16 yp of
    moe_experts_w8a8) are refused: moe_unpermute takes those."""
    import torch
    T, topk = route.T, route.topk
    for name, t in (("yp", yp), ("shared", shared)):
        if t is not None and t.dtype != torch.float32 and t.dtype != torch.float16:
            raise TypeError(f"moe_combine: {name} is {t.dtype}, not torch.float32 or torch.float16 (moe_unpermute "
                            "takes bfloat16 rows)")
    if tok_w is not None:
        _whole("moe_combine", "tok_w", tok_w, (T, topk), torch.float32)
    elif route.top_w is None:
        raise ValueError("moe_combine: the route has no weights (moe_sort made it): give tok_w")
    else:
        tok_w = route.top_w
    if out is None:
        dt = out_dtype if out_dtype is not None else torch.bfloat16 if out_bf16 else torch.float32
        out = torch.empty((T, H), dtype=dt, device=yp.device)
    _dev(yp, shared, out, tok_w)
    rc = lib().qw_moe_combine(_ptr(yp), int(yp.dtype == torch.float16), _ptr(route.tok_slot), _ptr(tok_w),
                              _ptr(shared), int(shared is not None and shared.dtype == torch.float16), T, topk, H,
                              _ptr(out), _tcode(out), _stream())
    _check(rc, "qw_moe_combine")
    return out


# ------------------------------------------------------------------- W8A8
def _here(fn, *ts):
    """The raw handle of the current GPU's current stream (as _stream gives it); every tensor has to be on that GPU."""
    import torch
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{fn}: all tensors must be on the GPU")
        if dev is None:
            dev = torch.cuda.current_device()
        if t.get_device() != dev:
            raise RuntimeError(f"{fn}: a tensor is on GPU {t.get_device()}, the current one is {dev}")
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(dev) if raw is not None else torch.cuda.current_stream(dev).cuda_stream


_INT_MAX = 2**31 - 1


def _matrix(fn, name, t, rows, cols, dtype=None):
    """The row stride of a [rows][cols] tensor whose rows are contiguous (None: any number). Sizes and strides are
    passed on as 32-bit numbers."""
    shape = t.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (cols is not None and shape[1] != cols):
        raise ValueError(f"{fn}: {name} is {tuple(shape)}, not ({rows}, {cols})")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{fn}: {name} is {t.dtype}, not {dtype}")
    stride = t.stride()
    if stride[1] != 1 and shape[1] > 1:
        raise ValueError(f"{fn}: the rows of {name} must be contiguous")
    if shape[0] > 1:
        if shape[0] > _INT_MAX or stride[0] > _INT_MAX:
            raise ValueError(f"{fn}: {name} has {shape[0]} rows of stride {stride[0]}, more than 2^31 - 1")
        return stride[0]
    if shape[1] > _INT_MAX:
        raise ValueError(f"{fn}: {name} has rows of {shape[1]}, more than 2^31 - 1")
    return shape[1]


def _space(fn, workspace):
    """The bytes of a workspace (None: none)."""
    if workspace is None:
        return 0
    if not workspace.is_contiguous():
        raise ValueError(f"{fn}: workspace must be contiguous")
    return workspace.numel() * workspace.element_size()


def _whole(fn, name, t, shape, dtype):
    """A contiguous tensor of this shape and type."""
    if t.shape != shape:
        raise ValueError(f"{fn}: {name} is {tuple(t.shape)}, not {shape}")
    if t.dtype != dtype:
        raise TypeError(f"{fn}: {name} is {t.dtype}, not {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{fn}: {name} must be contiguous")


def quant_tokens_i8(x, q=None, scale=None):
    """Rows x [T][K] (float32, bfloat16 or float16) -> (q int8 [T][K], scale fp32 [T]), a scale per row:
    q = rint(x (1 / scale)), scale = max |x| / 127."""
    import torch
    fn = "quant_tokens_i8"
    ldx = _matrix(fn, "x", x, None, None)
    T, K = x.shape
    if q is None:
        q = torch.empty((T, K), dtype=torch.int8, device=x.device)
    if scale is None:
        scale = torch.empty(T, dtype=torch.float32, device=x.device)
    ldq = _matrix(fn, "q", q, T, K, torch.int8)
    _whole(fn, "scale", scale, (T,), torch.float32)
    code = _tcode(x)
    stream = _here(fn, x, q, scale)
    _check(lib().qw_quant_tokens_i8(_ptr(x), code, ldx, T, K, _ptr(q), ldq, _ptr(scale), stream),
           "qw_quant_tokens_i8")
    return q, scale


def _w8_out(fn, Y, y_dtype, T, N, default, device):
    """The output rows, their stride and their QW_T_* code."""
    import torch
    if Y is None:
        Y = torch.empty((T, N), dtype=y_dtype if y_dtype is not None else default, device=device)
    elif y_dtype is not None and Y.dtype != y_dtype:
        raise TypeError(f"{fn}: the output is {Y.dtype}, not {y_dtype}")
    return Y, _matrix(fn, "the output", Y, T, N), _tcode(Y)


def gemm_w8a8(W, sw, q, sx, Y=None, y_dtype=None):
    """Y[t][n] = (sum_k q[t][k] W[n][k]) sw[n] sx[t], the sum in whole numbers. W int8 [N][K] and sw fp32 [N] as the
    checkpoint holds them, (q, sx) from quant_tokens_i8; any T. Y bfloat16, or y_dtype / the dtype of a given Y."""
    import torch
    fn = "gemm_w8a8"
    ldq, ldw = _matrix(fn, "q", q, None, None, torch.int8), _matrix(fn, "W", W, None, q.shape[-1], torch.int8)
    (T, K), N = q.shape, W.shape[0]
    _whole(fn, "sw", sw, (N,), torch.float32)
    _whole(fn, "sx", sx, (T,), torch.float32)
    Y, ldy, code = _w8_out(fn, Y, y_dtype, T, N, torch.bfloat16, q.device)
    stream = _here(fn, W, sw, q, sx, Y)
    _check(lib().qw_w8a8_gemm(_ptr(W), ldw, _ptr(sw), _ptr(q), ldq, _ptr(sx), T, _ptr(Y), ldy, code, N, K, stream),
           "qw_w8a8_gemm")
    return Y


def w8a8_workspace_size(T, K):
    return lib().qw_w8a8_workspace_size(T, K)


def linear_w8a8(W, sw, x, Y=None, y_dtype=None, workspace=None):
    """gemm_w8a8(W, sw, *quant_tokens_i8(x)) in one call, bit for bit; x [T][K] float32, bfloat16 or float16. Y of
    x's type, or y_dtype / the dtype of a given Y."""
    import torch
    fn = "linear_w8a8"
    ldx, ldw = _matrix(fn, "x", x, None, None), _matrix(fn, "W", W, None, x.shape[-1], torch.int8)
    (T, K), N = x.shape, W.shape[0]
    _whole(fn, "sw", sw, (N,), torch.float32)
    code = _tcode(x)
    Y, ldy, ycode = _w8_out(fn, Y, y_dtype, T, N, x.dtype, x.device)
    if workspace is None:
        need = w8a8_workspace_size(T, K)
        if need:  # (one or two rows need none)
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    stream = _here(fn, W, sw, x, Y, workspace)
    _check(lib().qw_w8a8_linear(_ptr(W), ldw, _ptr(sw), _ptr(x), code, ldx, T, _ptr(Y), ldy, ycode, N, K,
                                _ptr(workspace), _space(fn, workspace), stream), "qw_w8a8_linear")
    return Y


def moe_w8a8_tile_m():
    return lib().qw_moe_w8a8_tile_m()


def moe_w8a8_workspace_size(T, topk, H, F):
    return lib().qw_moe_w8a8_workspace_size(T, topk, H, F)


def moe_experts_w8a8(gate, up, down, route, x, h=None, yp=None, yp_dtype=None, workspace=None):
    """The routed experts in W8A8 (route from moe_route or moe_sort with tile_m = moe_w8a8_tile_m()): gate and up
    (int8 [E][F][H], fp32 [E][F]), down (int8 [E][H][F], fp32 [E][H]), x [T][H] float32, bfloat16 or float16. Returns
    (h fp16 [T*k][F], yp [T*k][H]); yp float16, or yp_dtype / the dtype of a given yp. Rows that no choice has (behind
    route.offsets[E]) are left as they were, in a new h and yp not set: read yp through route.tok_slot."""
    import torch
    fn = "moe_experts_w8a8"
    T, topk, E = route.T, route.topk, route.E
    if gate[0].dim() != 3:
        raise ValueError(f"{fn}: gate is {tuple(gate[0].shape)}, not [E][F][H]")
    F, H = gate[0].shape[1:]
    for name, (w, s), n, k in (("gate", gate, F, H), ("up", up, F, H), ("down", down, H, F)):
        _whole(fn, name, w, (E, n, k), torch.int8)
        _whole(fn, name + " scales", s, (E, n), torch.float32)
    if route.tile_m != moe_w8a8_tile_m():
        raise ValueError(f"{fn}: route has the tile list of tile_m = {route.tile_m}, not moe_w8a8_tile_m()")
    code = _tcode(x)
    _whole(fn, "x", x, (T, H), x.dtype)
    if h is None:
        h = torch.empty((T * topk, F), dtype=torch.float16, device=x.device)
    if yp is None:
        yp = torch.empty((T * topk, H), dtype=yp_dtype if yp_dtype is not None else torch.float16, device=x.device)
    elif yp_dtype is not None and yp.dtype != yp_dtype:
        raise TypeError(f"{fn}: yp is {yp.dtype}, not {yp_dtype}")
    _whole(fn, "h", h, (T * topk, F), torch.float16)
    _whole(fn, "yp", yp, (T * topk, H), yp.dtype)
    ycode = _tcode(yp)
    if workspace is None:
        workspace = torch.empty(moe_w8a8_workspace_size(T, topk, H, F), dtype=torch.uint8, device=x.device)
    stream = _here(fn, x, h, yp, workspace, route.offsets, *gate, *up, *down)
    rc = lib().qw_moe_experts_w8a8(*[_ptr(t) for t in (*gate, *up, *down)], E, H, F, _ptr(route.offsets),
                                   _ptr(route.pair_tok), _ptr(route.tile_e), _ptr(route.tile_m0), _ptr(route.n_tiles),
                                   _ptr(x), code, T, topk, _ptr(h), _ptr(yp), ycode, _ptr(workspace),
                                   _space(fn, workspace), stream)
    _check(rc, "qw_moe_experts_w8a8")
    return h, yp


# ----------------------------------------- tokens sorted by expert and back
def moe_sort(top_e, E, tile_m=0, out=None):
    """The slots of given choices top_e int32 [T][k], as a Route (its top_e is the tensor given, top_w is None):
    experts ascending, within one the choices in order; a choice outside 0 .. E - 1 has slot -1, a place behind the
    last slot token -1. moe_combine and moe_unpermute take the choices' weights. A Route given as out has its own
    top_e and top_w back with the next moe_route into it."""
    import torch
    fn = "moe_sort"
    if top_e.dim() != 2:
        raise ValueError(f"{fn}: top_e is {tuple(top_e.shape)}, not [T][k]")
    T, k = top_e.shape
    if T * k >= 1 << 30 or not 1 <= E <= 1024 or abs(tile_m) >= 4096:
        raise ValueError(f"{fn}: T = {T}, k = {k}, E = {E}, tile_m = {tile_m} (need T * k below 2^30, E 1..1024, "
                         "|tile_m| below 4096)")
    _whole(fn, "top_e", top_e, (T, k), torch.int32)
    if out is None:
        r = Route.__new__(Route)
        r.T, r.E, r.topk, r.tile_m, r.top_w, r._router = T, E, k, tile_m, None, (None, None)
        P = T * k
        nt = P // abs(tile_m) + E if tile_m else 0
        # (one buffer for all of the lists: an allocation each would cost more than the sort)
        own = torch.empty(2 * P + 3 * E + 3 + 2 * nt, dtype=torch.int32, device=top_e.device)
        slot, r.pair_tok, r.counts, r.offsets, r.active, r.n_active, tile_e, tile_m0, n_tiles = own.split_with_sizes(
            (P, P, E, E + 1, E, 1, nt, nt, 1))
        r.tok_slot = slot.view(T, k)
        r.tile_e, r.tile_m0, r.n_tiles = (tile_e, tile_m0, n_tiles) if tile_m else (None, None, None)
    else:
        r = out
        if (r.T, r.E, r.topk, r.tile_m) != (T, E, k, tile_m):
            raise ValueError(f"{fn}: out was made for T, E, k, tile_m = {r.T, r.E, r.topk, r.tile_m}")
    stream = _here(fn, top_e, r.pair_tok)
    if getattr(r, "_router", None) is None:
        r._router = r.top_e, r.top_w  # (the router's own buffers, for the next moe_route)
    r.top_e, r.top_w = top_e, None
    rc = lib().qw_moe_sort(_ptr(top_e), T, E, k, tile_m, _ptr(r.counts), _ptr(r.offsets), _ptr(r.tok_slot),
                           _ptr(r.pair_tok), _ptr(r.active), _ptr(r.n_active), _ptr(r.tile_e), _ptr(r.tile_m0),
                           _ptr(r.n_tiles), stream)
    _check(rc, "qw_moe_sort")
    return r


def _slots(fn, tok_slot):
    import torch
    if tok_slot.dim() != 2:
        raise ValueError(f"{fn}: tok_slot is {tuple(tok_slot.shape)}, not [T][k]")
    _whole(fn, "tok_slot", tok_slot, tok_slot.shape, torch.int32)
    if tok_slot.numel() >= 1 << 30:
        raise ValueError(f"{fn}: tok_slot is {tuple(tok_slot.shape)}, need fewer than 2^30 choices")
    return tok_slot.shape


def _no_autograd(fn, *ts):
    """Nothing here is recorded for autograd: an input whose gradient torch follows is refused, not cut off silently."""
    import torch
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{fn}: an input requires grad, which this call does not record (use torch.no_grad(), "
                                   f"or a torch.autograd.Function with {fn}_backward)")


def moe_permute(x, tok_slot, xs=None):
    """The rows in slot order: xs[tok_slot[t][i]] = x[t] (x [T][H] of 1, 2 or 4 bytes an element). Rows of xs
    [T*k][H] that no choice has are left as they were; a new xs has zeros there, which a caller who does not need
    them saves by giving one. Its gradient is moe_permute_backward; autograd does not record the call."""
    import torch
    fn = "moe_permute"
    _no_autograd(fn, x)
    T, k = _slots(fn, tok_slot)
    ldx = _matrix(fn, "x", x, T, None)
    H = x.shape[1]
    if xs is None:
        xs = torch.zeros((T * k, H), dtype=x.dtype, device=x.device)
    ldxs = _matrix(fn, "xs", xs, T * k, H, x.dtype)
    stream = _here(fn, x, tok_slot, xs)
    _check(lib().qw_moe_permute(_ptr(x), ldx, x.element_size(), T, k, H, _ptr(tok_slot), _ptr(xs), ldxs, stream),
           "qw_moe_permute")
    return xs


def moe_unpermute(yp, tok_slot, tok_w=None, out=None, out_dtype=None):
    """out[t] = sum_i tok_w[t][i] yp[tok_slot[t][i]] over the choices with a slot, in order, in fp32 (tok_w None: all
    1); yp [T*k][H]. out of yp's type, or out_dtype / the dtype of a given out. moe_combine is the form with a shared
    expert's rows. Its gradients are moe_unpermute_backward; autograd does not record the call."""
    import torch
    fn = "moe_unpermute"
    _no_autograd(fn, yp, tok_w)
    T, k = _slots(fn, tok_slot)
    ldyp = _matrix(fn, "yp", yp, T * k, None)
    H = yp.shape[1]
    if tok_w is not None:
        _whole(fn, "tok_w", tok_w, (T, k), torch.float32)
    code = _tcode(yp)
    out, ldo, ocode = _w8_out(fn, out, out_dtype, T, H, yp.dtype, yp.device)
    stream = _here(fn, yp, tok_slot, tok_w, out)
    _check(lib().qw_moe_unpermute(_ptr(yp), code, ldyp, _ptr(tok_slot), _ptr(tok_w), T, k, H, _ptr(out), ocode, ldo,
                                  stream), "qw_moe_unpermute")
    return out


def moe_permute_backward(dxs, tok_slot, dx=None, dx_dtype=None):
    """The gradient of moe_permute: dx[t] = sum_i dxs[tok_slot[t][i]], summed and typed as moe_unpermute does, but
    float16 dx beyond +-65504 becomes infinite."""
    fn = "moe_permute_backward"
    T, k = _slots(fn, tok_slot)
    lddxs = _matrix(fn, "dxs", dxs, T * k, None)
    H = dxs.shape[1]
    code = _tcode(dxs)
    dx, lddx, xcode = _w8_out(fn, dx, dx_dtype, T, H, dxs.dtype, dxs.device)
    stream = _here(fn, dxs, tok_slot, dx)
    _check(lib().qw_moe_permute_backward(_ptr(dxs), code, lddxs, _ptr(tok_slot), T, k, H, _ptr(dx), xcode, lddx,
                                         stream), "qw_moe_permute_backward")
    return dx


def moe_unpermute_backward(dout, yp, tok_slot, tok_w=None, dyp=None, dw=None, need_dyp=True, need_dw=True):
    """The gradients of moe_unpermute from dout [T][H]: (dyp [T*k][H] of yp's type, dw fp32 [T][k]), either None
    where it is not needed. float16 dyp beyond +-65504 becomes infinite. Rows of dyp that no choice has are left as
    they were; a new dyp has zeros there."""
    import torch
    fn = "moe_unpermute_backward"
    T, k = _slots(fn, tok_slot)
    ldyp = _matrix(fn, "yp", yp, T * k, None)
    H = yp.shape[1]
    ldd = _matrix(fn, "dout", dout, T, H)
    dcode, code = _tcode(dout), _tcode(yp)
    if tok_w is not None:
        _whole(fn, "tok_w", tok_w, (T, k), torch.float32)
    if not need_dyp:
        dyp = None
    elif dyp is None:
        dyp = torch.zeros((T * k, H), dtype=yp.dtype, device=yp.device)
    if not need_dw:
        dw = None
    elif dw is None:
        dw = torch.empty((T, k), dtype=torch.float32, device=yp.device)
    lddyp = _matrix(fn, "dyp", dyp, T * k, H, yp.dtype) if dyp is not None else H
    if dw is not None:
        _whole(fn, "dw", dw, (T, k), torch.float32)
    stream = _here(fn, dout, yp, tok_slot, tok_w, dyp, dw)
    _check(lib().qw_moe_unpermute_backward(_ptr(dout), dcode, ldd, _ptr(yp), code, ldyp, _ptr(tok_slot), _ptr(tok_w), T,
                                           k, H, _ptr(dyp), lddyp, _ptr(dw), stream), "qw_moe_unpermute_backward")
    return dyp, dw


# ------------------------------------------------------ around a projection
def _norm_rows(fn, x, w, residual, residual_out):
    """(T, H, arguments of the C call up to eps, residual_out)"""
    _no_autograd(fn, x, w, residual)
    ldx = _matrix(fn, "x", x, None, None)
    T, H = x.shape
    if w.shape != (H,) or not w.is_contiguous():
        raise ValueError(f"{fn}: w is {tuple(w.shape)}, not ({H},), or not contiguous")
    if residual is None:
        if residual_out is not None:
            raise ValueError(f"{fn}: residual_out without a residual")
        return T, H, (_ptr(x), _tcode(x), ldx, None, 0, 0, None, 0, _ptr(w), _tcode(w)), None
    ldr = _matrix(fn, "residual", residual, T, H)
    if residual_out is None:
        residual_out = residual.new_empty((T, H))
    ldro = _matrix(fn, "residual_out", residual_out, T, H, residual.dtype)
    return T, H, (_ptr(x), _tcode(x), ldx, _ptr(residual), _tcode(residual), ldr, _ptr(residual_out), ldro, _ptr(w),
                  _tcode(w)), residual_out


def rms_norm(x, w, eps=1e-6, residual=None, y=None, y_dtype=None, residual_out=None):
    """y = h w / sqrt(mean(h^2) + eps) of rows x [T][H], w [H] (of x's type or float32), in fp32; y of x's type, or y_dtype / the dtype of a
    given y. With a residual (of x's type or float32) h = x + residual, and the result is (y, residual_out): h
    rounded to the residual's type, in a new tensor or the one given, which may be the residual. Its gradients are
    rms_norm_backward; autograd does not record the call."""
    fn = "rms_norm"
    T, H, args, residual_out = _norm_rows(fn, x, w, residual, residual_out)
    y, ldy, ycode = _w8_out(fn, y, y_dtype, T, H, x.dtype, x.device)
    stream = _here(fn, x, w, residual, residual_out, y)
    _check(lib().qw_rms_norm(*args, eps, T, H, _ptr(y), ycode, ldy, stream), "qw_rms_norm")
    return y if residual is None else (y, residual_out)


def rms_norm_i8(x, w, eps=1e-6, residual=None, q=None, scale=None, residual_out=None):
    """rms_norm with its rows in 8 bits, as gemm_w8a8 takes them: (q int8 [T][H], scale fp32 [T]), and residual_out
    behind them where there is a residual. The values of q are quant_tokens_i8's of the rows h w in fp32."""
    import torch
    fn = "rms_norm_i8"
    T, H, args, residual_out = _norm_rows(fn, x, w, residual, residual_out)
    if q is None:
        q = x.new_empty((T, H), dtype=torch.int8)
    if scale is None:
        scale = x.new_empty(T, dtype=torch.float32)
    ldq = _matrix(fn, "q", q, T, H, torch.int8)
    _whole(fn, "scale", scale, (T,), torch.float32)
    stream = _here(fn, x, w, residual, residual_out, q, scale)
    _check(lib().qw_rms_norm_i8(*args, eps, T, H, _ptr(q), ldq, _ptr(scale), stream), "qw_rms_norm_i8")
    return (q, scale) if residual is None else (q, scale, residual_out)


def rms_norm_backward_workspace_size(T, H):
    return lib().qw_rms_norm_backward_workspace_size(T, H)


def rms_norm_backward(dy, h, w, eps=1e-6, dres=None, dx=None, dw=None, need_dw=True, workspace=None):
    """The gradients of rms_norm from dy [T][H]: (dx of h's type, dw fp32 [H] or None where it is not needed). h
    [T][H], of dy's type or float32 as w is, is what was normalised (residual_out where there was a residual); dres, of h's
    type, is the gradient of residual_out and is added to dx, which is then that of x and of the residual alike.
    dx may be dy, h or dres. float16 dx beyond +-65504 becomes infinite."""
    import torch
    fn = "rms_norm_backward"
    lddy = _matrix(fn, "dy", dy, None, None)
    T, H = dy.shape
    ldh = _matrix(fn, "h", h, T, H)
    if w.shape != (H,) or not w.is_contiguous():
        raise ValueError(f"{fn}: w is {tuple(w.shape)}, not ({H},), or not contiguous")
    lddr = _matrix(fn, "dres", dres, T, H, h.dtype) if dres is not None else 0
    if dx is None:
        dx = h.new_empty((T, H))
    lddx = _matrix(fn, "dx", dx, T, H, h.dtype)
    if not need_dw:
        dw = None
    else:
        if dw is None:
            dw = h.new_empty(H, dtype=torch.float32)
        _whole(fn, "dw", dw, (H,), torch.float32)
        if workspace is None:
            workspace = h.new_empty(rms_norm_backward_workspace_size(T, H), dtype=torch.uint8)
    stream = _here(fn, dy, h, w, dres, dx, dw, workspace)
    _check(lib().qw_rms_norm_backward(_ptr(dy), _tcode(dy), lddy, _ptr(h), _tcode(h), ldh, _ptr(w), _tcode(w), eps,
                                      _ptr(dres), lddr, T, H, _ptr(dx), lddx, _ptr(dw), _ptr(workspace),
                                      _space(fn, workspace), stream), "qw_rms_norm_backward")
    return dx, dw


def _adapters(fn, x, A, B, ids, scaling):
    """(T, K, N, R, L, whether fp16) of an adapter call"""
    import torch
    if A.dim() != 3 or B.dim() != 3:
        raise ValueError(f"{fn}: A is {tuple(A.shape)}, B {tuple(B.shape)}, not [L][R][K] and [L][N][R]")
    (L, R, K), N, T = A.shape, B.shape[1], x.shape[0]
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{fn}: rows are {x.dtype}, not bfloat16 or float16")
    _whole(fn, "A", A, (L, R, K), x.dtype)
    _whole(fn, "B", B, (L, N, R), x.dtype)
    _whole(fn, "ids", ids, (T,), torch.int32)
    if scaling is not None:
        _whole(fn, "scaling", scaling, (L,), torch.float32)
    if max(T, L, R, K, N) > _INT_MAX:
        raise ValueError(f"{fn}: T, K, N, R, L = {T, K, N, R, L}, more than 2^31 - 1")
    return T, K, N, R, L, int(x.dtype == torch.float16)


def lora(x, A, B, ids, y, scaling=None, out=None, v=None):
    """Low-rank adapters beside a projection whose rows y [T][N] are given: out_t = y_t + scaling[i] B[i] (A[i] x_t),
    i = ids[t] (int32 [T]; outside 0 .. L - 1: no adapter, out_t = y_t). x [T][K], A [L][R][K], B [L][N][R] all
    bfloat16 or all float16; y of any type; scaling fp32 [L] (None: all 1). out is y unless another is given. v fp32
    [T][R] takes A[i] x_t, which lora_backward needs; rows without an adapter are left as they were. Its gradients are
    lora_backward; autograd does not record the call."""
    import torch
    fn = "lora"
    _no_autograd(fn, x, A, B, y, scaling)
    ldx = _matrix(fn, "x", x, None, None)
    T, K, N, R, L, f16 = _adapters(fn, x, A, B, ids, scaling)
    if x.shape[1] != K:
        raise ValueError(f"{fn}: x is {tuple(x.shape)}, not ({T}, {K})")
    ldy = _matrix(fn, "y", y, T, N)
    code = _tcode(y)
    if out is None:
        out = y
    ldo = _matrix(fn, "out", out, T, N, y.dtype)
    if v is None:
        v = x.new_empty((T, R), dtype=torch.float32)
    else:
        _whole(fn, "v", v, (T, R), torch.float32)
    stream = _here(fn, x, A, B, ids, y, scaling, out, v)
    _check(lib().qw_lora(_ptr(x), ldx, f16, _ptr(A), _ptr(B), _ptr(ids), _ptr(scaling), T, K, N, R, L, _ptr(v), _ptr(y),
                         ldy, _ptr(out), ldo, code, stream), "qw_lora")
    return out


def lora_backward_workspace_size(T, K, N, R, L):
    return lib().qw_lora_backward_workspace_size(T, K, N, R, L)


def lora_backward(dy, x, A, B, ids, v, scaling=None, dx=None, dx_out=None, dA=None, dB=None, need_weights=True,
                  workspace=None):
    """The gradients of lora from dy [T][N] (of x's type) and v as lora left it: (dx_out, dA fp32 [L][R][K], dB fp32
    [L][N][R]). dx [T][K], of x's type, is the gradient through the shared projection; the adapters' is added to it, in
    place unless another dx_out is given; None: not wanted. dA and dB are written whole, zeros for an adapter without
    tokens, and None with need_weights = False. float16 dx_out beyond +-65504 becomes infinite."""
    import torch
    fn = "lora_backward"
    lddy, ldx = _matrix(fn, "dy", dy, None, None, x.dtype), _matrix(fn, "x", x, None, None)
    T, K, N, R, L, f16 = _adapters(fn, x, A, B, ids, scaling)
    if x.shape[1] != K or dy.shape != (T, N):
        raise ValueError(f"{fn}: x is {tuple(x.shape)}, dy {tuple(dy.shape)}, not ({T}, {K}) and ({T}, {N})")
    _whole(fn, "v", v, (T, R), torch.float32)
    lddx = lddxo = 0
    if dx is not None:
        dx_out = dx if dx_out is None else dx_out
        lddx, lddxo = _matrix(fn, "dx", dx, T, K, x.dtype), _matrix(fn, "dx_out", dx_out, T, K, x.dtype)
    elif dx_out is not None:
        raise ValueError(f"{fn}: dx_out without dx")
    if need_weights:
        dA = x.new_empty((L, R, K), dtype=torch.float32) if dA is None else dA
        dB = x.new_empty((L, N, R), dtype=torch.float32) if dB is None else dB
        _whole(fn, "dA", dA, (L, R, K), torch.float32)
        _whole(fn, "dB", dB, (L, N, R), torch.float32)
    else:
        dA = dB = None
    if workspace is None:
        workspace = x.new_empty(lora_backward_workspace_size(T, K, N, R, L), dtype=torch.uint8)
    stream = _here(fn, dy, x, A, B, ids, v, scaling, dx, dx_out, dA, dB, workspace)
    _check(lib().qw_lora_backward(_ptr(dy), lddy, _ptr(x), ldx, f16, _ptr(A), _ptr(B), _ptr(ids), _ptr(v), _ptr(scaling),
                                  T, K, N, R, L, _ptr(dx), lddx, _ptr(dx_out), lddxo, _ptr(dA), _ptr(dB),
                                  _ptr(workspace), _space(fn, workspace), stream), "qw_lora_backward")
    return dx_out, dA, dB


def logprobs_workspace_size(T, V, top):
    return lib().qw_logprobs_workspace_size(T, V, top)


def logprobs(logits, tokens, top=0, workspace=None):
    """Of logits [T][V] and tokens int32 [T]: (logp, entropy, lse, top_ids, top_logp). logp = logits[t][tokens[t]] -
    lse (0 for a token outside 0 .. V - 1), entropy and lse fp32 [T]; top_ids int32 and top_logp fp32 [T][top]: the
    most likely tokens, largest first, ties by the lowest index (None with top = 0). Logits of -inf are masked; a row
    of only such has lse, logp and top_logp of -inf and entropy 0. Its gradient is logprobs_backward; autograd does
    not record the call."""
    import torch
    fn = "logprobs"
    _no_autograd(fn, logits)
    ld = _matrix(fn, "logits", logits, None, None)
    T, V = logits.shape
    _whole(fn, "tokens", tokens, (T,), torch.int32)
    if not 0 <= top <= min(64, V):
        raise ValueError(f"{fn}: top = {top} (0..64, at most V = {V})")
    code = _tcode(logits)
    # (tensors of their own: torch refuses in-place work on several views of one buffer, and each would keep all of it)
    logp = logits.new_empty(T, dtype=torch.float32)
    entropy, lse = logp.new_empty(T), logp.new_empty(T)
    top_ids, top_logp = (tokens.new_empty((T, top)), logp.new_empty((T, top))) if top else (None, None)
    stream = _here(fn, logits, tokens, workspace)  # (the outputs are where logits is)
    if workspace is None:
        space = lib().qw_logprobs_workspace_size(T, V, top)
        workspace = logp.new_empty((space + 3) // 4) if space else None
    else:
        space = _space(fn, workspace)
    _check(lib().qw_logprobs(logits.data_ptr(), code, ld, tokens.data_ptr(), T, V, top, logp.data_ptr(),
                             entropy.data_ptr(), lse.data_ptr(), _ptr(top_ids), _ptr(top_logp), _ptr(workspace), space,
                             stream), "qw_logprobs")
    return logp, entropy, lse, top_ids, top_logp


def logprobs_backward(logits, tokens, lse, entropy, dlogp=None, dentropy=None, dlogits=None):
    """The gradient of logprobs' logp and entropy (dlogp, dentropy fp32 [T], either None: none) in the logits' type,
    from lse and entropy as logprobs gave them (p is put right where lse is too large for its rounding not to show).
    dlogits may be the logits. float16 beyond +-65504 becomes infinite."""
    import torch
    fn = "logprobs_backward"
    ld = _matrix(fn, "logits", logits, None, None)
    T, V = logits.shape
    _whole(fn, "tokens", tokens, (T,), torch.int32)
    for name, t in (("lse", lse), ("entropy", entropy), ("dlogp", dlogp), ("dentropy", dentropy)):
        if t is not None:
            _whole(fn, name, t, (T,), torch.float32)
    if dlogits is None:
        dlogits = logits.new_empty((T, V))
    ldd = _matrix(fn, "dlogits", dlogits, T, V, logits.dtype)
    stream = _here(fn, logits, tokens, lse, entropy, dlogp, dentropy, dlogits)
    _check(lib().qw_logprobs_backward(_ptr(logits), _tcode(logits), ld, _ptr(tokens), _ptr(lse), _ptr(entropy),
                                      _ptr(dlogp), _ptr(dentropy), T, V, _ptr(dlogits), ldd, stream),
           "qw_logprobs_backward")
    return dlogits


def unpack(W, N, K):
    import torch
    out = torch.empty((N, K), dtype=torch.uint8, device=W.device)
    _check(lib().qw_q4_unpack(_ptr(W), N, K, _ptr(out), _stream()), "qw_q4_unpack")
    return out


def dequant(W, S, Z, N, K):
    import torch
    out = torch.empty((N, K), dtype=torch.float32, device=W.device)
    _check(lib().qw_q4_dequant(_ptr(W), _ptr(S), _ptr(Z), N, K, _ptr(out), _stream()), "qw_q4_dequant")
    return out


def from_engine_order(words):
    import torch
    out = torch.empty_like(words)
    _check(lib().qw_q4_from_engine_order(_ptr(words), _ptr(out), words.numel(), _stream()), "qw_q4_from_engine_order")
    return out


class MoeDecode:
    """Buffers of the fused decode block (qw_moe_decode) for T tokens."""

    def __init__(self, T, E, topk, H, F, device, yp_f16=False, Fs=0):
        """Fs > 0: also the shared expert's rows (sh_v [T][2 Fs + 1], sh_out [T][H], fp32) and the
        workspace of qw_moe_decode_with_shared."""
        import torch
        i32 = dict(dtype=torch.int32, device=device)
        self.T, self.E, self.topk, self.H, self.F, self.Fs = T, E, topk, H, F, Fs
        self.logits = torch.empty((T, E), dtype=torch.float32, device=device)
        self.top_e = torch.empty((T, topk), **i32)
        self.top_w = torch.empty((T, topk), dtype=torch.float32, device=device)
        self.tok_slot = torch.empty((T, topk), **i32)
        self.h = torch.empty((T * topk, F), dtype=torch.float16, device=device)
        self.yp = torch.empty((T * topk, H), dtype=torch.float16 if yp_f16 else torch.float32, device=device)
        # zero once: holds completion counters every call leaves at zero
        self.ws = torch.zeros(lib().qw_moe_decode_workspace_size(T, E, topk, H, F), dtype=torch.uint8, device=device)
        if Fs:
            self.sh_v = torch.empty((T, 2 * Fs + 1), dtype=torch.float32, device=device)
            self.sh_out = torch.empty((T, H), dtype=torch.float32, device=device)
            self.ws_sh = torch.zeros(lib().qw_moe_decode_with_shared_workspace_size(T, E, topk, H, F, Fs),
                                     dtype=torch.uint8, device=device)


def moe_decode(router_w, x, topk, gate, up, down, E, F, buf=None, shared=None, out=None, out_bf16=True, x_f16=None,
               out_dtype=None, yp_f16=False):
    """Router GEMV + routing + experts + combine for a decode batch (3 to 5 launches).
    router_w [E][H] float32, or float16 (the engine's router weights). out bf16 (out_bf16), fp32, or
    out_dtype / the dtype of a given out; yp fp32, or fp16 with yp_f16 (or a buf whose yp is float16)."""
    import torch
    T, H = x.shape
    buf = buf if buf is not None else MoeDecode(T, E, topk, H, F, x.device, yp_f16=yp_f16)
    if out is None:
        dt = out_dtype if out_dtype is not None else torch.bfloat16 if out_bf16 else torch.float32
        out = torch.empty((T, H), dtype=dt, device=x.device)
    _dev(router_w, x, shared, out, *gate, *up, *down)
    if router_w.dtype not in (torch.float32, torch.float16):
        raise TypeError(f"moe_decode: router_w must be float32 or float16, not {router_w.dtype}")
    rc = lib().qw_moe_decode(_ptr(router_w), int(router_w.dtype == torch.float16), _ptr(x), int(_is_f16(x, x_f16)), T, E, topk, *map(_ptr, gate), *map(_ptr, up), *map(_ptr, down),
                             H, F, _ptr(shared), _ptr(out), _tcode(out), _ptr(buf.logits), _ptr(buf.top_e),
                             _ptr(buf.top_w), _ptr(buf.tok_slot), _ptr(buf.h), _ptr(buf.yp),
                             int(buf.yp.dtype == torch.float16), _ptr(buf.ws), buf.ws.numel(), _stream())
    _check(rc, "qw_moe_decode")
    return out, buf


def moe_decode_with_shared(router_w, x, topk, gate, up, down, E, F, sh_gu, sh_down, Fs, buf=None, out=None,
                           out_bf16=True, x_f16=None, yp_f16=False):
    """moe_decode with the shared expert: sh_gu [2 Fs + 1][H] tiled 16-bit (w16_tile) of x's type,
    sh_down [H][Fs] tiled fp16. Returns (out, buf, sh_v, sh_out): the shared expert's gate/up/gate-logit
    rows and output rows (fp32) beside the block's output."""
    import torch
    T, H = x.shape
    buf = buf if buf is not None else MoeDecode(T, E, topk, H, F, x.device, yp_f16=yp_f16, Fs=Fs)
    if buf.Fs != Fs:
        raise ValueError(f"moe_decode_with_shared: buf was made for Fs = {buf.Fs}, not {Fs}")
    if out is None:
        out = torch.empty((T, H), dtype=torch.bfloat16 if out_bf16 else torch.float32, device=x.device)
    if router_w.dtype not in (torch.float32, torch.float16):
        raise TypeError(f"moe_decode_with_shared: router_w must be float32 or float16, not {router_w.dtype}")
    sh_v, sh_out, ws = buf.sh_v, buf.sh_out, buf.ws_sh
    _dev(router_w, x, out, sh_gu, sh_down, *gate, *up, *down)
    rc = lib().qw_moe_decode_with_shared(
        _ptr(router_w), int(router_w.dtype == torch.float16), _ptr(x), int(_is_f16(x, x_f16)), T, E, topk,
        *map(_ptr, gate), *map(_ptr, up), *map(_ptr, down), H, F, _ptr(sh_gu), _ptr(sh_down), Fs, _ptr(sh_v),
        _ptr(sh_out), _ptr(out), _tcode(out), _ptr(buf.logits), _ptr(buf.top_e), _ptr(buf.top_w), _ptr(buf.tok_slot),
        _ptr(buf.h), _ptr(buf.yp), int(buf.yp.dtype == torch.float16), _ptr(ws), ws.numel(), _stream())
    _check(rc, "qw_moe_decode_with_shared")
    return out, buf, sh_v, sh_out


# -------------------------------------------------------- checkpoint loading
def bf16_to_f16(x, out=None):
    """bf16 bits (int16/uint16 or bfloat16 tensor) -> fp16 bits, saturating as
    the reference converts scales at load."""
    import torch
    out = out if out is not None else torch.empty(x.shape, dtype=torch.int16, device=x.device)
    _dev(x, out)
    _check(lib().qw_bf16_to_f16(_ptr(x), _ptr(out), x.numel(), _stream()), "qw_bf16_to_f16")
    return out


def read_probe(t=None):
    """Measurement aid: read tensor t's bytes (a multiple of 32768) with the
    dense GEMV's load shape and nothing else; t=None launches one empty block."""
    if t is None:
        _check(lib().qw_read_probe(None, 0, _stream()), "qw_read_probe")
        return
    _dev(t)
    _check(lib().qw_read_probe(_ptr(t), t.numel() * t.element_size(), _stream()), "qw_read_probe")


class StFile:
    """A safetensors file mapped by the library (host side)."""

    def __init__(self, path):
        h = ctypes.c_void_p()
        _check(lib().qw_st_open(os.fsencode(path), ctypes.byref(h)), "qw_st_open")
        self._h = h

    def close(self):
        if self._h:
            lib().qw_st_close(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def names(self):
        return [lib().qw_st_name(self._h, i).decode() for i in range(lib().qw_st_count(self._h))]

    def info(self, name):
        """(dtype, shape, nbytes) of one tensor."""
        dt = ctypes.create_string_buffer(16)
        shape = (ctypes.c_int64 * 8)()
        nd, nb, data = ctypes.c_int(), ctypes.c_size_t(), ctypes.c_void_p()
        _check(lib().qw_st_tensor(self._h, name.encode(), dt, shape, ctypes.byref(nd), ctypes.byref(data),
                                  ctypes.byref(nb)), "qw_st_tensor")
        return dt.value.decode(), tuple(shape[i] for i in range(nd.value)), nb.value


def tiled_offset(row0, K):
    a, b, c = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    lib().qw_q4_tiled_offset(row0, K, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c))
    return a.value, b.value, c.value


def load_q4(st, prefix, N, K, out=None, row0=0, device=None, cache=None):
    """Loads "<prefix>.weight_packed/.weight_scale" of an StFile into tiled
    device tensors (Wt, St, None). With out=(Wt, St, Zt) of a larger tiled
    matrix, writes rows row0 .. row0 + N - 1 of it (stacked experts).
    With a WCache: replaying, the rows come from the cache (st may be None);
    recording, they are converted and appended to it."""
    import torch
    device = device or torch.device("cuda", torch.cuda.current_device())
    if out is None:
        wb, sb, _ = tiled_size(N, K)
        out = (torch.empty(wb // 4, dtype=torch.int32, device=device),
               torch.empty(sb // 2, dtype=torch.int16, device=device), None)
    Wt, St_ = out[0], out[1]
    _dev(Wt, St_)
    ow, os_, _ = tiled_offset(row0, K)
    nw, ns, _ = tiled_size(N, K)
    if ow + nw > Wt.numel() * Wt.element_size() or os_ + ns > St_.numel() * St_.element_size():
        raise ValueError("load_q4: rows beyond the output tensors")
    wp, sp = Wt.data_ptr() + ow, St_.data_ptr() + os_
    if cache is not None and cache.mode == "replay":
        cache.get_ptr(wp, nw)
        cache.get_ptr(sp, ns)
        return out
    staging = torch.empty(lib().qw_q4_load_staging_size(N, K), dtype=torch.uint8, device=Wt.device)
    rc = lib().qw_q4_load(st._h, prefix.encode(), N, K, ctypes.c_void_p(wp), ctypes.c_void_p(sp), _ptr(staging),
                          staging.numel(), _stream())
    _check(rc, "qw_q4_load")
    torch.cuda.current_stream().synchronize()  # staging is freed on return
    if cache is not None:
        cache.put_ptr(wp, nw)
        cache.put_ptr(sp, ns)
    return out


def checkpoint_key(paths, options=""):
    """A 64-bit cache key for a checkpoint: names, sizes and modification
    times of its files plus the caller's conversion options."""
    import hashlib
    h = hashlib.blake2b(digest_size=8)
    for p in sorted(os.fspath(x) for x in paths):
        st = os.stat(p)
        h.update(f"{os.path.basename(p)}\0{st.st_size}\0{st.st_mtime_ns}\0".encode())
    h.update(options.encode())
    return int.from_bytes(h.digest(), "little")


class WCache:
    """Converted-weights cache file (qw_wcache_*). mode is "replay" when the
    file is a complete cache for `key`, "record" while writing it (completed
    by finish()), or "off" (reason in `why`)."""

    _MODES = {0: "off", 1: "record", 2: "replay"}

    def __init__(self, path, key):
        h, m = ctypes.c_void_p(), ctypes.c_int()
        _check(lib().qw_wcache_open(os.fsencode(path), ctypes.c_uint64(key), ctypes.byref(h), ctypes.byref(m)),
               "qw_wcache_open")
        self._h, self.mode = h, self._MODES[m.value]
        self.why = lib().qw_q4_last_error().decode() if self.mode == "off" else ""

    def put_ptr(self, ptr, nbytes, on_device=True):
        _check(lib().qw_wcache_put(self._h, ctypes.c_void_p(ptr), nbytes, int(on_device),
                                   _stream() if on_device else None), "qw_wcache_put")

    def get_ptr(self, ptr, nbytes, on_device=True):
        _check(lib().qw_wcache_get(self._h, ctypes.c_void_p(ptr), nbytes, int(on_device),
                                   _stream() if on_device else None), "qw_wcache_get")

    def put(self, t):
        """Appends a contiguous tensor (device or host) while recording."""
        if not t.is_contiguous():
            raise ValueError("WCache.put: tensor must be contiguous")
        self.put_ptr(t.data_ptr(), t.numel() * t.element_size(), t.is_cuda)

    def get(self, t):
        """Fills a contiguous tensor (device or host) with the next piece."""
        if not t.is_contiguous():
            raise ValueError("WCache.get: tensor must be contiguous")
        self.get_ptr(t.data_ptr(), t.numel() * t.element_size(), t.is_cuda)

    def finish(self):
        _check(lib().qw_wcache_finish(self._h), "qw_wcache_finish")
        if self.mode == "record":
            self.mode = "off"

    def close(self):
        if self._h:
            lib().qw_wcache_close(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
