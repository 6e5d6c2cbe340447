"""NumPy / torch front-ends over the C ABI, shaped like the calls the
reference's parity scripts make (ctypes into ck_test_* and the kernel symbols,
e.g. unittest/test_q4_k_q8_k_matvec.py:93-132, unittest/test_parallel_gemv.py:112-170).

Host functions take NumPy arrays and go through the drop-in (host-pointer)
symbols; `dev_*` functions take torch CUDA tensors and go through the
device-resident entry points on torch's current stream."""
import ctypes
import importlib.util
import os
import struct
import sys
import warnings

import numpy as np

from .api import BLOCK_ELEMS, CSRC, FMT, STEP, CkqError, MatmulOp, check, dump_lib, lib, row_bytes

_vp = ctypes.c_void_p


def _p(a):
    if a is None:
        return None
    assert a.flags.c_contiguous
    p = _vp(a.__array_interface__["data"][0])     # what a.ctypes.data_as(_vp) gives, at half its cost (1.3 us against 2.4)
    p._arr = a                                    # the array lives as long as the pointer
    return p


def act_format(wfmt):
    return "q8_0" if wfmt in ("q8_0", "q5_0") else "q8_k"


# ---- host-pointer (drop-in) path ------------------------------------------------

def quantize(x, fmt="q8_k", rows=1):
    """fp32 [rows*k] -> Q8_K / Q8_0 bytes via quantize_batch_*."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    k = x.size // rows
    out = np.zeros(rows * row_bytes(fmt, k), dtype=np.uint8)
    fn = lib().quantize_batch_q8_k if fmt == "q8_k" else lib().quantize_batch_q8_0
    fn(_p(x), _p(out), rows, k)
    return out


_GEMV = {"q4_k": "gemv_q4_k_q8_k", "q5_k": "gemv_q5_k_q8_k", "q6_k": "gemv_q6_k_q8_k", "q8_0": "gemv_q8_0_q8_0",
         "q5_0": "gemv_q5_0_q8_0"}
_GEMM_NT = {"q4_k": "gemm_nt_q4_k_q8_k", "q5_k": "gemm_nt_q5_k_q8_k", "q6_k": "gemm_nt_q6_k_q8_k",
            "q8_0": "gemm_nt_q8_0_q8_0", "q5_0": "gemm_nt_q5_0_q8_0"}


def gemv(fmt, W, x_q8, M, K, name=None):
    y = np.zeros(M, dtype=np.float32)
    getattr(lib(), name or _GEMV[fmt])(_p(y), _p(W), _p(x_q8), M, K)
    return y


def gemv_parallel(fmt, W, x_q8, M, K, nth, simd=True, y=None):
    """Union over ith of the thread-split entry point."""
    y = np.zeros(M, dtype=np.float32) if y is None else y
    fn = getattr(lib(), _GEMV[fmt] + ("_parallel_simd" if simd else "_parallel"))
    for ith in range(nth):
        fn(_p(y), _p(W), _p(x_q8), M, K, ith, nth)
    return y


def gemm_nt(fmt, A_q8, B, bias, M, N, K):
    c = np.zeros(M * N, dtype=np.float32)
    getattr(lib(), _GEMM_NT[fmt])(_p(A_q8), _p(B), _p(bias), _p(c), M, N, K)
    return c.reshape(M, N)


def dequant_row(fmt, src, n):
    out = np.zeros(n, dtype=np.float32)
    getattr(lib(), "dequant_%s_row" % fmt)(_p(src), _p(out), n)
    return out


def embedding_forward(fmt, ids, token_count, vocab, table, pos, embed_dim, aligned, context, add_pos, fill=0.0):
    out = np.full(context * aligned, fill, dtype=np.float32)
    getattr(lib(), "embedding_forward_" + fmt)(_p(ids), token_count, vocab, _p(table), _p(pos), _p(out),
                                               embed_dim, aligned, context, add_pos)
    return out.reshape(context, aligned)


def rmsnorm_q8_k_fused(x, gamma, tokens, d_model, aligned=None, eps=1e-6):
    aligned = aligned or d_model
    out = np.zeros(tokens * row_bytes("q8_k", d_model), dtype=np.uint8)
    lib().rmsnorm_q8_k_fused(_p(x), _p(gamma), _p(out), tokens, d_model, aligned, ctypes.c_float(eps))
    return out


CK_DT = {"q4_k": 7, "q6_k": 8, "q8_0": 9, "q8_k": 10, "q5_0": 11}   # the reference's CKDataType values


def fused_mlp_swiglu_prefill_w1w2_quant(x, W1, B1, w1_fmt, W2, B2, w2_fmt, seq_len, embed, aligned_embed,
                                        inter, aligned_inter, output=None, scratch=True):
    """Mirror of the reference symbol; returns the [seq_len, aligned_embed] output
    (or the untouched `output` passed in when the call rejects its arguments)."""
    out = output if output is not None else np.zeros(seq_len * aligned_embed, dtype=np.float32)
    scr = np.zeros(16, dtype=np.uint8) if scratch else None
    lib().fused_mlp_swiglu_prefill_w1w2_quant(_p(x), _p(W1), _p(B1), CK_DT[w1_fmt], _p(W2), _p(B2), CK_DT[w2_fmt],
                                              _p(out), seq_len, embed, aligned_embed, inter, aligned_inter, _p(scr))
    return out.reshape(seq_len, aligned_embed) if out.size == seq_len * aligned_embed else out


def gemv_f32act(fmt, W, x_f32, M, K):
    """gemv_q4_k / gemv_q6_k / gemv_q8_0: fp32 activations, nothing quantized."""
    y = np.zeros(M, dtype=np.float32)
    getattr(lib(), "gemv_" + fmt)(_p(y), _p(W), _p(x_f32), M, K)
    return y


def gemm_nt_f32act(fmt, A_f32, B, bias, M, N, K):
    c = np.zeros(M * N, dtype=np.float32)
    getattr(lib(), "gemm_nt_" + fmt)(_p(A_f32), _p(B), _p(bias), _p(c), M, N, K)
    return c.reshape(M, N)


def gemm_f32act(fmt, W, X_f32, M, N, K):
    """gemm_q4_k / gemm_q6_k / gemm_q8_0: Y[n*M + row]."""
    y = np.zeros(N * M, dtype=np.float32)
    getattr(lib(), "gemm_" + fmt)(_p(y), _p(W), _p(X_f32), M, N, K)
    return y.reshape(N, M)


# ---- device-resident path ---------------------------------------------------------

def _stream():
    import torch
    return _vp(torch.cuda.current_stream().cuda_stream)


def _dp(t):
    return None if t is None else _vp(t.data_ptr())


def to_device(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def dev_quantize(x_t, fmt="q8_k", rows=1):
    import torch
    k = x_t.numel() // rows
    out = torch.empty(rows * row_bytes(fmt, k), dtype=torch.uint8, device=x_t.device)
    fn = lib().ckq_quantize_q8_k_dev if fmt == "q8_k" else lib().ckq_quantize_q8_0_dev
    check(fn(_dp(x_t), _dp(out), rows, k, _stream()), "quantize_dev")
    return out


ACT_F32 = 0x200


def fmt_tag(name):
    """Weight-format tag of a format name; "<fmt>+f32" adds CKQ_ACT_F32 (a sequence entry
    with fp32 activations, no quantization)."""
    return FMT[name[:-4]] | ACT_F32 if name.endswith("+f32") else FMT[name]


def dev_gemm_nt(fmt, A_t, B_t, bias_t, M, N, K, out=None):
    """C[M,N] on the device; M = 1 is the GEMV."""
    import torch
    c = out if out is not None else torch.empty(M * N, dtype=torch.float32, device=B_t.device)
    check(lib().ckq_gemm_nt_dev(fmt_tag(fmt), _dp(A_t), _dp(B_t), _dp(bias_t), _dp(c), M, N, K, N, _stream()),
          "ckq_gemm_nt_dev")
    return c.view(M, N)


def dev_gemv_q8_0_f32(W_t, x_t, M, K):
    import torch
    y = torch.empty(M, dtype=torch.float32, device=W_t.device)
    check(lib().ckq_gemv_q8_0_dev(_dp(y), _dp(W_t), _dp(x_t), M, K, _stream()), "ckq_gemv_q8_0_dev")
    return y


def dev_dequant_rows(fmt, table_t, ids_t, vocab, pos_t, n_valid, n_row, tokens, n_out_rows):
    import torch
    out = torch.full((n_out_rows * n_row,), 7.0, dtype=torch.float32, device=table_t.device)
    check(lib().ckq_dequant_rows_dev(FMT[fmt], _dp(table_t), _dp(ids_t), vocab, _dp(pos_t), _dp(out), n_valid, n_row,
                                     tokens, n_out_rows, _stream()), "ckq_dequant_rows_dev")
    return out.view(n_out_rows, n_row)


def dev_rmsnorm_q8_k_fused(x_t, gamma_t, tokens, d_model, aligned=None, eps=1e-6):
    import torch
    aligned = aligned or d_model
    out = torch.zeros(tokens * row_bytes("q8_k", d_model), dtype=torch.uint8, device=x_t.device)
    check(lib().ckq_rmsnorm_q8_k_fused_dev(_dp(x_t), _dp(gamma_t), _dp(out), tokens, d_model, aligned,
                                           ctypes.c_float(eps), _stream()), "ckq_rmsnorm_q8_k_fused_dev")
    return out


def dev_swiglu_q8_k(gate_t, up_t, rows, k, ld):
    import torch
    out = torch.zeros(rows * row_bytes("q8_k", k), dtype=torch.uint8, device=gate_t.device)
    check(lib().ckq_swiglu_q8_k_dev(_dp(gate_t), _dp(up_t), _dp(out), rows, k, ld, _stream()), "ckq_swiglu_q8_k_dev")
    return out


def dev_gemm_nt_f32act(fmt, A_t, B_t, bias_t, M, N, K, out=None):
    import torch
    c = out if out is not None else torch.empty(M * N, dtype=torch.float32, device=B_t.device)
    check(lib().ckq_gemm_nt_f32act_dev(FMT[fmt], _dp(A_t), _dp(B_t), _dp(bias_t), _dp(c), M, N, K, N, _stream()),
          "ckq_gemm_nt_f32act_dev")
    return c


# ---- rows of int8 with one scale each ---------------------------------------------
# A decode step makes these calls one by one, each for a kernel of a few microseconds.  So a call looks at a tensor's
# shape, strides, type and device once each, in one expression without calls of functions in Python (a matmul's checks 0.6 us less);
# what that expression does not take goes to _i8_refuse, which looks again and says why.

_torch, _INT8, _F8, _I32, _F32, _started, _device, _raw_stream, _I8_TYPES = None, None, None, None, None, None, None, None, {}


def _i8_torch():
    """torch, and what every call needs of it, once: an import statement in each call costs it 0.3 us a time, a chain of names 0.05."""
    global _torch, _INT8, _F8, _I32, _F32, _started, _device, _raw_stream
    import torch
    _INT8, _F8, _I32, _F32 = torch.int8, torch.float8_e4m3fn, torch.int32, torch.float32
    _I8_TYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})   # CKDataType values
    _started = torch.cuda.is_initialized
    _device, _raw_stream = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)
    _torch = torch
    return torch


def _i8_where():
    """The current device and its current stream (what torch.cuda.current_device and current_stream say, a tenth of their cost);
    without a device, a number that no tensor's device has."""
    if _torch is None:
        _i8_torch()
    if not _started():
        if not _torch.cuda.is_available():
            return -2, None
        _torch.cuda.init()
    dev = _device()
    return dev, _raw_stream(dev)


def _i8_refuse(dev, rows, floats):
    """Says what is wrong with a call: rows, 2-d tensors (tensor, name, shape or None, type; None: one of floats), elements of a row side by
    side; floats, contiguous float32 vectors (tensor, name, shape).  All on device `dev`."""
    for t, what, shape, dtype in rows:
        if t.dim() != 2 or (shape is not None and tuple(t.shape) != tuple(shape)):
            raise CkqError("%s has the shape %s, not %s" % (what, tuple(t.shape), "rows x k" if shape is None else tuple(shape)))
        if dtype is None and t.dtype not in _I8_TYPES:
            raise CkqError("%s is %s: float32, bfloat16 or float16 are taken" % (what, t.dtype))
        if dtype is not None and t.dtype is not dtype:
            raise CkqError("%s is %s, not %s" % (what, t.dtype, dtype))
        if t.get_device() != dev:
            raise CkqError("%s is on %s, not on the current device" % (what, t.device))
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise CkqError("%s: the elements of a row have to lie side by side" % what)
    for t, what, shape in floats:
        if t.dtype is not _F32 or t.shape != shape or not t.is_contiguous():
            raise CkqError("%s has to be contiguous float32 of the shape %s" % (what, tuple(shape)))
        if t.get_device() != dev:
            raise CkqError("%s is on %s, not on the current device" % (what, t.device))
    raise CkqError("two tensors of this call need one pitch")


def _i8_too_many(*sizes):
    raise CkqError("sizes %s: the library takes 2^31 - 1 at most (ctypes would pass their lowest 32 bits)" % (sizes,))


def empty_i8(rows, k, device="cuda"):
    """int8 [rows, k] whose rows begin at multiples of 16 bytes, as dev_gemm_nt_i8 takes them."""
    torch = _torch or _i8_torch()
    return torch.empty(rows, -(-k // 16) * 16, dtype=torch.int8, device=device)[:, :k]


def _i8_new(x):
    if x.dim() != 2:
        raise CkqError("a tensor of the shape %s, not rows x k" % (tuple(x.shape),))
    return empty_i8(*x.shape, x.device), _torch.empty(x.shape[0], dtype=_F32, device=x.device)


# A single row has any stride in torch: its pitch counts as its length.

def dev_quantize_i8(x, out=None):
    """Rows of x [rows, k] in 8 bits: (q int8 [rows, k], scale float32 [rows])."""
    dev, stream = _i8_where()
    q, scale = out if out is not None else _i8_new(x)
    shape, kind = x.shape, _I8_TYPES.get(x.dtype)
    if (len(shape) != 2 or q.shape != shape or kind is None or q.dtype is not _INT8 or scale.dtype is not _F32 or scale.shape != shape[:1]
            or not scale.is_contiguous() or not x.get_device() == q.get_device() == scale.get_device() == dev):
        _i8_refuse(dev, [(x, "x", None, None), (q, "q", shape, _INT8)], [(scale, "scale", shape[:1])])
    rows, k = shape
    if (rows | k) >> 31:
        _i8_too_many(rows, k)
    (ldx, ex), (ldq, eq) = x.stride(), q.stride()
    if (ex != 1 or eq != 1) and k > 1:
        _i8_refuse(dev, [(x, "x", None, None), (q, "q", shape, _INT8)], [])
    if rows == 1:
        ldx = ldq = k
    rc = lib().ckq_quantize_i8_dev(kind, x.data_ptr(), ldx, q.data_ptr(), ldq, scale.data_ptr(), rows, k, stream)
    if rc:
        check(rc, "ckq_quantize_i8_dev")
    return q, scale


def dev_dequantize_i8(q, scale, dtype=None, out=None):
    """scale * q as rows of dtype (float32), or into `out`."""
    dev, stream = _i8_where()
    shape = q.shape
    y = out if out is not None else _torch.empty(shape, dtype=dtype or _F32, device=q.device)
    t = y.dtype
    kind = _I8_TYPES.get(t)
    if (len(shape) != 2 or y.shape != shape or kind is None or (dtype is not None and t is not dtype) or q.dtype is not _INT8 or scale.dtype is not _F32
            or scale.shape != shape[:1] or not scale.is_contiguous() or not q.get_device() == scale.get_device() == y.get_device() == dev):
        _i8_refuse(dev, [(q, "q", None, _INT8), (y, "out", shape, None), (y, "out", shape, dtype)], [(scale, "scale", shape[:1])])
    rows, k = shape
    if (rows | k) >> 31:
        _i8_too_many(rows, k)
    (ldq, eq), (ldy, ey) = q.stride(), y.stride()
    if (eq != 1 or ey != 1) and k > 1:
        _i8_refuse(dev, [(q, "q", None, _INT8), (y, "out", shape, None)], [])
    if rows == 1:
        ldq = ldy = k
    rc = lib().ckq_dequantize_i8_dev(q.data_ptr(), ldq, scale.data_ptr(), kind, y.data_ptr(), ldy, rows, k, stream)
    if rc:
        check(rc, "ckq_dequantize_i8_dev")
    return y


def dev_rmsnorm_i8(x, gamma, eps=1e-6, residual=None, residual_out=None, out=None):
    """RMSNorm(x (+ residual)) * gamma in 8 bits: (q, scale), or (q, scale, x + residual) with a residual; residual_out
    may be the residual itself, or x."""
    dev, stream = _i8_where()
    q, scale = out if out is not None else _i8_new(x)
    shape, t = x.shape, x.dtype
    kind = _I8_TYPES.get(t)
    if (len(shape) != 2 or q.shape != shape or kind is None or q.dtype is not _INT8 or scale.dtype is not _F32 or gamma.dtype is not _F32
            or scale.shape != shape[:1] or gamma.shape != shape[1:] or not scale.is_contiguous() or not gamma.is_contiguous()
            or not x.get_device() == q.get_device() == scale.get_device() == gamma.get_device() == dev):
        _i8_refuse(dev, [(x, "x", None, None), (q, "q", shape, _INT8)], [(scale, "scale", shape[:1]), (gamma, "gamma", shape[1:])])
    rows, k = shape
    if (rows | k) >> 31:
        _i8_too_many(rows, k)
    (ldx, ex), (ldq, eq) = x.stride(), q.stride()
    ldr, rp, hp = 0, None, None
    if residual is not None:
        if residual_out is None:
            residual_out = _torch.empty_strided(residual.shape, residual.stride(), dtype=t, device=x.device)
        if (residual.shape != shape or residual_out.shape != shape or residual.dtype is not t or residual_out.dtype is not t
                or not residual.get_device() == residual_out.get_device() == dev):
            _i8_refuse(dev, [(residual, "residual", shape, t), (residual_out, "residual_out", shape, t)], [])
        (ldr, er), (ldh, eh) = residual.stride(), residual_out.stride()
        if (er != 1 or eh != 1) and k > 1 or ldr != ldh and rows > 1:
            _i8_refuse(dev, [(residual, "residual", shape, t), (residual_out, "residual_out", shape, t)], [])
        rp, hp = residual.data_ptr(), residual_out.data_ptr()
    elif residual_out is not None:
        raise CkqError("residual_out without a residual")
    if (ex != 1 or eq != 1) and k > 1:
        _i8_refuse(dev, [(x, "x", None, None), (q, "q", shape, _INT8)], [])
    if rows == 1:
        ldx = ldq = ldr = k
    rc = lib().ckq_rmsnorm_i8_dev(kind, x.data_ptr(), ldx, rp, hp, ldr, gamma.data_ptr(), eps, q.data_ptr(), ldq, scale.data_ptr(), rows, k, stream)
    if rc:
        check(rc, "ckq_rmsnorm_i8_dev")
    return (q, scale) if residual is None else (q, scale, residual_out)


def dev_swiglu_i8(gate, up, out=None):
    """SiLU(gate) * up in 8 bits: (q, scale); gate and up have one pitch (halves of one tensor, say)."""
    dev, stream = _i8_where()
    q, scale = out if out is not None else _i8_new(gate)
    shape, t = gate.shape, gate.dtype
    kind = _I8_TYPES.get(t)
    if (len(shape) != 2 or q.shape != shape or up.shape != shape or kind is None or up.dtype is not t or q.dtype is not _INT8 or scale.dtype is not _F32
            or scale.shape != shape[:1] or not scale.is_contiguous() or not gate.get_device() == up.get_device() == q.get_device() == scale.get_device() == dev):
        _i8_refuse(dev, [(gate, "gate", None, None), (up, "up", shape, t), (q, "q", shape, _INT8)], [(scale, "scale", shape[:1])])
    rows, k = shape
    if (rows | k) >> 31:
        _i8_too_many(rows, k)
    (ld, eg), (ldu, eu), (ldq, eq) = gate.stride(), up.stride(), q.stride()
    if (eg != 1 or eu != 1 or eq != 1) and k > 1 or ldu != ld and rows > 1:
        _i8_refuse(dev, [(gate, "gate", None, None), (up, "up", shape, t), (q, "q", shape, _INT8)], [])
    if rows == 1:
        ld = ldq = k
    rc = lib().ckq_swiglu_i8_dev(kind, gate.data_ptr(), up.data_ptr(), ld, q.data_ptr(), ldq, scale.data_ptr(), rows, k, stream)
    if rc:
        check(rc, "ckq_swiglu_i8_dev")
    return q, scale


def dev_gemm_nt_i8(a, sa, b, sb, bias=None, dtype=None, out=None):
    """C [M, N] = sa[m] * sb[n] * (a b^T) (+ bias[n]): int8 rows a [M, K] (tokens), b [N, K] (channels); C of dtype (float32),
    or into `out`."""
    dev, stream = _i8_where()
    of_a, of_b = a.shape, b.shape
    if len(of_a) != 2 or len(of_b) != 2 or of_a[1] != of_b[1]:
        _i8_refuse(dev, [(a, "a", None, _INT8), (b, "b", (of_b[0], of_a[1]) if a.dim() == b.dim() == 2 else None, _INT8)], [])
    M, K = of_a
    N = of_b[0]
    if (M | N | K) >> 31:
        _i8_too_many(M, N, K)
    c = out if out is not None else _torch.empty(M, N, dtype=dtype or _F32, device=b.device)
    t = c.dtype
    kind = _I8_TYPES.get(t)
    if (c.shape != (M, N) or kind is None or (dtype is not None and t is not dtype) or a.dtype is not _INT8 or b.dtype is not _INT8 or sa.dtype is not _F32 or sb.dtype is not _F32
            or sa.shape != (M,) or sb.shape != (N,) or not sa.is_contiguous() or not sb.is_contiguous()
            or not a.get_device() == b.get_device() == c.get_device() == sa.get_device() == sb.get_device() == dev):
        _i8_refuse(dev, [(a, "a", None, _INT8), (b, "b", None, _INT8), (c, "out", (M, N), None), (c, "out", (M, N), dtype)], [(sa, "sa", (M,)), (sb, "sb", (N,))])
    bp = None
    if bias is not None:
        if bias.dtype is not _F32 or bias.shape != (N,) or not bias.is_contiguous() or bias.get_device() != dev:
            _i8_refuse(dev, [], [(bias, "bias", (N,))])
        bp = bias.data_ptr()
    (lda, ea), (ldb, eb), (ldc, ec) = a.stride(), b.stride(), c.stride()
    if (ea != 1 or eb != 1) and K > 1 or ec != 1 and N > 1:
        _i8_refuse(dev, [(a, "a", None, _INT8), (b, "b", None, _INT8), (c, "out", (M, N), None)], [])
    if M == 1:
        lda, ldc = -(-K // 16) * 16, N
    if N == 1:
        ldb = -(-K // 16) * 16
    rc = lib().ckq_gemm_nt_i8_dev(a.data_ptr(), lda, sa.data_ptr(), b.data_ptr(), ldb, sb.data_ptr(), bp, kind, c.data_ptr(), ldc, M, N, K, stream)
    if rc:
        check(rc, "ckq_gemm_nt_i8_dev")
    return c


# ---- rows in e4m3 with one scale for each 128 elements, tokens sorted by expert --------------
# The manner of the int8 rows above: one expression of checks a call, the reasons of a refusal looked for afterwards.
# Scales are float32 [rows, groups] whose first index runs fastest (those of a group side by side), as empty_f8 makes them.

def _f8_refuse(dev, rows, scales=(), wholes=()):
    """Says what is wrong with a call: rows as _i8_refuse takes them; scales (tensor, name, shape), float32, the first index fastest; wholes,
    contiguous tensors (tensor, name, shape, type).  All on device `dev`."""
    for t, what, shape in scales:
        if t.dtype is not _F32 or tuple(t.shape) != tuple(shape):
            raise CkqError("%s has to be float32 of the shape %s, not %s %s" % (what, tuple(shape), t.dtype, tuple(t.shape)))
        if t.get_device() != dev:
            raise CkqError("%s is on %s, not on the current device" % (what, t.device))
        if (t.shape[0] > 1 and t.stride(0) != 1) or (t.shape[1] > 1 and t.stride(1) < t.shape[0]):
            raise CkqError("%s: the scales of a group have to lie side by side (empty_f8 makes them so)" % what)
    for t, what, shape, dtype in wholes:
        if t.dtype is not dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
            raise CkqError("%s has to be contiguous %s of the shape %s, not %s %s" % (what, dtype, tuple(shape), t.dtype, tuple(t.shape)))
        if t.get_device() != dev:
            raise CkqError("%s is on %s, not on the current device" % (what, t.device))
    _i8_refuse(dev, rows, [])


# With `out` given, a call is first offered to csrc/ckq_tensors.so, which reads the same of the tensors in C++ (a call of dev_gemm_nt_f8_experts 6.1 -> 3.5 us, of dev_moe_gather 4.7 -> 3.0); what that does not take, or the library
# refuses, comes back and is looked at here.  Without that module all of it happens here, and with one that was built for another torch or Python, or cannot be loaded.

class _Fast:
    """Stands for the module until the first call, and for good where there is none that can be used."""
    absent = False

    def __getattr__(self, name):
        return (lambda *a: -1000) if self.absent else getattr(_load_fast(), name)


_fast = _Fast()


def _load_fast():
    global _fast
    torch = _i8_torch()
    path = os.path.join(CSRC, "ckq_tensors.so")
    why, here = None, "torch-%s-python-%d.%d" % (torch.__version__, *sys.version_info[:2])
    if os.path.exists(path):
        try:
            spec = importlib.util.spec_from_file_location("ckq_tensors", path)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
        except ImportError as e:
            why = str(e)
        else:
            built = getattr(module, "built_for", None)
            if built == here:
                module.bind(ctypes.cast(lib().ckq_call_dev, _vp).value)
                _fast = module
                return _fast
            why = "it was built for %s, this is %s" % (built, here)
    if why:
        warnings.warn("%s is not used, calls go through ctypes (`make tensors` builds it anew): %s" % (path, why))
    _fast = _Fast()
    _fast.absent = True
    return _fast


# The calls go through ckq_call_dev, which number and arguments in one string of bytes: an argument costs ctypes 0.09 us and struct 0.01.
_PACK_8, _PACK_10, _PACK_11, _PACK_12, _PACK_13, _PACK_15, _PACK_16, _PACK_20 = (struct.Struct("%dq" % (n + 1)).pack for n in (8, 10, 11, 12, 13, 15, 16, 20))


def empty_f8(rows, k, device="cuda"):
    """(codes, scales) for rows of k: float8_e4m3fn [rows, k] whose rows begin at multiples of 16 bytes, as dev_gemm_nt_f8 takes them, and float32
    [rows, ceil(k / 128)] with the scales of a group side by side."""
    torch = _torch or _i8_torch()
    return (torch.empty(rows, -(-k // 16) * 16, dtype=torch.float8_e4m3fn, device=device)[:, :k],
            torch.empty(-(-k // 128), rows, dtype=torch.float32, device=device).t())


def _f8_new(x, rows=None):
    """`rows` given: some of them may be written by nothing, and are zeros."""
    if x.dim() != 2:
        raise CkqError("a tensor of the shape %s, not rows x k" % (tuple(x.shape),))
    if rows is None:
        return empty_f8(*x.shape, x.device)
    q, scale = empty_f8(rows, x.shape[1], x.device)
    q.view(_torch.uint8).zero_()
    return q, scale.zero_()


def _f8_side(scale, rows, groups):
    """The pitch of scales [rows, groups], 0 where they do not lie as the library takes them."""
    if scale.dtype is not _F32 or scale.shape != (rows, groups):
        return 0
    s0, s1 = scale.stride()
    if groups == 1:
        s1 = rows
    return s1 if (s0 == 1 or rows == 1) and s1 >= rows else 0


def dev_quantize_f8(x, out=None):
    """Rows of x [rows, k] in e4m3: (q float8_e4m3fn [rows, k], scale float32 [rows, ceil(k / 128)])."""
    if out is not None and _fast.quantize(x, *out) == 0:
        return out
    dev, stream = _i8_where()
    q, scale = out if out is not None else _f8_new(x)
    shape, kind = x.shape, _I8_TYPES.get(x.dtype)
    if (len(shape) != 2 or q.shape != shape or kind is None or q.dtype is not _F8 or not x.get_device() == q.get_device() == scale.get_device() == dev):
        _f8_refuse(dev, [(x, "x", None, None), (q, "q", shape, _F8)], [(scale, "scale", (shape[0], -(-shape[-1] // 128)))])
    rows, k = shape
    if (rows | k) >> 31:
        _i8_too_many(rows, k)
    lds = _f8_side(scale, rows, -(-k // 128))
    (ldx, ex), (ldq, eq) = x.stride(), q.stride()
    if (ex != 1 or eq != 1) and k > 1 or not lds:
        _f8_refuse(dev, [(x, "x", None, None), (q, "q", shape, _F8)], [(scale, "scale", (rows, -(-k // 128)))])
    if rows == 1:
        ldx = ldq = k
    rc = lib().ckq_call_dev(_PACK_10(0, kind, x.data_ptr(), ldx, q.data_ptr(), ldq, scale.data_ptr(), lds, rows, k, stream))
    if rc:
        check(rc, "ckq_quantize_f8_dev")
    return q, scale


def dev_dequantize_f8(q, scale, dtype=None, out=None):
    """scale * q as rows of dtype (float32), or into `out`."""
    if out is not None and dtype is None and _fast.dequantize(q, scale, out) == 0:
        return out
    dev, stream = _i8_where()
    shape = q.shape
    y = out if out is not None else _torch.empty(shape, dtype=dtype or _F32, device=q.device)
    kind = _I8_TYPES.get(y.dtype)
    if (len(shape) != 2 or y.shape != shape or kind is None or (dtype is not None and y.dtype is not dtype) or q.dtype is not _F8
            or not q.get_device() == scale.get_device() == y.get_device() == dev):
        _f8_refuse(dev, [(q, "q", None, _F8), (y, "out", shape, None), (y, "out", shape, dtype)], [(scale, "scale", (shape[0], -(-shape[-1] // 128)))])
    rows, k = shape
    if (rows | k) >> 31:
        _i8_too_many(rows, k)
    lds = _f8_side(scale, rows, -(-k // 128))
    (ldq, eq), (ldy, ey) = q.stride(), y.stride()
    if (eq != 1 or ey != 1) and k > 1 or not lds:
        _f8_refuse(dev, [(q, "q", None, _F8), (y, "out", shape, None)], [(scale, "scale", (rows, -(-k // 128)))])
    if rows == 1:
        ldq = ldy = k
    rc = lib().ckq_call_dev(_PACK_10(1, q.data_ptr(), ldq, scale.data_ptr(), lds, kind, y.data_ptr(), ldy, rows, k, stream))
    if rc:
        check(rc, "ckq_dequantize_f8_dev")
    return y


def dev_swiglu_f8(gate, up, out=None):
    """SiLU(gate) * up in e4m3: (q, scale); gate and up have one pitch (halves of one tensor, say)."""
    if out is not None and _fast.swiglu(gate, up, *out) == 0:
        return out
    dev, stream = _i8_where()
    q, scale = out if out is not None else _f8_new(gate)
    shape, t = gate.shape, gate.dtype
    kind = _I8_TYPES.get(t)
    if (len(shape) != 2 or q.shape != shape or up.shape != shape or kind is None or up.dtype is not t or q.dtype is not _F8
            or not gate.get_device() == up.get_device() == q.get_device() == scale.get_device() == dev):
        _f8_refuse(dev, [(gate, "gate", None, None), (up, "up", shape, t), (q, "q", shape, _F8)], [(scale, "scale", (shape[0], -(-shape[-1] // 128)))])
    rows, k = shape
    if (rows | k) >> 31:
        _i8_too_many(rows, k)
    lds = _f8_side(scale, rows, -(-k // 128))
    (ld, eg), (ldu, eu), (ldq, eq) = gate.stride(), up.stride(), q.stride()
    if (eg != 1 or eu != 1 or eq != 1) and k > 1 or ldu != ld and rows > 1 or not lds:
        _f8_refuse(dev, [(gate, "gate", None, None), (up, "up", shape, t), (q, "q", shape, _F8)], [(scale, "scale", (rows, -(-k // 128)))])
    if rows == 1:
        ld = ldq = k
    rc = lib().ckq_call_dev(_PACK_11(2, kind, gate.data_ptr(), up.data_ptr(), ld, q.data_ptr(), ldq, scale.data_ptr(), lds, rows, k, stream))
    if rc:
        check(rc, "ckq_swiglu_f8_dev")
    return q, scale


def dev_gemm_nt_f8(a, sa, b, sb, bias=None, dtype=None, out=None, fp32_sums=False):
    """C [M, N] = a b^T (+ bias[n]) of the values that the codes stand for: float8_e4m3fn rows a [M, K] (tokens) with scales sa [M, ceil(K / 128)], b [N, K]
    (channels) with float32 scales sb [ceil(N / 128), ceil(K / 128)]; C of dtype (float32), or into `out`.  A C of 16 bits may come from instructions that drop, of each eight products, what is under 2^-13
    of their largest; with fp32_sums it does not (2048 x 11008 x 4096 twice the time)."""
    if out is not None and dtype is None and not fp32_sums and _fast.gemm(a, sa, b, sb, bias, out) == 0:
        return out
    dev, stream = _i8_where()
    of_a, of_b = a.shape, b.shape
    if len(of_a) != 2 or len(of_b) != 2 or of_a[1] != of_b[1]:
        _f8_refuse(dev, [(a, "a", None, _F8), (b, "b", (of_b[0], of_a[1]) if a.dim() == b.dim() == 2 else None, _F8)])
    M, K = of_a
    N = of_b[0]
    if (M | N | K) >> 31:
        _i8_too_many(M, N, K)
    G, blocks = -(-K // 128), -(-N // 128)
    c = out if out is not None else _torch.empty(M, N, dtype=dtype or _F32, device=b.device)
    t = c.dtype
    kind = _I8_TYPES.get(t)
    ldsa = _f8_side(sa, M, G)
    if (c.shape != (M, N) or kind is None or (dtype is not None and t is not dtype) or a.dtype is not _F8 or b.dtype is not _F8 or not ldsa
            or sb.dtype is not _F32 or sb.shape != (blocks, G) or not sb.is_contiguous()
            or not a.get_device() == b.get_device() == c.get_device() == sa.get_device() == sb.get_device() == dev):
        _f8_refuse(dev, [(a, "a", None, _F8), (b, "b", None, _F8), (c, "out", (M, N), None), (c, "out", (M, N), dtype)], [(sa, "sa", (M, G))], [(sb, "sb", (blocks, G), _F32)])
    bp = 0
    if bias is not None:
        if bias.dtype is not _F32 or bias.shape != (N,) or not bias.is_contiguous() or bias.get_device() != dev:
            _i8_refuse(dev, [], [(bias, "bias", (N,))])
        bp = bias.data_ptr()
    (lda, ea), (ldb, eb), (ldc, ec) = a.stride(), b.stride(), c.stride()
    if (ea != 1 or eb != 1) and K > 1 or ec != 1 and N > 1:
        _f8_refuse(dev, [(a, "a", None, _F8), (b, "b", None, _F8), (c, "out", (M, N), None)])
    if M == 1:
        lda, ldc = -(-K // 16) * 16, N
    if N == 1:
        ldb = -(-K // 16) * 16
    rc = lib().ckq_call_dev(_PACK_16(3, a.data_ptr(), lda, sa.data_ptr(), ldsa, b.data_ptr(), ldb, sb.data_ptr(), G, bp, kind | 256 if fp32_sums else kind, c.data_ptr(), ldc, M, N, K, stream))
    if rc:
        check(rc, "ckq_gemm_nt_f8_dev")
    return c


def dev_gemm_nt_f8_experts(a, sa, b, sb, offsets, bias=None, dtype=None, out=None):
    """Rows offsets[e] .. offsets[e + 1] - 1 of C [M, N] as dev_gemm_nt_f8 has them with b[e], sb[e], bias[e]: b float8_e4m3fn [E, N, K], sb float32 [E, ceil(N / 128),
    ceil(K / 128)], bias float32 [E, N], offsets int32 [E + 1].  Rows that no expert has stay as they are in `out`, and are zeros without it."""
    if out is not None and dtype is None and _fast.experts(a, sa, b, sb, offsets, bias, out) == 0:
        return out
    dev, stream = _i8_where()
    of_a, of_b = a.shape, b.shape
    if len(of_a) != 2 or len(of_b) != 3 or of_a[1] != of_b[2]:
        raise CkqError("a of the shape %s and b of the shape %s, not rows x k and experts x rows x k" % (tuple(of_a), tuple(of_b)))
    M, K = of_a
    E, N = of_b[:2]
    if (M | N | K | E) >> 31:
        _i8_too_many(M, N, K, E)
    G, blocks = -(-K // 128), -(-N // 128)
    c = out if out is not None else _torch.zeros(M, N, dtype=dtype or _F32, device=b.device)
    t = c.dtype
    kind = _I8_TYPES.get(t)
    ldsa = _f8_side(sa, M, G)
    if (c.shape != (M, N) or kind is None or (dtype is not None and t is not dtype) or a.dtype is not _F8 or b.dtype is not _F8 or not ldsa
            or sb.dtype is not _F32 or sb.shape != (E, blocks, G) or not sb.is_contiguous() or offsets.dtype is not _I32 or offsets.shape != (E + 1,) or not offsets.is_contiguous()
            or not a.get_device() == b.get_device() == c.get_device() == sa.get_device() == sb.get_device() == offsets.get_device() == dev):
        _f8_refuse(dev, [(a, "a", None, _F8), (b[0] if E else b, "b[e]", None, _F8), (c, "out", (M, N), None), (c, "out", (M, N), dtype)], [(sa, "sa", (M, G))],
                   [(sb, "sb", (E, blocks, G), _F32), (offsets, "offsets", (E + 1,), _I32)])
    bp = 0
    if bias is not None:
        if bias.dtype is not _F32 or bias.shape != (E, N) or not bias.is_contiguous() or bias.get_device() != dev:
            _f8_refuse(dev, [], [], [(bias, "bias", (E, N), _F32)])
        bp = bias.data_ptr()
    (lda, ea), (per, ldb, eb), (ldc, ec) = a.stride(), b.stride(), c.stride()
    if (ea != 1 or eb != 1) and K > 1 or ec != 1 and N > 1:
        _f8_refuse(dev, [(a, "a", None, _F8), (b[0], "b[e]", None, _F8), (c, "out", (M, N), None)])
    if M == 1:
        lda, ldc = -(-K // 16) * 16, N
    if N == 1:
        ldb = -(-K // 16) * 16
    if E == 1:
        per = 0
    rc = lib().ckq_call_dev(_PACK_20(4, a.data_ptr(), lda, sa.data_ptr(), ldsa, b.data_ptr(), ldb, per, sb.data_ptr(), G, blocks * G, bp, offsets.data_ptr(), E, kind,
                                          c.data_ptr(), ldc, M, N, K, stream))
    if rc:
        check(rc, "ckq_gemm_nt_f8_experts_dev")
    return c


def dev_moe_sort(ids, experts, out=None):
    """Slots (t, j) of ids int32 [tokens, choices] in the order of their experts, those of one expert as they come: (offsets int32 [experts + 1], order int32 [tokens * choices],
    position int32 [tokens, choices]); -1 in position, and at the end of order, for ids outside 0 .. experts - 1."""
    if out is not None and _fast.sort(ids, experts, *out) == 0:
        return out
    dev, stream = _i8_where()
    shape = ids.shape
    if len(shape) != 2 or experts < 1:
        raise CkqError("ids of the shape %s, not tokens x choices, or %s experts" % (tuple(shape), experts))
    T, c = shape
    if out is None:
        out = (_torch.empty(experts + 1, dtype=_I32, device=ids.device), _torch.empty(T * c, dtype=_I32, device=ids.device), _torch.empty(T, c, dtype=_I32, device=ids.device))
    offsets, order, position = out
    if (not ids.dtype is offsets.dtype is order.dtype is position.dtype is _I32 or offsets.shape != (experts + 1,) or order.shape != (T * c,) or position.shape != shape
            or not (ids.is_contiguous() and offsets.is_contiguous() and order.is_contiguous() and position.is_contiguous())
            or not ids.get_device() == offsets.get_device() == order.get_device() == position.get_device() == dev):
        _f8_refuse(dev, [], [], [(ids, "ids", shape, _I32), (offsets, "offsets", (experts + 1,), _I32), (order, "order", (T * c,), _I32), (position, "position", shape, _I32)])
    if (T | c | experts) >> 31:
        _i8_too_many(T, c, experts)
    rc = lib().ckq_call_dev(_PACK_8(5, ids.data_ptr(), T, c, experts, offsets.data_ptr(), order.data_ptr(), position.data_ptr(), stream))
    if rc:
        check(rc, "ckq_moe_sort_dev")
    return out


def _moe_refuse(dev, x, tokens, position, others, weights=()):
    """Says what is wrong with rows there and back: x [tokens (None: any), k] of floats, position int32 [tokens, choices], others (tensor, name, rows or None) of x's type and
    width, weights (tensor, name) like position."""
    places = position.shape
    if len(places) != 2:
        raise CkqError("position has the shape %s, not tokens x choices" % (tuple(places),))
    sizes = [n for t in [x, position] + [o[0] for o in others] for n in t.shape]
    if any(n >> 31 for n in sizes):
        _i8_too_many(*sizes)
    _f8_refuse(dev, [(x, "the rows", None if tokens is None or x.dim() != 2 else (tokens, x.shape[1]), None)]
               + [(t, what, (t.shape[0] if rows is None and t.dim() else rows, x.shape[-1]), x.dtype) for t, what, rows in others], [],
               [(position, "position", places, _I32)] + [(t, what, places, _F32) for t, what in weights])


def dev_moe_gather(x, position, out=None):
    """y[position[t][j]] = x[t]: x [tokens, k], position as dev_moe_sort has it; y [tokens * choices, k], or into the rows of `out`.  Rows that have no slot stay as they are in `out`, and
    are zeros without it."""
    if out is not None and _fast.gather(x, position, out) == 0:
        return out
    dev, stream = _i8_where()
    shape, places, t = x.shape, position.shape, x.dtype
    if out is None and len(shape) == 2:
        out = _torch.zeros(position.numel(), shape[1], dtype=t, device=x.device)
    into, kind = out.shape if out is not None else (), _I8_TYPES.get(t)
    if (len(shape) != 2 or len(places) != 2 or len(into) != 2 or shape[0] != places[0] or into[1] != shape[1] or kind is None or out.dtype is not t or position.dtype is not _I32
            or not position.is_contiguous() or not x.get_device() == position.get_device() == out.get_device() == dev):
        _moe_refuse(dev, x, places[0] if places else 0, position, [(out, "out", None)] if out is not None else [])
    (T, k), c, rows = shape, places[1], into[0]
    (ldx, ex), (ldy, ey) = x.stride(), out.stride()
    if (ex != 1 or ey != 1) and k > 1 or (T | k | c | rows) >> 31:
        _moe_refuse(dev, x, T, position, [(out, "out", None)])
    rc = lib().ckq_call_dev(_PACK_11(6, kind, x.data_ptr(), ldx if T > 1 else k, position.data_ptr(), out.data_ptr(), ldy if rows > 1 else k, T, c, rows, k, stream))
    if rc:
        check(rc, "ckq_moe_gather_dev")
    return out


def dev_moe_gather_f8(x, position, out=None):
    """The same in e4m3: (q [tokens * choices, k], scale); codes and scales of rows that have no slot as there."""
    if out is not None and _fast.gather_f8(x, position, *out) == 0:
        return out
    dev, stream = _i8_where()
    q, scale = out if out is not None else _f8_new(x, position.numel())
    shape, places, into = x.shape, position.shape, q.shape
    kind = _I8_TYPES.get(x.dtype)
    if (len(shape) != 2 or len(places) != 2 or len(into) != 2 or shape[0] != places[0] or into[1] != shape[1] or kind is None or q.dtype is not _F8 or position.dtype is not _I32
            or not position.is_contiguous() or not x.get_device() == position.get_device() == q.get_device() == scale.get_device() == dev):
        _f8_refuse(dev, [(q, "q", (into[0], shape[-1]), _F8)], [(scale, "scale", (into[0], -(-shape[-1] // 128)))]) if q.dtype is not _F8 or into[1:] != shape[1:] else None
        _moe_refuse(dev, x, places[0] if places else 0, position, [])
    (T, k), c, rows = shape, places[1], into[0]
    if (T | k | c | rows) >> 31:
        _i8_too_many(T, k, c, rows)
    lds = _f8_side(scale, rows, -(-k // 128))
    (ldx, ex), (ldq, eq) = x.stride(), q.stride()
    if (ex != 1 or eq != 1) and k > 1 or not lds:
        _f8_refuse(dev, [(x, "x", shape, None), (q, "q", into, _F8)], [(scale, "scale", (rows, -(-k // 128)))])
    rc = lib().ckq_call_dev(_PACK_13(7, kind, x.data_ptr(), ldx if T > 1 else k, position.data_ptr(), q.data_ptr(), ldq if rows > 1 else k, scale.data_ptr(), lds, T, c, rows, k, stream))
    if rc:
        check(rc, "ckq_moe_gather_f8_dev")
    return q, scale


def dev_moe_combine(y, position, weights=None, out=None):
    """out[t] = sum over j of weights[t][j] * y[position[t][j]]: [tokens, k].  Without weights (ones) the gradient of dev_moe_gather."""
    if out is not None and _fast.combine(y, position, weights, out) == 0:
        return out
    dev, stream = _i8_where()
    shape, places, t = y.shape, position.shape, y.dtype
    if out is None and len(shape) == len(places) == 2:
        out = _torch.empty(places[0], shape[1], dtype=t, device=y.device)
    into, kind = out.shape if out is not None else (), _I8_TYPES.get(t)
    if (len(shape) != 2 or len(places) != 2 or into != (places[0], shape[1]) or kind is None or out.dtype is not t or position.dtype is not _I32
            or not position.is_contiguous() or not y.get_device() == position.get_device() == out.get_device() == dev
            or weights is not None and (weights.dtype is not _F32 or weights.shape != places or not weights.is_contiguous() or weights.get_device() != dev)):
        _moe_refuse(dev, y, None, position, [(out, "out", places[0] if places else 0)] if out is not None else [], [(weights, "weights")] if weights is not None else ())
    (rows, k), (T, c) = shape, places
    (ldy, ey), (ldo, eo) = y.stride(), out.stride()
    if (ey != 1 or eo != 1) and k > 1 or (T | k | c | rows) >> 31:
        _moe_refuse(dev, y, None, position, [(out, "out", T)])
    rc = lib().ckq_call_dev(_PACK_12(8, kind, y.data_ptr(), ldy if rows > 1 else k, position.data_ptr(), weights.data_ptr() if weights is not None else 0, out.data_ptr(),
                                   ldo if T > 1 else k, T, c, rows, k, stream))
    if rc:
        check(rc, "ckq_moe_combine_dev")
    return out


def dev_moe_combine_backward(dout, y, position, weights, out=None):
    """Of dout [tokens, k], the gradient of dev_moe_combine's result: (dy, of y's shape, dweights float32 [tokens, choices]).  Rows of dy that have no slot stay as they
    are in `out`, where dy may be y, and are zeros, their gradient, without it."""
    if out is not None and _fast.backward(dout, y, position, weights, *out) == 0:
        return out
    dev, stream = _i8_where()
    made = out is None
    if made:
        out = _torch.empty_strided(y.shape, y.stride(), dtype=y.dtype, device=y.device), _torch.empty(position.shape, dtype=_F32, device=y.device)
    dy, dw = out
    shape, places, of_y, t = dout.shape, position.shape, y.shape, dout.dtype
    kind = _I8_TYPES.get(t)
    if (len(shape) != 2 or len(places) != 2 or len(of_y) != 2 or shape[0] != places[0] or of_y[1] != shape[1] or dy.shape != of_y or kind is None or not y.dtype is dy.dtype is t
            or position.dtype is not _I32 or not weights.dtype is dw.dtype is _F32 or weights.shape != places or dw.shape != places
            or not (position.is_contiguous() and weights.is_contiguous() and dw.is_contiguous())
            or not dout.get_device() == y.get_device() == dy.get_device() == position.get_device() == weights.get_device() == dw.get_device() == dev):
        _moe_refuse(dev, dout, places[0] if places else 0, position, [(y, "y", None), (dy, "dy", of_y[0] if of_y else 0)], [(weights, "weights"), (dw, "dweights")])
    (T, k), c, rows = shape, places[1], of_y[0]
    (ldd, ed), (ldy, ey), (ldg, eg) = dout.stride(), y.stride(), dy.stride()
    if (ed != 1 or ey != 1 or eg != 1) and k > 1 or (T | k | c | rows) >> 31:
        _moe_refuse(dev, dout, T, position, [(y, "y", None), (dy, "dy", rows)])
    if rows == 1:
        ldy = ldg = k
    if made:
        dy.zero_()
    rc = lib().ckq_call_dev(_PACK_15(9, kind, dout.data_ptr(), ldd if T > 1 else k, y.data_ptr(), ldy, position.data_ptr(), weights.data_ptr(), dy.data_ptr(), ldg,
                                            dw.data_ptr(), T, c, rows, k, stream))
    if rc:
        check(rc, "ckq_moe_combine_backward_dev")
    return dy, dw


def dev_subblock_dots(fmt, W_t, x_t, M, K):
    import torch
    per = (K // 16) if fmt == "q6_k" else (K // 32)
    out = torch.zeros(M * per, dtype=torch.int32, device=W_t.device)
    check(dump_lib().ckq_subblock_dots_dev(FMT[fmt], _dp(out), _dp(W_t), _dp(x_t), M, K, _stream()),
          "ckq_subblock_dots_dev")
    return out.view(M, per)


def dev_subblock_dots_tokens(fmt, W_t, X_t, M, K, ntok):
    """Raw integer sub-block dots of every (token, row), from the instantiation of
    the streaming kernel a matmul of this shape and token count runs: [ntok, M, K/sub]."""
    import torch
    per = (K // 16) if fmt == "q6_k" else (K // 32)
    out = torch.zeros(ntok * M * per, dtype=torch.int32, device=W_t.device)
    check(dump_lib().ckq_subblock_dots_tokens_dev(FMT[fmt], _dp(out), _dp(W_t), _dp(X_t), M, K, ntok, _stream()),
          "ckq_subblock_dots_tokens_dev")
    return out.view(ntok, M, per)


def dev_subblock_dots_group(fmt, W_ts, X_ts, rows, K, ntok):
    """The same dump from ONE grouped launch over the problems (W_ts[g], X_ts[g],
    rows[g]): [n, ntok, max(rows), K/sub]; rows beyond rows[g] stay zero."""
    import torch
    n, per, mx = len(W_ts), (K // 16) if fmt == "q6_k" else (K // 32), max(rows)
    out = torch.zeros(n * ntok * mx * per, dtype=torch.int32, device=W_ts[0].device)
    Wp = (_vp * n)(*[w.data_ptr() for w in W_ts])
    Xp = (_vp * n)(*[x.data_ptr() for x in X_ts])
    rp = (ctypes.c_int * n)(*rows)
    check(dump_lib().ckq_subblock_dots_group_dev(FMT[fmt], n, _dp(out), ctypes.cast(Wp, _vp), ctypes.cast(Xp, _vp),
                                            ctypes.cast(rp, _vp), K, ntok, _stream()), "ckq_subblock_dots_group_dev")
    return out.view(n, ntok, mx, per)


def dev_gemm_block_sums(fmt, A_t, B_t, bias_t, M, N, K):
    """The matrix-core GEMM with its integer block sums: (C [M,N], sums [M,N,nblk,per])."""
    import torch
    nblk, per = (K // 32, 1) if fmt == "q8_0" else (K // 256, 1 if fmt == "q6_k" else 2)
    c = torch.empty(M * N, dtype=torch.float32, device=B_t.device)
    sums = torch.zeros(M * N * nblk * per, dtype=torch.int32, device=B_t.device)
    check(dump_lib().ckq_gemm_block_sums_dev(FMT[fmt], _dp(A_t), _dp(B_t), _dp(bias_t), _dp(c), _dp(sums), M, N, K, _stream()),
          "ckq_gemm_block_sums_dev")
    return c.view(M, N), sums.view(M, N, nblk, per)


def dev_matmul_sequence(ops, repeat=1):
    """ops: list of matmul entries (fmt, A_t, B_t, bias_t, C_t, M, N, K[, ldc]) and producer
    entries (step, A_t, B_t or None, C_t, M, K[, ld[, eps]]) with step one of
    "quantize_q8_k", "quantize_q8_0", "rmsnorm_q8_k", "swiglu_q8_k"; enqueued
    back-to-back `repeat` times by one C call (no Python between launches)."""
    arr = (MatmulOp * len(ops))()
    for i, op in enumerate(ops):
        if op[0] in STEP:
            step, A_t, B_t, C_t, M, K = op[:6]
            ld = op[6] if len(op) > 6 else 0
            eps = op[7] if len(op) > 7 else 0.0
            arr[i] = MatmulOp(STEP[step], M, 0, K, ld, A_t.data_ptr(), B_t.data_ptr() if B_t is not None else None,
                              None, C_t.data_ptr(), eps)
        else:
            fmt, A_t, B_t, bias_t, C_t, M, N, K = op[:8]
            ldc = op[8] if len(op) > 8 else N
            arr[i] = MatmulOp(fmt_tag(fmt), M, N, K, ldc, A_t.data_ptr(), B_t.data_ptr(),
                              bias_t.data_ptr() if bias_t is not None else None, C_t.data_ptr(), 0.0)
    check(lib().ckq_matmul_sequence_dev(ctypes.cast(arr, _vp), len(ops), repeat, _stream()), "ckq_matmul_sequence_dev")
