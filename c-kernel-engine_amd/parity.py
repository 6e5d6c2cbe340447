"""NumPy / torch front-ends over the C ABI, shaped like the calls the
reference's parity scripts make (ctypes into ck_test_* and the kernel symbols,
e.g. unittest/test_q4_k_q8_k_matvec.py:93-132, unittest/test_parallel_gemv.py:112-170).

Host functions take NumPy arrays and go through the drop-in (host-pointer)
symbols; `dev_*` functions take torch CUDA tensors and go through the
device-resident entry points on torch's current stream."""
import ctypes

import numpy as np

from .api import BLOCK_ELEMS, FMT, STEP, CkqError, MatmulOp, check, dump_lib, lib, row_bytes

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

_torch, _INT8, _F32, _started, _device, _raw_stream, _I8_TYPES = None, None, None, None, None, None, {}


def _i8_torch():
    """torch, and what every call needs of it, once: an import statement in each call costs it 0.3 us a time, a chain of names 0.05."""
    global _torch, _INT8, _F32, _started, _device, _raw_stream
    import torch
    _INT8, _F32 = torch.int8, torch.float32
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
