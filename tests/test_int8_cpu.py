"""CPU checks of the int8 entry points: what they refuse, before anything touches a device, and with which code.  No
kernel is launched here."""
import ctypes
import importlib
import os
import re
import subprocess

import pytest

ckq = importlib.import_module("c-kernel-engine_amd")
EINVAL, EFORMAT, EROWS = -1, -3, -8
F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(ckq.lib_path()):
        ckq.build()
    return ckq.lib()


@pytest.fixture(autouse=True)
def _kernel_by_shape(L):
    yield
    L.ckq_launch_set_i8_kernel(-1)


P = ctypes.c_void_p(4096)


def odd(n):
    return ctypes.c_void_p(4096 + n)


def test_quantize_and_dequantize_refusals(L):
    def quantize(t=BF16, x=P, ldx=64, q=P, ldq=64, scale=P, rows=2, k=64):
        return L.ckq_quantize_i8_dev(t, x, ldx, q, ldq, scale, rows, k, None)

    def dequantize(q=P, ldq=64, scale=P, t=BF16, y=P, ldy=64, rows=2, k=64):
        return L.ckq_dequantize_i8_dev(q, ldq, scale, t, y, ldy, rows, k, None)

    for bad in ({"x": None}, {"q": None}, {"scale": None}, {"rows": 0}, {"rows": -1}, {"k": 0}, {"k": -5}, {"ldx": 63}, {"ldq": 63}):
        assert quantize(**bad) == EINVAL, bad
    for bad in ({"q": None}, {"y": None}, {"scale": None}, {"rows": 0}, {"k": 0}, {"ldq": 63}, {"ldy": 63}):
        assert dequantize(**bad) == EINVAL, bad
    for t in (-1, 3, 7, 9, 13):
        assert quantize(t=t) == EFORMAT and dequantize(t=t) == EFORMAT
    assert quantize(x=odd(1)) == EROWS and quantize(scale=odd(2)) == EROWS
    assert quantize(t=F32, x=odd(2)) == EROWS
    assert dequantize(y=odd(1)) == EROWS and dequantize(t=F32, y=odd(2)) == EROWS and dequantize(scale=odd(3)) == EROWS


def test_rmsnorm_refusals(L):
    def norm(t=F16, x=P, ldx=64, residual=P, out=P, ldr=64, gamma=P, eps=1e-5, q=P, ldq=64, scale=P, rows=2, k=64):
        return L.ckq_rmsnorm_i8_dev(t, x, ldx, residual, out, ldr, gamma, ctypes.c_float(eps), q, ldq, scale, rows, k, None)

    for bad in ({"x": None}, {"gamma": None}, {"q": None}, {"scale": None}, {"residual": None}, {"out": None}, {"rows": 0}, {"k": 0},
                {"ldx": 63}, {"ldr": 63}, {"ldq": 63}, {"eps": -1e-5}, {"eps": float("nan")}, {"eps": float("inf")}):
        assert norm(**bad) == EINVAL, bad
    assert norm(t=5) == EFORMAT
    for bad in ({"x": odd(1)}, {"residual": odd(1)}, {"out": odd(1)}, {"gamma": odd(2)}, {"scale": odd(2)}, {"t": F32, "residual": odd(2)}):
        assert norm(**bad) == EROWS, bad


def test_rmsnorm_refuses_a_sum_that_lies_across_the_rows_of_x(L):
    """`sum` may be x only with one pitch, where each row lies in its own place."""
    for ldx, ldr in ((64, 80), (128, 64)):
        assert L.ckq_rmsnorm_i8_dev(F16, P, ldx, odd(1 << 20), P, ldr, P, ctypes.c_float(1e-5), P, 64, P, 2, 64, None) == EINVAL


def test_swiglu_refusals(L):
    def swiglu(t=BF16, gate=P, up=P, ld=128, q=P, ldq=64, scale=P, rows=2, k=64):
        return L.ckq_swiglu_i8_dev(t, gate, up, ld, q, ldq, scale, rows, k, None)

    for bad in ({"gate": None}, {"up": None}, {"q": None}, {"scale": None}, {"rows": 0}, {"k": 0}, {"ld": 63}, {"ldq": 63}):
        assert swiglu(**bad) == EINVAL, bad
    assert swiglu(t=4) == EFORMAT
    for bad in ({"gate": odd(1)}, {"up": odd(1)}, {"scale": odd(1)}, {"t": F32, "up": odd(2)}):
        assert swiglu(**bad) == EROWS, bad


def test_matmul_refusals(L):
    def gemm(a=P, lda=64, sa=P, b=P, ldb=64, sb=P, bias=P, t=BF16, c=P, ldc=32, M=2, N=32, K=50):
        return L.ckq_gemm_nt_i8_dev(a, lda, sa, b, ldb, sb, bias, t, c, ldc, M, N, K, None)

    for bad in ({"a": None}, {"sa": None}, {"b": None}, {"sb": None}, {"c": None}, {"M": 0}, {"N": 0}, {"K": 0}, {"M": -1}, {"K": 65},
                {"lda": 48}, {"ldb": 48}, {"ldc": 31}):
        assert gemm(**bad) == EINVAL, bad
    assert gemm(t=3) == EFORMAT and gemm(t=-1) == EFORMAT
    long = {"lda": 131072, "ldb": 131072}
    for bad in ({"a": odd(8)}, {"b": odd(4)}, {"lda": 72}, {"ldb": 50}, {"lda": (1 << 22) + 16}, {"ldb": 1 << 30}, {"K": 131072, **long},
                {"c": odd(1)}, {"t": F32, "c": odd(2)}, {"sa": odd(2)}, {"sb": odd(1)}, {"bias": odd(3)}):
        assert gemm(**bad) == EROWS, bad
    assert b"16 bytes" in L.ckq_error_string(EROWS)


def test_front_ends_refuse_what_a_pointer_cannot_tell():
    import torch
    par, err = ckq.parity, ckq.CkqError
    x = torch.zeros(3, 32)
    with pytest.raises(err, match="not on the current device"):
        par.dev_quantize_i8(x)
    with pytest.raises(err, match="shape"):
        par.dev_quantize_i8(x[0])
    with pytest.raises(err):
        par.dev_rmsnorm_i8(x, torch.ones(32))
    with pytest.raises(err):
        par.dev_gemm_nt_i8(torch.zeros(2, 32, dtype=torch.uint8), x[0], x, x[0])
    assert par.empty_i8(3, 33, device="cpu").shape == (3, 33) and par.empty_i8(3, 33, device="cpu").stride() == (48, 1)


def test_front_ends_refuse_sizes_beyond_31_bits(monkeypatch):
    """ctypes passes the lowest 32 bits of an int: 2^32 + 16 rows would be 16.  Memory that nothing touches, and a library that nothing reaches."""
    import torch
    par, err = ckq.parity, ckq.CkqError
    if torch.cuda.is_available():
        pytest.skip("the memory of a host without a device is meant")

    class Library:
        def __getattr__(self, name):
            return lambda *a: 0
    monkeypatch.setattr(par, "lib", Library)
    monkeypatch.setattr(par, "_i8_where", lambda: (-1, None))            # the device of host tensors
    par._i8_torch()
    f, q = torch.zeros(64), torch.zeros(64, dtype=torch.int8)
    assert par.dev_quantize_i8(f.view(4, 16))[0].shape == (4, 16)        # sizes as they should be get through
    for shape in (((1 << 32) + 16, 1), (1, (1 << 32) + 16), (1 << 31, 1), (1, 1 << 31)):
        rows, k = shape
        x, y = torch.empty(shape, dtype=torch.bfloat16), torch.empty(shape, dtype=torch.int8)
        out = (y, torch.empty(rows))
        gamma = torch.empty(k)
        for call in (lambda: par.dev_quantize_i8(x, out=out), lambda: par.dev_dequantize_i8(*out, out=x), lambda: par.dev_swiglu_i8(x, x, out=out),
                     lambda: par.dev_rmsnorm_i8(x, gamma, out=out)):
            with pytest.raises(err, match="2\\^31"):
                call()
    many = torch.empty((1 << 32) + 32, dtype=torch.int8)
    far, few, scales = many.as_strided(((1 << 32) + 16, 16), (1, 1)), q.view(4, 16), torch.empty((1 << 32) + 16)
    for call in (lambda: par.dev_gemm_nt_i8(far, scales, few, f[:4], out=scales), lambda: par.dev_gemm_nt_i8(few, f[:4], far, scales, out=scales)):
        with pytest.raises(err, match="2\\^31"):
            call()


def test_kernel_of_a_matmul(L):
    """One or two tokens stream, four if rows are short; then the cheapest by the estimate, which has to be one of the kernels at every size."""
    assert all(L.ckq_launch_i8_kernel(M, N, K) == 12 for N in (1, 5000, 151936) for M, K in ((1, 1), (1, 131071), (2, 896), (2, 131071), (3, 1024), (4, 1)))
    assert all(L.ckq_launch_i8_kernel(M, N, 1025) < 12 for M in (3, 4) for N in (1, 5000, 151936))
    seen = {L.ckq_launch_i8_kernel(M, N, K) for M in (5, 12, 16, 17, 40, 64, 100, 128, 200, 333, 512, 800, 1024, 1500, 2048, 5000) for N in (1, 64, 200, 512, 896, 1001, 1504, 2048, 3500, 4096, 4864, 8000, 11008, 17000, 28000, 151936)
            for K in (1, 64, 200, 512, 896, 1500, 2048, 4096, 4847, 11008, 131071)}
    assert seen == set(range(12)), seen
    assert L.ckq_launch_i8_kernel(2048, 11008, 4096) == 11          # 344 tiles of 256 x 256: 256 of them, the rest smaller
    assert L.ckq_launch_i8_kernel(2048, 8192, 4096) == 0            # one round of them
    assert L.ckq_launch_i8_kernel(1 << 22, 1 << 22, 64) in range(12)
    for forced in range(13):
        L.ckq_launch_set_i8_kernel(forced)
        assert L.ckq_launch_i8_kernel(2048, 11008, 4096) == (forced if forced != 12 else 11)
    L.ckq_launch_set_i8_kernel(-1)


def test_exported_launches_are_declared(L):
    """What the library exports of its kernels' interface stands in ckq_launch.h, the switches of the tests too."""
    text = open(os.path.join(ckq.api.CSRC, "ckq_launch.h")).read()
    names = subprocess.run(["nm", "-D", "--defined-only", ckq.lib_path()], capture_output=True, text=True, check=True).stdout.split()
    launches = {n for n in names if n.startswith("ckq_launch_")}
    assert len(launches) > 20
    assert not {n for n in launches if not re.search(r"\b%s\(" % n, text)}
