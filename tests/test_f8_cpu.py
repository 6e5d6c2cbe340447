"""CPU checks of the entry points of e4m3 rows and of tokens sorted by expert: what they refuse, before anything touches a device, and with
which code.  No kernel is launched here."""
import ctypes
import importlib
import os

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
    L.ckq_launch_set_f8_kernel(-1)


P = ctypes.c_void_p(4096)


def odd(n):
    return ctypes.c_void_p(4096 + n)


def refuses(call, invalid, format_, rows):
    for bad in invalid:
        assert call(**bad) == EINVAL, bad
    for bad in format_:
        assert call(**bad) == EFORMAT, bad
    for bad in rows:
        assert call(**bad) == EROWS, bad


TYPES_THAT_ARE_NONE = [{"t": t} for t in (-1, 3, 7, 9, 13)]


def test_rows_refusals(L):
    def quantize(t=BF16, x=P, ldx=64, q=P, ldq=64, scale=P, lds=2, rows=2, k=64):
        return L.ckq_quantize_f8_dev(t, x, ldx, q, ldq, scale, lds, rows, k, None)

    def dequantize(q=P, ldq=64, scale=P, lds=2, t=BF16, y=P, ldy=64, rows=2, k=64):
        return L.ckq_dequantize_f8_dev(q, ldq, scale, lds, t, y, ldy, rows, k, None)

    def swiglu(t=BF16, gate=P, up=P, ld=128, q=P, ldq=64, scale=P, lds=2, rows=2, k=64):
        return L.ckq_swiglu_f8_dev(t, gate, up, ld, q, ldq, scale, lds, rows, k, None)

    sizes = [{"rows": 0}, {"rows": -1}, {"k": 0}, {"k": -5}, {"lds": 1}, {"ldq": 63}, {"q": None}, {"scale": None}]
    refuses(quantize, sizes + [{"x": None}, {"ldx": 63}], TYPES_THAT_ARE_NONE, [{"x": odd(1)}, {"scale": odd(2)}, {"t": F32, "x": odd(2)}])
    refuses(dequantize, sizes + [{"y": None}, {"ldy": 63}], TYPES_THAT_ARE_NONE, [{"y": odd(1)}, {"scale": odd(2)}, {"t": F32, "y": odd(2)}])
    refuses(swiglu, sizes + [{"gate": None}, {"up": None}, {"ld": 63}], TYPES_THAT_ARE_NONE, [{"gate": odd(1)}, {"up": odd(1)}, {"scale": odd(1)}, {"t": F32, "up": odd(2)}])


def test_matmul_refusals(L):
    def gemm(a=P, lda=64, sa=P, ldsa=2, b=P, ldb=64, sb=P, ldsb=1, bias=P, t=BF16, c=P, ldc=32, M=2, N=32, K=50):
        return L.ckq_gemm_nt_f8_dev(a, lda, sa, ldsa, b, ldb, sb, ldsb, bias, t, c, ldc, M, N, K, None)

    def experts(a=P, lda=64, sa=P, ldsa=2, b=P, ldb=64, eb=2048, sb=P, ldsb=1, esb=1, bias=P, o=P, E=3, t=BF16, c=P, ldc=32, M=2, N=32, K=50):
        return L.ckq_gemm_nt_f8_experts_dev(a, lda, sa, ldsa, b, ldb, eb, sb, ldsb, esb, bias, o, E, t, c, ldc, M, N, K, None)

    invalid = [{"a": None}, {"sa": None}, {"b": None}, {"sb": None}, {"c": None}, {"M": 0}, {"N": 0}, {"K": 0}, {"M": -1}, {"K": 65}, {"lda": 48}, {"ldb": 48}, {"ldc": 31}, {"ldsa": 1},
               {"ldsb": 0}, {"K": 129, "lda": 144, "ldb": 144}]
    rows = [{"a": odd(8)}, {"b": odd(4)}, {"lda": 72}, {"ldb": 50}, {"lda": (1 << 22) + 16}, {"ldb": 1 << 30}, {"c": odd(1)}, {"t": F32, "c": odd(2)}, {"sa": odd(2)}, {"sb": odd(1)}, {"bias": odd(3)}]
    refuses(gemm, invalid, TYPES_THAT_ARE_NONE, rows)
    refuses(experts, invalid + [{"o": None}, {"E": 0}, {"E": -2}, {"E": 65536}, {"eb": -16}, {"esb": -1}], TYPES_THAT_ARE_NONE, rows + [{"eb": 2040}, {"o": odd(2)}])
    assert b"16 bytes" in L.ckq_error_string(EROWS)


def test_sort_and_rows_there_and_back_refusals(L):
    def sort(ids=P, T=2, c=2, E=3, offsets=P, order=P, position=P):
        return L.ckq_moe_sort_dev(ids, T, c, E, offsets, order, position, None)

    refuses(sort, [{"ids": None}, {"offsets": None}, {"order": None}, {"position": None}, {"T": 0}, {"c": 0}, {"E": 0}, {"T": -1}, {"E": 65536}, {"T": 1 << 20, "c": 1025}, {"T": (1 << 31) - 1, "c": (1 << 31) - 1}],
            [], [{"ids": odd(1)}, {"offsets": odd(2)}, {"order": odd(2)}, {"position": odd(2)}])

    def gather(t=BF16, x=P, ldx=64, pos=P, y=P, ldy=64, T=2, c=2, rows=4, k=64):
        return L.ckq_moe_gather_dev(t, x, ldx, pos, y, ldy, T, c, rows, k, None)

    def gather_f8(t=BF16, x=P, ldx=64, pos=P, q=P, ldq=64, scale=P, lds=4, T=2, c=2, rows=4, k=64):
        return L.ckq_moe_gather_f8_dev(t, x, ldx, pos, q, ldq, scale, lds, T, c, rows, k, None)

    def combine(t=BF16, y=P, ldy=64, pos=P, w=P, out=P, ldo=64, T=2, c=2, rows=4, k=64):
        return L.ckq_moe_combine_dev(t, y, ldy, pos, w, out, ldo, T, c, rows, k, None)

    def backward(t=BF16, dout=P, ldd=64, y=P, ldy=64, pos=P, w=P, dy=P, lddy=64, dw=P, T=2, c=2, rows=4, k=64):
        return L.ckq_moe_combine_backward_dev(t, dout, ldd, y, ldy, pos, w, dy, lddy, dw, T, c, rows, k, None)

    sizes = [{"T": 0}, {"c": 0}, {"rows": 0}, {"k": 0}, {"T": -1}, {"k": -1}, {"pos": None}]
    refuses(gather, sizes + [{"x": None}, {"y": None}, {"ldx": 63}, {"ldy": 63}], TYPES_THAT_ARE_NONE, [{"x": odd(1)}, {"y": odd(1)}, {"pos": odd(2)}, {"t": F32, "y": odd(2)}])
    refuses(gather_f8, sizes + [{"x": None}, {"q": None}, {"scale": None}, {"ldx": 63}, {"ldq": 63}, {"lds": 3}], TYPES_THAT_ARE_NONE, [{"x": odd(1)}, {"scale": odd(1)}, {"pos": odd(2)}])
    refuses(combine, sizes + [{"y": None}, {"out": None}, {"ldy": 63}, {"ldo": 63}], TYPES_THAT_ARE_NONE, [{"y": odd(1)}, {"out": odd(1)}, {"pos": odd(2)}, {"w": odd(2)}])
    refuses(backward, sizes + [{"dout": None}, {"y": None}, {"w": None}, {"dy": None}, {"dw": None}, {"ldd": 63}, {"ldy": 63}, {"lddy": 63}, {"lddy": 80}], TYPES_THAT_ARE_NONE,
            [{"dout": odd(1)}, {"y": odd(1)}, {"dy": odd(1)}, {"pos": odd(2)}, {"w": odd(2)}, {"dw": odd(1)}])


def test_any_call_by_its_number(L):
    """ckq_call_dev takes each entry point's arguments in its order: what that refuses, with its code."""
    import struct
    call = lambda *a: L.ckq_call_dev(struct.pack("%dq" % len(a), *a))
    p, n = 4096, 0
    good = [(BF16, p, 64, p, 64, p, 2, 2, 64, n), (p, 64, p, 2, BF16, p, 64, 2, 64, n), (BF16, p, p, 64, p, 64, p, 2, 2, 64, n), (p, 64, p, 2, p, 64, p, 1, p, BF16, p, 32, 2, 32, 64, n),
            (p, 64, p, 2, p, 64, 2048, p, 1, 1, p, p, 3, BF16, p, 32, 2, 32, 64, n), (p, 2, 2, 3, p, p, p, n), (BF16, p, 64, p, p, 64, 2, 2, 4, 64, n), (BF16, p, 64, p, p, 64, p, 4, 2, 2, 4, 64, n),
            (BF16, p, 64, p, p, p, 64, 2, 2, 4, 64, n), (BF16, p, 64, p, 64, p, p, p, 64, p, 2, 2, 4, 64, n)]
    pointers = [(1, 3, 5), (0, 2, 5), (1, 2, 4, 6), (0, 2, 4, 6, 10), (0, 2, 4, 7, 11, 14), (0, 4, 5, 6), (1, 3, 4), (1, 3, 4, 6), (1, 3, 5), (1, 3, 5, 6, 7, 9)]
    types = [0, 4, 0, 9, 13, None, 0, 0, 0, 0]
    for which, (a, at, t) in enumerate(zip(good, pointers, types)):
        for i in at:
            assert call(which, *a[:i], 0, *a[i + 1:]) == EINVAL, (which, i)
        if t is not None:
            assert call(which, *a[:t], 5, *a[t + 1:]) == EFORMAT
    assert call(-1, *good[4]) == EINVAL and call(10, *good[4]) == EINVAL and L.ckq_call_dev(None) == EINVAL


def test_a_call_by_its_number_refuses_what_no_int_holds(L):
    """64 bits come in and 32 go on: 2^32 + 2 rows would be 2.  Each size and type alone, in calls that are refused for their type if they get that far."""
    import struct
    call = lambda *a: L.ckq_call_dev(struct.pack("%dq" % len(a), *a))
    p, n, far = 4096, 0, 1 << 40                               # pitches and pointers are 64 bits wide
    bad = 5                                                    # no type of a row
    calls = [(bad, p, far, p, far, p, far, 2, 64, n), (p, far, p, far, bad, p, far, 2, 64, n), (bad, p, p, far, p, far, p, far, 2, 64, n),
             (p, far, p, far, p, far, p, far, p, bad, p, far, 2, 32, 64, n), (p, far, p, far, p, far, 2048, p, far, 1, p, p, 3, bad, p, far, 2, 32, 64, n), None,
             (bad, p, far, p, p, far, 2, 2, 4, 64, n), (bad, p, far, p, p, far, p, far, 2, 2, 4, 64, n), (bad, p, far, p, p, p, far, 2, 2, 4, 64, n), (bad, p, far, p, far, p, p, p, far, p, 2, 2, 4, 64, n)]
    sizes = [(7, 8), (7, 8), (8, 9), (12, 13, 14), (12, 16, 17, 18), (), (6, 7, 8, 9), (8, 9, 10, 11), (7, 8, 9, 10), (10, 11, 12, 13)]
    for which, (a, at) in enumerate(zip(calls, sizes)):
        if a is None:
            continue
        assert call(which, *a) == EFORMAT
        for i in (*at, a.index(bad)):
            for add in (1 << 32, 1 << 31, -(1 << 32), 1 << 62):
                assert call(which, *a[:i], a[i] + add, *a[i + 1:]) == EINVAL, (which, i, add)
    sort = (p + 2, 2, 2, 3, p, p, p, n)                        # refused for its pointer
    assert call(5, *sort) == EROWS
    for i in (1, 2, 3):
        assert call(5, *sort[:i], sort[i] + (1 << 32), *sort[i + 1:]) == EINVAL


def test_front_ends_refuse_what_a_pointer_cannot_tell():
    import torch
    par, err = ckq.parity, ckq.CkqError
    x, pos = torch.zeros(3, 32), torch.zeros(3, 2, dtype=torch.int32)
    if not torch.cuda.is_available():
        for call in (lambda: par.dev_quantize_f8(x), lambda: par.dev_moe_sort(pos, 4), lambda: par.dev_moe_gather(x, pos), lambda: par.dev_moe_combine(x, pos)):
            with pytest.raises(err, match="not on the current device"):
                call()
    for call in (lambda: par.dev_quantize_f8(x[0]), lambda: par.dev_swiglu_f8(x[0], x[0]), lambda: par.dev_moe_sort(pos[0], 4), lambda: par.dev_moe_gather(x, pos[0]),
                 lambda: par.dev_moe_gather_f8(x[0], pos), lambda: par.dev_gemm_nt_f8_experts(x, x, x, x, pos)):
        with pytest.raises(err, match="shape"):
            call()
    q, s = par.empty_f8(3, 200, device="cpu")
    assert q.shape == (3, 200) and q.stride() == (208, 1) and s.shape == (3, 2) and s.stride() == (1, 3) and q.dtype == torch.float8_e4m3fn


def without_module(par):
    none = par._Fast()
    none.absent = True
    return none


def test_the_module_that_reads_tensors_takes_none_of_the_host(L):
    """It is there, and whatever it is given that is not for it comes back untouched, as does a call of something that is no tensor."""
    import torch
    par = ckq.parity
    m = par._load_fast()
    names = ("quantize", "dequantize", "swiglu", "gemm", "experts", "sort", "gather", "gather_f8", "combine", "backward")
    assert os.path.exists(os.path.join(ckq.api.CSRC, "ckq_tensors.so")) and par._fast is m and all(hasattr(m, n) for n in names)
    x = torch.ones(3, 32)
    for n in names:
        for args in ((), (x,), (x,) * 7, (None,) * 7, (3, "a", 2.5, x, [x], None, x), (x.to_sparse(),) * 7, (x.to("meta"),) * 7):
            assert getattr(m, n)(*args) == -1000
    assert without_module(par).gemm(x) == -1000


def test_make_leaves_the_module_out_where_there_is_no_torch_and_builds_it_anew_for_another(tmp_path):
    """A compiler that only says that it was called; a Python without site packages, and one with another torch."""
    import shutil
    import subprocess
    import sys
    for f in ("Makefile", "ckq_tensors.cpp"):
        shutil.copy(os.path.join(ckq.api.CSRC, f), tmp_path)
    (tmp_path / "g++").write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\necho made > "$2"\n')
    (tmp_path / "g++").chmod(0o755)
    other = tmp_path / "other"
    (other / "torch" / "include" / "c10" / "hip").mkdir(parents=True)
    (other / "torch" / "include" / "c10" / "hip" / "HIPStream.h").write_text("")
    (other / "torch" / "__init__.py").write_text('__version__ = "0.1.2"\n')
    so, env = tmp_path / "ckq_tensors.so", dict(os.environ, PATH="%s:%s" % (tmp_path, os.environ["PATH"]))

    def make(python=sys.executable, **more):
        r = subprocess.run(["make", "-f", str(tmp_path / "Makefile"), "tensors", "PYTHON=" + python], env=dict(env, **more), capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return r.stdout

    assert "left out" in make(sys.executable + " -S") and not so.exists()
    make()
    assert so.read_text() == "made\n"
    so.write_text("kept\n")
    make()
    assert so.read_text() == "kept\n"                          # nothing has changed
    make(PYTHONPATH=str(other))
    assert so.read_text() == "made\n"
    assert "left out" in make(sys.executable + " -S") and not so.exists()          # none that is of neither


@pytest.mark.parametrize("what", ["cut short", "no library", "of another torch"])
def test_a_module_that_cannot_be_used_leaves_the_python_checks(L, monkeypatch, tmp_path, what):
    """Each call with `out` then goes the way that it has without the module."""
    import shutil
    import torch
    par = ckq.parity
    so, made = tmp_path / "ckq_tensors.so", os.path.join(ckq.api.CSRC, "ckq_tensors.so")
    if what == "cut short":
        so.write_bytes(open(made, "rb").read()[:50])
    elif what == "no library":
        so.write_text("not a library")
    else:
        shutil.copy(made, so)
        monkeypatch.setattr(torch, "__version__", "0.1.2")
    monkeypatch.setattr(par, "CSRC", str(tmp_path))
    monkeypatch.setattr(par, "_fast", par._Fast())
    x = torch.zeros(3, 32)
    with pytest.warns(UserWarning, match="built for" if what == "of another torch" else "is not used"):
        with pytest.raises(ckq.CkqError, match="not on the current device"):
            par.dev_quantize_f8(x, out=par.empty_f8(3, 32, device="cpu"))
    assert par._fast.absent
    with pytest.raises(ckq.CkqError, match="not on the current device"):        # and again, without another word
        par.dev_moe_gather(x, torch.zeros(3, 1, dtype=torch.int32), out=x)


def test_front_ends_refuse_sizes_beyond_31_bits(monkeypatch):
    """ctypes passes the lowest 32 bits of an int: 2^32 + 16 rows would be 16.  Memory that nothing touches, and a library that nothing reaches."""
    import torch
    par, err = ckq.parity, ckq.CkqError
    if torch.cuda.is_available():
        pytest.skip("the memory of a host without a device is meant")

    class Library:
        def __getattr__(self, name):
            return lambda *a: 0
    monkeypatch.setattr(par, "_fast", without_module(par))
    monkeypatch.setattr(par, "lib", Library)
    monkeypatch.setattr(par, "_i8_where", lambda: (-1, 0))               # the device of host tensors
    par._i8_torch()
    many = (1 << 32) + 16
    f, q, s = torch.empty(many, 1), torch.empty(many, 1, dtype=torch.float8_e4m3fn), torch.empty(1, many).t()
    assert par.dev_quantize_f8(torch.zeros(4, 16))[0].shape == (4, 16)   # sizes as they should be get through
    for call in (lambda: par.dev_quantize_f8(f, out=(q, s)), lambda: par.dev_dequantize_f8(q, s, out=f), lambda: par.dev_swiglu_f8(f, f, out=(q, s)),
                 lambda: par.dev_gemm_nt_f8(q, s, q[:2], torch.empty(1, 1), out=f.view(many, 1).expand(many, 2)),
                 lambda: par.dev_moe_sort(torch.empty(many, 1, dtype=torch.int32), 2), lambda: par.dev_moe_combine(f, torch.zeros(1, 1, dtype=torch.int32)),
                 lambda: par.dev_moe_gather_f8(f[:2], torch.zeros(2, 1, dtype=torch.int32), out=(q, s))):
        with pytest.raises(err, match="2\\^31"):
            call()


def test_kernel_of_a_matmul(L):
    """One token streams; fp32 results and experts stay on the fp16 instructions; every kernel has its sizes."""
    k = L.ckq_launch_f8_kernel
    assert all(k(t, 1, N, K, 0) == 16 for t in (F32, BF16, F16) for N in (1, 5000, 151936) for K in (1, 896, 131072))
    Ms, Ns, Ks = (2, 5, 12, 16, 17, 40, 64, 100, 128, 200, 333, 512, 800, 1024, 1500, 2048, 5000, 1 << 19), (1, 64, 200, 512, 896, 1001, 1504, 2048, 3500, 4096, 4864, 8000, 11008, 17000, 28000, 151936), \
        (1, 64, 200, 512, 896, 1500, 2048, 4096, 4847, 11008, 131071)
    seen = {t: {k(t, M, N, K, 0) for M in Ms for N in Ns for K in Ks} for t in (F32, BF16)}
    experts = {k(t, M, N, K, E) for t in (F32, F16) for M in Ms + (1,) for N in Ns for K in Ks for E in (1, 2, 8, 60, 256)}
    assert seen[F32] == set(range(9)) and experts <= set(range(9)) and seen[F32] | seen[BF16] | experts == set(range(16))
    assert k(F32, 1 << 22, 151936, 64, 0) == k(BF16, 1, 1 << 30, 64, 0) == k(BF16, 1 << 29, 4096, 64, 8) == -1          # in parts
    assert 0 <= k(F32, 1 << 29, 16, 64, 1 << 15) < 9
    assert k(BF16, 2048, 11008, 4096, 0) == 15                # 344 tiles of 256 x 256: 256 of them, the rest smaller
    assert k(BF16, 2048, 8192, 4096, 0) == 9                  # one round of them
    for forced in range(17):
        L.ckq_launch_set_f8_kernel(forced)
        assert k(BF16, 2048, 11008, 4096, 0) == (forced if forced != 16 else 15)
        assert k(BF16, 2048, 11008, 4096, 8) in ((forced,) if forced < 15 else range(9))
    L.ckq_launch_set_f8_kernel(-1)


def test_kernel_of_a_matmul_with_fp32_sums(L):
    """The fp32 result's choice, whatever the type and whichever kernel is forced on those that may have it."""
    k, wide = L.ckq_launch_f8_kernel, 256
    for M in (1, 2, 40, 300, 2048, 1 << 19):
        for N in (64, 1001, 11008):
            for K in (64, 4096):
                for E in (0, 8):
                    L.ckq_launch_set_f8_kernel(-1)
                    want = k(F32, M, N, K, E)
                    assert want < 9 or want == 16 and M == 1
                    for forced in (-1, *range(9, 16)):
                        L.ckq_launch_set_f8_kernel(forced)
                        assert k(BF16 | wide, M, N, K, E) == k(F16 | wide, M, N, K, E) == k(F32 | wide, M, N, K, E) == want
    L.ckq_launch_set_f8_kernel(3)
    assert k(BF16 | wide, 300, 1001, 4096, 0) == 3
    gemm = lambda t, b=P: L.ckq_gemm_nt_f8_dev(P, 64, P, 2, b, 64, P, 1, P, t, P, 32, 2, 32, 50, None)
    assert all(gemm(t | wide) == EFORMAT for t in (-1, 3, 7, 9)) and gemm(BF16 | wide, odd(4)) == EROWS and gemm(BF16 | 512) == EFORMAT
