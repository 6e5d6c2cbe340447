"""Rows in e4m3 with one scale for each 128 elements, and tokens sorted by expert, on the GPU against their definitions in 64 bits: quantizer
and rows read back, SwiGLU, the matmul and the one over experts, sort, gather, combine and their gradients, and all of them together.

What each result may be off follows from the operations that produce it.  U = 2^-24 is half a step of fp32 relative to the
value; a result of type T adds half a step of T."""
import importlib
import os
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ckq = importlib.import_module("c-kernel-engine_amd")
P = ckq.parity

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = 2.0 ** -100
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _lib():
    assert os.path.exists(ckq.lib_path()), "the HIP library has to be built"
    assert torch.cuda.is_available()
    assert ckq.lib().ckq_init() == 0
    yield
    torch.cuda.synchronize()


def normal(rows, k, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, k, generator=g, dtype=torch.float32) * std


def codes(rows, k, seed, pitch=None, rest=0x7F):
    """Random codes on the GPU; the bytes behind a row's last are `rest` (0x7F: a NaN)."""
    q = (normal(rows, k, seed) * 112).clamp(-448, 448).to(F8)
    pitch = pitch or -(-k // 16) * 16
    all_ = torch.full((rows, pitch), rest, dtype=torch.uint8)
    all_[:, :k] = q.view(torch.uint8)
    return all_.cuda().view(F8)[:, :k]


def side(rows, k, seed, extra=0):
    """Random scales [rows, groups], those of a group side by side."""
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(-(-k // 128), rows + extra, generator=g) + 0.5).cuda()[:, :rows].t()


def blocks(n, k, seed, *experts):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(*experts, -(-n // 128), -(-k // 128), generator=g) + 0.5).mul_(0.01).cuda()


def half_step(t):
    return torch.finfo(t).eps / 2


def rounding(t, v):
    """What rounding a value near v to the type t changes at most: half a step, which under the smallest normal number is that number's eps / 2 (the steps there
    are all the same)."""
    return half_step(t) * v.abs().clamp_min(torch.finfo(t).smallest_normal)


def pitched(x, extra, lead=0):
    """x on the GPU with rows `extra` elements further apart than they are long, the first `lead` elements into the memory."""
    rows, k = x.shape
    flat = torch.full((lead + rows * (k + extra) + 8,), 7.0, device="cuda").to(x.dtype)
    v = flat[lead:lead + rows * (k + extra)].view(rows, k + extra)[:, :k]
    v.copy_(x)
    return v


def values(q, scale):
    """What the codes stand for, in 64 bits on the CPU."""
    q, scale = q.cpu(), scale.cpu()
    return q.float().double() * scale.double().repeat_interleave(128, 1)[:, :q.shape[1]]


def block_values(b, sb):
    return b.cpu().float().double() * sb.cpu().double().repeat_interleave(128, 0)[:b.shape[0]].repeat_interleave(128, 1)[:, :b.shape[1]]


def e4m3(t):
    """The nearest code's value of float64, ties to even, and half the distance of the codes there."""
    step = np.ldexp(1.0, np.maximum(np.frexp(t)[1] - 1, -6) - 3)
    return np.rint(t / step) * step, step / 2


def grouped(v):
    """[rows, groups, 128] of a float64 array, zeros behind a row's last."""
    rows, k = v.shape
    out = np.zeros((rows, -(-k // 128) * 128))
    out[:, :k] = v
    return out.reshape(rows, -1, 128)


ROWS_K = [(1, 1), (2, 2), (3, 7), (5, 8), (1, 127), (4, 128), (3, 129), (9, 64), (7, 500), (33, 130), (31, 256), (67, 896), (2, 2048), (3, 2049), (70, 1001), (2, 4863), (300, 520), (2, 16391), (1, 40003)]


# ---- quantizer ----------------------------------------------------------------------

def expected_codes(x):
    """Quantizer's codes and scales of rows of floats, operation by operation: a' and 448 * 2^-e are exact, the product is exact or rounded to fp32, the
    quotient of two fp32 numbers in 64 bits and then in 32 is the correctly rounded one."""
    g = grouped(x.double().numpy())
    a = np.maximum(np.abs(g).max(2), TINY)
    e = np.frexp(a)[1] - 1
    n = np.ldexp(g * 448, -e[:, :, None]).astype(np.float32)
    t = (n.astype(np.float64) / np.ldexp(a, -e)[:, :, None]).astype(np.float32)
    q = e4m3(t.astype(np.float64))[0].reshape(x.shape[0], -1)[:, :x.shape[1]]
    return q, (a.astype(np.float32) / np.float32(448)).astype(np.float32)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k", ROWS_K)
def test_quantize(t, rows, k):
    x = normal(rows, k, 100 * rows + k, 3.0).to(TYPES[t])
    q, s = P.dev_quantize_f8(x.cuda())
    assert q.dtype == F8 and q.shape == (rows, k) and q.stride(0) % 16 == 0 and s.shape == (rows, -(-k // 128)) and (rows == 1 or s.stride(0) == 1)
    wq, ws = expected_codes(x)
    assert np.array_equal(q.cpu().float().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws)


@pytest.mark.parametrize("t", TYPES)
def test_quantize_strides_alignment_and_bytes_beside(t):
    for rows, k, extra, lead in ((5, 100, 3, 1), (3, 515, 1, 3), (6, 8, 1, 1), (40, 300, 5, 5), (2, 4096, 5, 5), (4, 9000, 7, 1)):
        x = normal(rows, k, k).to(TYPES[t])
        xd = pitched(x, extra, lead)
        base = torch.full((3 + (rows + 1) * (k + 5),), 77, dtype=torch.uint8, device="cuda")
        q = base[3:3 + rows * (k + 5)].view(rows, k + 5)[:, :k].view(F8)
        groups = -(-k // 128)
        sides = torch.full((groups + 1, rows + 3), -3.0, device="cuda")
        s = sides[:groups, 1:rows + 1].t()
        P.dev_quantize_f8(xd, out=(q, s))
        want, ws = P.dev_quantize_f8(x.cuda())
        assert torch.equal(q.view(torch.uint8), want.view(torch.uint8)) and torch.equal(s, ws)
        left = base.clone()
        left[3:3 + rows * (k + 5)].view(rows, k + 5)[:, :k] = 77
        sides[:groups, 1:rows + 1] = -3
        assert (left == 77).all() and (sides == -3).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", [5, 640, 3000])
def test_quantize_groups_of_zeros_infinities_nan_and_extremes(t, k):
    T = TYPES[t]
    x = normal(9, k, k).to(T)
    x[0] = 0
    x[1, k // 2] = float("inf")
    x[2, k - 1] = float("-inf")
    x[3, 0] = float("nan")
    x[4, 0], x[4, k - 1] = float("nan"), float("inf")
    x[5] = torch.finfo(T).max
    x[5, 1] = torch.finfo(T).min
    x[6] *= torch.finfo(T).tiny
    x[7] = 1.0
    q, s = P.dev_quantize_f8(x.cuda())
    y = P.dev_dequantize_f8(q, s).cpu()
    q, s = q.cpu().float(), s.cpu()
    assert (q[0] == 0).all() and (s[0] == np.float32(TINY) / np.float32(448)).all() and (y[0] == 0).all()
    for r, at, kind in ((1, k // 2, torch.isinf), (2, k - 1, torch.isinf), (3, 0, torch.isnan), (4, 0, torch.isnan)):
        g = at // 128
        assert kind(s[r, g]) and (q[r, 128 * g:128 * g + 128] == 0).all() and y[r, 128 * g:128 * g + 128].isnan().all()
        if r < 4:                                             # the other groups of the row are as they were
            keep = [i for i in range(s.shape[1]) if i != g]
            assert s[r, keep].isfinite().all()
    assert (q[5, 2:] == 448).all() and q[5, 1] == -448 and (q[7] == 448).all()
    for r in (5, 6, 7, 8):
        wq, ws = expected_codes(x[r:r + 1])
        assert np.array_equal(q[r:r + 1].numpy(), wq) and np.array_equal(s[r:r + 1].numpy(), ws)


def test_quantize_ties_go_to_even_codes():
    """With a = 1.25 the quotients 448 x / a of these are halfway between two codes, though 448 / a is no fp32 number."""
    x = torch.zeros(1, 128)
    t = torch.tensor([17.0, 19.0, 21.0, -17.0, 9.5, 8.5, 2.0 ** -10, 3 * 2.0 ** -10, 416.0 + 16.0])
    x[0, :9] = (t.double() * 1.25 / 448 * 7).float()          # times 7 is exact; divided again by the scale of the largest element
    x[0, 127] = 1.25 * 7
    q, s = P.dev_quantize_f8(x.cuda())
    assert q.cpu().float()[0, :9].tolist() == [16.0, 20.0, 20.0, -16.0, 10.0, 8.0, 0.0, 2.0 ** -8, 448.0]
    for T in (torch.bfloat16, torch.float16):
        top = 1.25 * 7
        y = torch.zeros(1, 128, dtype=T)
        y[0, 0], y[0, 1] = top, 17 * top / 448 if T is torch.float16 else 0
        wq, _ = expected_codes(y)
        assert np.array_equal(P.dev_quantize_f8(y.cuda())[0].cpu().float().numpy(), wq)


@pytest.mark.parametrize("rows,k", [(40, 128), (33, 500), (300, 1001)])
def test_quantize_fp32_next_to_ties(rows, k):
    """Quotients within two steps of fp32 of a tie between two codes: 448 x is no fp32 number there, the quotient is rounded once all the same."""
    g = torch.Generator().manual_seed(k)
    top = torch.rand(rows, -(-k // 128), generator=g, dtype=torch.float32) + 1
    tie = (17 + 2 * torch.randint(0, 8, (rows, k), generator=g)).double() * 2.0 ** torch.randint(-5, 4, (rows, k), generator=g).double()
    x = (tie * top.double().repeat_interleave(128, 1)[:, :k] / 448).float()
    x = (x.view(torch.int32) + torch.randint(-2, 3, (rows, k), generator=g, dtype=torch.int32)).view(torch.float32)
    x[:, ::128] = top
    x *= torch.where(torch.rand(rows, k, generator=g) < 0.5, -1.0, 1.0)
    v = grouped(x.double().numpy())
    t = (v * 448 / np.abs(v).max(2)[:, :, None]).astype(np.float32)        # 448 v is exact in 64 bits
    want = e4m3(t.astype(np.float64))[0].reshape(rows, -1)[:, :k]
    assert np.array_equal(P.dev_quantize_f8(x.cuda())[0].cpu().float().numpy(), want)
    back = torch.arange(rows - 1, -1, -1, device="cuda", dtype=torch.int32)[:, None]
    assert np.array_equal(P.dev_moe_gather_f8(x.cuda(), back)[0].cpu().float().numpy()[::-1], want)


def test_every_code_is_read_back():
    q = torch.arange(256, dtype=torch.uint8).view(2, 128).cuda()
    s = torch.tensor([[0.375], [3.0]]).cuda()
    for T in TYPES.values():
        y = P.dev_dequantize_f8(q.view(F8), s, dtype=T).cpu()
        want = (q.cpu().view(F8).float() * s.cpu()).to(T)
        assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(0), want.nan_to_num(0))
        assert y.isnan().sum() == 2
    # and in the products: each code against one
    one = torch.zeros(1, 128)
    one[0, 5] = 1
    a = torch.zeros(256, 128, dtype=torch.uint8)
    a[:, 5] = torch.arange(256, dtype=torch.uint8)
    c = P.dev_gemm_nt_f8(a.cuda().view(F8), torch.ones(1, 256, device="cuda").t(), one.to(F8).cuda(), torch.ones(1, 1, device="cuda")).cpu()
    want = torch.arange(256, dtype=torch.uint8).view(F8).float()
    assert torch.equal(c[:, 0].isnan(), want.isnan()) and torch.equal(c[:, 0].nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 8), (9, 1000), (2, 4097), (300, 520)])
def test_dequantize(t, rows, k):
    T = TYPES[t]
    q, s = codes(rows, k, rows + k, pitch=k + 3), side(rows, k, k, 2)
    y = P.dev_dequantize_f8(q, s, dtype=T)
    want = values(q, s)
    assert y.dtype == T and ((y.cpu().double() - want).abs() <= U * (1 + half_step(T)) * want.abs() + rounding(T, want * (1 + U))).all()
    out = pitched(torch.zeros(rows, k).to(T), 5, 1)
    P.dev_dequantize_f8(q, s, out=out)
    assert torch.equal(out, y)


# ---- SwiGLU ---------------------------------------------------------------------------

def check_swiglu(q, s, gate, up):
    """A value of the function is (4 + |gate|) 2^-23 of itself off (two more roundings in the product); the scale has the largest's, a code half a
    step and what is put on t by its value, the largest and the rounded quotient."""
    g, u = gate.double().numpy(), up.double().numpy()
    with np.errstate(over="ignore"):
        v = g / (1 + np.exp(-g)) * u
    rel = (5 + np.abs(g)) * 2 * U
    gv, gr = grouped(v), grouped(rel)
    a = np.maximum(np.abs(gv).max(2), TINY)
    worst = gr.max(2)
    s, q = s.cpu().double().numpy(), grouped(q.cpu().float().double().numpy())
    assert (np.abs(s - a / 448) <= (worst + U) * 1.01 * a / 448).all()
    t = gv * 448 / a[:, :, None]
    _, half = e4m3(np.abs(t) * (1 + 2.0 ** -10))
    assert (np.abs(q - t) <= half + (gr + worst[:, :, None] + 2 * U) * 1.01 * np.abs(t) + 1e-12).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k", ROWS_K)
def test_swiglu(t, rows, k):
    T = TYPES[t]
    both = normal(rows, 2 * k, 7 * k + rows, 3.0).to(T)
    dev = pitched(both, 1, 1)
    q, s = P.dev_swiglu_f8(dev[:, :k], dev[:, k:])
    check_swiglu(q, s, both[:, :k], both[:, k:])


def test_swiglu_of_far_gates():
    gate = torch.tensor([[0.0, 40.0, -40.0, 88.0, -80.0, 1e4, -1e4, -0.0] * 20])
    up = normal(1, 160, 3)
    q, s = P.dev_swiglu_f8(gate.cuda(), up.cuda())
    check_swiglu(q, s, gate, up)
    gate[0, 3] = float("nan")
    q, s = P.dev_swiglu_f8(gate.cuda(), up.cuda())
    assert s[0, 0].isnan() and (q[0, :128].float() == 0).all() and s[0, 1].isfinite()


# ---- matmul ---------------------------------------------------------------------------

def product(a, sa, b, sb, bias, cores=False):
    """The result in 64 bits and what a kernel may be off before it rounds to its type: the additions of a group's 128 products, each of them a step (2 U) off at
    most, scales and groups; with `cores` the matrix cores' own e4m3 sums, eight products less what is under 2^-13 of the largest."""
    x, w = values(a, sa), block_values(b, sb)
    c = x @ w.T
    size = x.abs() @ w.abs().T
    G = sa.shape[1]
    off = (2 * 128 + 2 * G + 4) * U * size + (8 * 2.0 ** -13 * size if cores else 0)
    if bias is not None:
        c = c + bias.cpu().double()
        off = off + U * (c.abs() + off)
    return c, off


def check_matmul(c, a, sa, b, sb, bias, cores=None):
    want, off = product(a, sa, b, sb, bias, c.dtype is not torch.float32 if cores is None else cores)
    h = half_step(c.dtype)
    d = (c.cpu().double() - want).abs()
    assert (d <= off * (1 + h) + rounding(c.dtype, want)).all(), (d - off - rounding(c.dtype, want)).max().item()


MATMULS = [(1, 1, 1), (1, 3, 16), (1, 128, 128), (1, 1000, 2048), (2, 129, 127), (3, 77, 129), (4, 64, 1024), (5, 300, 640), (13, 1000, 1500), (16, 16, 128), (17, 257, 384), (33, 500, 777),
           (64, 128, 4096), (65, 130, 65), (100, 1001, 260), (128, 256, 512), (129, 255, 1000), (200, 700, 2000), (256, 512, 896), (333, 1001, 1111), (520, 384, 640), (700, 1024, 300)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", MATMULS)
def test_matmul(t, M, N, K):
    a, sa, b, sb = codes(M, K, M + K), side(M, K, M), codes(N, K, N + K), blocks(N, K, N)
    bias = normal(1, N, N)[0].cuda() if (M + N) % 2 else None
    c = P.dev_gemm_nt_f8(a, sa, b, sb, bias, dtype=TYPES[t])
    check_matmul(c, a, sa, b, sb, bias)
    assert torch.equal(c, P.dev_gemm_nt_f8(a, sa, b, sb, bias, dtype=TYPES[t]))


@pytest.mark.parametrize("M,N,K", [(1, 50, 70), (5, 33, 200), (40, 130, 300), (140, 257, 129), (300, 300, 515)])
def test_matmul_strides_and_bytes_beside(M, N, K):
    """Pitches of every operand, bytes behind K that are NaNs, C starting at any element, scales among others."""
    pitch = -(-K // 16) * 16 + 48
    a, b = codes(M, K, 3, pitch), codes(N, K, 4, pitch + 16)
    sa, sb = side(M, K, 1, 5), blocks(N, K, 2)
    bias = normal(1, N, 5)[0].cuda()
    for t in TYPES.values():
        base = torch.full((M + 2, N + 3), 7.0, device="cuda").to(t)
        out = base.view(-1)[N + 4:N + 4 + M * (N + 3)].view(M, N + 3)[:, :N]
        P.dev_gemm_nt_f8(a, sa, b, sb, bias, out=out)
        check_matmul(out, a, sa, b, sb, bias)
        assert torch.equal(out, P.dev_gemm_nt_f8(codes(M, K, 3, rest=0), sa, codes(N, K, 4, rest=0), sb, bias, dtype=t))
        out.fill_(7.0)
        assert (base == 7).all()


def test_matmul_scales_and_codes_that_are_not_finite_stay_in_their_rows():
    for M, N, K in ((3, 40, 64), (20, 70, 300), (150, 300, 200)):
        for t in TYPES.values():
            a, b, sa, sb = codes(M, K, 1), codes(N, K, 2), side(M, K, 3), blocks(N, K, 4)
            a = a.clone()
            sa = sa.clone(memory_format=torch.preserve_format)
            sa[1, 0] = float("nan")
            sa[2, -1] = float("inf")
            a[2, 128 * (sa.shape[1] - 1):] = 0
            a = torch.nn.functional.pad(a.view(torch.uint8), (0, -K % 16)).view(F8)[:, :K]
            c = P.dev_gemm_nt_f8(a, sa, b, sb, dtype=t)
            assert c[1].isnan().all() and c[2].isnan().all() and c[0].isfinite().all()
            keep = [i for i in range(M) if i not in (1, 2)]
            check_matmul(c[keep], a[keep], sa.t()[:, keep].contiguous().t(), b, sb, None)


def test_matmul_transposed_weights_give_the_gradient():
    """dX = dY W: blocks of 128 x 128 transpose into themselves, so do the scales; against differences of the product too, which is linear in x."""
    M, N, K = 20, 300, 200
    w, sw = codes(N, K, 1), blocks(N, K, 2)
    dy, sy = P.dev_quantize_f8(normal(M, N, 3).cuda())
    wt = P.empty_f8(K, N)[0]
    wt.view(torch.uint8).copy_(w.view(torch.uint8).t())
    dx = P.dev_gemm_nt_f8(dy, sy, wt, sw.t().contiguous())
    want, off = product(dy, sy, wt, sw.t().contiguous(), None)
    assert (want - values(dy, sy) @ block_values(w, sw)).abs().max() <= 1e-12 * want.abs().max()
    assert ((dx.cpu().double() - want).abs() <= off).all()
    # d/dx_k of sum(dY * (x W^T)) at one element: the difference of two products whose inputs differ there
    x = normal(M, K, 5).mul_(30).clamp_(-448, 448).to(F8)
    one = torch.ones(-(-K // 128), M, device="cuda").t()
    for k in (0, 130, K - 1):
        up, down = x.clone().float(), x.clone().float()
        up[4, k], down[4, k] = 8, -8
        cu, cd = (P.dev_gemm_nt_f8(torch.nn.functional.pad(v, (0, -K % 16)).to(F8).cuda()[:, :K], one, w, sw) for v in (up, down))
        slope = ((cu - cd).cpu().double()[4] * values(dy, sy)[4]).sum() / 16
        _, o = product(x.cuda(), one, w, sw, None)
        slack = ((2 * o[4] + 16 * o.new_tensor(2.0 ** -20)) * values(dy, sy)[4].abs()).sum() / 16
        assert (slope - dx[4, k].cpu().double()).abs() <= slack + off[4, k]


def test_offsets_beyond_32_bits():
    """Rows whose distance from the first does not fit in 32 bits."""
    far = (1 << 30) + 24
    x = torch.empty(4 * far, dtype=torch.float16, device="cuda").as_strided((5, 300), (far - 300, 1))
    x.copy_(normal(5, 300, 1).half())
    q = torch.empty(4 * far, dtype=torch.uint8, device="cuda").as_strided((5, 300), (far - 300, 1)).view(F8)
    s = torch.empty(3, far, device="cuda")[:, :5].t()
    q, s = P.dev_quantize_f8(x, out=(q, s))
    q2, s2 = P.dev_quantize_f8(x.contiguous())
    assert torch.equal(q.float(), q2.float()) and torch.equal(s, s2)
    y = P.dev_dequantize_f8(q, s, out=x)
    assert torch.equal(y.contiguous(), P.dev_dequantize_f8(q2, s2, dtype=torch.float16))
    pos = torch.tensor([[3], [0], [-1], [4], [1]], dtype=torch.int32, device="cuda")
    y = P.dev_moe_gather(q2.float().half(), pos, out=x)
    assert torch.equal(y[pos[[0, 1, 3, 4], 0].long()].float(), q2.float()[[0, 1, 3, 4]])
    back = P.dev_moe_combine(x, pos)
    assert torch.equal(back[[0, 1, 3, 4]].float(), q2.float()[[0, 1, 3, 4]]) and (back[2] == 0).all()
    del x, q, y
    pitch = 1 << 22                                           # the longest that a matmul's operands may have
    a = torch.empty(1100 * pitch, dtype=torch.uint8, device="cuda").as_strided((1100, 200), (pitch, 1)).view(F8)
    a.copy_(codes(1100, 200, 3))
    b, sa, sb = codes(70, 200, 4), side(1100, 200, 5, far), blocks(70, 200, 6)
    sa1, sb1 = side(70, 200, 7), blocks(1100, 200, 8)
    for T in (torch.float32, torch.bfloat16):
        check_matmul(P.dev_gemm_nt_f8(a, sa, b, sb, dtype=T), a, sa, b, sb, None)
        check_matmul(P.dev_gemm_nt_f8(b, sa1, a, sb1, dtype=T), b, sa1, a, sb1, None)
        check_matmul(P.dev_gemm_nt_f8(b[:3], sa1[:3], a, sb1, dtype=T), b[:3], sa1[:3], a, sb1, None)
    out = torch.empty(3 * far, dtype=torch.float16, device="cuda").as_strided((4, 1100), (far - 1100, 1))
    for rows in (1, 4):
        P.dev_gemm_nt_f8(b[:rows], sa1[:rows], a, sb1, out=out[:rows])
        check_matmul(out[:rows], b[:rows], sa1[:rows], a, sb1, None)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 300, 640), (40, 130, 300), (300, 520, 1000), (2048, 8300, 640)])
def test_16_bit_results_of_fp32_sums(t, M, N, K):
    """Where the caller says so no product is dropped: the fp32 result's bits, rounded; kernels on the e4m3 instructions do not take such a call even if forced."""
    a, sa, b, sb = codes(M, K, 1).clone(), side(M, K, 2), codes(N, K, 3).clone(), blocks(N, K, 4)
    a, b = (torch.nn.functional.pad(v.view(torch.uint8), (0, -K % 16)).view(F8)[:, :K] for v in (a, b))
    a.view(torch.uint8)[:, 8], a.view(torch.uint8)[:, 9], b.view(torch.uint8)[:, 8:10] = 0x7E, 0xFE, 0x7E            # 448^2 - 448^2 among each eight's products
    bias = normal(1, N, 5)[0].cuda()
    whole = P.dev_gemm_nt_f8(a, sa, b, sb, bias)
    check_matmul(whole, a, sa, b, sb, bias)
    want = whole.to(TYPES[t])
    assert torch.equal(P.dev_gemm_nt_f8(a, sa, b, sb, bias, dtype=TYPES[t], fp32_sums=True), want)
    out = torch.empty_like(want)
    assert P.dev_gemm_nt_f8(a, sa, b, sb, bias, out=out, fp32_sums=True) is out and torch.equal(out, want)
    assert torch.equal(P.dev_gemm_nt_f8(a, sa, b, sb, bias, fp32_sums=True), whole)
    for kernel in CORES:
        ckq.lib().ckq_launch_set_f8_kernel(kernel)
        try:
            assert torch.equal(P.dev_gemm_nt_f8(a, sa, b, sb, bias, dtype=TYPES[t], fp32_sums=True), want)
        finally:
            ckq.lib().ckq_launch_set_f8_kernel(-1)


# ---- matmul over experts ----------------------------------------------------------------

def experts(M, N, K, counts, t, bias, seed=0):
    E = len(counts)
    a, sa = codes(M, K, seed + 1), side(M, K, seed + 2)
    b = torch.stack([codes(N, K, seed + 10 + e, -(-K // 16) * 16).view(torch.uint8) if 0 else torch.nn.functional.pad(codes(N, K, seed + 10 + e).view(torch.uint8), (0, -K % 16), value=0x7F)
                     for e in range(E)]).view(F8)[:, :, :K]
    sb = blocks(N, K, seed + 3, E)
    offsets = torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int32, device="cuda")
    bias = normal(E, N, seed + 4).cuda() if bias else None
    out = torch.full((M, N), 7.0, device="cuda").to(t)
    P.dev_gemm_nt_f8_experts(a, sa, b, sb, offsets, bias, out=out)
    return a, sa, b, sb, offsets, bias, out


def check_experts(out, a, sa, b, sb, offsets, bias, cores=False):
    o = offsets.cpu().tolist()
    for e in range(b.shape[0]):
        lo, hi = o[e], o[e + 1]
        if hi > lo:
            rows = slice(lo, hi)
            check_matmul(out[rows], a[rows], sa.t()[:, rows].contiguous().t(), b[e], sb[e], None if bias is None else bias[e], cores)
    assert (out[o[-1]:] == 7).all()                           # as they were


EXPERTS = [(1, 40, 64, [0, 1, 0]), (8, 300, 256, [1, 0, 2, 0, 0, 1, 3, 1]), (30, 129, 130, [0] * 40 + [7] + [0] * 40 + [3, 5] + [0] * 50), (100, 260, 300, [100]), (90, 70, 200, [0, 64, 1, 0, 15]),
           (64, 128, 512, [16, 16, 16, 16]), (200, 1000, 77, [3, 60, 0, 17, 33, 1]), (300, 384, 1000, [0, 299, 0, 1]), (700, 256, 640, [130, 1, 0, 256, 65, 127, 64]), (50, 64, 128, [0, 0, 0]),
           (1500, 200, 256, [700, 100, 5, 300, 257])]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K,counts", EXPERTS)
def test_experts(t, M, N, K, counts):
    for bias in (False, True):
        a, sa, b, sb, offsets, bias, out = experts(M, N, K, counts, TYPES[t], bias)
        check_experts(out, a, sa, b, sb, offsets, bias)


def test_transposed_weights_of_experts_give_the_gradient():
    """dX = dY W of each expert's rows, against the product of the values and against differences of the product."""
    M, N, K, counts = 150, 300, 200, [40, 0, 3, 100, 1]
    E, o = len(counts), [0] + np.cumsum(counts).tolist()
    offsets = torch.tensor(o, dtype=torch.int32, device="cuda")
    w = torch.stack([torch.nn.functional.pad(codes(N, K, e).view(torch.uint8), (0, -K % 16)) for e in range(E)]).view(F8)[:, :, :K]
    sw = blocks(N, K, 2, E)
    dy, sy = P.dev_quantize_f8(normal(M, N, 3).cuda())
    wt = torch.nn.functional.pad(w.view(torch.uint8).transpose(1, 2), (0, -N % 16)).contiguous().view(F8)[:, :, :N]
    dx = P.dev_gemm_nt_f8_experts(dy, sy, wt, sw.transpose(1, 2).contiguous(), offsets)
    x, one = normal(M, K, 5).mul_(30).clamp_(-448, 448).to(F8).float(), torch.ones(-(-K // 128), M, device="cuda").t()
    product_of = lambda v: P.dev_gemm_nt_f8_experts(torch.nn.functional.pad(v, (0, -K % 16)).to(F8).cuda()[:, :K], one, w, sw, offsets).cpu().double()
    for e in range(E):
        rows = slice(o[e], o[e + 1])
        v, m = values(dy, sy)[rows], block_values(w[e], sw[e])
        # one sum of 128 at a time, scales and groups, as `product` counts them
        off = (2 * 128 + 2 * -(-N // 128) + 4) * U * (v.abs() @ m.abs())
        assert ((dx.cpu().double()[rows] - v @ m).abs() <= off).all()
    for k in (0, 130, K - 1):
        up, down = x.clone(), x.clone()
        up[:, k], down[:, k] = 8, -8
        slope = ((product_of(up) - product_of(down)) * values(dy, sy)).sum(1) / 16
        for e in range(E):
            rows = slice(o[e], o[e + 1])
            m, v = block_values(w[e], sw[e]), values(dy, sy)[rows].abs()
            size = up[rows].double().abs() @ m.abs().T                             # |up| and |down| are alike
            slack = ((2 * (2 * 128 + 2 * 2 + 4) * U * size) * v).sum(1) / 16 + (2 * 128 + 2 * -(-N // 128) + 4) * U * (v @ m.abs()[:, k])
            assert ((slope[rows] - dx.cpu().double()[rows, k]).abs() <= slack).all()


KERNELS = range(17)             # CKQ_F8_* of ckq_launch.h
CORES = range(9, 16)              # those on the e4m3 instructions


@pytest.fixture
def kernel(request):
    ckq.lib().ckq_launch_set_f8_kernel(request.param)
    yield request.param
    ckq.lib().ckq_launch_set_f8_kernel(-1)


@pytest.mark.parametrize("kernel", KERNELS, indirect=True)
@pytest.mark.parametrize("M,N,K", [(1, 3, 16), (1, 128, 128), (2, 129, 127), (5, 300, 640), (17, 257, 384), (65, 130, 65), (129, 255, 1000), (200, 700, 2000), (257, 513, 896), (333, 1001, 1111), (520, 384, 129)])
def test_matmul_on_every_kernel(kernel, M, N, K):
    a, sa, b, sb = codes(M, K, M + K, -(-K // 16) * 16 + 32), side(M, K, M, 3), codes(N, K, N + K), blocks(N, K, N)
    bias = normal(1, N, N)[0].cuda() if M % 2 else None
    for t in TYPES.values():
        c = P.dev_gemm_nt_f8(a, sa, b, sb, bias, dtype=t)
        check_matmul(c, a, sa, b, sb, bias, cores=kernel in CORES)
        assert torch.equal(c, P.dev_gemm_nt_f8(a, sa, b, sb, bias, dtype=t))


@pytest.mark.parametrize("kernel", KERNELS, indirect=True)
@pytest.mark.parametrize("M,N,K,counts", EXPERTS)
def test_experts_on_every_kernel(kernel, M, N, K, counts):
    a, sa, b, sb, offsets, bias, out = experts(M, N, K, counts, torch.bfloat16, M % 2)
    check_experts(out, a, sa, b, sb, offsets, bias, cores=kernel in CORES)


@pytest.mark.parametrize("kernel", [8, 6, 0], indirect=True)
def test_matmul_launches_in_parts(kernel):
    """More tiles than one launch has blocks, of 16 x 16 and 16 x 32: whole numbers, whose sums are exact in any order."""
    def whole(*shape):
        return torch.randint(-4, 5, shape, device="cuda", generator=g).to(torch.float16)

    g = torch.Generator(device="cuda").manual_seed(1)
    for M, N, E in ((4100, (1 << 19) + 77, 0), ((1 << 19) + 77, 4100, 0), (3000, (1 << 18) + 130, 300), (1, (1 << 24) + 9, 0)):
        a, b, K = whole(M, 16), whole(*((E, N, 16) if E else (N, 16))), 16
        sa, sb = torch.full((1, M), 2.0, device="cuda").t(), torch.full((*b.shape[:-2], -(-N // 128), 1), 0.25, device="cuda")
        sa[M // 2:] = 4.0
        sb[..., 5::3, :] = 0.5
        bias = torch.randint(-3, 4, b.shape[:-1], device="cuda", generator=g).float()
        out = torch.full((M, N), 7.0, device="cuda", dtype=torch.float16)
        aw, bw = a * sa.half(), b * sb.half().repeat_interleave(128, -2)[..., :N, :]           # |sums| <= 16 * 16 * 2 + 3 in steps of 1/2: exact in fp16
        if E:
            counts = torch.full((E,), M // E)
            counts[3], counts[7] = 0, 2 * (M // E)
            offsets = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).int().cuda()
            P.dev_gemm_nt_f8_experts(a.to(F8), sa, b.to(F8), sb, offsets, bias, out=out)
            at = [0] + counts.cumsum(0).tolist()
            for e in range(E):
                assert torch.equal(out[at[e]:at[e + 1]], aw[at[e]:at[e + 1]] @ bw[e].t() + bias[e].half()), e
        else:
            P.dev_gemm_nt_f8(a.to(F8), sa, b.to(F8), sb, bias, out=out)
            for m in range(0, M, 1 << 16):
                assert torch.equal(out[m:m + (1 << 16)], aw[m:m + (1 << 16)] @ bw.t() + bias.half()), m
        del out, aw, bw


def whole_product(M, N, K, seed, t, E=0):
    """Operands of small whole numbers, scales that are powers of two, and their product: every sum is a multiple of 1/8 below 2^18, exact in fp32 in any order, and no
    product is below 2^-13 of another.  Bytes behind K are NaNs."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    whole = lambda *s: torch.randint(-4, 5, s, device="cuda", generator=g).float()
    power = lambda *s: 2.0 ** torch.randint(-1, 2, s, device="cuda", generator=g).float()
    held = lambda v: torch.nn.functional.pad(v.to(F8).view(torch.uint8), (0, -K % 16), value=0x7F).view(F8)[..., :K]
    lead = (E,) if E else ()
    a, b, sa, sb, bias = whole(M, K), whole(*lead, N, K), power(-(-K // 128), M).t(), 0.5 * power(*lead, -(-N // 128), -(-K // 128)), whole(*lead, N)
    x = a * sa.repeat_interleave(128, 1)[:, :K]
    w = b * sb.repeat_interleave(128, -1)[..., :K].repeat_interleave(128, -2)[..., :N, :]
    return held(a), sa, held(b), sb, bias, lambda rows=slice(None), e=None: ((x[rows] @ (w if e is None else w[e]).t().contiguous()) + (bias if e is None else bias[e])).to(t)


EXACT = [(2, 129, 127), (65, 130, 65), (129, 255, 1000), (257, 513, 896), (333, 1001, 1111), (520, 390, 1284)]
# at least 256 tiles of 256 x 256; N that ends within a tile of 192 and a block of 128, and a whole column of tiles less
TWO_EXACT = [(4000, 4300, 300), (4100, 3900, 1000), (2048, 8300, 640), (2000, 8500, 129), (9000, 2100, 77)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kernel", KERNELS, indirect=True)
def test_matmul_is_exact_on_whole_numbers_on_every_kernel(kernel, t):
    sizes = [(1, N, K) for _, N, K in EXACT] if kernel == 16 else TWO_EXACT if kernel == 15 else EXACT
    for M, N, K in sizes:
        assert ckq.lib().ckq_launch_f8_kernel(list(TYPES).index(t), M, N, K, 0) == kernel            # and no other one
        a, sa, b, sb, bias, want = whole_product(M, N, K, M + N, TYPES[t])
        assert torch.equal(P.dev_gemm_nt_f8(a, sa, b, sb, bias, dtype=TYPES[t]), want()), (M, N, K)


@pytest.mark.parametrize("kernel", range(15), indirect=True)
def test_experts_are_exact_on_whole_numbers_on_every_kernel(kernel):
    for M, N, K, counts in ((700, 256, 640, [130, 1, 0, 256, 65, 127, 64]), (300, 390, 1001, [0, 290, 0, 1]), (90, 70, 200, [0, 64, 1, 0, 15])):
        assert ckq.lib().ckq_launch_f8_kernel(1, M, N, K, len(counts)) == kernel
        a, sa, b, sb, bias, want = whole_product(M, N, K, M + N, torch.bfloat16, len(counts))
        o = [0] + np.cumsum(counts).tolist()
        out = torch.full((M, N), 7.0, device="cuda", dtype=torch.bfloat16)
        P.dev_gemm_nt_f8_experts(a, sa, b, sb, torch.tensor(o, dtype=torch.int32, device="cuda"), bias, out=out)
        for e in range(len(counts)):
            assert torch.equal(out[o[e]:o[e + 1]], want(slice(o[e], o[e + 1]), e)), e
        assert (out[o[-1]:] == 7).all()


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_a_long_prompt_is_exact_on_whole_numbers(t):
    """The size for which two sizes of tiles are chosen without being forced."""
    M, N, K = 2048, 11008, 4096
    assert ckq.lib().ckq_launch_f8_kernel(list(TYPES).index(t), M, N, K, 0) == 15
    a, sa, b, sb, bias, want = whole_product(M, N, K, 1, TYPES[t])
    assert torch.equal(P.dev_gemm_nt_f8(a, sa, b, sb, bias, dtype=TYPES[t]), want())


@pytest.mark.parametrize("kernel", range(9, 15), indirect=True)
def test_sums_of_the_e4m3_instructions_lose_no_more_than_they_may(kernel):
    """Codes of every size, signs that cancel: each eight products may lose eight times 2^-13 of their largest, and nothing else."""
    M, N, K = 70, 90, 500
    g = torch.Generator().manual_seed(kernel)

    def any_codes(n):
        q = torch.randint(0, 256, (n, 512), generator=g, dtype=torch.uint8)
        return torch.where((q & 0x7F) == 0x7F, 0x7E, q).to(torch.uint8).cuda().view(F8)[:, :K]

    a, b, sa, sb = any_codes(M), any_codes(N), side(M, K, 1), blocks(N, K, 2)
    assert ckq.lib().ckq_launch_f8_kernel(0, M, N, K, 0) == kernel
    c = P.dev_gemm_nt_f8(a, sa, b, sb).cpu().double()
    want, off = product(a, sa, b, sb, None)
    x, w = values(a, sa), block_values(b, sb)
    largest = torch.nn.functional.pad((x[:, None] * w).abs(), (0, -K % 8)).view(M, N, -1, 8).amax(3)
    off = off + 8 * 2.0 ** -13 * largest.sum(2)
    assert ((c - want).abs() <= off).all(), ((c - want).abs() / off).max().item()
    assert (((c - want).abs() - product(a, sa, b, sb, None)[1]) > 0).any()         # and it is them that are meant


def test_experts_without_rows_and_as_many_experts_as_there_can_be():
    a, sa, b, sb = codes(7, 300, 1), side(7, 300, 2), codes(50, 300, 3), blocks(50, 300, 4, 4)
    out = torch.full((7, 50), 3.0, device="cuda")
    P.dev_gemm_nt_f8_experts(a, sa, b[None].expand(4, -1, -1), sb, torch.zeros(5, dtype=torch.int32, device="cuda"), out=out)
    assert (out == 3).all()
    E, T = 65535, 3000
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, E, (T, 2), device="cuda", dtype=torch.int32, generator=g)
    ids[5], ids[6, 0] = E - 1, E
    offsets, order, position = P.dev_moe_sort(ids, E)
    key = ids.flatten().long()
    key, slots = torch.sort(key, stable=True)
    n = int((key < E).sum())
    assert n == 2 * T - 1 and torch.equal(order[:n].long(), slots[:n]) and (order[n:] == -1).all()
    assert torch.equal(offsets.long(), torch.searchsorted(key, torch.arange(E + 1, device="cuda")))
    # whole numbers, scales that are powers of two: exact
    b = torch.randint(-4, 5, (E, 16, 32), device="cuda", generator=g).float()
    x = torch.randint(-4, 5, (T, 32), device="cuda", generator=g).to(F8)
    rows = torch.zeros(2 * T, 32, device="cuda", dtype=torch.uint8)
    rows[:n] = x.view(torch.uint8)[slots[:n] // 2]
    y = P.dev_gemm_nt_f8_experts(rows.view(F8), torch.full((1, 2 * T), 2.0, device="cuda").t(), b.to(F8), torch.full((E, 1, 1), 0.5, device="cuda"), offsets)
    assert torch.equal(y[:n], (b[key[:n]] * rows[:n].view(F8).float()[:, None]).sum(2))


def test_a_hundred_choices_with_the_gradient_in_place():
    T, c, k = 50, 100, 77
    g = torch.Generator(device="cuda").manual_seed(2)
    position = torch.randperm(T * c, device="cuda", generator=g).int().view(T, c)
    position[3, 50:] = -1
    there, slots = position.flatten() >= 0, position.flatten().long()
    w, y, d = (torch.randn(*n, device="cuda", generator=g) for n in ((T, c), (T * c, k), (T, k)))
    terms = torch.where(position[:, :, None] < 0, 0.0, y.double()[position.clamp(min=0).long()])
    # c products and sums, each a half step of what they add up to
    bound = (terms * w.double()[:, :, None]).abs().sum(1) * 2 * c * U
    assert ((P.dev_moe_combine(y, position, w).double() - (terms * w.double()[:, :, None]).sum(1)).abs() <= bound).all()
    dy, dw = y.clone(), torch.empty_like(w)
    P.dev_moe_combine_backward(d, dy, position, w, out=(dy, dw))
    products = terms * d.double()[:, None]
    assert ((dw.double() - products.sum(2)).abs() <= products.abs().sum(2) * 2 * k * U).all()
    assert torch.equal(dy[slots[there]], (w[:, :, None] * d[:, None]).reshape(-1, k)[there])
    assert torch.equal(P.dev_moe_gather(d, position, dy)[slots[there]], d.repeat_interleave(c, 0)[there])


def test_rows_launches_in_parts():
    """Rows of one element, more than a launch has threads for."""
    rows = (1 << 28) + 45
    x = torch.randn(rows, 1, device="cuda", dtype=torch.bfloat16)
    q, s = torch.empty(rows, 1, device="cuda", dtype=F8), torch.empty(1, rows, device="cuda").t()
    top = torch.tensor(448.0, device="cuda")                   # a number would be multiplied by its inverse

    def check():
        for i in range(0, rows, 1 << 26):
            part = x[i:i + (1 << 26)]
            assert torch.equal(q[i:i + (1 << 26)].view(torch.uint8), torch.where(part < 0, 0xFE, torch.where(part > 0, 0x7E, 0)).to(torch.uint8) | torch.signbit(part) * 128)
            assert torch.equal(s[i:i + (1 << 26)], part.float().abs().clamp(min=TINY) / top)

    P.dev_quantize_f8(x, (q, s))
    check()
    y = torch.empty_like(x)
    P.dev_dequantize_f8(q, s, out=y)
    for i in range(0, rows, 1 << 26):                         # scale * 448: an eighth of a step of bf16 off, at most
        assert torch.equal(x[i:i + (1 << 26)], y[i:i + (1 << 26)])
    q.view(torch.uint8).zero_()
    s.zero_()
    back = torch.arange(rows - 1, -1, -1, device="cuda", dtype=torch.int32)[:, None]
    P.dev_moe_gather_f8(x, back, out=(q, s))
    x = x.flip(0)
    check()
    del q, s
    P.dev_moe_gather(x, back, y)
    assert torch.equal(y, x.flip(0))
    # a block has a token: 2^23 of them a launch
    T = (1 << 23) + 9
    d, rows_ = x[:T].contiguous(), y[:T].contiguous()
    w = torch.rand(T, 1, device="cuda")
    dy, dw = P.dev_moe_combine_backward(d, rows_, back[-T:].contiguous(), w)
    assert torch.equal(dy, (d.float() * w).bfloat16().flip(0)) and torch.equal(dw, d.float() * rows_.flip(0).float())
    del x, y, d, rows_, dy, dw, w, back
    # two threads a row: 2^30 rows a launch
    T = (1 << 30) + 5
    x, back = torch.randn(T, 9, device="cuda", dtype=torch.bfloat16), torch.arange(T - 1, -1, -1, device="cuda", dtype=torch.int32)[:, None]
    y, out = torch.empty_like(x), torch.empty_like(x)
    P.dev_moe_gather(x, back, y)
    P.dev_moe_combine(y, back, None, out=out)
    for part in (slice(0, 5000), slice((1 << 30) - 5000, None)):
        assert torch.equal(y[part], x[T - (part.stop or T):T - part.start].flip(0)) and torch.equal(out[part], x[part])


def test_experts_of_one_matrix_and_of_offsets_out_of_range():
    a, sa, b, sb = codes(40, 200, 1), side(40, 200, 2), codes(130, 200, 3), blocks(130, 200, 4)
    # experts side by side in one tensor whose rows are further apart, one matrix for all of them
    out = P.dev_gemm_nt_f8_experts(a, sa, b[None].expand(3, -1, -1), sb[None].expand(3, -1, -1).contiguous(), torch.tensor([0, 7, 7, 40], dtype=torch.int32, device="cuda"))
    check_matmul(out, a, sa, b, sb, None)
    # offsets beyond the rows there are: as many as there are
    bb, ssb = torch.stack([b.view(torch.uint8)] * 3).view(F8), torch.stack([sb] * 3)
    pad = torch.nn.functional.pad(bb.view(torch.uint8), (0, -200 % 16)).view(F8)[:, :, :200]
    for o in ([-5, 9, 50, 1000], [0, 2000, 2000, 2000], [-9, -9, 41, 41]):
        out = torch.full((40, 130), 7.0, device="cuda")
        P.dev_gemm_nt_f8_experts(a, sa, pad, ssb, torch.tensor(o, dtype=torch.int32, device="cuda"), out=out)
        check_matmul(out, a, sa, b, sb, None)
    # the other way round: nothing outside the rows is touched
    out = torch.full((42, 130), 7.0, device="cuda")
    P.dev_gemm_nt_f8_experts(a, sa, pad, ssb, torch.tensor([30, 5, 40, 2], dtype=torch.int32, device="cuda"), out=out[1:41])
    assert (out[0] == 7).all() and (out[41] == 7).all()


# ---- tokens sorted by expert -----------------------------------------------------------------

def random_ids(T, c, E, seed, none=0.1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, E, (T, c), generator=g, dtype=torch.int32)
    ids[torch.rand(T, c, generator=g) < none] = -1
    return ids


def sorted_slots(ids, E):
    flat = ids.reshape(-1).numpy().astype(np.int64)
    key = np.where((flat >= 0) & (flat < E), flat, E)
    order = np.argsort(key, kind="stable")
    have = int((key < E).sum())
    position = np.empty(flat.size, np.int64)
    position[order] = np.arange(flat.size)
    position[key == E] = -1
    order = order.copy()
    order[have:] = -1
    return np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])]), order, position.reshape(ids.shape)


@pytest.mark.parametrize("T,c,E", [(1, 1, 1), (1, 8, 64), (3, 2, 2), (7, 6, 64), (63, 1, 5), (64, 4, 3), (65, 4, 256), (129, 2, 7), (300, 7, 16), (1000, 3, 100), (2049, 8, 128), (5000, 8, 4), (9000, 2, 300), (20000, 6, 60)])
def test_sort(T, c, E):
    for none in (0.0, 0.1, 1.0):
        ids = random_ids(T, c, E, T + E, none)
        if T > 2:
            ids[1], ids[2, 0] = E, 2 ** 31 - 1                # no such experts either
        got = P.dev_moe_sort(ids.cuda(), E)
        for g, w in zip(got, sorted_slots(ids, E)):
            assert g.dtype == torch.int32 and np.array_equal(g.cpu().numpy(), w)


def test_sort_one_expert_twice_and_all_in_one():
    ids = torch.tensor([[3, 3], [0, 3], [3, 3]], dtype=torch.int32)
    for got, want in zip(P.dev_moe_sort(ids.cuda(), 4), ([0, 1, 1, 1, 6], [2, 0, 1, 3, 4, 5], [[1, 2], [0, 3], [4, 5]])):
        assert got.cpu().tolist() == want
    ids = torch.full((3000, 2), 200, dtype=torch.int32)
    offsets, order, position = P.dev_moe_sort(ids.cuda(), 300)
    assert order.cpu().tolist() == list(range(6000)) and torch.equal(position.cpu().view(-1), order.cpu()) and offsets.cpu().tolist() == [0] * 201 + [6000] * 100


TOKENS = [(1, 1, 1), (1, 8, 2048), (2, 3, 7), (5, 2, 8), (7, 6, 129), (33, 4, 1001), (64, 8, 256), (100, 1, 4099), (300, 9, 72), (3, 20, 33)]


def placed(T, c, seed):
    ids = random_ids(T, c, 6, seed)
    return P.dev_moe_sort(ids.cuda(), 6)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,c,k", TOKENS)
def test_gather(t, T, c, k):
    x = normal(T, k, T * k).to(TYPES[t])
    offsets, order, position = placed(T, c, k)
    have = int(offsets[-1])
    y = torch.full((T * c, k), 7.0, device="cuda").to(TYPES[t])
    P.dev_moe_gather(x.cuda(), position, out=y)
    assert torch.equal(y[:have].cpu(), x[order[:have].cpu().long() // c]) and (y[have:] == 7).all()
    # rows anywhere, fewer of them than places: those are left out, the others stay in their rows
    some = max(1, have // 2)
    out = pitched(torch.full((some, k), 5.0).to(TYPES[t]), 3, 1)
    P.dev_moe_gather(pitched(x, 1, 1), position, out=out)
    assert torch.equal(out[:min(some, have)], y[:min(some, have)])
    # in 8 bits: the rows' own codes
    q, s = P.empty_f8(T * c, k)
    q.view(torch.uint8).fill_(77)
    s.fill_(-3)
    P.dev_moe_gather_f8(x.cuda(), position, out=(q, s))
    wq, ws = P.dev_quantize_f8(x.cuda())
    at = order[:have].long() // c
    assert torch.equal(q[:have].view(torch.uint8), wq.view(torch.uint8)[at]) and torch.equal(s[:have], ws[at])
    assert (q[have:].view(torch.uint8) == 77).all() and (s[have:] == -3).all()


def back64(y, position, w):
    y, position = y.cpu().double(), position.cpu().long()
    there = (position >= 0) & (position < y.shape[0])
    rows = y[position.clamp(0, y.shape[0] - 1)] * (w.cpu().double() * there)[:, :, None]
    return rows.sum(1), rows.abs().sum(1)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,c,k", TOKENS)
def test_combine(t, T, c, k):
    D = TYPES[t]
    y = normal(T * c, k, T + k).to(D)
    _, _, position = placed(T, c, k)
    w = torch.rand(T, c, generator=torch.Generator().manual_seed(k))
    h = half_step(D)
    for weights in (w, None):
        out = P.dev_moe_combine(y.cuda(), position, weights.cuda() if weights is not None else None)
        want, size = back64(y, position, torch.ones(T, c) if weights is None else weights)
        off = c * U * size                                    # a rounding for each of the c multiply-adds
        assert ((out.cpu().double() - want).abs() <= off * (1 + h) + rounding(D, want)).all()
        strided = pitched(torch.zeros(T, k).to(D), 3, 1)
        P.dev_moe_combine(pitched(y, 1, 1), position, weights.cuda() if weights is not None else None, out=strided)
        assert torch.equal(strided, out)
    none = torch.full_like(position, -1)
    assert (P.dev_moe_combine(y.cuda(), none, w.cuda()) == 0).all()
    # rows that no token has may hold anything, and so may the weights of slots without a place
    if (position < 0).any():
        y2, w2 = y.cuda().clone(), w.cuda().clone()
        y2[int((position >= 0).sum()):] = float("nan")
        w2[position < 0] = float("nan")
        assert torch.equal(P.dev_moe_combine(y2, position, w2), P.dev_moe_combine(y.cuda(), position, w.cuda()))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,c,k", TOKENS)
def test_combine_backward(t, T, c, k):
    D = TYPES[t]
    dout, y = normal(T, k, T + k).to(D), normal(T * c, k, T + k + 1).to(D)
    offsets, _, position = placed(T, c, k)
    have = int(offsets[-1])
    w = torch.rand(T, c, generator=torch.Generator().manual_seed(k)).cuda()
    dy = torch.full((T * c, k), 7.0, device="cuda").to(D)
    dw = torch.empty(T, c, device="cuda")
    P.dev_moe_combine_backward(dout.cuda(), y.cuda(), position, w, out=(dy, dw))
    pos = position.cpu().long()
    h = half_step(D)
    for tok in range(min(T, 40)):
        for j in range(c):
            p = int(pos[tok, j])
            if p < 0:
                assert dw[tok, j] == 0
                continue
            want = dout[tok].double() * float(w[tok, j])
            assert ((dy[p].cpu().double() - want).abs() <= U * (1 + h) * want.abs() + rounding(D, want * (1 + U))).all()
            terms = dout[tok].double() * y[p].double()
            # every thread's chain, the tree of a wave, four waves
            depth = 8 * -(-k // 2048) + 6 + 4
            assert (dw[tok, j].cpu().double() - terms.sum()).abs() <= depth * U * terms.abs().sum()
    assert (dy[have:] == 7).all()
    # again, strided, and into y itself
    sy, sd = pitched(y, 3, 1), pitched(torch.full((T * c, k), 7.0).to(D), 5, 3)
    dw2 = torch.empty_like(dw)
    P.dev_moe_combine_backward(pitched(dout, 1, 1), sy, position, w, out=(sd, dw2))
    assert torch.equal(sd, dy) and torch.equal(dw2, dw)
    P.dev_moe_combine_backward(dout.cuda(), sy, position, w, out=(sy, dw2))
    assert torch.equal(sy[:have], dy[:have]) and torch.equal(dw2, dw) and torch.equal(sy[have:].cpu(), y[have:])


@pytest.mark.parametrize("t", TYPES)
def test_rows_without_a_slot_are_zeros_where_the_call_makes_the_tensor(t):
    """The gradient of a row that no token has is zero, and no caller may get what the memory held before."""
    T, c, E, k, N = 40, 3, 5, 300, 70
    S = T * c
    offsets, order, position = P.dev_moe_sort(random_ids(T, c, E, 3, 0.4).cuda(), E)
    have = int(offsets[-1])
    assert 0 < have < S
    x, y, w = normal(T, k, 1).to(TYPES[t]).cuda(), pitched(normal(S, k, 2).to(TYPES[t]), 8), torch.rand(T, c, device="cuda")
    a, sa, b, sb = codes(S, k, 3), side(S, k, 4), codes(E * N, k, 5).view(torch.uint8), blocks(N, k, 6, E)
    b = torch.nn.functional.pad(b, (0, -k % 16)).view(F8).view(E, N, -1)[:, :, :k]

    def made(call):
        nan = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for n in 4 * [2 ** i for i in range(9, 22)]]        # what the next tensors get
        del nan
        return call()

    for i in range(3):
        dy, dw = made(lambda: P.dev_moe_combine_backward(x, y, position, w))
        want = torch.zeros_like(dy)
        P.dev_moe_combine_backward(x, y, position, w, out=(want, torch.empty_like(dw)))
        assert dy.shape == y.shape and torch.equal(dy, want) and (dy[have:] == 0).all()
        g = made(lambda: P.dev_moe_gather(x, position))
        assert torch.equal(g, P.dev_moe_gather(x, position, out=torch.zeros_like(g))) and (g[have:] == 0).all()
        q, s = made(lambda: P.dev_moe_gather_f8(x, position))
        assert (q[have:].view(torch.uint8) == 0).all() and (s[have:] == 0).all() and q[:have].float().abs().max() == 448
        o = made(lambda: P.dev_gemm_nt_f8_experts(a, sa, b, sb, offsets, dtype=TYPES[t]))
        assert (o[have:] == 0).all()
        check_experts(torch.cat([o[:have], torch.full_like(o[have:], 7)]), a, sa, b, sb, offsets, None)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("k", [2048, 2047, 2044])
def test_rows_there_and_back_beyond_the_cache(t, k):
    """Rows of 16 bits, more than 192 MB of them, which leave past the caches; the same in place."""
    D, T, c, E = TYPES[t], 7000, 8, 40
    g = torch.Generator(device="cuda").manual_seed(k)
    assert T * c * k * 2 > 192 << 20
    rows = lambda n, fill=None: (torch.randn(n, 2048, device="cuda", generator=g) if fill is None else torch.full((n, 2048), fill, device="cuda")).to(D)[:, :k]
    ids = torch.randint(-1, E, (T, c), device="cuda", generator=g, dtype=torch.int32)
    offsets, order, position = P.dev_moe_sort(ids, E)
    have = int(offsets[-1])
    assert have < T * c
    x, w, y = rows(T), torch.rand(T, c, device="cuda", generator=g), rows(T * c)
    out = P.dev_moe_gather(x, position, out=rows(T * c, 7.0))
    slots = order[:have].long()
    assert torch.equal(out[:have], x[slots // c]) and (out[have:] == 7).all()
    del out
    dy, dw = P.dev_moe_combine_backward(x, y, position, w, out=(rows(T * c, 7.0), torch.empty(T, c, device="cuda")))
    assert (dy[have:] == 7).all()
    h, depth = half_step(D), 8 * -(-k // 2048) + 6 + 4        # every thread's chain, the tree of a wave, four waves
    for part in slots.split(1 << 13):
        # w * dout has 24 + 11 bits: rounded to fp32 first (U of it) and then to the type, or at once
        want = w.view(-1)[part, None].double() * x[part // c].double()
        d = dy[position.view(-1)[part].long()].double()
        assert ((d - want).abs() <= U * (1 + h) * want.abs() + rounding(D, want * (1 + U))).all()
        terms = x[part // c].double() * y[position.view(-1)[part].long()].double()
        assert ((dw.view(-1)[part].double() - terms.sum(1)).abs() <= depth * U * terms.abs().sum(1)).all()
    assert (dw[position < 0] == 0).all()
    again, behind = torch.empty_like(dw), y[have:].clone()
    P.dev_moe_combine_backward(x, y, position, w, out=(y, again))
    assert torch.equal(y[:have], dy[:have]) and torch.equal(y[have:], behind) and torch.equal(again, dw)


def test_gradients_against_differences():
    """Both functions are linear in each argument, so a difference of any width is the derivative; on fp32 whole numbers of few bits nothing is rounded, and the
    two agree to the last bit."""
    g = torch.Generator().manual_seed(1)
    T, c, k = 9, 3, 40
    whole = lambda *s: torch.randint(-8, 9, s, generator=g).float().cuda()
    x, y, dout, w, gy = whole(T, k), whole(T * c, k), whole(T, k), whole(T, c), whole(T * c, k)
    _, _, position = placed(T, c, 5)
    dy, dw = P.dev_moe_combine_backward(dout, y, position, w, out=(torch.zeros_like(y), torch.empty_like(w)))
    dx = P.dev_moe_combine(gy, position)
    loss = lambda y, w: (P.dev_moe_combine(y, position, w) * dout).sum()
    there = lambda x: (P.dev_moe_gather(x, position, out=torch.zeros(T * c, k, device="cuda")) * gy).sum()
    for v, d, f in ((y, dy, lambda v: loss(v, w)), (w, dw, lambda v: loss(y, v)), (x, dx, there)):
        for i in torch.randint(0, v.numel(), (25,), generator=g).tolist():
            up, down = v.clone(), v.clone()
            up.view(-1)[i] += 4
            down.view(-1)[i] -= 4
            assert (f(up) - f(down)) / 8 == d.view(-1)[i]


def test_front_ends_refuse_on_the_device():
    a, sa = codes(2, 32, 1), side(2, 32, 1)
    x = torch.zeros(2, 32, device="cuda")
    b, sb, o = codes(4, 32, 2).view(torch.uint8).view(2, 2, 32).view(F8), torch.ones(2, 1, 1, device="cuda"), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    pos, w = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, 1, device="cuda")
    wide, many = codes(2, 256, 1), side(2, 256, 1)
    bad = [lambda: P.dev_quantize_f8(x.double()), lambda: P.dev_quantize_f8(x.t()), lambda: P.dev_quantize_f8(x[:0]), lambda: P.dev_quantize_f8(x[:, ::2]),
           lambda: P.dev_quantize_f8(x, out=(a, sa[:1])), lambda: P.dev_quantize_f8(x, out=(a.view(torch.uint8), sa)), lambda: P.dev_quantize_f8(x, out=(a, sa.double())),
           lambda: P.dev_quantize_f8(torch.zeros(2, 256, device="cuda"), out=(wide, many.contiguous())), lambda: P.dev_dequantize_f8(a, sa, out=x.double()),
           lambda: P.dev_dequantize_f8(wide, many[:, :1]), lambda: P.dev_swiglu_f8(x, x[:, :16]), lambda: P.dev_swiglu_f8(x, pitched(x, 4)),
           lambda: P.dev_gemm_nt_f8(a, sa, codes(3, 16, 1), torch.ones(1, 1, device="cuda")), lambda: P.dev_gemm_nt_f8(a[:, 1:], sa, a[:, 1:], torch.ones(1, 1, device="cuda")),
           lambda: P.dev_gemm_nt_f8(a, sa, a, torch.ones(2, 1, device="cuda")), lambda: P.dev_gemm_nt_f8(a, sa.cpu(), a, sb[0]), lambda: P.dev_gemm_nt_f8(a, sa, a, sb[0], bias=x[0]),
           lambda: P.dev_gemm_nt_f8(wide, many.contiguous(), wide, torch.ones(1, 2, device="cuda")), lambda: P.dev_gemm_nt_f8(a, sa, a, sb[0], out=torch.zeros(2, 1, device="cuda").expand(2, 2)),
           lambda: P.dev_gemm_nt_f8_experts(a, sa, b, sb, o[:2]), lambda: P.dev_gemm_nt_f8_experts(a, sa, b, sb, o.long()), lambda: P.dev_gemm_nt_f8_experts(a, sa, b[0], sb[0], o),
           lambda: P.dev_gemm_nt_f8_experts(a, sa, b, sb, o, bias=w), lambda: P.dev_gemm_nt_f8_experts(a, sa, b[:, :, :16], sb, o),
           lambda: P.dev_moe_sort(pos.long(), 2), lambda: P.dev_moe_sort(pos, 0), lambda: P.dev_moe_sort(pos, 70000), lambda: P.dev_moe_sort(pos.t()[0], 2), lambda: P.dev_moe_sort(pos[:0], 2),
           lambda: P.dev_moe_sort(torch.zeros(4, 4, dtype=torch.int32, device="cuda")[:, :2], 2), lambda: P.dev_moe_gather(x[:1], pos), lambda: P.dev_moe_gather(x, pos.long()),
           lambda: P.dev_moe_gather(x, pos, out=x.half()), lambda: P.dev_moe_gather(x, pos, out=x[:, :16]), lambda: P.dev_moe_gather_f8(x, pos, out=(wide, many)),
           lambda: P.dev_moe_combine(x, pos, w[:1]), lambda: P.dev_moe_combine(x, pos, w.double()), lambda: P.dev_moe_combine(x, pos, out=x[:1]), lambda: P.dev_moe_combine(x, pos.cpu()),
           lambda: P.dev_moe_combine_backward(x, x, pos, w, out=(x.half(), w)), lambda: P.dev_moe_combine_backward(x, x, pos, w, out=(x, w[:1])), lambda: P.dev_moe_combine_backward(x[:1], x, pos, w)]
    for i, f in enumerate(bad):
        with pytest.raises(ckq.CkqError):
            f()
            pytest.fail("call %d" % i)


# ---- all of them together -------------------------------------------------------------------------

class Moe:
    """The MLP half of a decoder layer with experts on the buffers of a serving loop."""

    def __init__(self, T, c, E, D, F, t, seed=5):
        self.F, self.E, self.c, S = F, E, c, T * c
        self.x = normal(T, D, seed).to(t).cuda()
        self.ids = random_ids(T, c, E, seed).cuda()
        self.w = torch.rand(T, c, generator=torch.Generator().manual_seed(seed)).cuda()
        stack = lambda n, k, s: torch.stack([torch.nn.functional.pad(codes(n, k, s + e).view(torch.uint8), (0, -k % 16)) for e in range(E)]).view(F8)[:, :, :k]
        self.w1, self.s1, self.w2, self.s2 = stack(2 * F, D, seed), blocks(2 * F, D, seed, E), stack(D, F, seed + 100), blocks(D, F, seed + 1, E)
        self.place = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, S)] + [torch.empty(T, c, dtype=torch.int32, device="cuda")]
        self.q, self.s = P.empty_f8(S, D)
        self.gu = torch.empty(S, 2 * F, dtype=t, device="cuda")
        self.qf, self.sf = P.empty_f8(S, F)
        self.y = torch.empty(S, D, dtype=t, device="cuda")
        self.out = torch.empty(T, D, dtype=t, device="cuda")
        self.bufs = [*self.place, self.q.view(torch.uint8), self.s, self.gu, self.qf.view(torch.uint8), self.sf, self.y, self.out]
        for b in self.bufs:
            b.zero_()

    def run(self):
        P.dev_moe_sort(self.ids, self.E, out=self.place)
        offsets, _, position = self.place
        P.dev_moe_gather_f8(self.x, position, out=(self.q, self.s))
        P.dev_gemm_nt_f8_experts(self.q, self.s, self.w1, self.s1, offsets, out=self.gu)
        P.dev_swiglu_f8(self.gu[:, :self.F], self.gu[:, self.F:], out=(self.qf, self.sf))
        P.dev_gemm_nt_f8_experts(self.qf, self.sf, self.w2, self.s2, offsets, out=self.y)
        P.dev_moe_combine(self.y, position, self.w, out=self.out)
        return [b.clone() for b in self.bufs]


@pytest.mark.parametrize("T,c,E,D,F,t", [(1, 4, 8, 256, 200, "bf16"), (9, 2, 5, 300, 77, "f16"), (60, 3, 70, 256, 128, "f32"), (200, 4, 6, 384, 260, "bf16")])
def test_mlp_of_a_layer_with_experts(T, c, E, D, F, t):
    """Each step is held to what it got from the one before."""
    m = Moe(T, c, E, D, F, TYPES[t])
    m.run()
    offsets, order, position = m.place
    for g, w in zip(m.place, sorted_slots(m.ids.cpu(), E)):
        assert np.array_equal(g.cpu().numpy(), w)
    have = int(offsets[-1])
    wq, ws = P.dev_quantize_f8(m.x)
    at = order[:have].long() // c
    assert torch.equal(m.q[:have].view(torch.uint8), wq[:].view(torch.uint8)[at]) and torch.equal(m.s[:have], ws[at])
    part = lambda s: s.t()[:, :have].contiguous().t()
    seven = lambda v: torch.cat([v[:have], torch.full_like(v[have:], 7)])
    check_experts(seven(m.gu), m.q, m.s, m.w1, m.s1, offsets, None)
    check_swiglu(m.qf[:have], part(m.sf), m.gu[:have, :F].cpu(), m.gu[:have, F:].cpu())
    check_experts(seven(m.y), m.qf, m.sf, m.w2, m.s2, offsets, None)
    want, size = back64(m.y, position, m.w)
    h = half_step(TYPES[t])
    assert ((m.out.cpu().double() - want).abs() <= c * U * size * (1 + h) + rounding(TYPES[t], want)).all()


@pytest.mark.parametrize("T", [1, 9, 140])
def test_experts_captured_replayed_and_on_two_streams(T):
    m, n = Moe(T, 3, 6, 256, 200, torch.bfloat16), Moe(T, 3, 6, 256, 200, torch.bfloat16, seed=500)
    want, other = m.run(), n.run()
    torch.cuda.synchronize()
    stream, second = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for layer in (m, n):
        with torch.cuda.stream(stream):
            layer.run()
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                layer.run()
            graphs.append(g)
    for _ in range(4):
        for layer in (m, n):
            for buf in layer.bufs:
                buf.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):                      # two replays at once: the calls share no scratch
            graphs[0].replay()
        with torch.cuda.stream(second):
            graphs[1].replay()
        torch.cuda.synchronize()
        for layer, ref in ((m, want), (n, other)):
            assert all(torch.equal(got, w) for got, w in zip(layer.bufs, ref))
        again = m.run()                                       # eager work between the replays
        assert all(torch.equal(a, b) for a, b in zip(again, want))
    # other tokens for other experts through the same graph
    m.x.copy_(n.x)
    m.ids.copy_(n.ids)
    for buf in m.bufs:
        buf.zero_()
    graphs[0].replay()
    torch.cuda.synchronize()
    got = [b.clone() for b in m.bufs]
    for buf in m.bufs:
        buf.zero_()
    assert all(torch.equal(a, b) for a, b in zip(m.run(), got))


def test_captured_calls_that_make_their_tensors():
    """Rows without a slot are zeros in every replay, also where the replay before had written them."""
    T, c, E, k, N = 40, 3, 5, 300, 70
    x, w, y, b, sb = normal(T, k, 1).cuda(), torch.rand(T, c, device="cuda"), normal(T * c, k, 2).cuda(), codes(E * N, k, 5).view(torch.uint8), blocks(N, k, 6, E)
    b = torch.nn.functional.pad(b, (0, -k % 16)).view(F8).view(E, N, -1)[:, :, :k]
    ids = torch.zeros(T, c, dtype=torch.int32, device="cuda")

    def all_of_them():
        offsets, order, position = P.dev_moe_sort(ids, E)
        q, s = P.dev_moe_gather_f8(x, position)
        return [offsets, order, position, q.view(torch.uint8), s, P.dev_moe_gather(x, position), P.dev_gemm_nt_f8_experts(q, s, b, sb, offsets), *P.dev_moe_combine_backward(x, y, position, w)]

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        all_of_them()
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            made = all_of_them()
    for none in (0.0, 0.5, 1.0, 0.2):
        ids.copy_(random_ids(T, c, E, 7, none))
        want = all_of_them()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(made, want))
        have = int(want[0][-1])
        assert all((v[have:] == 0).all() for v in made[3:8])


def test_the_same_with_and_without_the_module_that_reads_tensors(monkeypatch):
    """Every call that it takes is made by the Python checks with the same result; what those refuse it does not take."""
    assert P._fast.gemm() == -1000 and P._fast.__name__ == "ckq_tensors"
    took = []

    class Watch:
        def __getattr__(self, name):
            f = getattr(module, name)
            return lambda *a: took.append((name, f(*a))) or took[-1][1]
    module, none = P._fast, P._Fast()
    none.absent = True

    def everything():
        m = Moe(9, 2, 5, 300, 77, torch.float16)
        out = m.run()
        a, sa, b, sb, x = codes(9, 200, 1), side(9, 200, 2, 3), codes(70, 200, 3), blocks(70, 200, 4), normal(9, 200, 5).cuda()
        q, s, y, c = *P.empty_f8(9, 200), torch.zeros(9, 200, device="cuda"), torch.zeros(9, 70, device="cuda")
        P.dev_quantize_f8(x, out=(q, s))
        P.dev_dequantize_f8(q, s, out=y)
        P.dev_gemm_nt_f8(a, sa, b, sb, sb.new_ones(70), out=c)
        rows, dy, dw = torch.zeros(18, 300, dtype=torch.float16, device="cuda"), torch.zeros(18, 300, dtype=torch.float16, device="cuda"), torch.zeros(9, 2, device="cuda")
        P.dev_moe_gather(m.x, m.place[2], out=rows)
        P.dev_moe_combine_backward(m.x, m.y, m.place[2], m.w, out=(dy, dw))
        one = P.dev_gemm_nt_f8(a[:1], sa[:1], b, sb, out=c[:1].clone())
        return out + [v.float() for v in (q, s, y, c, rows, dy, dw, one)]

    monkeypatch.setattr(P, "_fast", Watch())
    got = everything()
    assert {n for n, rc in took if rc == 0} == {"quantize", "dequantize", "swiglu", "gemm", "experts", "sort", "gather", "gather_f8", "combine", "backward"} and all(rc == 0 for _, rc in took)
    monkeypatch.setattr(P, "_fast", none)
    assert all(torch.equal(a, b) for a, b in zip(got, everything()))
    monkeypatch.setattr(P, "_fast", Watch())
    del took[:]
    test_front_ends_refuse_on_the_device()
    assert took and all(rc != 0 for _, rc in took)


def test_two_host_threads_on_streams_of_their_own():
    layers = [Moe(T, 3, 6, 256, 200, torch.bfloat16, seed=10 * T) for T in (1, 40)]
    wants = [m.run() for m in layers]
    torch.cuda.synchronize()
    failed = []

    def work(layer, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not all(torch.equal(a, b) for a, b in zip(layer.run(), want)):
                    failed.append(layer)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=pair) for pair in zip(layers, wants)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed
