"""Rows of int8 with one scale each, on the GPU against their definitions in 64 bits: the quantizer and its inverse, RMSNorm
with the residual's addition, SwiGLU, the matmul, and all of them together.

What each result may be off follows from the operations that produce it.  U = 2^-24 is half a step of fp32 relative to the
value; a result of type T adds half a step of T.  A quant is the nearest integer to t = v * 127 / a: it may be half off t, and
127 times what the fp32 operations before the rounding put on t (their number is at each test)."""
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


def codes(rows, k, seed, pitch=None):
    g = torch.Generator().manual_seed(seed)
    pitch = pitch or -(-k // 16) * 16
    q = torch.randint(-128, 128, (rows, pitch), generator=g, dtype=torch.int8)     # bytes behind a row's last are not zero
    return q.cuda()[:, :k]


def half_step(t):
    return torch.finfo(t).eps / 2


def pitched(x, extra, lead=0):
    """x on the GPU with rows `extra` elements further apart than they are long, the first `lead` elements into the memory."""
    rows, k = x.shape
    flat = torch.full((lead + rows * (k + extra) + 8,), 7.0, device="cuda").to(x.dtype)
    v = flat[lead:lead + rows * (k + extra)].view(rows, k + extra)[:, :k]
    v.copy_(x)
    return v


def check_codes(q, scale, v64, rel, scale_rel):
    """Quants and scales of rows whose values in 64 bits are v64; rel: what the operations before the rounding put on t,
    a number or one for each element."""
    q, scale = q.cpu().double(), scale.cpu().double()
    a = v64.abs().amax(1, keepdim=True).clamp_min(TINY)
    t = v64 * 127 / a
    assert (q.abs() <= 127).all()
    off = (q - t).abs()
    assert (off <= 0.5 + 127 * torch.as_tensor(rel, dtype=torch.float64) * 1.01).all(), (off.max() - 0.5).item()
    assert ((scale - a[:, 0] / 127).abs() <= scale_rel * 1.01 * a[:, 0] / 127).all()


ROWS_K = [(1, 1), (2, 2), (3, 7), (5, 8), (4, 9), (1, 17), (9, 64), (5, 127), (7, 511), (3, 512), (2, 513), (67, 896), (2, 2048), (3, 2049), (5, 4096),
          (2, 4863), (2, 8192), (3, 8193), (2, 16384), (1, 16391), (2, 32768), (2, 40003)]


# ---- quantizer ----------------------------------------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k", ROWS_K)
def test_quantize(t, rows, k):
    x = normal(rows, k, 100 * rows + k, 3.0).to(TYPES[t])
    q, s = P.dev_quantize_i8(x.cuda())
    assert q.dtype == torch.int8 and q.shape == (rows, k) and q.stride(0) % 16 == 0
    check_codes(q, s, x.double(), 2 * U, U)                 # 127 / a and its product with x
    # the largest element of a row is 127 steps
    top = x.double().abs().argmax(1)
    assert (q.cpu()[torch.arange(rows), top].abs() == 127).all()


@pytest.mark.parametrize("t", TYPES)
def test_quantize_strides_alignment_and_bytes_beside(t):
    for rows, k, extra, lead in ((5, 100, 3, 1), (3, 515, 1, 3), (6, 8, 1, 1), (2, 4096, 5, 5), (4, 9000, 7, 1)):
        x = normal(rows, k, k).to(TYPES[t])
        xd = pitched(x, extra, lead)
        base = torch.full((3 + (rows + 1) * (k + 5),), 77, dtype=torch.int8, device="cuda")
        q = base[3:3 + rows * (k + 5)].view(rows, k + 5)[:, :k]
        s = torch.full((rows + 2,), -3.0, device="cuda")
        P.dev_quantize_i8(xd, out=(q, s[1:-1]))
        want, ws = P.dev_quantize_i8(x.cuda())
        assert torch.equal(q, want) and torch.equal(s[1:-1], ws)
        left = base.clone()
        left[3:3 + rows * (k + 5)].view(rows, k + 5)[:, :k] = 77
        assert (left == 77).all() and s[0] == -3 and s[-1] == -3


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", [5, 640, 3000, 20000, 40000])
def test_quantize_rows_of_zeros_infinities_nan_and_extremes(t, k):
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
    q, s = (v.cpu() for v in P.dev_quantize_i8(x.cuda()))
    assert (q[:5] == 0).all() and s[0] == np.float32(TINY / 127) and s[1] == float("inf") and s[2] == float("inf") and s[3].isnan() and s[4].isnan()
    assert (q[5, 2:] == 127).all() and q[5, 1] == -127 and (q[7] == 127).all()
    for r in (5, 6, 7, 8):
        check_codes(q[r:r + 1], s[r:r + 1], x[r:r + 1].double(), 2 * U, U)
    y = P.dev_dequantize_i8(q.cuda(), s.cuda()).cpu()
    assert (y[0] == 0).all() and y[1].isnan().all() and y[3].isnan().all()      # infinity times zero


def test_quantize_ties_go_to_even():
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5, 0.49999997, 3.5]])
    q, s = P.dev_quantize_i8(x.cuda())
    assert q.cpu().tolist() == [[127, 0, 2, 2, 0, -2, -2, 126, -126, 0, 4]] and s.item() == 1.0


# ---- rows read back --------------------------------------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 8), (9, 1000), (2, 4097), (300, 520)])
def test_dequantize(t, rows, k):
    T = TYPES[t]
    q = codes(rows, k, rows + k, pitch=k + 3)                 # rows begin anywhere
    s = (torch.rand(rows, generator=torch.Generator().manual_seed(k)) + 0.01).cuda()
    y = P.dev_dequantize_i8(q, s, dtype=T)
    assert y.dtype == T
    want = q.cpu().double() * s.cpu().double()[:, None]
    assert ((y.cpu().double() - want).abs() <= (U + half_step(T)) * (1 + half_step(T)) * want.abs()).all()
    out = pitched(torch.zeros(rows, k).to(T), 5, 1)
    P.dev_dequantize_i8(q, s, out=out)
    assert torch.equal(out, y)


# ---- RMSNorm with the residual's addition ---------------------------------------------------

def norm64(h, gamma, eps):
    h = h.double()
    return h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * gamma.double()


def check_norm(q, s, h, gamma, eps):
    """t has six fp32 operations on it: h gamma, the largest of them and its product with r, 127 / a, and the products with r
    and with h gamma; r itself cancels.  The scale has r's: a sum of k squares whose deepest chain of additions is d long, the
    division by k, eps, the root and its inverse, and four more."""
    k = h.shape[1]
    nvec = -(-k // 8)
    wpr = 1 if nvec <= 64 else 4 if nvec <= 256 else 16
    d = 8 * -(-nvec // (64 * wpr)) + 6 + 16
    check_codes(q, s, norm64(h, gamma, eps), 6 * U, ((d + 2) / 2 + 2 + 4) * U)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k", ROWS_K)
def test_rmsnorm_with_residual(t, rows, k):
    T = TYPES[t]
    x, res = normal(rows, k, 3 * k + rows).to(T), normal(rows, k, 5 * k + rows, 2.0).to(T)
    gamma = torch.rand(k, generator=torch.Generator().manual_seed(k)) + 0.25
    q, s, h = P.dev_rmsnorm_i8(x.cuda(), gamma.cuda(), 1e-5, residual=res.cuda())
    want = x.double() + res.double()
    assert ((h.cpu().double() - want).abs() <= (U + half_step(T) * (1 + U)) * want.abs()).all()
    check_norm(q, s, h.cpu(), gamma, 1e-5)
    # without one: the norm of the stream as it is stored, the same bits
    q2, s2 = P.dev_rmsnorm_i8(h, gamma.cuda(), 1e-5)
    assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", [96, 1111, 4096, 33000])
def test_rmsnorm_in_place(t, k):
    T, rows = TYPES[t], 6
    x, res = normal(rows, k, k).to(T).cuda(), normal(rows, k, k + 1).to(T).cuda()
    gamma = torch.linspace(0.5, 2.0, k, device="cuda")
    q, s, h = P.dev_rmsnorm_i8(x, gamma, 1e-6, residual=res)
    into_residual, into_x = res.clone(), x.clone()
    q1, s1, h1 = P.dev_rmsnorm_i8(x, gamma, 1e-6, residual=into_residual, residual_out=into_residual)
    q2, s2, h2 = P.dev_rmsnorm_i8(into_x, gamma, 1e-6, residual=res, residual_out=into_x)
    for a, b, c in ((q, q1, q2), (s, s1, s2), (h, h1, h2)):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert h1.data_ptr() == into_residual.data_ptr() and h2.data_ptr() == into_x.data_ptr()


@pytest.mark.parametrize("k", [40, 700, 5000, 35000])
def test_rmsnorm_pitches_zero_rows_and_rows_that_are_not_finite(k):
    rows, T = 7, torch.bfloat16
    x, res = normal(rows, k, k).to(T), normal(rows, k, k + 1).to(T)
    x[1], res[1] = 0, 0
    x[2, k - 1] = float("nan")
    res[3, 0] = float("inf")
    x[4, 1], res[4, 1] = float("inf"), float("-inf")
    gamma = torch.ones(k)
    gamma[3] = 0
    xd, rd = pitched(x, 3, 1), pitched(res, 5, 3)
    out = pitched(torch.zeros(rows, k).to(T), 5, 1)
    q, s, h = P.dev_rmsnorm_i8(xd, gamma.cuda(), 1e-6, residual=rd, residual_out=out)
    assert torch.equal(xd.cpu().nan_to_num(9), x.nan_to_num(9)) and torch.equal(rd.cpu(), res)
    q, s, h = q.cpu(), s.cpu(), h.cpu()
    assert (q[1] == 0).all() and s[1] == np.float32(TINY / 127)
    for r in (2, 3, 4):
        assert (q[r] == 0).all() and not s[r].isfinite()
    for r in (0, 5, 6):
        check_norm(q[r:r + 1], s[r:r + 1], h[r:r + 1], gamma, 1e-6)
    # eps = 0 and a row of zeros: 0 * infinity; squares beyond fp32: no norm either
    for x, eps in ((torch.zeros(1, k), 0.0), (torch.full((1, k), 1e25), 1e-6)):
        q, s = P.dev_rmsnorm_i8(x.cuda(), gamma.cuda(), eps)
        assert (q == 0).all() and s.isnan().all()


# lengths on both sides of each change of the waves that share a row, of few rows and of more than 256
SWITCHES = [512, 513, 1024, 1025, 1536, 1537, 2049, 3000, 3080, 4096, 4097, 6144, 6145, 8192, 8193, 11008, 12288, 12289, 16385, 24577, 32768, 32769]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", SWITCHES)
def test_rmsnorm_has_the_same_bits_in_any_batch(t, k):
    """The number of rows decides how many waves share one, and nothing of what they compute."""
    x, res = normal(300, k, k).to(TYPES[t]).cuda(), normal(300, k, k + 1).to(TYPES[t]).cuda()
    gamma = (torch.rand(k, generator=torch.Generator().manual_seed(k)) + 0.25).cuda()
    q, s, h = P.dev_rmsnorm_i8(x, gamma, 1e-6, residual=res)
    for rows in (slice(0, 256), slice(0, 257), slice(7, 8), slice(290, 300)):
        q1, s1, h1 = P.dev_rmsnorm_i8(x[rows], gamma, 1e-6, residual=res[rows])
        assert torch.equal(s1, s[rows]) and torch.equal(q1, q[rows]) and torch.equal(h1, h[rows]), rows


@pytest.mark.parametrize("k", [9, 600, 40000])
def test_rmsnorm_of_small_rows_without_eps(k):
    x = normal(3, k, k) * 2.0 ** -60
    for gamma in (torch.zeros(k), torch.rand(k, generator=torch.Generator().manual_seed(k)) + 0.5):
        q, s = P.dev_rmsnorm_i8(x.cuda(), gamma.cuda(), 0.0)
        check_norm(q, s, x, gamma, 0.0)


def test_rmsnorm_in_place_of_x_in_a_single_row():
    """Which has no pitch: any will do."""
    x, res, gamma = normal(1, 500, 1).cuda(), normal(1, 500, 2).cuda(), torch.ones(500, device="cuda")
    q, s, h = P.dev_rmsnorm_i8(x, gamma, residual=res)
    assert ckq.lib().ckq_rmsnorm_i8_dev(0, x.data_ptr(), 500, res.data_ptr(), x.data_ptr(), 700, gamma.data_ptr(), 1e-6, q.zero_().data_ptr(), q.stride(0), s.data_ptr(), 1, 500,
                                        torch.cuda.current_stream().cuda_stream) == 0
    q1, s1 = P.dev_rmsnorm_i8(h, gamma)
    assert torch.equal(x, h) and torch.equal(q, q1) and torch.equal(s, s1)


SMALL = [(2.0 ** -60, 2.0 ** -65, 0.0), (2.0 ** -60, 2.0 ** -80, 0.0), (2.0 ** -74, 1.0, 0.0), (2.0 ** -100, 2.0 ** 60, 0.0), (2.0 ** -118, 1.0, 0.0), (1.0, 2.0 ** -104, 1e-6),
         (2.0 ** -60, 1.0, 1e-30), (2.0 ** -100, 2.0 ** 40, 1e-38), (2.0 ** -110, 2.0 ** 100, 2.0 ** -140), (2.0 ** -45, 2.0 ** -90, 2.0 ** -90)]


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("size,gsize,eps", SMALL)
def test_rmsnorm_of_rows_whose_squares_or_products_are_below_fp32(t, size, gsize, eps):
    """The same bounds as of any row, with and without a residual, in place, and the same bits in any batch."""
    for k in (5, 256, 1001, 4096, 11001, 40000):
        x = (normal(300 if k < 5000 else 3, k, k) * size).to(TYPES[t])
        gamma = (torch.rand(k, generator=torch.Generator().manual_seed(k)) + 0.5) * gsize
        x[1] *= 2.0 ** 20 if size < 1 else 1.0
        q, s = P.dev_rmsnorm_i8(x.cuda(), gamma.cuda(), eps)
        check_norm(q, s, x, gamma, eps)
        for rows in (slice(0, 1), slice(1, 3)):
            q1, s1 = P.dev_rmsnorm_i8(x[rows].cuda(), gamma.cuda(), eps)
            assert torch.equal(q1, q[rows]) and torch.equal(s1, s[rows])
        half = (x.double() / 2).to(TYPES[t])
        into = half[:3].cuda()
        q2, s2, h2 = P.dev_rmsnorm_i8(half[:3].cuda(), gamma.cuda(), eps, residual=into, residual_out=into)
        check_norm(q2, s2, h2.cpu(), gamma, eps)


def test_rmsnorm_of_small_rows_in_half_precision():
    for size, gsize in ((2.0 ** -20, 2.0 ** -100), (2.0 ** -22, 2.0 ** -80), (1.0, 2.0 ** -102)):
        for k in (300, 9000):
            x = (normal(3, k, k) * size).half()
            gamma = (torch.rand(k, generator=torch.Generator().manual_seed(k)) + 0.5) * gsize
            q, s = P.dev_rmsnorm_i8(x.cuda(), gamma.cuda(), 0.0)
            check_norm(q, s, x, gamma, 0.0)


@pytest.mark.parametrize("k", [7, 512, 3000, 12000, 40000])
def test_rmsnorm_zeros_and_infinities_among_small_rows(k):
    x = normal(6, k, k) * 2.0 ** -80
    x[1] = 0
    x[2, 1] = float("inf")
    x[3, k - 1] = float("nan")
    ones = torch.ones(k)
    q, s = (v.cpu() for v in P.dev_rmsnorm_i8(x.cuda(), ones.cuda(), 0.0))
    assert (q[1:4] == 0).all() and s[1].isnan() and not s[2].isfinite() and s[3].isnan()
    check_norm(q[[0, 4, 5]], s[[0, 4, 5]], x[[0, 4, 5]], ones, 0.0)
    q, s = (v.cpu() for v in P.dev_rmsnorm_i8(x.cuda(), ones.cuda(), 2.0 ** -120))      # zeros over sqrt(eps)
    assert (q[1] == 0).all() and s[1] == np.float32(TINY / 127)
    for bad in (float("nan"), float("inf")):
        ones[0] = bad
        q, s = (v.cpu() for v in P.dev_rmsnorm_i8(x[4:].cuda(), ones.cuda(), 0.0))
        assert (q == 0).all() and not s.isfinite().any()


# ---- SwiGLU ----------------------------------------------------------------------------------

def check_swiglu(q, s, gate, up):
    """v: the exponent has two roundings, so e is |g| 2 U off, and the instruction's ulp (2 U); of that e / (1 + e) gets into v,
    with the sum's U, the reciprocal's 2 U and two products.  t has those twice (its own and the largest's), the division and the
    last product."""
    g, u = gate.double(), up.double()
    e = torch.exp(-g)
    v = g / (1 + e) * u
    rel = (1 - 1 / (1 + e)) * (2 * g.abs() + 2) * U + 5 * U
    a = v.abs().amax(1, keepdim=True)
    rel_top = torch.where(v.abs() >= a * (1 - 2.0 ** -18), rel, torch.zeros_like(rel)).amax(1, keepdim=True)
    check_codes(q, s, v, rel + rel_top + 2 * U, (rel_top[:, 0] + U))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k", ROWS_K)
def test_swiglu(t, rows, k):
    both = normal(rows, 2 * k, 7 * k + rows, 3.0).to(TYPES[t])
    d = both.cuda()
    q, s = P.dev_swiglu_i8(d[:, :k], d[:, k:])               # halves of one tensor
    check_swiglu(q, s, both[:, :k], both[:, k:])
    gate, up = both[:, :k].contiguous().cuda(), both[:, k:].contiguous().cuda()
    q2, s2 = P.dev_swiglu_i8(gate, up)
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_swiglu_far_gates_count_where_up_is_large():
    """1 + exp(-gate) up to the end of fp32, whose reciprocal is below its normal numbers."""
    for rows, k in ((3, 40), (2, 20000)):
        gate = -86.0 - 2.7 * torch.rand(rows, k, generator=torch.Generator().manual_seed(k))
        up = normal(rows, k, k + 1) * 2.0 ** 120
        q, s = P.dev_swiglu_i8(gate.cuda(), up.cuda())
        check_swiglu(q, s, gate, up)


def test_swiglu_far_gates():
    gate = torch.tensor([[-200.0, -100.0, -88.0, -30.0, 0.0, 30.0, 100.0, 200.0]])
    up = torch.ones(1, 8)
    q, s = P.dev_swiglu_i8(gate.cuda(), up.cuda())
    assert q.cpu().tolist() == [[0, 0, 0, 0, 0, 19, 64, 127]] and s.item() == np.float32(200.0) / np.float32(127.0)
    gate[0, 3] = float("nan")
    q, s = P.dev_swiglu_i8(gate.cuda(), up.cuda())
    assert (q == 0).all() and s.isnan().all()


# ---- more than 256 rows: fewer waves share a row, with two to four vectors a thread ------------------

def norm_chain(k):
    """Longest chain of additions of a row's sum of squares, a function of its length alone: a thread's elements, the tree of a wave,
    groups of 512 sixteen apart, and up to sixteen of these sums; rows that are read twice: a thread's elements, the tree, the waves."""
    nvec, groups = -(-k // 8), -(-k // 512)
    return 8 * -(-nvec // 1024) + 6 + 16 if k < 8 or k > 32768 else 8 + 6 + -(-groups // 16) + min(16, groups)


def check_many_norm(q, s, h, gamma, eps):
    check_codes(q, s, norm64(h, gamma, eps), 6 * U, ((norm_chain(h.shape[1]) + 2) / 2 + 2 + 4) * U)


MANY = SWITCHES + [5, 100, 777, 1531, 2001, 3071, 5999, 9001, 12281, 20001]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", MANY)
def test_quantize_many_rows(t, k):
    x = normal(259, k, k, 3.0).to(TYPES[t])
    q, s = P.dev_quantize_i8(x.cuda())
    check_codes(q, s, x.double(), 2 * U, U)
    base = torch.full((259, k + 5), 77, dtype=torch.int8, device="cuda")
    q2, s2 = P.dev_quantize_i8(pitched(x, 3, 1), out=(base[:, :k], torch.empty_like(s)))
    assert torch.equal(q, q2) and torch.equal(s, s2) and (base[:, k:] == 77).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", MANY)
def test_rmsnorm_many_rows(t, k):
    T, rows = TYPES[t], 258
    x, res = normal(rows, k, 3 * k).to(T), normal(rows, k, 5 * k, 2.0).to(T)
    gamma = torch.rand(k, generator=torch.Generator().manual_seed(k)) + 0.25
    q, s, h = P.dev_rmsnorm_i8(x.cuda(), gamma.cuda(), 1e-5, residual=res.cuda())
    want = x.double() + res.double()
    assert ((h.cpu().double() - want).abs() <= (U + half_step(T) * (1 + U)) * want.abs()).all()
    check_many_norm(q, s, h.cpu(), gamma, 1e-5)
    for out in (P.dev_rmsnorm_i8(h, gamma.cuda(), 1e-5), P.dev_rmsnorm_i8(pitched(h.cpu(), 5, 3), gamma.cuda(), 1e-5)):
        assert torch.equal(out[0], q) and torch.equal(out[1], s)
    for into in ("x", "residual"):                            # in place, at a pitch
        xd, rd = pitched(x, 3, 1), pitched(res, 3, 1)
        q1, s1, h1 = P.dev_rmsnorm_i8(xd, gamma.cuda(), 1e-5, residual=rd, residual_out=xd if into == "x" else rd)
        assert torch.equal(q1, q) and torch.equal(s1, s) and torch.equal(h1, h), into


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", MANY)
def test_swiglu_many_rows(t, k):
    both = normal(257, 2 * k, 7 * k, 3.0).to(TYPES[t])
    d = both.cuda()
    q, s = P.dev_swiglu_i8(d[:, :k], d[:, k:])
    check_swiglu(q, s, both[:, :k], both[:, k:])
    q2, s2 = P.dev_swiglu_i8(d[40:41, :k], d[40:41, k:])
    assert torch.equal(q2, q[40:41]) and torch.equal(s2, s[40:41])


# ---- matmul ------------------------------------------------------------------------------------

def check_matmul(c, a, sa, b, sb, bias):
    """The sum is exact; it is converted, scaled twice, the bias added (U each) and the result rounded to its type: to an infinity
    from half a step beyond the type's largest value on (65520 in half precision, whose last step is 32)."""
    T = c.dtype
    p = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    want = p if bias is None else p + bias.double()
    got = c.double()
    tol = 3 * U * 1.01 * p.abs() + (U + half_step(T)) * 1.01 * (want.abs() + 3 * U * p.abs()) + (2.0 ** -25 if T == torch.float16 else 0)
    off = (got - want).abs()
    top = torch.finfo(T).max * (1 + half_step(T) / 2)
    beyond = want.abs() - 4 * U * p.abs() - 4 * U * want.abs() >= top
    near = want.abs() + 4 * U * p.abs() + 4 * U * want.abs() >= top
    assert (got[beyond] == torch.sign(want[beyond]) * float("inf")).all()
    fine = (off <= tol) | beyond | (near & got.isinf())
    assert fine.all(), (off / tol.clamp_min(1e-30)).max().item()


def matmul_case(M, N, K, t, bias, seed=1, pitch_a=0, pitch_b=0, pitch_c=0):
    a = codes(M, K, seed, -(-K // 16) * 16 + 16 * pitch_a)
    b = codes(N, K, seed + 1, -(-K // 16) * 16 + 16 * pitch_b)
    g = torch.Generator().manual_seed(seed + 2)
    sa = (torch.rand(M, generator=g) * 0.01 + 0.001).cuda()
    sb = (torch.rand(N, generator=g) * 0.01 + 0.001).cuda()
    bv = torch.randn(N, generator=g).cuda() if bias else None
    out = torch.full((M, N + pitch_c), 5.0, device="cuda").to(TYPES[t])
    c = P.dev_gemm_nt_i8(a, sa, b, sb, bv, out=out[:, :N])
    check_matmul(c, a, sa, b, sb, bv)
    assert (out[:, N:] == 5).all()
    return c


MNK = [(1, 1, 1), (1, 5, 15), (1, 130, 16), (1, 300, 4096), (1, 1001, 4847), (2, 33, 64), (3, 100, 1000), (4, 257, 513), (5, 64, 130), (7, 129, 2049), (8, 896, 4864),
       (9, 40, 333), (13, 300, 1024), (16, 128, 256), (17, 31, 127), (31, 200, 65), (32, 64, 128), (33, 257, 1025), (63, 500, 700), (64, 192, 896), (65, 64, 64),
       (100, 333, 2047), (127, 127, 127), (128, 256, 512), (129, 1001, 129), (255, 250, 300), (256, 256, 1024), (257, 257, 257), (333, 1001, 4847), (513, 800, 640)]


@pytest.mark.parametrize("M,N,K", MNK)
def test_matmul(M, N, K):
    for i, t in enumerate(TYPES):
        matmul_case(M, N, K, t, bias=i != 1, seed=M + N + K + i)


@pytest.mark.parametrize("M,N,K", [(1, 70, 100), (3, 65, 200), (6, 33, 90), (14, 100, 77), (40, 130, 300), (130, 150, 170), (300, 270, 400)])
@pytest.mark.parametrize("t", TYPES)
def test_matmul_pitches(M, N, K, t):
    matmul_case(M, N, K, t, bias=True, pitch_a=3, pitch_b=5, pitch_c=3)


@pytest.mark.parametrize("M", [1, 4, 11, 40, 150, 300])
def test_matmul_tail_of_k(M):
    """Every length of a last piece: bytes behind a row's last take no part."""
    for K in list(range(1, 34)) + [47, 63, 64, 65, 79, 80, 81, 95, 97, 111, 112, 127, 128, 129, 143, 145, 160, 191, 193, 255, 257]:
        matmul_case(M, 37, K, "f32", bias=False, seed=K)


# the kernels that a call may be sent to (ckq_launch_i8_kernel), by the tokens and the rows of their tiles
KERNELS = [(256, 256), (256, 192), (256, 128), (128, 192), (128, 128), (64, 128), (64, 64), (32, 48), (32, 32), (16, 16), (16, 32)]
TWO, STREAM = 11, 12


@pytest.fixture
def kernel():
    yield ckq.lib().ckq_launch_set_i8_kernel
    ckq.lib().ckq_launch_set_i8_kernel(-1)


@pytest.mark.parametrize("which", range(len(KERNELS)))
def test_matmul_every_kernel(kernel, which):
    bt, bn = KERNELS[which]
    kernel(which)
    L = ckq.lib()
    assert L.ckq_launch_i8_kernel(5, 5, 5) == which
    for i, (M, N, K) in enumerate([(1, 1, 1), (bt, bn, 128), (bt + 1, bn + 1, 129), (2 * bt - 1, 3 * bn - 5, 300), (3, 9 * bn + 7, 1100), (9 * bt + 3, 5, 700),
                                   (bt - 1, bn - 1, 127), (2 * bt + 5, 2 * bn + 8, 2048), (17 * bt + 9, 3 * bn, 256)]):
        matmul_case(M, N, K, list(TYPES)[i % 3], bias=i % 2 == 0, seed=i, pitch_a=i % 3, pitch_b=i % 2, pitch_c=i % 4)


@pytest.mark.parametrize("which", range(len(KERNELS)))
def test_matmul_every_kernel_tail_of_k(kernel, which):
    kernel(which)
    for K in list(range(1, 18)) + [31, 33, 47, 63, 64, 65, 111, 112, 113, 127, 128, 129, 143, 145, 255, 256, 257, 383, 384, 385, 400, 511, 512, 513, 640, 641, 895, 1023, 1025, 1151]:
        matmul_case(5, 37, K, "f32", bias=False, seed=K)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", [(4, 300, 1100), (150, 333, 2049)])
def test_matmul_every_kernel_has_the_same_bits(kernel, M, N, K, t):
    """And a token the same results alone, in any company."""
    a, b = codes(M, K, 1), codes(N, K, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    sa, sb, bias = (torch.rand(n, device="cuda", generator=g) for n in (M, N, N))
    want = [P.dev_gemm_nt_i8(a, sa, b, sb, v, dtype=TYPES[t]) for v in (None, bias)]
    for which in range(len(KERNELS)):
        kernel(which)
        for v, w in zip((None, bias), want):
            assert torch.equal(P.dev_gemm_nt_i8(a, sa, b, sb, v, dtype=TYPES[t]), w), which
    kernel(-1)
    for rows in (slice(0, 1), slice(1, 3), slice(0, 4), slice(M // 2, M), slice(0, min(M, 17))):
        assert torch.equal(P.dev_gemm_nt_i8(a[rows], sa[rows], b, sb, bias, dtype=TYPES[t]), want[1][rows])


@pytest.mark.parametrize("M,N,K", [(4000, 4300, 130), (2048, 8193, 128), (8100, 2100, 200)])
def test_matmul_two_sizes_of_tiles(kernel, M, N, K):
    kernel(TWO)
    assert ckq.lib().ckq_launch_i8_kernel(M, N, K) == TWO
    matmul_case(M, N, K, "bf16", bias=True)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", [(2048, 8500, 4096), (2040, 11008, 1111), (300, 40000, 2049)])
def test_matmul_two_sizes_of_tiles_over_long_rows(kernel, M, N, K, t):
    """And the bits of a launch of one size."""
    kernel(TWO)
    assert ckq.lib().ckq_launch_i8_kernel(M, N, K) == TWO
    c = matmul_case(M, N, K, t, bias=True, pitch_a=1, pitch_c=1)
    for which in (0, 3, 9):
        kernel(which)
        a, b = codes(M, K, 1, -(-K // 16) * 16 + 16), codes(N, K, 2)
        g = torch.Generator().manual_seed(3)
        sa, sb = (torch.rand(M, generator=g) * 0.01 + 0.001).cuda(), (torch.rand(N, generator=g) * 0.01 + 0.001).cuda()
        assert torch.equal(P.dev_gemm_nt_i8(a, sa, b, sb, torch.randn(N, generator=g).cuda(), dtype=TYPES[t]), c), which


@pytest.mark.parametrize("K", [1, 15, 16, 17, 100, 1008, 1023, 1024, 1025, 1040, 2047, 2048, 2049, 4095, 4097, 6000, 8191, 8193, 11008])
def test_matmul_rows_streamed(kernel, K):
    for M in (1, 2, 3, 4):
        assert (ckq.lib().ckq_launch_i8_kernel(M, 100, K) == STREAM) == (M <= 2 or K <= 1024)
        for i, N in enumerate((1, 3, 4, 5, 16, 18, 61)):
            matmul_case(M, N, K, list(TYPES)[i % 3], bias=i % 2 == 0, seed=K + N, pitch_b=i % 2, pitch_c=i % 3)


@pytest.mark.parametrize("M", [1, 2, 6, 16, 33, 130, 260])
def test_matmul_sums_are_exact_to_the_longest_row(kernel, M):
    for which in [-1] + list(range(len(KERNELS))) * (M == 6):
        kernel(which)
        longest_row(M)


def longest_row(M):
    K, N = 131071, 19
    a = torch.full((M, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    b = torch.full((N, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    b[1] = 127
    b[2, 1::2] = 127
    one = torch.ones(max(M, N), device="cuda")
    c = P.dev_gemm_nt_i8(a, one[:M], b, one[:N]).double()
    assert (c[:, 0] == 128.0 * 128 * K).all() or ((c[:, 0] - 128.0 * 128 * K).abs() <= U * 128 * 128 * K).all()
    assert ((c[:, 1] + 128.0 * 127 * K).abs() <= U * 128 * 127 * K).all()
    s2 = float((a[:1].double() @ b[2:3].double().t()).item())
    assert ((c[:, 2] - s2).abs() <= U * abs(s2)).all()


def test_matmul_scales_that_are_not_finite_stay_in_their_rows():
    for M, N, K in ((3, 40, 64), (20, 70, 100), (150, 140, 200)):
        a, b = codes(M, K, 1), codes(N, K, 2)
        sa, sb = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
        a[1] = 0
        sa[1] = float("nan")
        a[2] = 0
        sa[2] = float("inf")
        c = P.dev_gemm_nt_i8(a, sa, b, sb)
        assert c[1].isnan().all() and c[2].isnan().all() and c[0].isfinite().all()
        keep = [i for i in range(M) if i not in (1, 2)]
        check_matmul(c[keep], a[keep], sa[keep], b, sb, None)


def test_matmul_unaligned_results():
    """C of any pitch, starting at any element."""
    for M, N, K in ((1, 50, 64), (5, 33, 80), (40, 130, 128), (140, 257, 64)):
        a, b = codes(M, K, 3), codes(N, K, 4)
        sa, sb = torch.rand(M, device="cuda"), torch.rand(N, device="cuda")
        for t in TYPES.values():
            out = pitched(torch.zeros(M, N).to(t), 1, 1)
            P.dev_gemm_nt_i8(a, sa, b, sb, out=out)
            assert torch.equal(out, P.dev_gemm_nt_i8(a, sa, b, sb, dtype=t))


def test_launches_in_parts():
    """More rows than one launch has (2^22 of a matmul, 2^21 of the producers)."""
    a, b = codes(2, 16, 1), codes((1 << 22) + 37, 16, 2)
    sa, sb, bias = torch.rand(2, device="cuda"), torch.rand(b.shape[0], device="cuda"), torch.rand(b.shape[0], device="cuda")
    check_matmul(P.dev_gemm_nt_i8(a[:1], sa[:1], b, sb, bias), a[:1], sa[:1], b, sb, bias)
    c = P.dev_gemm_nt_i8(b, sb, a, sa, dtype=torch.float16)
    check_matmul(c, b, sb, a, sa, None)
    x = torch.randn((1 << 21) + 3, 9, device="cuda")
    q, s = P.dev_quantize_i8(x)
    for part in (slice(0, 50), slice((1 << 21) - 7, None)):
        q2, s2 = P.dev_quantize_i8(x[part].contiguous())
        assert torch.equal(q[part], q2) and torch.equal(s[part], s2)
    res = torch.ones_like(x)
    qn, sn, h = P.dev_rmsnorm_i8(x, torch.ones(9, device="cuda"), residual=res)
    q2, s2, h2 = P.dev_rmsnorm_i8(x[-9:].contiguous(), torch.ones(9, device="cuda"), residual=res[-9:].contiguous())
    assert torch.equal(qn[-9:], q2) and torch.equal(sn[-9:], s2) and torch.equal(h, x + res) and torch.equal(h[-9:], h2)


def test_offsets_beyond_32_bits():
    """Rows whose distance from the first does not fit in 32 bits of elements."""
    far = (1 << 30) + 24
    x = torch.empty(4 * far, dtype=torch.float16, device="cuda").as_strided((5, 100), (far - 100, 1))
    x.copy_(normal(5, 100, 1).half())
    q = torch.empty(4 * far, dtype=torch.int8, device="cuda").as_strided((5, 100), (far - 100, 1))
    q, s = P.dev_quantize_i8(x, out=(q, torch.empty(5, device="cuda")))
    q2, s2 = P.dev_quantize_i8(x.contiguous())
    assert torch.equal(q, q2) and torch.equal(s, s2)
    y = P.dev_dequantize_i8(q, s, out=x)
    assert torch.equal(y.contiguous(), P.dev_dequantize_i8(q2, s2, dtype=torch.float16))
    r = P.dev_rmsnorm_i8(x, torch.ones(100, device="cuda"), residual=x, residual_out=x)
    r2 = P.dev_rmsnorm_i8(y2 := P.dev_dequantize_i8(q2, s2, dtype=torch.float16), torch.ones(100, device="cuda"), residual=y2)
    assert all(torch.equal(u.contiguous(), v) for u, v in zip(r, r2))
    del x, q, y, r
    pitch = 1 << 22                                           # the longest that a matmul's operands may have
    big = torch.empty(1100 * pitch, dtype=torch.int8, device="cuda")
    a = big.as_strided((1100, 200), (pitch, 1))
    a.copy_(codes(1100, 200, 3))
    b, sa, sb = codes(70, 200, 4), torch.rand(1100, device="cuda"), torch.rand(70, device="cuda")
    check_matmul(P.dev_gemm_nt_i8(a, sa, b, sb), a, sa, b, sb, None)
    check_matmul(P.dev_gemm_nt_i8(b, sb, a, sa), b, sb, a, sa, None)
    check_matmul(P.dev_gemm_nt_i8(b[:3], sb[:3], a, sa), b[:3], sb[:3], a, sa, None)
    out = torch.empty(3 * far, dtype=torch.float16, device="cuda").as_strided((4, 1100), (far - 1100, 1))
    for rows in (1, 4):
        P.dev_gemm_nt_i8(b[:rows], sb[:rows], a, sa, out=out[:rows])
        check_matmul(out[:rows], b[:rows], sb[:rows], a, sa, None)
    P.dev_gemm_nt_i8(codes(4, 200, 9), sb[:4], a, sa, out=out)
    check_matmul(out, codes(4, 200, 9), sb[:4], a, sa, None)


def test_front_ends_refuse_on_the_device():
    a, s = codes(2, 32, 1), torch.ones(2, device="cuda")
    x = torch.zeros(2, 32, device="cuda")
    bad = [lambda: P.dev_quantize_i8(x.double()), lambda: P.dev_quantize_i8(x.t()), lambda: P.dev_quantize_i8(x[:0]),
           lambda: P.dev_quantize_i8(x[:, ::2]), lambda: P.dev_quantize_i8(x, out=(a, s[:1])), lambda: P.dev_quantize_i8(x.expand(4, 2, 32)),
           lambda: P.dev_gemm_nt_i8(a, s, codes(3, 16, 1), s), lambda: P.dev_gemm_nt_i8(a[:, 1:], s, a[:, 1:], s),
           lambda: P.dev_gemm_nt_i8(a, s, a, s, bias=x[0]), lambda: P.dev_gemm_nt_i8(a, s.cpu(), a, s),
           lambda: P.dev_gemm_nt_i8(torch.zeros(2, 31, dtype=torch.int8, device="cuda"), s, codes(2, 31, 1), s),
           lambda: P.dev_rmsnorm_i8(x, x[0], residual=x.half()), lambda: P.dev_rmsnorm_i8(x, x[0], residual_out=x),
           lambda: P.dev_swiglu_i8(x, x[:, :16]), lambda: P.dev_swiglu_i8(x, pitched(x, 4)), lambda: P.dev_dequantize_i8(a, s, out=x.double()),
           lambda: P.dev_gemm_nt_i8(a, s, a, s, out=torch.zeros(2, 1, device="cuda").expand(2, 2))]
    for i, f in enumerate(bad):
        with pytest.raises(ckq.CkqError):
            f()
            pytest.fail("call %d" % i)


# ---- all of them together -------------------------------------------------------------------------

class Mlp:
    """The MLP half of a decoder layer on the buffers of a serving loop."""

    def __init__(self, M, D, F, T, seed=5):
        self.T, self.F, self.eps = T, F, 1e-5
        self.x, self.res = normal(M, D, seed).to(T).cuda(), normal(M, D, seed + 1).to(T).cuda()
        self.gamma = (torch.rand(D, generator=torch.Generator().manual_seed(seed)) + 0.5).cuda()
        self.w1, self.s1 = P.dev_quantize_i8(normal(2 * F, D, seed + 2, 0.05).cuda())
        self.w2, self.s2 = P.dev_quantize_i8(normal(D, F, seed + 3, 0.05).cuda())
        self.h = torch.empty_like(self.res)
        self.q, self.s = P.empty_i8(M, D), torch.empty(M, device="cuda")
        self.gu = torch.empty(M, 2 * F, dtype=T, device="cuda")
        self.qf, self.sf = P.empty_i8(M, F), torch.empty(M, device="cuda")
        self.c = torch.empty(M, D, dtype=T, device="cuda")

    def run(self):
        P.dev_rmsnorm_i8(self.x, self.gamma, self.eps, residual=self.res, residual_out=self.h, out=(self.q, self.s))
        P.dev_gemm_nt_i8(self.q, self.s, self.w1, self.s1, out=self.gu)
        P.dev_swiglu_i8(self.gu[:, :self.F], self.gu[:, self.F:], out=(self.qf, self.sf))
        P.dev_gemm_nt_i8(self.qf, self.sf, self.w2, self.s2, out=self.c)
        return [v.clone() for v in (self.h, self.q, self.s, self.gu, self.qf, self.sf, self.c)]


@pytest.mark.parametrize("M,D,F,t", [(1, 256, 640, "bf16"), (5, 896, 1001, "f16"), (70, 500, 777, "f32"), (300, 512, 1408, "bf16")])
def test_mlp_of_a_layer(M, D, F, t):
    m = Mlp(M, D, F, TYPES[t])
    h, q, s, gu, qf, sf, c = m.run()
    check_norm(q, s, h.cpu(), m.gamma.cpu(), m.eps)
    check_matmul(gu, q, s, m.w1, m.s1, None)
    check_swiglu(qf, sf, gu[:, :F].cpu(), gu[:, F:].cpu())
    check_matmul(c, qf, sf, m.w2, m.s2, None)


@pytest.mark.parametrize("M", [1, 9, 140])
def test_mlp_captured_replayed_and_on_two_streams(M):
    m, n = Mlp(M, 512, 1000, torch.bfloat16), Mlp(M, 512, 1000, torch.bfloat16, seed=50)
    want, other = m.run(), n.run()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graphs = []
    for layer in (m, n):
        with torch.cuda.stream(stream):
            layer.run()
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                layer.run()
            graphs.append(g)
    second = torch.cuda.Stream()
    for _ in range(4):
        for layer in (m, n):
            for buf in (layer.h, layer.q, layer.gu, layer.qf, layer.c):
                buf.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):                      # two replays at once: the calls share no scratch
            graphs[0].replay()
        with torch.cuda.stream(second):
            graphs[1].replay()
        torch.cuda.synchronize()
        for layer, ref in ((m, want), (n, other)):
            for got, w in zip((layer.h, layer.q, layer.s, layer.gu, layer.qf, layer.sf, layer.c), ref):
                assert torch.equal(got, w)
        again = m.run()                                       # eager work between the replays
        assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_two_host_threads_on_streams_of_their_own():
    layers = [Mlp(M, 512, 1000, torch.bfloat16, seed=10 * M) for M in (1, 40)]
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
