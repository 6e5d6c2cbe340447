"""The operators of the int8 path (int8 weights with one scale a channel, int8 activations with one scale a token): what is measured of them.

Five kinds of work:

  matmul     C = (A B^T) * (scale of the token) * (scale of the channel) + bias, A and B in int8.
  norm       the residual's addition, RMSNorm and its rows in 8 bits.
  swiglu     SiLU(gate) * up in 8 bits, gate and up side by side as the projection before leaves them.
  quantize   rows of floats (attention outputs, weights) in 8 bits.
  mlp        the MLP half of a decoder layer, all of them together: norm, gate and up, SwiGLU, down.

8-bit rows come back as the values they stand for, in bfloat16, beside their scales.  Where rows are of an odd length the
next one begins at a multiple of 16 bytes, as the library's own allocation has it."""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
TINY = 2.0 ** -100            # no row is scaled by less


# ---- cases --------------------------------------------------------------------------

def listed():
    return [
        # interactive decode: the gate projection of a 7B model, one token
        {"name": "matmul_t1_11008x4096", "kind": "matmul", "M": 1, "N": 11008, "K": 4096, "t": "bf16", "bias": False},
        # continuous batching: the down projection, an odd number of sequences
        {"name": "matmul_t13_4096x11008", "kind": "matmul", "M": 13, "N": 4096, "K": 11008, "t": "f32", "bias": True},
        # a prompt whose length, and a layer whose sizes, fit no tile
        {"name": "matmul_t333_1001x4847", "kind": "matmul", "M": 333, "N": 1001, "K": 4847, "t": "f16", "bias": True},
        # a prompt of ordinary length
        {"name": "matmul_t512_11008x4096", "kind": "matmul", "M": 512, "N": 11008, "K": 4096, "t": "bf16", "bias": False},
        # a long prompt
        {"name": "matmul_t2048_11008x4096", "kind": "matmul", "M": 2048, "N": 11008, "K": 4096, "t": "bf16", "bias": False},
        # decode: the norm before a projection, one token, where latency is all there is
        {"name": "norm_t1_4096", "kind": "norm", "M": 1, "K": 4096, "t": "bf16"},
        # a long prompt through the same norm
        {"name": "norm_t2048_4096", "kind": "norm", "M": 2048, "K": 4096, "t": "bf16"},
        # a short prompt through a small model whose rows are odd, fp32 activations
        {"name": "swiglu_t93_4863", "kind": "swiglu", "M": 93, "K": 4863, "t": "f32"},
        # a long prompt between gate/up and down
        {"name": "swiglu_t2048_11008", "kind": "swiglu", "M": 2048, "K": 11008, "t": "bf16"},
        # batched decode of a small model: the attention outputs of five sequences on their way into the output projection
        {"name": "quantize_t5_896", "kind": "quantize", "M": 5, "K": 896, "t": "f16"},
        # a weight matrix, a row a channel, when a model is loaded
        {"name": "quantize_w_11008x4096", "kind": "quantize", "M": 11008, "K": 4096, "t": "f32"},
        # one token through the MLP half of a 7B layer
        {"name": "mlp_t1_4096x11008", "kind": "mlp", "M": 1, "K": 4096, "F": 11008, "t": "bf16"},
    ]


MOST = 2 * 2048 * 11008 * 4096           # operations of the longest listed prompt


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["matmul", "matmul", "matmul", "norm", "swiglu", "quantize", "mlp"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "matmul":
        N, K = _log(rng, 32, 32000), _log(rng, 32, 11008)
        if rng.random() < 0.5:               # as often as not a width that a model would have
            K = max(64, K - K % 64)
        M = max(1, min(_log(rng, 1, 2048), MOST // (2 * N * K)))
        return {"kind": kind, "M": M, "N": N, "K": K, "t": t, "bias": rng.random() < 0.5}
    if kind == "mlp":
        K = max(64, 64 * round(_log(rng, 256, 4096) / 64))
        F = max(64, 16 * round(K * rng.uniform(2.0, 2.6875) / 16))
        return {"kind": kind, "M": max(1, min(_log(rng, 1, 512), MOST // (6 * K * F))), "K": K, "F": F, "t": rng.choice(["bf16", "f16"])}
    K = _log(rng, 64, 11008)
    if rng.random() < 0.5:
        K = max(64, K - K % 64)
    return {"kind": kind, "M": _log(rng, 1, 11008 if kind == "quantize" else 2048), "K": K, "t": t}


# ---- inputs ---------------------------------------------------------------------------

def _pitch(k):
    return -(-k // 16) * 16


def _rows(gen, m, k, t):
    """Activations: N(0, 1) with every 61st channel some ten times larger, as the residual stream of a trained model has them."""
    x = torch.randn(m, k, device="cuda", generator=gen)
    x[:, 17::61] *= 10
    return x.to(t)


def _codes(gen, n, k):
    """int8 rows as quantized weights and activations are: normal, the largest of a row near 127."""
    q = torch.randn(n, _pitch(k), device="cuda", generator=gen).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
    return q[:, :k]


def _scales(gen, n, size):
    return torch.rand(n, device="cuda", generator=gen).add_(0.5).mul_(size)


def _i8(m, k):
    return torch.empty(m, _pitch(k), dtype=torch.int8, device="cuda")[:, :k]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    M, K, t = case["M"], case["K"], DTYPES[case["t"]]
    s = {"kind": case["kind"], "t": t}
    if case["kind"] == "matmul":
        N = case["N"]
        s.update(a=_codes(gen, M, K), sa=_scales(gen, M, 1 / 32), b=_codes(gen, N, K), sb=_scales(gen, N, 0.02 / 32),
                 bias=torch.randn(N, device="cuda", generator=gen) if case["bias"] else None,
                 c=torch.empty(M, N, dtype=t, device="cuda"))
        return s
    # the buffers that a serving loop keeps
    s.update(q=_i8(M, K), scale=torch.empty(M, device="cuda"), values=torch.empty(M, K, dtype=torch.bfloat16, device="cuda"))
    if case["kind"] in ("norm", "mlp"):
        s.update(x=_rows(gen, M, K, t), residual=_rows(gen, M, K, t), out=torch.empty(M, K, dtype=t, device="cuda"),
                 gamma=torch.rand(K, device="cuda", generator=gen).add_(0.5))
    elif case["kind"] == "swiglu":
        s["gate_up"] = torch.randn(M, 2 * K, device="cuda", generator=gen).mul_(2).to(t)
    else:
        s["x"] = _rows(gen, M, K, t)
    if case["kind"] == "mlp":
        F = case["F"]
        s.update(w1=_codes(gen, 2 * F, K), s1=_scales(gen, 2 * F, 0.02 / 32), w2=_codes(gen, K, F), s2=_scales(gen, K, 0.02 / 32),
                 gate_up=torch.empty(M, 2 * F, dtype=t, device="cuda"), qf=_i8(M, F), scalef=torch.empty(M, device="cuda"),
                 c=torch.empty(M, K, dtype=t, device="cuda"))
    return s


# ---- one pass: the plain forms ----------------------------------------------------------

def _eight_bits(v):
    """The codes of fp32 rows, and their scales."""
    a = v.abs().amax(1, keepdim=True).clamp_min(TINY)
    return (v * (127.0 / a)).round(), a / 127.0


def _norm(x, residual, gamma):
    h = (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    return h, f * torch.rsqrt(f.square().mean(1, keepdim=True) + EPS) * gamma


def _swiglu(gate_up):
    g, u = gate_up.float().chunk(2, 1)
    return g / (1.0 + torch.exp(-g)) * u


def _matmul(a, sa, b, sb, bias, t):
    c = torch.mm(a.float(), b.float().t()) * sa * sb
    return (c if bias is None else c + bias).to(t)


def _plain(s):
    if s["kind"] == "matmul":
        return {"c": _matmul(s["a"], s["sa"][:, None], s["b"], s["sb"], s["bias"], s["t"])}
    if s["kind"] == "mlp":
        h, v = _norm(s["x"], s["residual"], s["gamma"])
        gate_up = _matmul(*_eight_bits(v), s["w1"], s["s1"], None, s["t"])
        return {"residual": h, "c": _matmul(*_eight_bits(_swiglu(gate_up)), s["w2"], s["s2"], None, s["t"])}
    out = {}
    if s["kind"] == "norm":
        out["residual"], v = _norm(s["x"], s["residual"], s["gamma"])
    else:
        v = _swiglu(s["gate_up"]) if s["kind"] == "swiglu" else s["x"].float()
    q, scale = _eight_bits(v)
    return {**out, "values": (q * scale).to(torch.bfloat16), "scale": scale[:, 0]}


# ---- one pass: the library's calls ------------------------------------------------------

_parity = None


def _library():
    global _parity
    if _parity is None:
        _parity = importlib.import_module("c-kernel-engine_amd").parity
    return _parity


def _calls(s):
    P = _library()
    if s["kind"] == "matmul":
        return {"c": P.dev_gemm_nt_i8(s["a"], s["sa"], s["b"], s["sb"], s["bias"], out=s["c"])}
    out = {}
    if s["kind"] in ("norm", "mlp"):
        P.dev_rmsnorm_i8(s["x"], s["gamma"], EPS, residual=s["residual"], residual_out=s["out"], out=(s["q"], s["scale"]))
        out["residual"] = s["out"]
    elif s["kind"] == "swiglu":
        k = s["q"].shape[1]
        P.dev_swiglu_i8(s["gate_up"][:, :k], s["gate_up"][:, k:], out=(s["q"], s["scale"]))
    else:
        P.dev_quantize_i8(s["x"], out=(s["q"], s["scale"]))
    if s["kind"] == "mlp":
        f = s["qf"].shape[1]
        P.dev_gemm_nt_i8(s["q"], s["scale"], s["w1"], s["s1"], out=s["gate_up"])
        P.dev_swiglu_i8(s["gate_up"][:, :f], s["gate_up"][:, f:], out=(s["qf"], s["scalef"]))
        return {**out, "c": P.dev_gemm_nt_i8(s["qf"], s["scalef"], s["w2"], s["s2"], out=s["c"])}
    return {**out, "values": P.dev_dequantize_i8(s["q"], s["scale"], out=s["values"]), "scale": s["scale"]}


def run(s):
    return _calls(s) if own else _plain(s)


# ---- what a pass cannot do without -------------------------------------------------------

def work(case):
    M, K, e = case["M"], case["K"], SIZE[case["t"]]
    if case["kind"] == "matmul":
        N = case["N"]
        return {"bytes": M * K + N * K + 4 * (M + N) + (4 * N if case["bias"] else 0) + e * M * N, "flops": 2 * M * N * K}
    if case["kind"] == "mlp":
        F = case["F"]
        return {"bytes": 4 * e * M * K + 4 * K + 3 * F * K + 8 * F + 4 * K, "flops": 6 * M * F * K}
    inputs = {"norm": 2 * e * M * K + 4 * K, "swiglu": 2 * e * M * K, "quantize": e * M * K}[case["kind"]]
    outputs = (e if case["kind"] == "norm" else 0) * M * K + 2 * M * K + 4 * M
    return {"bytes": inputs + outputs, "flops": {"norm": 8, "swiglu": 12, "quantize": 4}[case["kind"]] * M * K}


# ---- the definitions in 64 bits ------------------------------------------------------------

def _row_codes64(v):
    top = torch.maximum(v.abs().max(dim=1).values, torch.full((), TINY, dtype=torch.float64, device=v.device))
    step = top / 127
    return torch.round(v / step.unsqueeze(1)), step


def _sum_of_squares_norm64(h, gamma):
    h = h.double()
    return h / torch.sqrt((h * h).sum(1) / h.shape[1] + EPS).unsqueeze(1) * gamma.double()


def _products64(a, b):
    return a.double() @ b.double().transpose(0, 1).contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "matmul":
        c = torch.einsum("mn,m,n->mn", _products64(s["a"], s["b"]), s["sa"].double(), s["sb"].double())
        return {"c": c if s["bias"] is None else c + s["bias"].double()}
    result = {}
    if case["kind"] in ("norm", "mlp"):
        total = s["x"].double() + s["residual"].double()
        result["residual"] = total
        v = _sum_of_squares_norm64(total.to(s["t"]), s["gamma"])       # the norm is of the stream as it is stored
    elif case["kind"] == "swiglu":
        g, u = s["gate_up"].double().split(case["K"], dim=1)
        v = g * torch.sigmoid(g) * u
    else:
        v = s["x"].double()
    q, step = _row_codes64(v)
    if case["kind"] == "mlp":
        y = (_products64(q, s["w1"]) * step.unsqueeze(1) * s["s1"].double()).to(s["t"]).double()
        g, u = y.split(case["F"], dim=1)
        q, step = _row_codes64(g * torch.sigmoid(g) * u)
        result["c"] = _products64(q, s["w2"]) * step.unsqueeze(1) * s["s2"].double()
        return result
    result["values"], result["scale"] = q * step.unsqueeze(1), step
    return result
