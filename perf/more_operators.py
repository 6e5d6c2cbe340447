"""The operators of the 8-bit floating point path and of its experts: what is measured of them.

Rows are in e4m3 with one fp32 scale for each 128 elements of a row (activations) or for each block of 128 x 128 (weights).
Five kinds of work:

  matmul     C = the sum over groups of 128 of (scale of the token's group) * (scale of the weights' block) * A B^T, + bias.
  quantize   rows of floats in 8 bits, and read back.
  dispatch   tokens sorted by expert, their rows brought there, the experts' rows brought back with weights.
  grad       the gradients of both: of the experts' rows and the weights, and of the tokens.
  moe        the MLP half of a decoder layer with experts, all of it together: sort, rows in 8 bits, gate and up, SwiGLU, down,
             and back.

8-bit rows come back as the values they stand for, in bfloat16, beside their scales.  A row begins at a multiple of 16 bytes and
the scales of one group lie side by side, as the library's own allocation has them."""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
F8 = torch.float8_e4m3fn
GROUP = 128
MOST_F8 = 448.0
TINY = 2.0 ** -100            # no group is scaled by less


# ---- cases --------------------------------------------------------------------------

def listed():
    return [
        # interactive decode: the gate projection of a 7B model, one token
        {"name": "matmul_t1_11008x4096", "kind": "matmul", "M": 1, "N": 11008, "K": 4096, "t": "bf16", "bias": False},
        # a prompt whose length, and a layer whose sizes, fit no tile and no group
        {"name": "matmul_t333_1001x4847", "kind": "matmul", "M": 333, "N": 1001, "K": 4847, "t": "f32", "bias": True},
        # a long prompt
        {"name": "matmul_t2048_11008x4096", "kind": "matmul", "M": 2048, "N": 11008, "K": 4096, "t": "bf16", "bias": False},
        # batched decode of a small model: the attention outputs of five sequences on their way into the output projection
        {"name": "quantize_t5_896", "kind": "quantize", "M": 5, "K": 896, "t": "f16"},
        # a long prompt on its way into the down projection
        {"name": "quantize_t2048_11008", "kind": "quantize", "M": 2048, "K": 11008, "t": "bf16"},
        # batched decode of seven sequences, six experts each
        {"name": "dispatch_t7_2048", "kind": "dispatch", "T": 7, "K": 2048, "E": 64, "top": 6, "t": "bf16"},
        # a batch of prompts, the last of it padding
        {"name": "dispatch_t8192_2048", "kind": "dispatch", "T": 8192, "K": 2048, "E": 128, "top": 8, "t": "bf16"},
        # a short sequence through a small layer of odd width, in fp32
        {"name": "grad_t93_1001", "kind": "grad", "T": 93, "K": 1001, "E": 16, "top": 3, "t": "f32"},
        # a training batch
        {"name": "grad_t4096_2048", "kind": "grad", "T": 4096, "K": 2048, "E": 64, "top": 8, "t": "bf16"},
        # interactive decode: one token through eight of 64 experts
        {"name": "moe_t1_2048x1408", "kind": "moe", "T": 1, "K": 2048, "F": 1408, "E": 64, "top": 8, "t": "bf16"},
        # continuous batching, a small model whose experts end within a group of 128
        {"name": "moe_t61_896x608", "kind": "moe", "T": 61, "K": 896, "F": 608, "E": 32, "top": 4, "t": "f16"},
        # a long prompt
        {"name": "moe_t2048_2048x1408", "kind": "moe", "T": 2048, "K": 2048, "F": 1408, "E": 64, "top": 8, "t": "bf16"},
    ]


MOST = 2 * 2048 * 11008 * 4096           # operations of the longest listed prompt
MOST_ROWS = 65536 * 2048                 # elements of the longest listed dispatch
MOST_EXPERTS = 64 * 2048 * 1408 * 3      # weights of the listed experts


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["matmul", "matmul", "quantize", "dispatch", "grad", "moe", "moe"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "matmul":
        N, K = _log(rng, 32, 32000), _log(rng, 32, 11008)
        if rng.random() < 0.5:               # as often as not a width that a model would have
            K = max(64, K - K % 64)
        M = max(1, min(_log(rng, 1, 2048), MOST // (2 * N * K)))
        return {"kind": kind, "M": M, "N": N, "K": K, "t": t, "bias": rng.random() < 0.5}
    if kind == "quantize":
        K = _log(rng, 64, 11008)
        if rng.random() < 0.5:
            K = max(64, K - K % 64)
        return {"kind": kind, "M": _log(rng, 1, 2048), "K": K, "t": t}
    if kind == "moe":
        K = max(64, 64 * round(_log(rng, 256, 4096) / 64))
        F = max(64, 16 * round(_log(rng, 128, 2048) / 16))
        E = max(2, min(_log(rng, 4, 128), MOST_EXPERTS // (3 * K * F)))
        top = rng.randint(1, min(8, E))
        T = max(1, min(_log(rng, 1, 2048), MOST // (6 * top * K * F)))
        return {"kind": kind, "T": T, "K": K, "F": F, "E": E, "top": top, "t": rng.choice(["bf16", "f16"])}
    K = _log(rng, 64, 8192)
    if rng.random() < 0.5:
        K = max(64, K - K % 64)
    E = _log(rng, 4, 256)
    top = rng.randint(1, min(8, E))
    most = MOST_ROWS // (2 if t == "f32" else 1)
    T = max(1, min(_log(rng, 1, 8192 if kind == "dispatch" else 4096), most // (top * K)))
    return {"kind": kind, "T": T, "K": K, "E": E, "top": top, "t": t}


# ---- inputs ---------------------------------------------------------------------------

def _groups(k):
    return -(-k // GROUP)


def _f8(rows, k):
    return torch.empty(rows, -(-k // 16) * 16, dtype=F8, device="cuda")[:, :k]


def _f8_scales(rows, k):
    return torch.empty(_groups(k), rows, device="cuda").t()


def _rows(gen, m, k, t):
    """Activations: N(0, 1) with every 61st channel some ten times larger, as the residual stream of a trained model has them."""
    x = torch.randn(m, k, device="cuda", generator=gen)
    x[:, 17::61] *= 10
    return x.to(t)


def _codes(gen, *shape):
    """e4m3 rows as quantized weights and activations are: normal, the largest of a block near 448."""
    q = torch.randn(*shape[:-1], -(-shape[-1] // 16) * 16, device="cuda", generator=gen).mul_(112).clamp_(-MOST_F8, MOST_F8).to(F8)
    return q[..., :shape[-1]]


def _block_scales(gen, *shape):
    return torch.rand(*shape, device="cuda", generator=gen).add_(0.5).mul_(0.02 / 112)


def _router(gen, T, E, top, padding):
    """The experts of each token and their weights as a router gives them: some experts more popular than others, a softmax over
    those chosen; tokens that are padding have none."""
    logits = torch.randn(T, E, device="cuda", generator=gen) + 0.5 * torch.randn(E, device="cuda", generator=gen)
    best = logits.topk(top, dim=1)
    ids = best.indices.to(torch.int32)
    if padding:
        ids[T - T // 16:] = -1
    return ids, torch.softmax(best.values, dim=1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    K, t, kind = case["K"], DTYPES[case["t"]], case["kind"]
    s = {"kind": kind, "t": t}
    if kind == "matmul":
        M, N = case["M"], case["N"]
        sa = _f8_scales(M, K)
        sa.copy_(torch.rand(M, _groups(K), device="cuda", generator=gen).add_(0.5).mul_(1 / 112))
        s.update(a=_codes(gen, M, K), sa=sa, b=_codes(gen, N, K), sb=_block_scales(gen, _groups(N), _groups(K)),
                 bias=torch.randn(N, device="cuda", generator=gen) if case["bias"] else None, c=torch.empty(M, N, dtype=t, device="cuda"))
        return s
    if kind == "quantize":
        M = case["M"]
        s.update(x=_rows(gen, M, K, t), q=_f8(M, K), scale=_f8_scales(M, K), values=torch.empty(M, K, dtype=torch.bfloat16, device="cuda"))
        return s
    T, E, top = case["T"], case["E"], case["top"]
    S = T * top
    ids, weights = _router(gen, T, E, top, kind != "moe")
    s.update(E=E, ids=ids, weights=weights, offsets=torch.zeros(E + 1, dtype=torch.int32, device="cuda"),
             order=torch.zeros(S, dtype=torch.int32, device="cuda"), position=torch.zeros(T, top, dtype=torch.int32, device="cuda"))
    if kind == "dispatch":
        s.update(x=_rows(gen, T, K, t), rows=torch.zeros(S, K, dtype=t, device="cuda"), back=_rows(gen, S, K, t), out=torch.zeros(T, K, dtype=t, device="cuda"))
    elif kind == "grad":
        # what a training step has kept of its forward pass: where each slot went
        s["position"] = _plain_sort(ids, E)[2]
        s.update(dout=_rows(gen, T, K, t), y=_rows(gen, S, K, t), g=_rows(gen, S, K, t), dy=torch.zeros(S, K, dtype=t, device="cuda"),
                 dw=torch.zeros(T, top, device="cuda"), dx=torch.zeros(T, K, dtype=t, device="cuda"))
    else:
        F = case["F"]
        s.update(x=_rows(gen, T, K, t), w1=_codes(gen, E, 2 * F, K), s1=_block_scales(gen, E, _groups(2 * F), _groups(K)),
                 w2=_codes(gen, E, K, F), s2=_block_scales(gen, E, _groups(K), _groups(F)), q=_f8(S, K), scale=_f8_scales(S, K),
                 gate_up=torch.zeros(S, 2 * F, dtype=t, device="cuda"), qf=_f8(S, F), scalef=_f8_scales(S, F),
                 y=torch.zeros(S, K, dtype=t, device="cuda"), out=torch.zeros(T, K, dtype=t, device="cuda"))
    return s


# ---- one pass: the plain forms ----------------------------------------------------------

def _eight_bits(v):
    """The codes of fp32 rows as floats, and the scales of their groups.  The quotients in 64 bits: those of values with few bits
    are often halfway between two codes."""
    m, k = v.shape
    g = torch.nn.functional.pad(v, (0, -k % GROUP)).view(m, -1, GROUP)
    a = g.abs().amax(2, keepdim=True).clamp_min(TINY)
    q = (g.double() * MOST_F8 / a).float().to(F8).float()
    return q.view(m, -1)[:, :k], (a / MOST_F8)[:, :, 0]


def _spread(scale, k):
    return scale.repeat_interleave(GROUP, dim=-1)[..., :k]


def _weights(b, sb):
    n, k = b.shape[-2:]
    return b.float() * _spread(sb.repeat_interleave(GROUP, dim=-2)[..., :n, :], k)


def _matmul(a, sa, b, sb, bias, t):
    c = torch.mm(a.float() * _spread(sa, a.shape[1]), _weights(b, sb).t())
    return (c if bias is None else c + bias).to(t)


def _plain_sort(ids, E):
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(E + 1, dtype=torch.long, device=ids.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([counts.new_zeros(1), counts[:E].cumsum(0)])
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=ids.device)
    position = torch.where(key < E, position, -1)
    order = torch.where(torch.arange(order.numel(), device=ids.device) < offsets[E], order, -1)
    return offsets.int(), order.int(), position.view(ids.shape).int()


def _plain_gather(x, order, top):
    return x[torch.div(order.clamp_min(0), top, rounding_mode="floor").long()] * (order >= 0)[:, None].to(x.dtype)


def _plain_combine(y, position, weights, t):
    w = (position >= 0).float() if weights is None else weights * (position >= 0)
    return (y[position.clamp_min(0).long()].float() * w[:, :, None]).sum(1).to(t)


def _plain_experts(a, sa, b, sb, offsets, t):
    """Rows of each expert in tiles, a tile's matrix beside it; rows without an expert are zeros."""
    m, k = a.shape
    E, n = b.shape[:2]
    bt = 1 << max(0, math.ceil(math.log2(m / E)))
    tiles = m // bt + min(E, m)
    offsets = offsets.long()
    count = offsets[1:] - offsets[:-1]
    each = (count + bt - 1) // bt
    ends = each.cumsum(0)
    i = torch.arange(tiles, device=a.device)
    e = torch.searchsorted(ends, i, right=True).clamp_max(E - 1)
    rows = (offsets[e] + (i - (ends - each)[e]) * bt)[:, None] + torch.arange(bt, device=a.device)
    rows = torch.where((rows < offsets[e + 1][:, None]) & (i < ends[-1])[:, None], rows, m)
    x = torch.nn.functional.pad(a.float() * _spread(sa, k), (0, 0, 0, 1))[rows]
    w = _weights(b.view(torch.uint8)[e].view(F8), sb[e])
    c = torch.bmm(w, x.transpose(1, 2).contiguous()).transpose(1, 2)
    out = torch.zeros(m + 1, n, device=a.device)
    out[rows.reshape(-1)] = c.reshape(-1, n)
    return out[:m].to(t)


def _swiglu(gate_up):
    g, u = gate_up.float().chunk(2, 1)
    return g / (1.0 + torch.exp(-g)) * u


def _plain(s):
    kind = s["kind"]
    if kind == "matmul":
        return {"c": _matmul(s["a"], s["sa"], s["b"], s["sb"], s["bias"], s["t"])}
    if kind == "quantize":
        q, scale = _eight_bits(s["x"].float())
        return {"values": (q * _spread(scale, q.shape[1])).to(torch.bfloat16), "scale": scale}
    if kind == "grad":
        position, dout, weights = s["position"], s["dout"].float(), s["weights"]
        there = position >= 0
        S = s["y"].shape[0]
        dy = torch.zeros(S + 1, dout.shape[1], device=dout.device)
        dy[torch.where(there, position, S).long().view(-1)] = (weights[:, :, None] * dout[:, None]).flatten(0, 1)
        dw = (dout[:, None] * s["y"][position.clamp_min(0).long()].float()).sum(2) * there
        return {"dy": dy[:S].to(s["t"]), "dw": dw, "dx": _plain_combine(s["g"], position, None, s["t"])}
    offsets, order, position = _plain_sort(s["ids"], s["E"])
    if kind == "dispatch":
        return {"offsets": offsets, "order": order, "position": position, "rows": _plain_gather(s["x"], order, s["ids"].shape[1]),
                "out": _plain_combine(s["back"], position, s["weights"], s["t"])}
    a, sa = _eight_bits(_plain_gather(s["x"], order, s["ids"].shape[1]).float())
    gate_up = _plain_experts(a, sa, s["w1"], s["s1"], offsets, s["t"])
    y = _plain_experts(*_eight_bits(_swiglu(gate_up)), s["w2"], s["s2"], offsets, s["t"])
    return {"offsets": offsets, "out": _plain_combine(y, position, s["weights"], s["t"])}


# ---- one pass: the library's calls ------------------------------------------------------

_parity = None


def _library():
    global _parity
    if _parity is None:
        _parity = importlib.import_module("c-kernel-engine_amd").parity
    return _parity


def _calls(s):
    P = _library()
    kind = s["kind"]
    if kind == "matmul":
        return {"c": P.dev_gemm_nt_f8(s["a"], s["sa"], s["b"], s["sb"], s["bias"], out=s["c"])}
    if kind == "quantize":
        P.dev_quantize_f8(s["x"], out=(s["q"], s["scale"]))
        return {"values": P.dev_dequantize_f8(s["q"], s["scale"], out=s["values"]), "scale": s["scale"]}
    if kind == "grad":
        P.dev_moe_combine_backward(s["dout"], s["y"], s["position"], s["weights"], out=(s["dy"], s["dw"]))
        return {"dy": s["dy"], "dw": s["dw"], "dx": P.dev_moe_combine(s["g"], s["position"], out=s["dx"])}
    P.dev_moe_sort(s["ids"], s["E"], out=(s["offsets"], s["order"], s["position"]))
    if kind == "dispatch":
        return {"offsets": s["offsets"], "order": s["order"], "position": s["position"], "rows": P.dev_moe_gather(s["x"], s["position"], out=s["rows"]),
                "out": P.dev_moe_combine(s["back"], s["position"], s["weights"], out=s["out"])}
    f = s["qf"].shape[1]
    P.dev_moe_gather_f8(s["x"], s["position"], out=(s["q"], s["scale"]))
    P.dev_gemm_nt_f8_experts(s["q"], s["scale"], s["w1"], s["s1"], s["offsets"], out=s["gate_up"])
    P.dev_swiglu_f8(s["gate_up"][:, :f], s["gate_up"][:, f:], out=(s["qf"], s["scalef"]))
    P.dev_gemm_nt_f8_experts(s["qf"], s["scalef"], s["w2"], s["s2"], s["offsets"], out=s["y"])
    return {"offsets": s["offsets"], "out": P.dev_moe_combine(s["y"], s["position"], s["weights"], out=s["out"])}


def run(s):
    return _calls(s) if own else _plain(s)


# ---- what a pass cannot do without -------------------------------------------------------

def work(case):
    K, e, kind = case["K"], SIZE[case["t"]], case["kind"]
    if kind == "matmul":
        M, N = case["M"], case["N"]
        scales = _groups(K) * (M + _groups(N))
        return {"bytes": M * K + N * K + 4 * scales + (4 * N if case["bias"] else 0) + e * M * N, "flops": 2 * M * N * K}
    if kind == "quantize":
        return {"bytes": (e + 2) * case["M"] * K + 4 * case["M"] * _groups(K), "flops": 4 * case["M"] * K}
    T, E, top = case["T"], case["E"], case["top"]
    S = (T - (T // 16 if kind != "moe" else 0)) * top                 # slots that have an expert
    if kind == "dispatch":
        return {"bytes": 16 * T * top + 4 * (E + 1) + 2 * e * (T + S) * K, "flops": 2 * S * K}
    if kind == "grad":
        return {"bytes": 12 * T * top + e * (3 * S + 2 * T) * K, "flops": 4 * S * K}
    F = case["F"]
    used = E * (1 - (1 - top / E) ** T)                               # experts that have a token, on average
    return {"bytes": used * (3 * K * F + 4 * (_groups(2 * F) * _groups(K) + _groups(K) * _groups(F))) + 8 * T * top + 2 * e * T * K, "flops": 6 * S * K * F}


# ---- the definitions in 64 bits ------------------------------------------------------------

def _e4m3_64(t):
    """The nearest e4m3 value, ties to even: three bits behind the leading one, none smaller than 2^-9."""
    exponent = (torch.frexp(t)[1] - 1).clamp_min(-6)
    step = torch.ldexp(torch.ones_like(t), exponent - 3)
    return torch.round(t / step) * step


def _group_codes64(v):
    q, scale = torch.empty_like(v), torch.empty(v.shape[0], _groups(v.shape[1]), dtype=torch.float64, device=v.device)
    for g in range(scale.shape[1]):
        part = v[:, g * GROUP:(g + 1) * GROUP]
        top = part.abs().max(dim=1).values.clamp_min(TINY)
        scale[:, g] = top / MOST_F8
        q[:, g * GROUP:(g + 1) * GROUP] = _e4m3_64(part * MOST_F8 / top.unsqueeze(1))       # a tie stays one
    return q, scale


def _values64(q, scale):
    v = q.double().clone()
    for g in range(scale.shape[1]):
        v[:, g * GROUP:(g + 1) * GROUP] *= scale[:, g, None].double()
    return v


def _block_values64(b, sb):
    v = b.double().clone()
    for i in range(sb.shape[0]):
        for g in range(sb.shape[1]):
            v[i * GROUP:(i + 1) * GROUP, g * GROUP:(g + 1) * GROUP] *= sb[i, g].double()
    return v


def _sorted_slots(ids, E):
    """Experts in turn, each with its slots as they come."""
    flat = ids.reshape(-1)
    slots = [torch.nonzero(flat == e)[:, 0] for e in range(E)]
    offsets = [0]
    for v in slots:
        offsets.append(offsets[-1] + v.numel())
    order = torch.full_like(flat, -1)
    order[:offsets[-1]] = torch.cat(slots).to(order.dtype)
    position = torch.full_like(flat, -1)
    position[order[:offsets[-1]].long()] = torch.arange(offsets[-1], dtype=position.dtype, device=ids.device)
    return torch.tensor(offsets, dtype=torch.int32, device=ids.device), order, position.view(ids.shape)


def _back64(y, position, weights):
    out = torch.zeros(position.shape[0], y.shape[1], dtype=torch.float64, device=y.device)
    for j in range(position.shape[1]):
        p = position[:, j]
        row = y[p.clamp_min(0).long()].double()
        if weights is not None:
            row *= weights[:, j, None].double()
        out += torch.where((p >= 0)[:, None], row, torch.zeros_like(row))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind, K = case["kind"], case["K"]
    if kind == "matmul":
        c = _values64(s["a"], s["sa"]) @ _block_values64(s["b"], s["sb"]).transpose(0, 1).contiguous()
        return {"c": c if s["bias"] is None else c + s["bias"].double()}
    if kind == "quantize":
        q, scale = _group_codes64(s["x"].double())
        return {"values": _values64(q, scale), "scale": scale}
    if kind == "grad":
        position, dout = s["position"], s["dout"].double()
        dy = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros(position.shape, dtype=torch.float64, device="cuda")
        for j in range(position.shape[1]):
            t = torch.nonzero(position[:, j] >= 0)[:, 0]
            p = position[t, j].long()
            dy[p] = dout[t] * s["weights"][t, j, None].double()
            dw[t, j] = (dout[t] * s["y"][p].double()).sum(1)
        return {"dy": dy, "dw": dw, "dx": _back64(s["g"], position, None)}
    offsets, order, position = _sorted_slots(s["ids"], case["E"])
    have = int(offsets[-1])
    rows = torch.zeros(order.numel(), K, dtype=torch.float64, device="cuda")
    rows[:have] = s["x"].double()[order[:have].long() // case["top"]]
    if kind == "dispatch":
        return {"offsets": offsets, "order": order, "position": position, "rows": rows, "out": _back64(s["back"], position, s["weights"])}
    F = case["F"]
    a = _values64(*_group_codes64(rows))
    y = torch.zeros_like(rows)
    for e in range(case["E"]):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if hi > lo:
            h = (a[lo:hi] @ _block_values64(s["w1"][e], s["s1"][e]).transpose(0, 1).contiguous()).to(s["t"]).double()
            v = h[:, :F] * torch.sigmoid(h[:, :F]) * h[:, F:]
            y[lo:hi] = _values64(*_group_codes64(v)) @ _block_values64(s["w2"][e], s["s2"][e]).transpose(0, 1).contiguous()
    return {"offsets": offsets, "out": _back64(y.to(s["t"]), position, s["weights"])}
