"""The 8-bit operators of the MoE FFN path, as cases to time and compare.

Four operators, each in its plain form (``own`` false: elementary torch operations
in 32 bits) and as a user's program calls it (``own`` true):

  linear   rows [R, K] times weights [E, N, K] held in e4m3 with a scale for each
           128 x 128 block; the rows are quantised in blocks of 128 first
  layer    the whole MoE layer for a few tokens: router, top-k, expert FFN with
           8-bit weights, sum over the chosen experts; as a sub-layer also the
           norms before and after, the gate and the residual scale
  experts  the expert FFN of a prompt with the routing given
  norm     residual_scale * residual + gate * rms_norm(y), and the next block's
           rms_norm of the sum

Quantisation (all of them): a block of 128 consecutive values along K shares the
scale 2^p, p the least integer with amax <= 448 * 2^p, and every value becomes
e4m3(v / 2^p) * 2^p, rounded to nearest even.
"""

import math
import os
import sys

import torch

own = False

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "frank-models_b200")
if PACKAGE not in sys.path:
    sys.path.append(PACKAGE)

BLOCK = 128
DEV = "cuda"
EPS = 1e-5


# ---------------------------------------------------------------- cases ----
def listed():
    return [
        # a decode batch's projection: one tile of rows, launch latency counts
        {"name": "linear_decode", "op": "linear", "E": 1, "rows": 5, "K": 2048, "N": 1536, "skew": 0.0, "out": "bf16"},
        # a prompt through one dense projection of the Mixtral-shaped block
        {"name": "linear_prompt", "op": "linear", "E": 1, "rows": 8192, "K": 4096, "N": 14336, "skew": 0.0,
         "out": "bf16"},
        # expert-sorted rows of a fine-grained router, ragged groups and empty ones, odd widths, fp32 out
        {"name": "linear_ragged", "op": "linear", "E": 128, "rows": 8191, "K": 2000, "N": 784, "skew": 1.2,
         "out": "f32"},
        # one token, the fine-grained block: eight experts' weights are all there is to read
        {"name": "layer_one_token", "op": "layer", "T": 1, "H": 2048, "F": 768, "E": 128, "k": 8, "normalize": False,
         "sub": False},
        # a small decode batch through the whole sub-layer: norms on both sides, gate and residual scale
        {"name": "layer_batch", "op": "layer", "T": 8, "H": 2048, "F": 768, "E": 128, "k": 8, "normalize": True,
         "sub": True},
        # an odd decode batch that reaches most experts, several rows for some of them
        {"name": "layer_wide_batch", "op": "layer", "T": 47, "H": 2048, "F": 768, "E": 128, "k": 8,
         "normalize": True, "sub": True},
        # few large experts, three tokens, long rows
        {"name": "layer_large_experts", "op": "layer", "T": 3, "H": 4096, "F": 14336, "E": 8, "k": 2,
         "normalize": False, "sub": False},
        # a prompt through small experts with a skewed router
        {"name": "experts_skewed", "op": "experts", "T": 8192, "H": 2048, "F": 768, "E": 128, "k": 8, "skew": 1.2},
        # a long prompt through the Mixtral-shaped experts: the tensor-bound end
        {"name": "experts_prompt", "op": "experts", "T": 16384, "H": 4096, "F": 14336, "E": 8, "k": 2, "skew": 0.0},
        # one token between two blocks
        {"name": "norm_one_token", "op": "norm", "T": 1, "H": 2048, "gates": 1, "next": True, "y": "f32"},
        # an odd number of rows, no following norm, a gate for each row
        {"name": "norm_ragged", "op": "norm", "T": 1021, "H": 2040, "gates": 1021, "next": False, "y": "bf16"},
        # a prompt between two blocks, one gate for each of 16 sequences
        {"name": "norm_prompt", "op": "norm", "T": 16384, "H": 4096, "gates": 16, "next": True, "y": "f32"},
    ]


def _log(rng, lo, hi, step=1):
    """A whole multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return min(hi, max(lo, int(v) // step * step))


def draw(rng):
    op = rng.choice(["linear", "linear", "layer", "layer", "experts", "norm"])
    if op == "linear":
        E = rng.choice([1, 1, _log(rng, 2, 160)])
        K, N = _log(rng, 64, 4096, 16), _log(rng, 64, 14336, 16)
        return {"op": op, "E": E, "rows": _log(rng, 1, 8192), "K": K, "N": N, "skew": rng.uniform(0.0, 1.4),
                "out": rng.choice(["bf16", "f32"])}
    if op == "layer":
        E = _log(rng, 4, 160)
        wide = 4096 if E <= 16 else 2048
        return {"op": op, "T": _log(rng, 1, 64), "H": _log(rng, 256, wide, 16), "F": _log(rng, 128, wide, 16),
                "E": E, "k": rng.randint(1, min(8, E)), "normalize": rng.random() < 0.5, "sub": rng.random() < 0.5}
    if op == "experts":
        E = _log(rng, 4, 128)
        wide = 4096 if E <= 16 else 1024
        return {"op": op, "T": _log(rng, 65, 8192), "H": _log(rng, 256, wide, 16), "F": _log(rng, 128, wide, 16),
                "E": E, "k": rng.randint(1, min(8, E)), "skew": rng.uniform(0.0, 1.4)}
    T = _log(rng, 1, 16384)
    return {"op": op, "T": T, "H": _log(rng, 64, 4096, 4), "gates": rng.choice([0, 1, T]), "next": rng.random() < 0.5,
            "y": rng.choice(["f32", "bf16"])}


# --------------------------------------------------------------- inputs ----
def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _weights(g, E, N, K):
    """Quantised weights as a checkpoint holds them: e4m3 values and one fp32 scale, no power of two, for each
    128 x 128 block; together about N(0, 0.02)."""
    q = (torch.randn((E, N, K), generator=g, device=DEV) * 112.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    s = torch.rand((E, -(-N // BLOCK), -(-K // BLOCK)), generator=g, device=DEV) * 0.6 + 0.7
    return q, s * (0.02 / 112.0)


def _popularity(E, skew, g):
    rank = torch.randperm(E, generator=g, device=DEV)
    return -skew * torch.log(rank.float() + 1.0)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "linear":
        E, rows, K, N = case["E"], case["rows"], case["K"], case["N"]
        s["x"] = _normal(g, rows, K, dtype=torch.bfloat16)
        s["w"] = _weights(g, E, N, K)
        s["offsets"], s["cap"] = None, rows
        if E > 1:
            p = torch.softmax(_popularity(E, case["skew"], g), 0)
            e = torch.multinomial(p, rows, replacement=True, generator=g)
            count = torch.bincount(e, minlength=E)
            s["offsets"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
            s["cap"] = int(count.max())
    elif op in ("layer", "experts"):
        T, H, F, E, k = case["T"], case["H"], case["F"], case["E"], case["k"]
        s["up"], s["gate"], s["down"] = _weights(g, E, F, H), _weights(g, E, F, H), _weights(g, E, H, F)
        s["wr"] = _normal(g, E, H, std=0.02)
        s["x"] = _normal(g, T, H, dtype=torch.bfloat16)
        if op == "experts":
            score = _popularity(E, case["skew"], g)[None, :] - torch.log(-torch.log(
                torch.rand((T, E), generator=g, device=DEV).clamp_(1e-20, 1 - 1e-7)))
            top, ids = score.topk(k, dim=1)
            s["route_w"] = torch.softmax(top, 1).t().contiguous()
            s["route_ids"] = ids.t().to(torch.int32).contiguous()
            s["cap"] = int(torch.bincount(ids.reshape(-1), minlength=E).max())
        elif case["sub"]:
            s["norm_w"] = 1.0 + _normal(g, H, std=0.1)
            s["post_w"] = 1.0 + _normal(g, H, std=0.1)
            s["g"] = 0.5 + _normal(g, H, std=0.1)
        if own:  # the handle that a program keeps; it holds the same tensors
            from frank_b200 import Fp8Experts, Fp8MoEFFNBlock
            s["block"] = Fp8MoEFFNBlock(s["wr"], Fp8Experts(*s["up"]), Fp8Experts(*s["gate"]), Fp8Experts(*s["down"]),
                                        E, k, bool(case.get("normalize", False)), out_dtype=torch.bfloat16)
    else:
        T, H = case["T"], case["H"]
        s["y"] = _normal(g, T, H, std=0.3, dtype=torch.float32 if case["y"] == "f32" else torch.bfloat16)
        s["residual"] = _normal(g, T, H, dtype=torch.bfloat16)
        s["w"] = 1.0 + _normal(g, H, std=0.1)
        s["g"] = 0.5 + _normal(g, case["gates"], H, std=0.1) if case["gates"] else None
        s["next_w"] = 1.0 + _normal(g, H, std=0.1) if case["next"] else None
    return s


RESIDUAL_SCALE = 0.75


# ----------------------------------------------------------- plain forms ----
def _quantised(x):
    """The fp32 values that the 8-bit form of `x` [..., K] stands for."""
    K = x.shape[-1]
    nb = -(-K // BLOCK)
    b = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - K)).unflatten(-1, (nb, BLOCK))
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    p = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-110)
    b = torch.ldexp(torch.ldexp(b, -p).to(torch.float8_e4m3fn).float(), p)
    return b.flatten(-2)[..., :K]


def _weights32(w, pick=None):
    q, s = w
    if pick is not None:
        q, s = q.view(torch.uint8)[pick].view(torch.float8_e4m3fn), s[pick]
    N, K = q.shape[-2:]
    s = s.repeat_interleave(BLOCK, -2)[..., :N, :].repeat_interleave(BLOCK, -1)[..., :K]
    return q.float().mul_(s)


def _grouped(xs, offsets, cap):
    """Expert-sorted rows laid out [E, cap, K], and where each row went."""
    start, end = offsets[:-1].long(), offsets[1:].long()
    at = start[:, None] + torch.arange(cap, device=DEV)
    r = torch.arange(xs.shape[0], device=DEV)
    e = torch.searchsorted(end, r, right=True)
    return xs[at.clamp_(max=xs.shape[0] - 1)], (e, r - start[e])


def _swiglu(gate, up):
    return gate * (up / (1.0 + torch.exp(-up)))


def _rms_norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _plain_linear(s):
    w = _weights32(s["w"])
    x = _quantised(s["x"])
    if s["offsets"] is None:
        y = x @ w[0].t()
    else:
        xg, at = _grouped(x, s["offsets"], s["cap"])
        y = torch.bmm(xg, w.transpose(1, 2))[at]
    return y.to(torch.bfloat16) if s["case"]["out"] == "bf16" else y


def _plain_few(s, x):
    """The MoE block of a few tokens, fp32 [T, H]."""
    c = s["case"]
    T, E, k = x.shape[0], c["E"], c["k"]
    p = torch.softmax(x.float() @ s["wr"].t(), 1)
    top, ids = torch.sort(p, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    if c["normalize"]:
        top = top / top.sum(1, keepdim=True)
    xq = _quantised(x)
    if k * T <= E:  # every slot with its own expert's matrices
        pick = ids.reshape(-1)
        xs = xq.repeat_interleave(k, 0)[:, :, None]
        gate, up = (torch.bmm(_weights32(s[n], pick), xs)[:, :, 0] for n in ("gate", "up"))
        d = torch.bmm(_weights32(s["down"], pick), _quantised(_swiglu(gate, up))[:, :, None])[:, :, 0].view(T, k, -1)
    else:  # every expert for every token, then the chosen ones
        h = _quantised(_swiglu(xq @ _weights32(s["gate"]).transpose(1, 2), xq @ _weights32(s["up"]).transpose(1, 2)))
        d = torch.bmm(h, _weights32(s["down"]).transpose(1, 2))[ids, torch.arange(T, device=DEV)[:, None]]
    return (d * top[:, :, None]).sum(1)


def _plain_layer(s):
    x = s["x"]
    if not s["case"]["sub"]:
        return _plain_few(s, x).to(torch.bfloat16)
    xn = _rms_norm(x.float(), s["norm_w"]).to(torch.bfloat16)
    y = _rms_norm(_plain_few(s, xn), s["post_w"])
    return (RESIDUAL_SCALE * x.float() + s["g"] * y).to(torch.bfloat16)


def _plain_experts(s):
    c = s["case"]
    T, E, k = c["T"], c["E"], c["k"]
    ids = s["route_ids"].reshape(-1).long()
    order = torch.sort(ids, stable=True)[1]
    offsets = torch.searchsorted(ids[order], torch.arange(E + 1, device=DEV))
    xg, at = _grouped(_quantised(s["x"])[order % T], offsets, s["cap"])
    h = _swiglu(torch.bmm(xg, _weights32(s["gate"]).transpose(1, 2)),
                torch.bmm(xg, _weights32(s["up"]).transpose(1, 2)))
    d = torch.bmm(_quantised(h), _weights32(s["down"]).transpose(1, 2))[at] * s["route_w"].reshape(-1)[order][:, None]
    back = torch.empty_like(order)
    back[order] = torch.arange(k * T, device=DEV)
    return d[back].view(k, T, -1).sum(0).to(torch.bfloat16)


def _plain_norm(s):
    y = _rms_norm(s["y"].float(), s["w"])
    if s["g"] is not None:
        G, H = s["g"].shape
        y = (y.view(G, -1, H) * s["g"][:, None, :]).view(-1, H)
    out = (RESIDUAL_SCALE * s["residual"].float() + y).to(torch.bfloat16)
    if s["next_w"] is None:
        return out
    return out, _rms_norm(out.float(), s["next_w"]).to(torch.bfloat16)


# ----------------------------------------------------------------- calls ----
def _own(s):
    from frank_b200 import Fp8Experts, fp8_matmul, post_norm_residual

    c = s["case"]
    op = c["op"]
    if op == "linear":
        return fp8_matmul(s["x"], Fp8Experts(*s["w"]), offsets=s["offsets"],
                          out_dtype=torch.bfloat16 if c["out"] == "bf16" else torch.float32)
    if op == "layer":
        if not c["sub"]:
            return s["block"](s["x"])
        return s["block"].sublayer(s["x"], s["norm_w"], EPS, post_norm_w=s["post_w"], gate=s["g"],
                                   residual_scale=RESIDUAL_SCALE)
    if op == "experts":
        return s["block"].experts(s["x"], s["route_w"], s["route_ids"])
    return post_norm_residual(s["y"], s["residual"], s["w"], EPS, gate=s["g"], residual_scale=RESIDUAL_SCALE,
                              next_weight=s["next_w"])


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "layer": _plain_layer, "experts": _plain_experts,
            "norm": _plain_norm}[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "linear":
        E, R, K, N = case["E"], case["rows"], case["K"], case["N"]
        used = E if case["skew"] == 0.0 else min(E, R)
        return {"bytes": 2 * R * K + used * N * K + R * N * (2 if case["out"] == "bf16" else 4),
                "flops": 2 * R * K * N}
    if op in ("layer", "experts"):
        T, H, F, E, k = case["T"], case["H"], case["F"], case["E"], case["k"]
        used = E * (1.0 - (1.0 - k / E) ** T)  # experts that T tokens reach
        router = 4 * E * H if op == "layer" else 8 * k * T
        return {"bytes": int(4 * T * H + used * 3 * H * F + router),
                "flops": 6 * k * T * H * F + (2 * T * H * E if op == "layer" else 0)}
    T, H, G = case["T"], case["H"], case["gates"]
    y = 4 if case["y"] == "f32" else 2
    return {"bytes": T * H * (y + 4 + (2 if case["next"] else 0)) + 4 * H * (1 + G + bool(case["next"])),
            "flops": T * H * (8 + (4 if case["next"] else 0))}


# ------------------------------------------------- the definition in 64 bits
def _power(p):
    return torch.ldexp(torch.ones_like(p), p.int())


def _q64(x):
    """Quantised values by arithmetic alone: the block's power of two, then the nearest multiple of the step that
    three mantissa bits leave at the value's exponent (never below 2^-6), halves to even."""
    out = torch.empty_like(x)
    for k0 in range(0, x.shape[1], BLOCK):
        b = x[:, k0:k0 + BLOCK]
        amax = b.abs().amax(1, keepdim=True)
        r = (amax / 448.0).clamp(min=2.0 ** -110)
        s = _power(torch.ceil(torch.log2(r)))
        s = torch.where(s < r, 2 * s, torch.where(s >= 2 * r, s / 2, s))  # log2 rounds
        v = b / s
        a = v.abs().clamp(min=2.0 ** -6)
        t = _power(torch.floor(torch.log2(a)))
        step = torch.where(t > a, t / 2, torch.where(2 * t <= a, 2 * t, t)) / 8
        out[:, k0:k0 + BLOCK] = torch.round(v / step) * step * s
    return out


def _w64(w, e):
    q, s = w[0][e].double(), w[1][e].double()
    return q * torch.kron(s, s.new_ones(BLOCK, BLOCK))[:q.shape[0], :q.shape[1]]


def _norm64(x, w):
    return x / torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPS) * w.double()


def _experts64(s, x, w, ids):
    """sum_j w[j, t] * down(q(gate(x) * silu(up(x)))), one expert after the other."""
    xq = _q64(x)
    y = torch.zeros_like(x)
    for e in ids.unique().tolist():
        j, t = torch.nonzero(ids == e, as_tuple=True)
        xe = xq[t]
        u = xe @ _w64(s["up"], e).T
        h = (xe @ _w64(s["gate"], e).T) * (u * torch.sigmoid(u))
        y.index_add_(0, t, (_q64(h) @ _w64(s["down"], e).T) * w[j, t][:, None])
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        x = _q64(s["x"].double())
        bounds = [0, x.shape[0]] if s["offsets"] is None else s["offsets"].tolist()
        return torch.cat([x[a:b] @ _w64(s["w"], e).T for e, (a, b) in enumerate(zip(bounds, bounds[1:])) if b > a])
    if op == "experts":
        return _experts64(s, s["x"].double(), s["route_w"].double(), s["route_ids"])
    if op == "layer":
        x = s["x"].double()
        xn = _norm64(x, s["norm_w"]).to(torch.bfloat16).double() if case["sub"] else x
        z = xn @ s["wr"].double().T
        ids = torch.sort(z, dim=1, descending=True, stable=True)[1][:, :case["k"]].T
        w = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)).T.gather(0, ids)
        if case["normalize"]:
            w = w / w.sum(0, keepdim=True)
        y = _experts64(s, xn, w, ids)
        if not case["sub"]:
            return y
        return RESIDUAL_SCALE * x + s["g"].double() * _norm64(y, s["post_w"])
    y = _norm64(s["y"].double(), s["w"])
    if s["g"] is not None:
        G = s["g"].shape[0]
        y = y * s["g"].double().repeat_interleave(y.shape[0] // G, 0)
    out = RESIDUAL_SCALE * s["residual"].double() + y
    if s["next_w"] is None:
        return out
    return out, _norm64(out.to(torch.bfloat16).double(), s["next_w"])
