"""The 8-bit path in float64 (torch, any device): quantisation, product, expert
FFN and norms as include/frank_fp8.h defines them, and how far a kernel that
sums in fp32 may be from them.

Test infrastructure; written from the definitions, without the kernels' code.
"""

from __future__ import annotations

import torch

BLOCK = 128
U32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype) -> float:
    """The largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def _blocked(x):
    K = x.shape[-1]
    nb = -(-K // BLOCK)
    return torch.nn.functional.pad(x, (0, nb * BLOCK - K)).unflatten(-1, (nb, BLOCK))


def block_scales(x):
    """[..., nb] power-of-two scales of float64 rows; NaN for a block that is not finite."""
    amax = _blocked(x).abs().amax(-1)
    return torch.where(torch.isfinite(amax), scale_of(amax), torch.full_like(amax, float("nan")))


def scale_of(amax):
    """2^p, p the least integer >= -110 with amax <= 448 * 2^p (exact: log2 would miss exact powers)."""
    m, e = torch.frexp((amax / 448.0).clamp(min=2.0 ** -110))  # m in [0.5, 1)
    return torch.ldexp(torch.ones_like(amax), torch.where(m == 0.5, e - 1, e))


def round_e4m3(v):
    """Nearest e4m3 value, ties to even, of float64 |v| <= 448 (arithmetic only)."""
    e = torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 1  # 2^e <= |v| < 2^(e+1)
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return torch.round(v / step) * step


def quantised(x, scales=None):
    """The float64 values that the 8-bit form of x stands for (with the given block scales)."""
    K = x.shape[-1]
    s = block_scales(x) if scales is None else scales
    s = s.repeat_interleave(BLOCK, -1)[..., :K]
    return round_e4m3((x / s).clamp(-448.0, 448.0)) * s


def quantised_slack(x, err):
    """How far the 8-bit form of a value within `err` of x can be from that of x: every value may round either
    way where a border lies within `err`, and a block whose maximum may cross a power of two may take either scale."""
    q = quantised(x)
    slack = torch.zeros_like(x)
    amax, aerr = _blocked(x).abs().amax(-1), _blocked(err).amax(-1)
    for a in (amax - aerr, amax + aerr):
        s = scale_of(a)
        for v in (x - err, x + err):
            slack = torch.maximum(slack, (quantised(v, s) - q).abs())
    return slack


def product(a, w, err_a=None):
    """(a @ w.T, its bound): a [R, K], w [N, K] float64.  The kernel adds K products in fp32 -- exact products of two
    4-bit significands, K additions of relative error U32 each, doubled for adders that truncate -- then scales and
    adds ceil(K/128) partial sums (three roundings each)."""
    K = a.shape[-1]
    gamma = (2 * K + 3 * (-(-K // BLOCK)) + 2) * U32
    bound = gamma * (a.abs() @ w.abs().T)
    if err_a is not None:
        bound = bound + err_a @ w.abs().T * (1 + gamma)
    return a @ w.T, bound


def swiglu(gate, up, err_gate, err_up):
    """gate * silu(up) and its bound.  |silu'| <= 1.1; silu itself and the product: expf, add, divide, multiply,
    16 units in all."""
    s = up * torch.sigmoid(up)
    h = gate * s
    return h, err_gate * (s.abs() + 1.1 * err_up) + gate.abs() * 1.1 * err_up + 16 * U32 * h.abs()


def expert_ffn(xq, w_gate, w_up, w_down):
    """down(q(gate(xq) * silu(up(xq)))) for rows xq that are 8-bit values, and its bound."""
    h, eh = swiglu(*_pair(product(xq, w_gate), product(xq, w_up)))
    return product(quantised(h), w_down, quantised_slack(h, eh))


def _pair(g, u):
    return g[0], u[0], g[1], u[1]


def moe_experts(x, route_w, route_ids, w_gate, w_up, w_down):
    """y[t] = sum_j w[j, t] * ffn(x[t]), its bound, and sum_j |w ffn|; x [T, H], weights [E, N, K] float64."""
    xq = quantised(x)
    y, bound, terms = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    k = route_ids.shape[0]
    for e in route_ids.unique().tolist():
        j, t = torch.nonzero(route_ids == e, as_tuple=True)
        d, b = expert_ffn(xq[t], w_gate[e], w_up[e], w_down[e])
        w = route_w[j, t][:, None]
        y.index_add_(0, t, d * w)
        terms.index_add_(0, t, (d * w).abs())
        bound.index_add_(0, t, (b + (k + 2) * U32 * d.abs()) * w.abs())
    return y, bound, terms


def rms_norm(x, w, eps, err=None):
    """x / sqrt(mean x^2 + eps) * w and its bound: the sum of H squares, the square root, the divide and two
    products in fp32, (H / 2 + 8) units; err: a bound on x's own error."""
    H = x.shape[-1]
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    y = x * r * w
    bound = (H / 2 + 8) * U32 * y.abs()
    if err is not None:  # d y = r w dx - x w r^3 mean(x dx)
        rms_err = torch.sqrt((err * err).mean(-1, keepdim=True))
        bound = bound + 1.1 * (r * w.abs() * err + y.abs() * r * rms_err)
    return y, bound


def post_norm_residual(y, residual, w, eps, gate=None, residual_scale=1.0, err_y=None):
    """residual_scale * residual + gate * rms_norm(y, w) before its last rounding, and its bound; w None: no norm."""
    if w is None:
        n, b = y, torch.zeros_like(y) if err_y is None else err_y
    else:
        n, b = rms_norm(y, w, eps, err_y)
    if gate is not None:
        g = gate.reshape(-1, gate.shape[-1]).repeat_interleave(y.shape[0] // gate.reshape(-1, gate.shape[-1]).shape[0], 0)
        n, b = n * g, b * g.abs() + 2 * U32 * (n * g).abs()
    out = residual_scale * residual + n
    return out, b + 3 * U32 * ((residual_scale * residual).abs() + n.abs())
