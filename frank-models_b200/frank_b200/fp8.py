"""The 8-bit path: rows and expert weights in e4m3 with a scale for each block
of 128 (include/frank_fp8.h has the formulas).

Functions take and return torch tensors, launch on the current stream of the
tensors' device and do not synchronise.  Inputs that are not contiguous or not
16-byte aligned are copied.  Every workspace comes from torch's caching
allocator in the call that uses it, so calls on several streams and captured
graphs do not share one.
"""

from __future__ import annotations

import contextlib

import torch

from . import _lib, ops
from .ops import _DT, _ptr

BLOCK = _lib.FP8_BLOCK
E4M3 = torch.float8_e4m3fn
FLOATS = (torch.float32, torch.bfloat16)


BF16_ONLY, F32_ONLY, I32_ONLY, E4M3_ONLY = ((t,) for t in (torch.bfloat16, torch.float32, torch.int32, E4M3))
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_SAME_DEVICE = contextlib.nullcontext()


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _on(device: torch.device):
    """The context in which the library's calls go to `device` (nothing to do where it is the current one)."""
    return _SAME_DEVICE if device.index == _current_device() else torch.cuda.device(device)


def _stream() -> int:
    """The current device's current stream, as a handle."""
    return torch._C._cuda_getCurrentRawStream(_current_device())


def _arg(t, name: str, shape=None, dtypes=FLOATS, device=None) -> torch.Tensor:
    """A checked input: dtype, shape (None: any extent) and device; contiguous and 16-byte aligned."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: unsupported dtype {t.dtype}; expected {' or '.join(str(d) for d in dtypes)}")
    if shape is not None:
        got = t.shape
        if got != shape and (len(got) != len(shape) or [s for s, n in zip(shape, got) if s is not None and s != n]):
            want = ", ".join("*" if s is None else str(s) for s in shape)
            raise ValueError(f"{name}: expected shape [{want}], got {tuple(got)}")
    if not t.is_cuda:
        raise ValueError(f"{name}: tensor must be on a CUDA device")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: tensor is on {t.device}, expected {device}")
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _new(rows: int, cols: int, dtype, device) -> torch.Tensor:
    """[rows, cols]; empty_strided costs the host two thirds of empty."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _out(out, name: str, shape, dtype, device, like: torch.Tensor | None = None) -> torch.Tensor:
    """The output: new, or the caller's (exact shape and dtype, contiguous, aligned).
    like: a contiguous tensor of the shape (empty_like costs the host half of empty)."""
    if out is None:
        return torch.empty_like(like) if like is not None and like.dtype == dtype else _new(*shape, dtype, device)
    if (not isinstance(out, torch.Tensor) or tuple(out.shape) != tuple(shape) or out.dtype != dtype
            or out.device != device or not out.is_contiguous() or out.data_ptr() % 16 != 0):
        raise ValueError(f"{name}: out must be contiguous, 16-byte aligned {dtype} {list(shape)} on {device}")
    return out


def _multiple(n: int, name: str) -> None:
    if n < 16 or n % 16 != 0:
        raise ValueError(f"{name}={n} is not a positive multiple of 16")


def quantize_fp8(x: torch.Tensor):
    """x [T, K] (float32 or bfloat16) -> (q float8_e4m3fn [T, K], scale float32
    [ceil(K/128), T]); x is about q * scale, the scales powers of two."""
    x = _arg(x, "quantize_fp8: x", (None, None))
    T, K = x.shape
    _multiple(K, "quantize_fp8: K")
    with _on(x.device):
        q = _new(T, K, E4M3, x.device)
        scale = _new(_blocks(K), T, torch.float32, x.device)
        _lib.check(_lib.load().frank_quantize_fp8(_DT[x.dtype], _ptr(x), T, K, _ptr(q), _ptr(scale), _stream()))
    return q, scale


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float, return_norm: bool = False):
    """xn = bfloat16(rms_norm(x, weight, eps)) of x [T, H] and its 8-bit form:
    (q, scale) as :func:`quantize_fp8` gives for xn, or (q, scale, xn)."""
    x = _arg(x, "rms_norm_fp8: x", (None, None))
    T, H = x.shape
    _multiple(H, "rms_norm_fp8: H")
    weight = _arg(weight, "rms_norm_fp8: weight", (H,), F32_ONLY, x.device)
    with _on(x.device):
        q = _new(T, H, E4M3, x.device)
        scale = _new(_blocks(H), T, torch.float32, x.device)
        xn = _new(T, H, torch.bfloat16, x.device) if return_norm else None
        _lib.check(_lib.load().frank_rms_norm_fp8(_DT[x.dtype], _ptr(x), _ptr(weight), T, H, float(eps), _ptr(xn),
                                                  _ptr(q), _ptr(scale), _stream()))
    return (q, scale, xn) if return_norm else (q, scale)


class Fp8Experts:
    """Expert weights in 8 bits: ``q`` float8_e4m3fn [E, N, K] and ``scale``
    float32 [E, ceil(N/128), ceil(K/128)], one for each 128 x 128 block (a quantised
    checkpoint's are used as they are; magnitudes below 2^8 serve every row).  The
    tensors are held, not copied, unless they are not contiguous or not 16-byte aligned;
    others of the same shape may be assigned."""

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        q = _arg(q, "Fp8Experts: q", (None, None, None), E4M3_ONLY)
        E, N, K = q.shape
        _multiple(N, "Fp8Experts: n_out")
        _multiple(K, "Fp8Experts: n_in")
        self._q = q
        self.scale = scale

    @property
    def q(self) -> torch.Tensor:
        return self._q

    @q.setter
    def q(self, q: torch.Tensor) -> None:
        self._q = _arg(q, "Fp8Experts: q", self._q.shape, E4M3_ONLY, self._q.device)

    @property
    def scale(self) -> torch.Tensor:
        return self._scale

    @scale.setter
    def scale(self, scale: torch.Tensor) -> None:
        E, N, K = self._q.shape
        self._scale = _arg(scale, "Fp8Experts: scale", (E, _blocks(N), _blocks(K)), F32_ONLY, self._q.device)

    @classmethod
    def from_reference(cls, w_oie: torch.Tensor) -> "Fp8Experts":
        """Quantise [O, I, E] expert-innermost weights (float32 or bfloat16)."""
        w = _arg(w_oie, "Fp8Experts: weights", (None, None, None))
        O, I, E = w.shape
        _multiple(O, "Fp8Experts: n_out")
        _multiple(I, "Fp8Experts: n_in")
        with _on(w.device):
            q = torch.empty((E, O, I), dtype=E4M3, device=w.device)
            scale = torch.empty((E, _blocks(O), _blocks(I)), dtype=torch.float32, device=w.device)
            _lib.check(_lib.load().frank_prepack_experts_fp8(_DT[w.dtype], _ptr(w), O, I, E, _ptr(q), _ptr(scale),
                                                             _stream()))
        return cls(q, scale)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weights [E, N, K] that the 8-bit form stands for."""
        E, N, K = self.q.shape
        s = self.scale.repeat_interleave(BLOCK, 1)[:, :N].repeat_interleave(BLOCK, 2)[:, :, :K]
        return (self.q.float() * s).to(dtype)

    @property
    def n_expert(self):
        return self.q.shape[0]

    @property
    def n_out(self):
        return self.q.shape[1]

    @property
    def n_in(self):
        return self.q.shape[2]


def fp8_matmul(x, weights: Fp8Experts, offsets: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows times 8-bit weights: x [R, K] (float32 or bfloat16, quantised here)
    or a (q, scale) pair of :func:`quantize_fp8` -> [R, N] in ``out_dtype``.
    ``offsets``: int32 [E+1], ascending from 0 to R, the first row of each expert's
    group; None for a single expert.  Rows of ``out`` outside every group are
    left as they were."""
    if not isinstance(weights, Fp8Experts):
        raise TypeError(f"fp8_matmul: weights must be Fp8Experts, got {type(weights).__name__}")
    wq = weights.q
    E, N, K = wq.shape
    dev = wq.device
    if out_dtype not in FLOATS:
        raise TypeError(f"fp8_matmul: unsupported output dtype {out_dtype}")
    quantised = isinstance(x, (tuple, list))
    if quantised:
        if len(x) != 2:
            raise ValueError("fp8_matmul: expected (q, scale)")
        q = _arg(x[0], "fp8_matmul: q", (None, K), E4M3_ONLY, dev)
        R = q.shape[0]
        scale = _arg(x[1], "fp8_matmul: scale", (_blocks(K), R), F32_ONLY, dev)
    else:
        x = _arg(x, "fp8_matmul: x", (None, K), FLOATS, dev)
        R = x.shape[0]
    if offsets is not None:
        offsets = _arg(offsets, "fp8_matmul: offsets", (E + 1,), I32_ONLY, dev)
    elif E != 1:
        raise ValueError(f"fp8_matmul: offsets may be omitted only for one expert, not {E}")
    lib = _lib.load()
    with _on(dev):
        y = _out(out, "fp8_matmul", (R, N), out_dtype, dev)
        if quantised:
            _lib.check(lib.frank_fp8_matmul(_ptr(q), _ptr(scale), _ptr(wq), _ptr(weights.scale),
                                            _ptr(offsets), E, R, N, K, _DT[out_dtype], _ptr(y), _stream()))
        else:
            need = lib.frank_fp8_linear_workspace_size(R, K)
            ws = wq.new_empty(need)
            _lib.check(lib.frank_fp8_linear(_DT[x.dtype], _ptr(x), _ptr(wq), _ptr(weights.scale),
                                            _ptr(offsets), E, R, N, K, _DT[out_dtype], _ptr(y), _ptr(ws), need,
                                            _stream()))
    return y


def _gate_arg(gate, name, T, H, device):
    """(gate, its rows): [H], or [G, H] with G dividing T."""
    if gate is None:
        return None, 1
    gate = _arg(gate, f"{name}: gate", None, F32_ONLY, device)
    shape = gate.shape
    rows = shape[0] if len(shape) == 2 else 1
    if not 1 <= len(shape) <= 2 or shape[-1] != H or rows < 1 or T % rows != 0:
        raise ValueError(f"{name}: gate must be [{H}] or [G, {H}] with G dividing {T}, got {tuple(shape)}")
    return gate, rows


class Fp8MoEFFNBlock(ops.MoEFFNBlock):
    """:class:`MoEFFNBlock` with 8-bit expert weights: tokens in bfloat16, rows
    and the hidden values quantised in blocks of 128 on the way, sums in fp32.
    The expert weights are :class:`Fp8Experts` or the reference layouts (up/gate
    [F, H, E], down [H, F, E]), which are quantised once here.  A call reads the
    expert weights that ``w_up``, ``w_gate`` and ``w_down`` are then, in-place changes
    included, and the router that ``wr`` was when it was last assigned.  A captured
    graph goes on reading the expert tensors that it was captured with."""

    def __init__(self, gate_inp_w, up_exps_w, gate_exps_w, down_exps_w, n_expert: int, n_expert_used: int,
                 normalize_weights: bool, out_dtype: torch.dtype = torch.float32):
        if out_dtype not in FLOATS:
            raise TypeError(f"Fp8MoEFFNBlock: unsupported output dtype {out_dtype}")
        self.dtype = torch.bfloat16
        self.out_dtype = out_dtype
        self.E, self.k, self.normalize = int(n_expert), int(n_expert_used), bool(normalize_weights)
        if not 1 <= self.k <= min(self.E, 32):
            raise ValueError(f"Fp8MoEFFNBlock: n_expert_used={self.k} outside [1, min({self.E}, 32)]")
        up, gate, down = (w if isinstance(w, Fp8Experts) else Fp8Experts.from_reference(w)
                          for w in (up_exps_w, gate_exps_w, down_exps_w))
        _, self.F, self.H = up.q.shape
        self.device = up.q.device
        self.w_up, self.w_gate, self.w_down = up, gate, down
        self.wr_pack = None
        self.wr = gate_inp_w

    @property
    def wr(self) -> torch.Tensor:
        """The router [E, H].  Calls read its packed form ``wr_pack``, which assigning ``wr`` rewrites in place on the
        current stream, so captured graphs take the new router up too.  After a change of ``wr`` in place, assign it
        again (``block.wr = block.wr``)."""
        return self._wr

    @wr.setter
    def wr(self, gate_inp_w: torch.Tensor) -> None:
        wr = _arg(gate_inp_w, "gate_inp_w", (self.E, self.H), device=self.device)
        with _on(self.device):
            if self.wr_pack is None:
                self.wr_pack = ops.router_pack(wr)
            else:
                _lib.check(_lib.load().frank_router_pack(_DT[wr.dtype], _ptr(wr), self.E, self.H, _ptr(self.wr_pack),
                                                         _stream()))
        self._wr = wr

    def _fit(self, weights: Fp8Experts, name: str, n_out: int, n_in: int) -> Fp8Experts:
        """Weights for this block: the kernels read them by the block's sizes."""
        if not isinstance(weights, Fp8Experts):
            raise TypeError(f"Fp8MoEFFNBlock: {name} must be Fp8Experts, got {type(weights).__name__}")
        q = weights.q
        if tuple(q.shape) != (self.E, n_out, n_in):
            raise ValueError(f"Fp8MoEFFNBlock: {name} has shape {tuple(q.shape)}, expected "
                             f"[{self.E}, {n_out}, {n_in}]")
        if q.device != self.device:
            raise ValueError(f"Fp8MoEFFNBlock: {name} is on device {q.device}, expected {self.device}")
        return weights

    w_up = property(lambda self: self._up, lambda self, w: setattr(self, "_up", self._fit(w, "w_up", self.F, self.H)))
    w_gate = property(lambda self: self._gate,
                      lambda self, w: setattr(self, "_gate", self._fit(w, "w_gate", self.F, self.H)))
    w_down = property(lambda self: self._down,
                      lambda self, w: setattr(self, "_down", self._fit(w, "w_down", self.H, self.F)))

    def _weights(self):
        return [_ptr(t) for w in (self._up, self._gate, self._down) for t in (w._q, w._scale)]

    def workspace_bytes(self, T: int) -> int:
        return _lib.load().frank_fp8_moe_workspace_size(T, self.H, self.F, self.E, self.k)

    def _workspace(self, T: int, device, need: int | None = None) -> torch.Tensor:
        """New for each call: ordered by the stream it is used on, kept by the graph that captures it."""
        return torch.empty(self.workspace_bytes(T) if need is None else need, dtype=torch.uint8, device=device)

    def _routing(self, T, wanted):
        if not wanted:
            return None, None
        return _new(self.k, T, torch.float32, self.device), _new(self.k, T, torch.int32, self.device)

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, return_routing: bool = False):
        """moe_ffn_block on tokens x [T, H] bfloat16 -> y [T, H] in ``out_dtype``."""
        x = _arg(x, "fp8_moe_block: x", (None, self.H), BF16_ONLY, self.device)
        T = x.shape[0]
        with _on(self.device):
            y = _out(out, "fp8_moe_block", (T, self.H), self.out_dtype, self.device, x)
            rw, rid = self._routing(T, return_routing)
            ws = self._workspace(T, self.device)
            _lib.check(_lib.load().frank_fp8_moe_block(
                _ptr(x), _lib.ROUTER_PACKED, _ptr(self.wr_pack), *self._weights(), T, self.E, self.k, self.H, self.F,
                int(self.normalize), _DT[self.out_dtype], _ptr(y), _ptr(rw), _ptr(rid), _ptr(ws), ws.numel(),
                _stream()))
        return (y, rw, rid) if return_routing else y

    def experts(self, x: torch.Tensor, route_w: torch.Tensor, route_ids: torch.Tensor,
                out: torch.Tensor | None = None, check_ids: bool = False) -> torch.Tensor:
        """The expert FFN with the routing given: x [T, H] bfloat16, route_w
        float32 [k, T], route_ids int32 [k, T] (one named twice counts twice) -> y
        [T, H] = sum_j route_w[j] * down(gate(x) * silu(up(x))).  With check_ids,
        ids outside [0, E) raise FrankError(EIDS) (this synchronises the stream);
        without, they are clamped."""
        x = _arg(x, "fp8_moe_experts: x", (None, self.H), BF16_ONLY, self.device)
        T = x.shape[0]
        route_w = _arg(route_w, "fp8_moe_experts: route_w", (self.k, T), F32_ONLY, self.device)
        route_ids = _arg(route_ids, "fp8_moe_experts: route_ids", (self.k, T), I32_ONLY, self.device)
        with _on(self.device):
            y = _out(out, "fp8_moe_experts", (T, self.H), self.out_dtype, self.device, x)
            err = torch.zeros(1, dtype=torch.int32, device=self.device) if check_ids else None
            ws = self._workspace(T, self.device)
            _lib.check(_lib.load().frank_fp8_moe_experts(
                _ptr(x), _ptr(route_w), _ptr(route_ids), *self._weights(), T, self.E, self.k, self.H, self.F,
                _DT[self.out_dtype], _ptr(y), _ptr(err), _ptr(ws), ws.numel(), _stream()))
            if check_ids and int(err.item()) != 0:
                raise _lib.FrankError(_lib.EIDS, f"fp8_moe_experts: an expert id is outside [0, {self.E})")
        return y

    def sublayer(self, residual: torch.Tensor, ffn_norm_w: torch.Tensor, rms_eps: float,
                 out: torch.Tensor | None = None, return_routing: bool = False,
                 post_norm_w: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                 residual_scale: float = 1.0):
        """The sub-layer: ``residual_scale * residual + gate * post(block(xn))``
        with xn = bfloat16(rms_norm(residual, ffn_norm_w, rms_eps)) and post the
        rms_norm by post_norm_w (nothing when None).  residual and the result are
        [T, H] in float32 or bfloat16; gate float32 [H], or [G, H] with one row for
        each T/G consecutive tokens.  ``out`` may be ``residual``."""
        res = _arg(residual, "fp8_moe_sublayer: residual", (None, self.H), device=self.device)
        T = res.shape[0]
        ffn_norm_w = _arg(ffn_norm_w, "fp8_moe_sublayer: ffn_norm_w", (self.H,), F32_ONLY, self.device)
        if post_norm_w is not None:
            post_norm_w = _arg(post_norm_w, "fp8_moe_sublayer: post_norm_w", (self.H,), F32_ONLY, self.device)
        gate, gate_rows = _gate_arg(gate, "fp8_moe_sublayer", T, self.H, self.device)
        with _on(self.device):
            y = _out(out, "fp8_moe_sublayer", (T, self.H), res.dtype, self.device, res)
            rw, rid = self._routing(T, return_routing)
            ws = self._workspace(T, self.device)
            _lib.check(_lib.load().frank_fp8_moe_sublayer(
                _DT[res.dtype], _ptr(res), _ptr(ffn_norm_w), float(rms_eps), _lib.ROUTER_PACKED, _ptr(self.wr_pack),
                *self._weights(), T, self.E, self.k, self.H, self.F, int(self.normalize), _ptr(post_norm_w),
                _ptr(gate), gate_rows, float(residual_scale), _ptr(y), _ptr(rw), _ptr(rid), _ptr(ws), ws.numel(),
                _stream()))
        return (y, rw, rid) if return_routing else y


def post_norm_residual(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float,
                       gate: torch.Tensor | None = None, residual_scale: float = 1.0,
                       next_weight: torch.Tensor | None = None, next_dtype: torch.dtype = torch.bfloat16,
                       out: torch.Tensor | None = None):
    """The end of a sub-layer: ``out = residual_scale * residual + gate *
    rms_norm(y, weight, eps)`` for y and residual [T, H] (float32 or bfloat16
    each; out has residual's dtype and may be residual), gate float32 [H] or
    [G, H] (one row for each T/G consecutive tokens).  With next_weight also the
    next block's input, rms_norm(out, next_weight, eps) in next_dtype: (out, next)."""
    y = _arg(y, "post_norm_residual: y", (None, None))
    T, H = y.shape
    if H % 4 != 0 or H < 4:
        raise ValueError(f"post_norm_residual: H={H} is not a positive multiple of 4")
    dev = y.device
    res = _arg(residual, "post_norm_residual: residual", (T, H), device=dev)
    weight = _arg(weight, "post_norm_residual: weight", (H,), F32_ONLY, dev)
    gate, gate_rows = _gate_arg(gate, "post_norm_residual", T, H, dev)
    if next_dtype not in FLOATS:
        raise TypeError(f"post_norm_residual: unsupported dtype {next_dtype}")
    if next_weight is not None:
        next_weight = _arg(next_weight, "post_norm_residual: next_weight", (H,), F32_ONLY, dev)
    with _on(dev):
        o = _out(out, "post_norm_residual", (T, H), res.dtype, dev, res)
        nxt = _out(None, "", (T, H), next_dtype, dev, res) if next_weight is not None else None
        _lib.check(_lib.load().frank_post_norm_residual(
            _DT[y.dtype], _ptr(y), _DT[res.dtype], _ptr(res), _ptr(weight), float(eps), _ptr(gate), gate_rows,
            float(residual_scale), _ptr(o), _ptr(next_weight), _DT[next_dtype], _ptr(nxt), T, H, _stream()))
    return o if nxt is None else (o, nxt)
