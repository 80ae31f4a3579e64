"""The 8-bit path on the GPU against its definition in float64 (oracle/fp8_oracle.py).

Quantisation is exact.  Everything else is held to the oracle's own error
bounds: fp32 sums in any order, one rounding of the output (half a step of its
type), and for the expert FFN the values of h that lie so near a rounding
border that an fp32 sum may take either side.
"""

import pytest
import torch

import frank_b200 as fb
from frank_b200 import ops
from oracle import fp8_oracle as Q
from tests.utils import strict_route

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, std=1.0, dtype=F32):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def weights(g, E, N, K):
    """8-bit weights with scales that are no powers of two."""
    q = (torch.randn((E, N, K), generator=g, device=DEV) * 100).clamp_(-448, 448).to(E4M3)
    s = (torch.rand((E, -(-N // 128), -(-K // 128)), generator=g, device=DEV) + 0.5) * 2e-4
    return fb.Fp8Experts(q, s)


def dense(w):
    s = w.scale.double().repeat_interleave(128, 1)[:, :w.n_out].repeat_interleave(128, 2)[:, :, :w.n_in]
    return w.q.double() * s


def values(q, scale):
    return q.double() * scale.double().t().repeat_interleave(128, 1)[:, :q.shape[1]]


def within(got, want, bound, what=""):
    """|got - want| <= bound + one rounding of the output to its type."""
    got64 = got.double()
    tol = bound + Q.half_step(got.dtype) * (want.abs() + bound) + 1e-37
    bad = ~((got64 - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(((got64 - want).abs() / tol).max()))


# ---------------------------------------------------------------- quantise --
@pytest.mark.parametrize("T,K", [(1, 16), (3, 128), (5, 144), (7, 2048), (1000, 272), (2, 4112)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize(T, K, dtype):
    g = gen(T + K)
    x = randn(g, T, K) * torch.exp2(torch.randint(-20, 20, (T, 1), generator=g, device=DEV).float())
    x[0, :16] = 0
    x = x.to(dtype)
    q, s = fb.quantize_fp8(x)
    want_s = Q.block_scales(x.double())
    assert torch.equal(s.double().t(), want_s)
    assert torch.equal(values(q, s), Q.quantised(x.double()))


def test_quantize_special_values():
    x = torch.zeros(8, 256, device=DEV)
    x[1, 3] = float("inf")
    x[2, 200] = float("nan")
    x[3] = 1e-42                      # denormal
    x[4, 0], x[4, 1] = 448.0, 17.0    # a tie, to even
    x[5, 0] = 3.4e38
    x[6, 0], x[6, 1] = 1.75, 1e-30
    x[7, 0] = -1.7500001
    q, s = fb.quantize_fp8(x)
    assert torch.isnan(s[0, 1]) and torch.isnan(s[1, 2]) and not torch.isnan(s[1, 1]) and not torch.isnan(s[0, 2])
    ok = torch.tensor([0, 3, 4, 5, 6, 7], device=DEV)
    assert torch.equal(values(q, s)[ok], Q.quantised(x.double())[ok])
    assert s[0, 6] == 2.0 ** -8 and s[0, 7] == 2.0 ** -7
    assert torch.isnan(values(q, s)[1, :128]).all() and torch.isnan(values(q, s)[2, 128:]).all()


def test_quantize_views():
    """A strided and a misaligned view give what their copies give."""
    base = randn(gen(1), 9 * 300 + 1)
    a = base[1:1 + 9 * 288].view(9, 288)       # 4 bytes off
    b = base[:2700].view(9, 300)[:, 4:276]     # rows apart
    c = randn(gen(2), 272, 6).t()
    for v in (a, b, c):
        q, s = fb.quantize_fp8(v)
        q2, s2 = fb.quantize_fp8(v.clone(memory_format=torch.contiguous_format))
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


@pytest.mark.parametrize("O,I,E", [(16, 16, 1), (144, 272, 3), (128, 384, 40), (400, 128, 8)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prepack(O, I, E, dtype):
    w = randn(gen(O), O, I, E, std=0.02, dtype=dtype)
    p = fb.Fp8Experts.from_reference(w)
    w64 = w.double().permute(2, 0, 1)
    for e in range(E):
        for o in range(0, O, 128):
            for i in range(0, I, 128):
                blk = w64[e, o:o + 128, i:i + 128]
                s = torch.exp2(torch.ceil(torch.log2(blk.abs().max() / 448.0)))
                assert p.scale[e, o // 128, i // 128].double() == s
                assert torch.equal(p.q[e, o:o + 128, i:i + 128].double(), Q.round_e4m3(blk / s))
    assert torch.equal(p.dequantize().double(), dense(p))


# ----------------------------------------------------------------- product --
PRODUCTS = [(1, 16, 16), (1, 1536, 2048), (5, 144, 272), (64, 256, 128), (130, 272, 400), (129, 528, 96),
            (300, 512, 1024), (257, 784, 2000), (1024, 1296, 640)]


@pytest.mark.parametrize("R,N,K", PRODUCTS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_matmul_dense(R, N, K, dtype):
    g = gen(R + N + K)
    x = randn(g, R, K, dtype=BF16)
    w = weights(g, 1, N, K)
    q, s = fb.quantize_fp8(x)
    want, bound = Q.product(values(q, s), dense(w)[0])
    y = fb.fp8_matmul(x, w, out_dtype=dtype)
    assert y.dtype == dtype
    within(y, want, bound)
    assert torch.equal(y, fb.fp8_matmul((q, s), w, out_dtype=dtype))


GROUPS = [([0, 5, 5, 128, 0], 272, 384), ([1] * 40, 256, 256), ([300, 0, 0, 700, 17, 1], 400, 272),
          ([0, 0, 3], 128, 128), ([2000, 1500, 513], 528, 256)]


@pytest.mark.parametrize("counts,N,K", GROUPS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_matmul_grouped(counts, N, K, dtype):
    g = gen(sum(counts) + N)
    E, R = len(counts), sum(counts)
    w = weights(g, E, N, K)
    q, s = fb.quantize_fp8(randn(g, R, K, dtype=BF16))
    off = torch.tensor([0] + counts, device=DEV).cumsum(0).to(torch.int32)
    y = fb.fp8_matmul((q, s), w, offsets=off, out_dtype=dtype)
    x64, w64 = values(q, s), dense(w)
    for e in range(E):
        a, b = int(off[e]), int(off[e + 1])
        within(y[a:b], *Q.product(x64[a:b], w64[e]), what=e)
    assert ops.read_device_error() == 0


def test_matmul_rows_outside_the_groups_stay():
    g = gen(7)
    w = weights(g, 2, 144, 256)
    q, s = fb.quantize_fp8(randn(g, 500, 256))
    off = torch.tensor([100, 230, 301], dtype=torch.int32, device=DEV)
    out = torch.full((500, 144), 7.5, device=DEV)
    fb.fp8_matmul((q, s), w, offsets=off, out_dtype=F32, out=out)
    assert (out[:100] == 7.5).all() and (out[301:] == 7.5).all()
    x64, w64 = values(q, s), dense(w)
    within(out[100:230], *Q.product(x64[100:230], w64[0]))
    within(out[230:301], *Q.product(x64[230:301], w64[1]))


def test_matmul_a_bad_row_stays_alone():
    """A NaN and an infinity reach their own rows only."""
    g = gen(8)
    x = randn(g, 200, 400)
    w = weights(g, 1, 272, 400)
    clean = fb.fp8_matmul(x, w, out_dtype=F32)
    x[17, 3], x[150, 399] = float("nan"), float("-inf")
    y = fb.fp8_matmul(x, w, out_dtype=F32)
    assert torch.isnan(y[17]).all() and torch.isnan(y[150]).all()
    keep = torch.ones(200, dtype=torch.bool, device=DEV)
    keep[17] = keep[150] = False
    assert torch.equal(y[keep], clean[keep])


def test_matmul_large_offsets():
    """Weights past 2^31 bytes: the last expert's are found."""
    E, N, K = 34, 8192, 8192
    q = torch.zeros((E, N, K), dtype=torch.uint8, device=DEV).view(E4M3)
    s = torch.ones((E, N // 128, K // 128), device=DEV)
    g = gen(9)
    q[E - 1, N - 128:] = (torch.randn((128, K), generator=g, device=DEV) * 100).clamp_(-448, 448).to(E4M3)
    w = fb.Fp8Experts(q, s)
    off = torch.tensor([0] * E + [3], dtype=torch.int32, device=DEV)
    xq, xs = fb.quantize_fp8(randn(g, 3, K))
    y = fb.fp8_matmul((xq, xs), w, offsets=off, out_dtype=F32)
    want, bound = Q.product(values(xq, xs), q[E - 1, N - 128:].double())
    within(y[:, N - 128:], want, bound)
    assert (y[:, :N - 128] == 0).all()


# ------------------------------------------------------------------- norms --
@pytest.mark.parametrize("T,H", [(1, 16), (3, 272), (9, 1024), (5, 1040), (2, 2048), (1000, 4096), (2, 16384),
                                 (19001, 48), (2501, 1040), (1301, 2064)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rms_norm_fp8(T, H, dtype):
    g = gen(T + H)
    x, w = randn(g, T, H, dtype=dtype), 1 + randn(g, H, std=0.1)
    q, s, xn = fb.rms_norm_fp8(x, w, 1e-5, return_norm=True)
    within(xn, *Q.rms_norm(x.double(), w.double(), 1e-5))
    q2, s2 = fb.quantize_fp8(xn)
    assert torch.equal(s, s2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
    q3, s3 = fb.rms_norm_fp8(x, w, 1e-5)
    assert torch.equal(s, s3) and torch.equal(q.view(torch.uint8), q3.view(torch.uint8))


@pytest.mark.parametrize("T,H,gates,nxt", [(1, 4, 1, True), (1, 2048, 0, True), (7, 100, 7, False), (6, 1028, 3, True),
                                           (12, 4096, 1, True), (3, 16384, 1, True), (1021, 2040, 1021, False),
                                           (19002, 36, 2, True), (2502, 1500, 1, False), (1302, 4100, 3, True),
                                           (1201, 16384, 0, True)])
@pytest.mark.parametrize("y_dtype,res_dtype", [(F32, BF16), (BF16, F32), (F32, F32), (BF16, BF16)])
def test_post_norm_residual(T, H, gates, nxt, y_dtype, res_dtype):
    g = gen(T + H)
    y, res = randn(g, T, H, std=0.3, dtype=y_dtype), randn(g, T, H, dtype=res_dtype)
    w, w2 = 1 + randn(g, H, std=0.1), 1 + randn(g, H, std=0.1)
    gate = randn(g, gates, H) if gates else None
    out = fb.post_norm_residual(y, res, w, 1e-5, gate=gate, residual_scale=0.75, next_weight=w2 if nxt else None,
                                next_dtype=y_dtype)
    out, xn = out if nxt else (out, None)
    want, bound = Q.post_norm_residual(y.double(), res.double(), w.double(), 1e-5,
                                       None if gate is None else gate.double(), 0.75)
    assert out.dtype == res_dtype
    within(out, want, bound)
    if nxt:
        assert xn.dtype == y_dtype
        within(xn, *Q.rms_norm(out.double(), w2.double(), 1e-5))
    # in place, the same bits
    again = res.clone()
    got = fb.post_norm_residual(y, again, w, 1e-5, gate=gate, residual_scale=0.75, out=again)
    assert got is again and torch.equal(again, out)


def test_post_norm_residual_special_rows():
    y = torch.zeros(4, 256, device=DEV)
    y[1, 0], y[2, 5], y[3] = float("nan"), float("inf"), 1e-30
    res = torch.ones(4, 256, device=DEV)
    out = fb.post_norm_residual(y, res, torch.ones(256, device=DEV), 1e-5)
    assert (out[0] == 1).all() and torch.isnan(out[1]).all() and torch.isnan(out[2, 5]) and (out[3] == 1).all()


# ------------------------------------------------------------- expert FFN ---
def block(g, T, H, F, E, k, normalize=True, out_dtype=BF16):
    up, gate, down = weights(g, E, F, H), weights(g, E, F, H), weights(g, E, H, F)
    wr = randn(g, E, H, std=0.05)
    return fb.Fp8MoEFFNBlock(wr, up, gate, down, E, k, normalize, out_dtype=out_dtype)


def prompt(T, b):
    """Whether T tokens run as a prompt: sorted rows, not the few tokens' kernels."""
    return T > 64 or b.k * T > 512 or b.k * T > 24 * b.E


def want_moe(b, x, rw, rid):
    """The block in float64 and its bound.  For a prompt and a bf16 result every slot's product is rounded to bf16
    before the fp32 sum: at most half a step of each term, |w d| with its own bound."""
    args = x.double(), rw.double(), rid, dense(b.w_gate), dense(b.w_up), dense(b.w_down)
    y, bound, terms = Q.moe_experts(*args)
    if b.out_dtype == BF16 and prompt(x.shape[0], b):
        bound = bound + Q.half_step(BF16) * (terms + bound)
    return y, bound


EXPERTS = [(64, 256, 272, 2, 2), (33, 128, 256, 1, 1), (24, 128, 256, 1, 1), (1, 128, 128, 1, 1), (1, 256, 144, 8, 2), (3, 272, 400, 16, 4), (40, 256, 256, 5, 3), (200, 144, 272, 12, 2),
           (700, 512, 384, 4, 2), (65, 1040, 96, 130, 6), (2, 16, 16, 3, 3)]


@pytest.mark.parametrize("T,H,F,E,k", EXPERTS)
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_experts(T, H, F, E, k, out_dtype):
    g = gen(T + H + F)
    b = block(g, T, H, F, E, k, out_dtype=out_dtype)
    x = randn(g, T, H, dtype=BF16)
    rid = torch.rand((T, E), generator=g, device=DEV).topk(k, 1)[1].t().to(torch.int32).contiguous()
    rw = torch.rand((k, T), generator=g, device=DEV)
    y = b.experts(x, rw, rid)
    within(y, *want_moe(b, x, rw, rid))
    assert torch.equal(y, b.experts(x, rw, rid)), "two runs differ"
    assert ops.read_device_error() == 0


def test_experts_all_tokens_on_one():
    g = gen(3)
    b = block(g, 300, 256, 272, 6, 1, out_dtype=F32)
    for T in (1, 33, 300):
        x = randn(g, T, 256, dtype=BF16)
        rid = torch.full((1, T), 4, dtype=torch.int32, device=DEV)
        rw = torch.rand((1, T), generator=g, device=DEV)
        within(b.experts(x, rw, rid), *want_moe(b, x, rw, rid))


def test_experts_ids_out_of_range():
    from frank_b200 import _lib

    g = gen(4)
    for T in (2, 300):
        b = block(g, T, 128, 128, 4, 2)
        x = randn(g, T, 128, dtype=BF16)
        rid = torch.tensor([[0], [3]], device=DEV).expand(2, T).to(torch.int32).contiguous()
        rw = torch.ones((2, T), device=DEV)
        b.experts(x, rw, rid, check_ids=True)
        for bad in (4, -1, 2 ** 31 - 1, -2 ** 31):
            rid[1, T - 1] = bad
            with pytest.raises(_lib.FrankError, match="outside"):
                b.experts(x, rw, rid, check_ids=True)


BLOCKS = [(1, 2048, 768, 128, 8, False), (1, 256, 128, 4, 4, True), (8, 512, 400, 64, 8, True), (3, 528, 272, 9, 2, True),
          (47, 256, 144, 128, 8, True), (64, 1024, 256, 160, 6, False), (5, 4096, 1040, 8, 2, False),
          (5, 4096, 1024, 8, 2, True), (20, 2048, 2064, 6, 2, False), (130, 272, 128, 16, 4, True), (1000, 256, 256, 8, 2, False), (17, 48, 80, 256, 32, True)]


@pytest.mark.parametrize("T,H,F,E,k,normalize", BLOCKS)
def test_block(T, H, F, E, k, normalize):
    g = gen(T + H + F)
    b = block(g, T, H, F, E, k, normalize, out_dtype=F32)
    x = randn(g, T, H, dtype=BF16)
    y, rw, rid = b(x, return_routing=True)
    w, ids, near, differ = strict_route(x.double().cpu().numpy(), b.wr.cpu().numpy(), rw.cpu().numpy(),
                                        rid.cpu().numpy(), k, normalize)
    print(f"near-tied {near}, routed differently {differ} of {T}")
    within(y, *want_moe(b, x, rw, rid))
    assert torch.equal(y, b(x)), "two runs differ"
    assert torch.equal(y, b.experts(x, rw, rid)), "the routing given and the routing made differ"
    assert ops.read_device_error() == 0


def test_block_no_tokens():
    b = block(gen(5), 1, 128, 128, 4, 2)
    assert b(torch.empty((0, 128), dtype=BF16, device=DEV)).shape == (0, 128)
    assert b.sublayer(torch.empty((0, 128), device=DEV), torch.ones(128, device=DEV), 1e-5).shape == (0, 128)


def test_block_bad_tokens_stay_alone():
    """Tokens with a NaN or an infinity: NaN there, the other tokens as without them, ids in range."""
    g = gen(6)
    for T in (6, 200):
        b = block(g, T, 256, 128, 16, 4, out_dtype=F32)
        x = randn(g, T, 256, dtype=BF16)
        clean = b(x)
        bad = x.clone()
        bad[1, 7], bad[T - 2, 255] = float("nan"), float("inf")
        y = b(bad)
        keep = torch.ones(T, dtype=torch.bool, device=DEV)
        keep[1] = keep[T - 2] = False
        assert torch.equal(y[keep], clean[keep])
        assert torch.isnan(y[1]).all() and torch.isnan(y[T - 2]).all()
        assert ops.read_device_error() == 0


# --------------------------------------------------------------- together ---
@pytest.mark.parametrize("T,H,F,E,k", [(1, 512, 256, 16, 4), (6, 272, 144, 8, 2), (48, 1024, 128, 64, 8),
                                       (300, 256, 272, 8, 2)])
@pytest.mark.parametrize("res_dtype", [F32, BF16])
@pytest.mark.parametrize("post,gates", [(True, 1), (True, 0), (False, 3), (False, 0)])
def test_sublayer_is_its_parts(T, H, F, E, k, res_dtype, post, gates):
    """The sub-layer against rms_norm_fp8, the block in fp32 and the end of the sub-layer in float64."""
    g = gen(T + H)
    b = block(g, T, H, F, E, k, out_dtype=F32)
    res = randn(g, T, H, dtype=res_dtype)
    nw, pw = 1 + randn(g, H, std=0.1), 1 + randn(g, H, std=0.1)
    gates = gates if gates and T % gates == 0 else int(gates > 0)
    gate = randn(g, gates, H) if gates else None
    out, rw, rid = b.sublayer(res, nw, 1e-5, post_norm_w=pw if post else None, gate=gate, residual_scale=0.5,
                              return_routing=True)
    xn = fb.rms_norm_fp8(res, nw, 1e-5, return_norm=True)[2]
    y, rw2, rid2 = b(xn, return_routing=True)
    assert torch.equal(rid, rid2) and torch.equal(rw, rw2)
    err = None
    if prompt(T, b) and res_dtype == BF16:  # the slots' products are rounded to bf16 there, half a step each
        _, e, terms = Q.moe_experts(xn.double(), rw.double(), rid, dense(b.w_gate), dense(b.w_up), dense(b.w_down))
        err = Q.half_step(BF16) * (terms + e)
    want, bound = Q.post_norm_residual(y.double(), res.double(), pw.double() if post else None, 1e-5,
                                       None if gate is None else gate.double(), 0.5, err)
    within(out, want, bound)
    if post and (not prompt(T, b) or res_dtype == F32):
        assert torch.equal(out, fb.post_norm_residual(y, res, pw, 1e-5, gate=gate, residual_scale=0.5))
    again = res.clone()
    assert torch.equal(b.sublayer(again, nw, 1e-5, post_norm_w=pw if post else None, gate=gate, residual_scale=0.5,
                                  out=again), out)


def test_two_layers_decoding():
    """Three steps of two sub-layers as a server runs them, each step one captured graph: the bits of eager calls."""
    g = gen(11)
    T, H = 4, 512
    layers = [(block(g, T, H, 256, 32, 4), 1 + randn(g, H, std=0.1), 1 + randn(g, H, std=0.1)) for _ in range(2)]

    def step(x):
        for b, nw, pw in layers:
            x = b.sublayer(x, nw, 1e-5, post_norm_w=pw)
        return x

    x = randn(g, T, H, dtype=BF16)
    step(x)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        buf = torch.zeros_like(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step(buf)
        graphs.append((graph, buf, y))
    xs = [randn(g, T, H, dtype=BF16) for _ in range(3)]
    want = [step(v).clone() for v in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for v, w in zip(xs, want):  # two graphs of the same layers at once
        for (graph, buf, y), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                buf.copy_(v)
                graph.replay()
        torch.cuda.synchronize()
        for _, _, y in graphs:
            assert torch.equal(y, w)


def test_two_streams_at_once():
    g = gen(12)
    b = block(g, 1, 512, 256, 32, 4, out_dtype=F32)
    xs = [randn(g, T, 512, dtype=BF16) for T in (1, 7, 50, 300)]
    want = [b(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(b(x))
        torch.cuda.synchronize()
        for y, w in zip(got, want):
            assert torch.equal(y, w)


def test_graphed_and_host_pipelines_take_the_block():
    """The framework's step graph and host pipeline run the 8-bit block as they run the bf16 one."""
    g = gen(13)
    b = block(g, 4, 256, 128, 16, 2, out_dtype=F32)
    x = randn(g, 4, 256, dtype=BF16)
    want = b(x)
    step = ops.GraphedMoEFFN(b, 4)
    assert torch.equal(step(x), want)
    pipe = ops.HostPipeline(b, 4, 256, BF16)
    xh, yh = x.cpu().pin_memory(), torch.zeros(4, 256).pin_memory()
    pipe.submit(xh, yh).synchronize()
    assert torch.equal(yh, want.cpu())


def test_layer_from_params():
    """The reference's parameter names give the 8-bit layer that the packed weights give."""
    import numpy as np

    from frank_b200.params import moe_layer_from_params

    rng = np.random.default_rng(3)
    E, H, F, k = 6, 144, 272, 2
    p = {"blk.0.ffn_norm.weight": np.ones(H, np.float32),
         "blk.0.ffn_gate_inp.weight": rng.standard_normal((E, H), dtype=np.float32) * 0.05,
         "blk.0.ffn_up_exps.weight": rng.standard_normal((F, H, E), dtype=np.float32) * 0.02,
         "blk.0.ffn_gate_exps.weight": rng.standard_normal((F, H, E), dtype=np.float32) * 0.02,
         "blk.0.ffn_down_exps.weight": rng.standard_normal((H, F, E), dtype=np.float32) * 0.02}
    layer = moe_layer_from_params(p, 0, k, dtype=E4M3, chunk_bytes=128 * H * E * 4)
    dev = {n: torch.from_numpy(v).to(DEV) for n, v in p.items()}
    b = fb.Fp8MoEFFNBlock(dev["blk.0.ffn_gate_inp.weight"], dev["blk.0.ffn_up_exps.weight"],
                          dev["blk.0.ffn_gate_exps.weight"], dev["blk.0.ffn_down_exps.weight"], E, k, False)
    x = randn(gen(14), 5, H, dtype=BF16)
    assert torch.equal(layer(x), b(x))
    res = randn(gen(15), 5, H)
    assert torch.equal(layer.sublayer(res, 1e-5), b.sublayer(res, dev["blk.0.ffn_norm.weight"], 1e-5))


def test_experts_the_same_id_twice():
    """A token that names an expert twice gets it twice, however many slots the expert has."""
    g = gen(16)
    for T, k, E in ((10, 8, 9), (64, 8, 8), (3, 2, 2), (200, 3, 4)):
        b = block(g, T, 256, 144, E, k, out_dtype=F32)
        x = randn(g, T, 256, dtype=BF16)
        rid = torch.randint(0, 2, (k, T), generator=g, device=DEV, dtype=torch.int32)
        rw = torch.rand((k, T), generator=g, device=DEV)
        within(b.experts(x, rw, rid), *want_moe(b, x, rw, rid))


def test_gate_refusals():
    y, w = torch.zeros(6, 64, device=DEV), torch.ones(64, device=DEV)
    for gate in (torch.ones(4, 64, device=DEV), torch.ones(63, device=DEV), torch.ones(6, 1, 64, device=DEV),
                 torch.ones(0, 64, device=DEV), torch.tensor(1.0, device=DEV)):
        with pytest.raises(ValueError, match="gate"):
            fb.post_norm_residual(y, y, w, 1e-5, gate=gate)
    with pytest.raises(TypeError, match="gate"):
        fb.post_norm_residual(y, y, w, 1e-5, gate=w.bfloat16())


def test_output_refusals():
    """A wrong out is refused, a right one is written and returned."""
    g = gen(17)
    b = block(g, 4, 128, 128, 4, 2, out_dtype=F32)
    x = randn(g, 4, 128, dtype=BF16)
    for bad in (torch.empty(4, 128, device=DEV, dtype=BF16), torch.empty(5, 128, device=DEV), torch.empty(4, 128),
                torch.empty(128, 4, device=DEV).t(), torch.empty(4 * 128 + 1, device=DEV)[1:].view(4, 128)):
        with pytest.raises(ValueError, match="out must be"):
            b(x, out=bad)
    out = torch.empty(4, 128, device=DEV)
    assert b(x, out=out) is out and torch.equal(out, b(x))


def test_calls_on_another_stream_and_device_context():
    """Calls follow the current stream of their tensors' device."""
    g = gen(18)
    b = block(g, 4, 256, 128, 8, 2, out_dtype=F32)
    x = randn(g, 4, 256, dtype=BF16)
    want = b(x)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        late = torch.zeros_like(x)
        torch.cuda._sleep(20_000_000)  # the input arrives late on this stream
        late.copy_(x)
        y = b(late)
        s = b.sublayer(late, torch.ones(256, device=DEV), 1e-5)
    st.synchronize()
    assert torch.equal(y, want)
    assert torch.equal(s, b.sublayer(x, torch.ones(256, device=DEV), 1e-5))


@pytest.mark.parametrize("T", [3, 100])
@pytest.mark.parametrize("std", [1e-3, 30.0, 1e4])
def test_experts_small_and_large_activations(T, std):
    """silu over its whole range: near zero, where it is u / 2, and where the exponential under- or overflows."""
    g = gen(T)
    b = block(g, T, 256, 272, 4, 2, out_dtype=F32)
    x = randn(g, T, 256, std=std, dtype=BF16)
    rw = torch.rand((2, T), generator=g, device=DEV)
    rid = torch.stack([torch.randperm(4, generator=g, device=DEV)[:2] for _ in range(T)], 1).to(torch.int32)
    within(b.experts(x, rw, rid), *want_moe(b, x, rw, rid))


def test_weights_replaced():
    """A block reads the weights it has when it is called."""
    g = gen(23)
    b, c = (block(g, 5, 256, 256, 4, 2) for _ in range(2))
    x = randn(g, 5, 256, dtype=BF16)
    b(x)
    c.wr, c.wr_pack = b.wr, b.wr_pack
    b.w_up, b.w_gate, b.w_down = c.w_up, c.w_gate, c.w_down
    assert torch.equal(b(x), c(x))


@pytest.mark.parametrize("T", [3, 100])
def test_chains_without_a_pause(T):
    """Calls that each read what the call before has just written, in buffers that are used again with new values
    every round: the bits of the same calls with a synchronisation after each."""
    g = gen(24)
    H = 512
    b = block(g, T, H, 256, 16, 4)
    nw, pw = 1 + randn(g, H, std=0.1), 1 + randn(g, H, std=0.1)
    lin = weights(g, 1, H, H)
    inputs = [randn(g, T, H, dtype=BF16) for _ in range(40)]
    buf, mid = torch.empty_like(inputs[0]), torch.empty_like(inputs[0])

    def chain(x, pause):
        buf.copy_(x)
        for _ in range(3):
            b.sublayer(buf, nw, 1e-5, post_norm_w=pw, out=buf)
            pause()
            fb.post_norm_residual(buf, buf, pw, 1e-5, out=mid)
            pause()
            q, s = fb.quantize_fp8(mid)
            pause()
            fb.fp8_matmul((q, s), lin, out=buf)
            pause()
        return buf.clone()

    want = [chain(x, torch.cuda.synchronize) for x in inputs]
    got = [chain(x, lambda: None) for x in inputs]
    for a, w in zip(got, want):
        assert torch.equal(a, w)


@pytest.mark.parametrize("T,H,F,E,k", [(64, 256, 272, 2, 2), (200, 144, 272, 12, 2), (700, 512, 384, 4, 2),
                                       (65, 1040, 96, 130, 6), (90, 256, 128, 32, 32)])
def test_prompt_slots_stay_in_fp32(T, H, F, E, k):
    """A prompt's products are summed over the slots in fp32 and a bf16 result is rounded once: the bound of the fp32
    result and half a step; a sub-layer's post-norm sees the fp32 sums."""
    g = gen(T + 25)
    b = block(g, T, H, F, E, k)
    assert prompt(T, b)
    x = randn(g, T, H, dtype=BF16)
    rid = torch.rand((T, E), generator=g, device=DEV).topk(k, 1)[1].t().to(torch.int32).contiguous()
    rw = torch.rand((k, T), generator=g, device=DEV)
    want, bound, _ = Q.moe_experts(x.double(), rw.double(), rid, dense(b.w_gate), dense(b.w_up), dense(b.w_down))
    y = b.experts(x, rw, rid)
    within(y, want, bound)
    f = fb.Fp8MoEFFNBlock(b.wr, b.w_up, b.w_gate, b.w_down, E, k, True, out_dtype=F32)
    assert torch.equal(y, f.experts(x, rw, rid).to(BF16))
    nw, pw = 1 + randn(g, H, std=0.1), 1 + randn(g, H, std=0.1)
    xn = fb.rms_norm_fp8(x, nw, 1e-5, return_norm=True)[2]
    assert torch.equal(b.sublayer(x, nw, 1e-5, post_norm_w=pw), fb.post_norm_residual(f(xn), x, pw, 1e-5))


@pytest.mark.parametrize("T", [3, 100])
def test_silu_up_to_the_largest_number(T):
    """Finite up-products to 3e38, past where their exponent overflows: silu(u) is u (or 0), not NaN."""
    g = gen(26)
    H, F, E = 144, 272, 2
    up, gate, down = weights(g, E, F, H), weights(g, E, F, H), weights(g, E, H, F)
    up.q[:, :, 0] = (torch.randn((E, F), generator=g, device=DEV) * 300).clamp_(-448, 448).to(E4M3)
    up.q[:, :4, 0] = torch.tensor([448.0, -448.0, 352.0, -352.0], device=DEV).to(E4M3)
    up.scale.fill_(3.2e38 / 448)
    gate.scale.fill_(1e-32)
    b = fb.Fp8MoEFFNBlock(randn(g, E, H), up, gate, down, E, 1, False, out_dtype=F32)
    x = torch.zeros((T, H), dtype=BF16, device=DEV)
    x[:, 0] = 1.0
    x[T - 1, 0] = -1.0
    rw = torch.ones((1, T), device=DEV)
    rid = torch.randint(0, E, (1, T), generator=g, device=DEV, dtype=torch.int32)
    y = b.experts(x, rw, rid)
    assert torch.isfinite(y).all() and (y != 0).any()
    within(y, *want_moe(b, x, rw, rid))


@pytest.mark.parametrize("T", [3, 200])
def test_router_replaced(T):
    """A block routes by the router it has when it is called; one changed in place is taken up by assigning it again."""
    g = gen(27)
    b = block(g, T, 256, 256, 8, 2, out_dtype=F32)
    x = randn(g, T, 256, dtype=BF16)
    b(x)
    fresh = lambda wr: fb.Fp8MoEFFNBlock(wr, b.w_up, b.w_gate, b.w_down, 8, 2, True, out_dtype=F32)  # noqa: E731
    step = ops.GraphedMoEFFN(b, T)
    for wr in (randn(g, 8, 256), randn(g, 8, 256, dtype=BF16), randn(g, 256, 8).t()):
        b.wr = wr
        want = fresh(wr)(x, return_routing=True)
        assert all(torch.equal(a, w) for a, w in zip(b(x, return_routing=True), want))
        assert torch.equal(step(x), want[0]), "a graph of the block takes the new router up"
    b.wr.copy_(randn(g, 8, 256))
    b.wr = b.wr
    assert torch.equal(b(x), fresh(b.wr)(x))
    for bad in (randn(g, 9, 256), randn(g, 8, 128), randn(g, 8, 256).half(), randn(g, 8, 256).cpu(), None):
        kept = b.wr
        with pytest.raises((TypeError, ValueError), match="gate_inp_w"):
            b.wr = bad
        assert b.wr is kept


def test_assigned_weights_fit_the_block():
    """Weights of other sizes are refused; tensors exchanged inside Fp8Experts are read by the next call."""
    g = gen(28)
    b, c = (block(g, 5, 256, 128, 4, 2) for _ in range(2))
    x = randn(g, 5, 256, dtype=BF16)
    with pytest.raises(ValueError, match="shape"):
        fb.Fp8MoEFFNBlock(b.wr, b.w_up, b.w_down, b.w_down, 4, 2, True)
    for bad in (weights(g, 3, 128, 256), weights(g, 4, 112, 256), b.w_down):
        with pytest.raises(ValueError, match="shape"):
            b.w_up = bad
    with pytest.raises(ValueError, match="shape"):
        b.w_up.q = b.w_down.q
    c.wr = b.wr
    for mine, other in ((b.w_up, c.w_up), (b.w_gate, c.w_gate), (b.w_down, c.w_down)):
        mine.q, mine.scale = other.q, other.scale
    assert torch.equal(b(x), c(x))


@pytest.mark.parametrize("R", [3, 300])
def test_scales_at_the_ends_of_their_range(R):
    """Rows of the largest scale with weights' scales just below 2^8: partial sums of 0 stay 0.  Rows and weights whose
    scales multiply to less than 2^-126: an absolute error of 2^-125 a block of K, and half a step of fp32's least number
    for each of its additions."""
    g = gen(29)
    K, N = 400, 272
    w = weights(g, 1, N, K)
    w.scale.fill_(255.0)
    w.q[:, :, :128] = torch.zeros((1, N, 128), device=DEV).to(E4M3)
    x = randn(g, R, K, std=1e-3)
    x[:, 3] = 3.3e38
    q, s = fb.quantize_fp8(x)
    assert s.max() == 2.0 ** 120
    within(fb.fp8_matmul((q, s), w, out_dtype=F32), *Q.product(values(q, s), dense(w)[0]))
    w = weights(g, 1, N, K)
    for scale in (1e-5, 1e-10, 1e-20, 1e-38):
        w.scale.fill_(scale)
        q, s = fb.quantize_fp8(randn(g, R, K, std=1e-33))
        assert s.min() == 2.0 ** -110
        want, bound = Q.product(values(q, s), dense(w)[0])
        within(fb.fp8_matmul((q, s), w, out_dtype=F32), want, bound + 4 * (2.0 ** -125 + 2.0 ** -150))


@pytest.mark.parametrize("T,chunks", [(200, 4), (130, 2), (9, 3)])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_host_chunks_across_the_rule(T, chunks, out_dtype):
    """Tokens from the host in chunks that take the few tokens' kernels, where one call for all takes a prompt's: the
    bits of a call for each chunk, and every chunk within the bounds of the definition for the routing that it took,
    which is the strict one but for near ties."""
    g = gen(T)
    b = block(g, T, 256, 128, 16, 4, out_dtype=out_dtype)
    x = randn(g, T, 256, dtype=BF16)
    xh, yh = x.cpu().pin_memory(), torch.zeros((T, 256), dtype=out_dtype).pin_memory()
    ops.moe_ffn_host(b, xh, yh, chunks=chunks).synchronize()
    bounds = [T * i // chunks for i in range(chunks + 1)]
    for lo, hi in zip(bounds, bounds[1:]):
        y, rw, rid = b(x[lo:hi], return_routing=True)
        assert torch.equal(yh[lo:hi], y.cpu())
        strict_route(x[lo:hi].double().cpu().numpy(), b.wr.cpu().numpy(), rw.cpu().numpy(), rid.cpu().numpy(), 4, True)
        within(y, *want_moe(b, x[lo:hi], rw, rid))


@pytest.mark.parametrize("T,H,F,E,k", [(3, 16384, 128, 8, 2), (5, 7168, 128, 256, 8), (2, 12304, 144, 16, 4),
                                       (64, 8208, 128, 24, 3), (70, 16384, 144, 8, 2), (90, 7168, 128, 256, 8)])
def test_long_rows_and_many_experts(T, H, F, E, k):
    """Rows up to 16384 and 256 experts: the router's slices of several blocks, the widest sums of squares and top-k."""
    g = gen(T + H)
    b = block(g, T, H, F, E, k, out_dtype=F32)
    b.wr = randn(g, E, H, std=0.02)
    # rows of +-1 have the mean square 1 exactly, so with eps = 0 and weights in bf16 every kernel's norm is res * nw
    res = torch.where(randn(g, T, H) > 0, 1.0, -1.0)
    nw, pw = (1 + randn(g, H, std=0.1)).to(BF16).float(), 1 + randn(g, H, std=0.1)
    x = (res * nw).to(BF16)
    assert torch.equal(fb.rms_norm_fp8(res, nw, 0.0, return_norm=True)[2], x)
    y, rw, rid = b(x, return_routing=True)
    _, _, near, differ = strict_route(x.double().cpu().numpy(), b.wr.cpu().numpy(), rw.cpu().numpy(),
                                      rid.cpu().numpy(), k, True)
    print(f"near-tied {near}, routed differently {differ} of {T}")
    within(y, *want_moe(b, x, rw, rid))
    out, rw2, rid2 = b.sublayer(res, nw, 0.0, post_norm_w=pw, return_routing=True)
    assert torch.equal(rw2, rw) and torch.equal(rid2, rid)
    assert torch.equal(out, fb.post_norm_residual(y, res, pw, 0.0))
    assert ops.read_device_error() == 0


@pytest.mark.parametrize("T", [3, 40, 100, 200])
@pytest.mark.parametrize("wr_dtype", [F32, BF16])
def test_router_weights_as_they_are(T, wr_dtype):
    """The C entries take the router in fp32 or bf16 without a pack: the bits of the packed call."""
    from frank_b200 import _lib

    g = gen(T + 30)
    H, F, E, k = 272, 144, 32, 4
    b = block(g, T, H, F, E, k)
    wr = randn(g, E, H, std=0.05, dtype=wr_dtype)
    b.wr = wr
    x = randn(g, T, H, dtype=BF16)
    nw = 1 + randn(g, H, std=0.1)
    lib, p = _lib.load(), lambda t: t.data_ptr()
    w = [p(t) for e in (b.w_up, b.w_gate, b.w_down) for t in (e.q, e.scale)]
    ws = torch.empty(b.workspace_bytes(T), dtype=torch.uint8, device=DEV)
    dt = {F32: _lib.F32, BF16: _lib.BF16}[wr_dtype]
    st = torch.cuda.current_stream().cuda_stream
    y, rw, rid = torch.empty_like(x), torch.empty(k, T, device=DEV), torch.empty(k, T, dtype=torch.int32, device=DEV)
    _lib.check(lib.frank_fp8_moe_block(p(x), dt, p(wr), *w, T, E, k, H, F, 1, _lib.BF16, p(y), p(rw), p(rid), p(ws),
                                       ws.numel(), st))
    want = b(x, return_routing=True)
    assert torch.equal(y, want[0]) and torch.equal(rw, want[1]) and torch.equal(rid, want[2])
    _lib.check(lib.frank_fp8_moe_sublayer(_lib.BF16, p(x), p(nw), 1e-5, dt, p(wr), *w, T, E, k, H, F, 1, None, None, 1,
                                          1.0, p(y), None, None, p(ws), ws.numel(), st))
    assert torch.equal(y, b.sublayer(x, nw, 1e-5))


def test_block_of_inference_mode():
    """A block made and called under inference mode; its router and weights are replaced and it is called outside."""
    g = gen(31)
    with torch.inference_mode():
        b = block(g, 3, 256, 128, 8, 2)
        x = randn(g, 3, 256, dtype=BF16)
        y = b(x)
    assert torch.equal(b(x), y)
    c = block(g, 3, 256, 128, 8, 2)
    b.wr, b.w_up, b.w_gate, b.w_down = c.wr, c.w_up, c.w_gate, c.w_down
    want = c(x)
    assert torch.equal(b(x), want)
    with torch.inference_mode():
        assert torch.equal(b(x), want)


def test_graphed_host_step_takes_the_block():
    """A step from pinned host tokens to the pinned host result as one graph: the bits of a call on the device."""
    g = gen(32)
    for T in (2, 80):
        b = block(g, T, 256, 128, 16, 2)
        step = ops.GraphedHostMoEFFN(b, T)
        for _ in range(2):
            x = randn(g, T, 256, dtype=BF16)
            step.x_host.copy_(x.cpu())
            step.replay().synchronize()
            assert torch.equal(step.y_host, b(x).cpu())
