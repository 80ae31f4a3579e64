"""The 8-bit path without a GPU: the oracle's own arithmetic, the library's
refusals (none reaches a device) and the Python argument checks."""

import pytest
import torch

from oracle import fp8_oracle as Q


def test_oracle_rounding_is_torchs_e4m3():
    """Rounding by arithmetic equals torch's conversion on a grid that holds every e4m3 value and midpoint."""
    v = torch.cat([torch.arange(0, 2 ** 12).double() / 2 ** 14, torch.arange(2 ** 7, 448 * 4).double() / 4])
    v = torch.cat([v, -v])
    assert torch.equal(Q.round_e4m3(v), v.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("amax,p", [(448.0, 0), (448.0000305, 1), (1.75, -8), (1.7500001, -7), (2.0, -7), (0.0, -110),
                                    (1e-42, -110), (3.0e38, 120)])
def test_oracle_scale(amax, p):
    x = torch.zeros(1, 128, dtype=torch.float64)
    x[0, 5] = -amax
    assert Q.block_scales(x).item() == 2.0 ** p


def test_oracle_slack_covers_a_flip():
    x = torch.tensor([[448.0, 17.0, 0.1] + [0.0] * 125], dtype=torch.float64)  # 17 lies between 16 and 18
    err = torch.full_like(x, 1e-6)
    err[0, 0] = 0.0
    s = Q.quantised_slack(x, err)
    assert s[0, 1] == 2.0 and s[0, 2] == 0.0


@pytest.fixture(scope="module")
def lib():
    from frank_b200 import _lib

    return _lib.load()


P = 4096  # stands for a 16-byte aligned device address; every call below is refused before one is used


def _refused(lib, status, text):
    from frank_b200 import _lib

    assert status == _lib.EINVAL, status
    assert text in lib.frank_last_error().decode(), lib.frank_last_error()


def test_library_refusals(lib):
    from frank_b200 import _lib

    _refused(lib, lib.frank_quantize_fp8(2, P, 1, 128, P, P, None), "dtype")
    _refused(lib, lib.frank_quantize_fp8(0, P, 1, 120, P, P, None), "multiple of 16")
    _refused(lib, lib.frank_quantize_fp8(0, None, 1, 128, P, P, None), "null")
    _refused(lib, lib.frank_quantize_fp8(0, P + 4, 1, 128, P, P, None), "aligned")
    _refused(lib, lib.frank_rms_norm_fp8(0, P, P, 1, 16400, 1e-5, None, P, P, None), "16384")
    _refused(lib, lib.frank_quantize_fp8(0, P, -1, 128, P, P, None), "out of range")
    _refused(lib, lib.frank_quantize_fp8(0, P, 1 << 31, 128, P, P, None), "out of range")
    _refused(lib, lib.frank_rms_norm_fp8(0, P, P, 1 << 32, 128, 1e-5, None, P, P, None), "out of range")
    _refused(lib, lib.frank_post_norm_residual(1, P, 1, P, P, 1e-5, P, 1, 1.0, P, None, 0, None, 1 << 32, 4, None),
             "out of range")
    _refused(lib, lib.frank_rms_norm_fp8(0, P, None, 1, 128, 1e-5, None, P, P, None), "null")
    _refused(lib, lib.frank_prepack_experts_fp8(0, P, 16, 16, 257, P, P, None), "extents")
    _refused(lib, lib.frank_fp8_matmul(P, P, P, P, None, 2, 4, 128, 128, 0, P, None), "offsets")
    _refused(lib, lib.frank_fp8_matmul(P, P, P, P, None, 1, 4, 120, 128, 0, P, None), "multiples of 16")
    _refused(lib, lib.frank_fp8_matmul(P, P, P, P, None, 1, 4, 128, 136, 0, P, None), "multiples of 16")
    _refused(lib, lib.frank_fp8_matmul(P, P, P, P, None, 1, 4, 128, 128, 2, P, None), "dtype")
    _refused(lib, lib.frank_fp8_matmul(P + 8, P, P, P, None, 1, 4, 128, 128, 0, P, None), "aligned")
    _refused(lib, lib.frank_fp8_matmul(P, P, P, P, P, 257, 4, 128, 128, 0, P, None), "E=257")
    _refused(lib, lib.frank_fp8_matmul(P, P, P, P, None, 1, 0x7fffff01, 16, 16, 0, P, None), "out of range")
    w = [P] * 6
    ws = 1 << 30
    for T in (-1, 0x7fffff00 // 2 + 1, 1 << 62):
        _refused(lib, lib.frank_fp8_moe_experts(P, P, P, *w, T, 8, 2, 128, 128, 0, P, None, P, ws, None), "out of range")
    _refused(lib, lib.frank_fp8_moe_experts(P, P, P, *w, 4, 8, 9, 128, 128, 0, P, None, P, ws, None), "n_expert_used")
    _refused(lib, lib.frank_fp8_moe_experts(P, P, P, *w, 4, 8, 2, 120, 128, 0, P, None, P, ws, None), "n_embd")
    _refused(lib, lib.frank_fp8_moe_experts(P, P, P, *w, 4, 8, 2, 128, 100, 0, P, None, P, ws, None), "n_ff")
    _refused(lib, lib.frank_fp8_moe_experts(None, P, P, *w, 4, 8, 2, 128, 128, 0, P, None, P, ws, None), "null")
    st = lib.frank_fp8_moe_experts(P, P, P, *w, 4, 8, 2, 128, 128, 0, P, None, P, 64, None)
    assert st == _lib.ENOSPC and b"workspace" in lib.frank_last_error()
    _refused(lib, lib.frank_fp8_moe_block(P, 7, P, *w, 4, 8, 2, 128, 128, 0, 0, P, None, None, P, ws, None), "dtype")
    _refused(lib, lib.frank_fp8_moe_block(P, 0, P, *w, 4, 300, 2, 128, 128, 0, 0, P, None, None, P, ws, None),
             "n_expert")
    sub = lambda gate_rows, res: lib.frank_fp8_moe_sublayer(  # noqa: E731
        res, P, P, 1e-5, 0, P, *w, 4, 8, 2, 128, 128, 0, None, P, gate_rows, 1.0, P, None, None, P, ws, None)
    _refused(lib, sub(3, 0), "gate_rows")
    _refused(lib, sub(1, 2), "dtype")
    _refused(lib, lib.frank_post_norm_residual(0, P, 0, P, P, 1e-5, None, 1, 1.0, P, None, 0, None, 4, 130, None),
             "multiple of 4")
    _refused(lib, lib.frank_post_norm_residual(0, P, 0, P, P, 1e-5, P, 3, 1.0, P, None, 0, None, 4, 128, None),
             "gate_rows")
    _refused(lib, lib.frank_post_norm_residual(0, P, 0, P, P, 1e-5, None, 1, 1.0, P, None, 0, P, 4, 128, None), "null")


def test_library_accepts_nothing_to_do(lib):
    """No rows: success without a launch."""
    assert lib.frank_quantize_fp8(0, None, 0, 128, None, None, None) == 0
    assert lib.frank_fp8_matmul(None, None, None, None, None, 1, 0, 128, 128, 0, None, None) == 0
    assert lib.frank_fp8_linear(0, None, None, None, None, 1, 0, 128, 128, 0, None, None, 0, None) == 0
    assert lib.frank_post_norm_residual(0, None, 0, None, None, 1e-5, None, 1, 1.0, None, None, 0, None, 0, 128,
                                        None) == 0
    assert lib.frank_fp8_moe_experts(*[None] * 9, 0, 8, 2, 128, 128, 0, None, None, None, 0, None) == 0


def test_workspace_size_of_anything(lib):
    """A size query is host arithmetic: it answers for no tokens, no experts and nonsense alike."""
    assert lib.frank_fp8_moe_workspace_size(1, 2048, 768, 128, 8) > 8 * 2048 * 4
    for shape in ((0, 128, 128, 8, 2), (4, 0, 0, 8, 2), (4, 128, 128, 0, 0), (4, 128, 128, 8, 0), (-1, 128, 128, 8, 2)):
        lib.frank_fp8_moe_workspace_size(*shape)


def test_python_refusals():
    import frank_b200 as fb

    x = torch.zeros(4, 128)
    with pytest.raises(ValueError, match="CUDA device"):
        fb.quantize_fp8(x)
    with pytest.raises(TypeError, match="dtype"):
        fb.quantize_fp8(x.half())
    with pytest.raises(ValueError, match="shape"):
        fb.quantize_fp8(x[0])
    with pytest.raises(TypeError, match="torch.Tensor"):
        fb.quantize_fp8(x.numpy())
    with pytest.raises(TypeError, match="Fp8Experts"):
        fb.fp8_matmul(x, x)
    with pytest.raises(TypeError, match="dtype"):
        fb.Fp8Experts(x[None], x)
    with pytest.raises(ValueError, match="CUDA device"):
        fb.post_norm_residual(x, x, x[0], 1e-5)
    with pytest.raises(TypeError, match="output dtype"):
        fb.Fp8MoEFFNBlock(x, x, x, x, 8, 2, False, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="n_expert_used"):
        fb.Fp8MoEFFNBlock(x, x, x, x, 8, 9, False)


def test_chained_kernels_read_what_may_change_coherently():
    """A kernel that starts before its predecessor has ended may take the read-only path (`__ldg`, or a pointer to const
    that is `__restrict__`) only for expert weights' scales: all else may be written while it runs."""
    import re
    from pathlib import Path

    csrc = Path(__file__).resolve().parent.parent / "frank-models_b200" / "csrc"
    scales = re.compile(r"p\.w2?_scale \+ |\(UP \? a\.s_gate : a\.s_down\) \+ |a\.s_up \+ ")
    for name in ("quantize_fp8.cu", "gemm_fp8.cu", "few_fp8.cu", "norm.cu"):
        code = re.sub(r"//[^\n]*", "", (csrc / name).read_text())
        for m in re.finditer(r"__ldg\(([^;]{0,60})", code):
            assert scales.match(m.group(1)), (name, m.group(0))
        for kernel in re.split(r"__global__", code)[1:]:
            params, _, body = kernel.partition("{")
            if "pdl_wait" in body:
                assert not re.search(r"const [\w:]+\s*\* ?__restrict__", params), (name, params)


def test_linear_refuses_before_it_launches(lib):
    """What the product would refuse, frank_fp8_linear refuses before the rows are quantised: no launch is tried."""
    from frank_b200 import _lib

    ws = 1 << 20
    linear = lambda off, E, rows, N, K, out_dtype=0, x=P, x_dtype=0, w=P, sw=P, out=P, ptr=P: lib.frank_fp8_linear(  # noqa: E731
        x_dtype, x, w, sw, off, E, rows, N, K, out_dtype, out, ptr, ws, None)
    _refused(lib, linear(None, 1, 4, 120, 128), "multiples of 16")
    _refused(lib, linear(None, 1, 4, 128, 136), "multiple")
    _refused(lib, linear(None, 2, 4, 128, 128), "offsets")
    _refused(lib, linear(P, 257, 4, 128, 128), "E=257")
    _refused(lib, linear(None, 1, 4, 128, 128, out_dtype=2), "dtype")
    _refused(lib, linear(None, 1, 4, 128, 128, x_dtype=2), "dtype")
    _refused(lib, linear(None, 1, 4, 128, 128, x=None), "null")
    _refused(lib, linear(None, 1, 4, 128, 128, w=None), "null")
    _refused(lib, linear(None, 1, 4, 128, 128, sw=None), "null")
    _refused(lib, linear(None, 1, 4, 128, 128, out=None), "null")
    _refused(lib, linear(None, 1, 4, 128, 128, x=P + 4), "aligned")
    _refused(lib, linear(None, 1, 4, 128, 128, w=P + 8), "aligned")
    _refused(lib, linear(None, 1, 4, 128, 128, out=P + 8), "aligned")
    _refused(lib, linear(None, 1, 4, 128, 128, ptr=P + 8), "aligned")
    _refused(lib, linear(None, 1, -1, 128, 128), "out of range")
    _refused(lib, linear(None, 1, 0x7fffff01, 16, 16), "out of range")
    _refused(lib, linear(None, 1, 4, 128, -16), "multiple")
    assert linear(None, 1, 4, 128, 128, ptr=None) == _lib.ENOSPC
    assert linear(None, 1, 1 << 20, 128, 128) == _lib.ENOSPC


def _experts_stand_in(E, N, K):
    """An Fp8Experts without a device: the checks of assignments read shapes and devices only."""
    import frank_b200 as fb

    w = fb.Fp8Experts.__new__(fb.Fp8Experts)
    w._q = torch.zeros((E, N, K), dtype=torch.uint8).view(torch.float8_e4m3fn)
    w._scale = torch.ones((E, -(-N // 128), -(-K // 128)))
    return w


def test_assigned_weights_are_checked():
    """Weights given to a block after its construction have to fit it: the kernels read them by the block's sizes."""
    import frank_b200 as fb

    b = fb.Fp8MoEFFNBlock.__new__(fb.Fp8MoEFFNBlock)
    b.E, b.H, b.F, b.device = 4, 256, 128, torch.device("cpu")
    good = {"w_up": _experts_stand_in(4, 128, 256), "w_gate": _experts_stand_in(4, 128, 256),
            "w_down": _experts_stand_in(4, 256, 128)}
    for name, w in good.items():
        setattr(b, name, w)
        assert getattr(b, name) is w
        for bad in ((3, 128, 256), (4, 256, 256), (4, 128, 128), (4, 112, 256)):
            with pytest.raises(ValueError, match="shape"):
                setattr(b, name, _experts_stand_in(*bad))
        with pytest.raises(TypeError, match="Fp8Experts"):
            setattr(b, name, w._q)
        assert getattr(b, name) is w
    b.device = torch.device("cuda", 0)
    with pytest.raises(ValueError, match="device"):
        b.w_up = good["w_up"]


def test_assigned_tensors_of_weights_are_checked():
    """An Fp8Experts keeps its sizes: another q or scale has to fit them."""
    w = _experts_stand_in(2, 144, 256)
    for bad in (torch.zeros(2, 144, 128), torch.zeros(2, 144, 256)):
        with pytest.raises((TypeError, ValueError)):
            w.q = bad.to(torch.float8_e4m3fn if bad.shape[2] == 128 else torch.float32)
    with pytest.raises(ValueError, match="shape"):
        w.scale = torch.ones(2, 1, 2)
    with pytest.raises(TypeError, match="dtype"):
        w.scale = torch.ones(2, 2, 2, dtype=torch.float64)
    assert tuple(w.q.shape) == (2, 144, 256) and tuple(w.scale.shape) == (2, 2, 2)
