"""MXFP4: the reference in the tests against the format's definition, the C ABI's
checks of arguments and the Python entry points' refusals; no GPU needed."""
import ctypes
import errno
import importlib

import numpy as np
import pytest
import torch

import mxfp4_ref as R
from _helpers import package


@pytest.fixture(scope="module")
def lib():
    package()
    return importlib.import_module("hrm-moe_b200._lib")


@pytest.fixture(scope="module")
def ops(lib):
    return importlib.import_module("hrm-moe_b200.ops")


def test_reference_values_and_ties():
    # scale 1 (largest magnitude in [4, 8)): ties go to the even code, 6 saturates
    x = np.zeros(32)
    x[:14] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 7.9, 0.26, 0.24, -6.5]
    codes, s = R.quantize(x)
    assert s.tolist() == [127]
    got = R.values(codes, s)[:14].tolist()
    assert got == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.0, -4.0, 6.0, 0.5, 0.0, -6.0]
    for amax, byte in [(0.0, 0), (2.0 ** -140, 0), (2.0 ** -125, 0), (2.0 ** -124, 1), (1.0, 125),
                       (1.999, 125), (2.0, 126), (3e38, 252), (np.inf, 255), (np.nan, 255)]:
        assert R.scale_bytes(np.array(amax)) == byte, amax
    assert R.rounded(np.array([[1.0, np.nan, 2.0]])).shape == (1, 3)
    assert np.isnan(R.rounded(np.array([1.0, np.inf]))).all()


def test_record_and_weight_sizes(lib):
    so = lib.load()
    for k in (8, 32, 40, 448, 512, 1280, 1536, 4096):
        blocks = -(-k // 32)
        size = so.hmoe_mxfp4_row_bytes(k)
        assert size % 16 == 0 and 17 * blocks <= size < 17 * blocks + 24
    for bad in (0, -8, 12, 1 << 25):
        assert so.hmoe_mxfp4_row_bytes(bad) == 0
        assert b"K must be" in so.hmoe_last_error()
    # XL gate_up: 64 x 1024 rows of 1536: half a byte of code and a 32nd of a scale each
    n = so.hmoe_mxfp4_weight_bytes(64, 512, 1536, 1)
    assert n == 64 * 1024 * 1536 * 17 // 32
    assert so.hmoe_mxfp4_weight_bytes(64, 1536, 512, 0) == 64 * 1536 * 512 * 17 // 32
    for args, word in [((0, 8, 8, 0), b"groups"), ((1025, 8, 8, 0), b"groups"),
                       ((4, 12, 8, 0), b"N must"), ((4, 8, 20, 0), b"K must"),
                       ((1024, 1 << 23, 8, 1), b"int32")]:
        assert so.hmoe_mxfp4_weight_bytes(*args) == 0
        assert word in so.hmoe_last_error()


def test_c_abi_refusals(lib):
    so = lib.load()
    p = ctypes.c_void_p(4096)       # never followed: the call fails before it touches memory
    odd = ctypes.c_void_p(4096 + 8)
    cases = [
        (so.hmoe_mxfp4_quantize, (p, 4, 12, 12, 0, p, None), b"K must"),
        (so.hmoe_mxfp4_quantize, (p, -1, 16, 16, 0, p, None), b"rows"),
        (so.hmoe_mxfp4_quantize, (p, 4, 16, 16, 2, p, None), b"dtype"),
        (so.hmoe_mxfp4_quantize, (None, 4, 16, 16, 0, p, None), b"required"),
        (so.hmoe_mxfp4_quantize, (p, 4, 16, 17, 0, p, None), b"aligned"),
        (so.hmoe_mxfp4_quantize, (odd, 4, 16, 16, 1, p, None), b"aligned"),
        (so.hmoe_mxfp4_dequantize, (p, 4, 16, 3, p, None), b"dtype"),
        (so.hmoe_mxfp4_dequantize, (p, 4, 16, 0, odd, None), b"aligned"),
        (so.hmoe_mxfp4_pack_weight, (p, 8, p, 1, 2, 8, 32, 0, p, None), b"strides"),
        (so.hmoe_mxfp4_pack_weight, (p, 24, p, 1, 2, 8, 32, 0, p, None), b"aligned"),
        (so.hmoe_mxfp4_pack_weight, (p, 16, None, 1, 2, 8, 32, 0, p, None), b"required"),
        (so.hmoe_grouped_linear_mxfp4, (p, p, p, -1, 8, 32, 2, p, None, 0, None), b"M must"),
        (so.hmoe_grouped_linear_mxfp4, (p, p, p, 4, 12, 32, 2, p, None, 0, None), b"N must"),
        (so.hmoe_grouped_linear_mxfp4, (p, p, p, 4, 8, 32, 0, p, None, 0, None), b"groups"),
        (so.hmoe_grouped_linear_mxfp4, (p, None, p, 4, 8, 32, 2, p, None, 0, None), b"NULL"),
        (so.hmoe_grouped_linear_mxfp4, (p, p, p, 4, 8, 32, 2, odd, None, 0, None), b"aligned"),
        (so.hmoe_grouped_swiglu_mxfp4, (p, p, None, 4, 8, 32, 2, 1, p, None, 0, None), b"NULL"),
        (so.hmoe_grouped_swiglu_mxfp4, (odd, p, p, 4, 8, 32, 2, 1, p, None, 0, None), b"aligned"),
    ]
    for fn, args, word in cases:
        assert fn(*args) == errno.EINVAL, (fn.__name__, args)
        assert word in so.hmoe_last_error(), (fn.__name__, args, so.hmoe_last_error())
    # nothing to do: no pointer is looked at
    assert so.hmoe_mxfp4_quantize(None, 0, 16, 16, 0, None, None) == 0
    assert so.hmoe_grouped_linear_mxfp4(None, None, None, 0, 8, 32, 2, None, None, 0, None) == 0
    f32 = lib.HmoeShape(16, 64, 8, 32, 2, 1, 1)
    bf16 = lib.HmoeShape(16, 64, 8, 32, 2, 0, 1)
    assert so.hmoe_experts_mxfp4_workspace_bytes(ctypes.byref(f32)) == 0
    assert b"bf16" in so.hmoe_last_error()
    need = so.hmoe_experts_mxfp4_workspace_bytes(ctypes.byref(bf16))
    assert need > 16 * 2 * 64 * 2
    assert so.hmoe_ffn_mxfp4_workspace_bytes(ctypes.byref(bf16)) > need
    rc = so.hmoe_experts_forward_mxfp4(ctypes.byref(bf16), p, p, p, p, None, None, p, None, None, p,
                                       need, None)
    assert rc == errno.EINVAL and b"required" in so.hmoe_last_error()
    rc = so.hmoe_ffn_forward_mxfp4(ctypes.byref(bf16), p, p, None, p, odd, p, 0, None, None, None,
                                   None, p, 1 << 30, None)
    assert rc == errno.EINVAL and b"aligned" in so.hmoe_last_error()


def test_python_refusals_without_a_gpu(ops):
    x = torch.randn(4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.quantize_mxfp4(x)
    with pytest.raises(TypeError):
        ops.quantize_mxfp4(x.half())
    with pytest.raises(RuntimeError, match="inference"):
        ops.quantize_mxfp4(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="records"):
        ops.Mxfp4Rows(torch.zeros((4, 16), dtype=torch.uint8), 64)
    with pytest.raises(TypeError):
        ops.Mxfp4Rows(torch.zeros((4, 48), dtype=torch.int32), 64)
    rows = ops.Mxfp4Rows(torch.zeros((4, 48), dtype=torch.uint8), 64)
    assert rows.shape == (4, 64) and rows.codes.shape == (4, 32) and rows.scales.shape == (4, 2)
    codes = torch.zeros((2, 8, 32), dtype=torch.uint8)
    scales = torch.zeros((2, 8, 2), dtype=torch.uint8)
    with pytest.raises(ValueError, match="k is required"):
        ops.pack_mxfp4_weight((codes, scales))
    with pytest.raises(TypeError):
        ops.pack_mxfp4_weight((codes.int(), scales), 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.pack_mxfp4_weight((codes, scales), 64)
    w = ops.Mxfp4Weight(torch.zeros(16, dtype=torch.uint8), 2, 8, 64, False)
    tpe = torch.tensor([2, 2])
    with pytest.raises(TypeError, match="pack_mxfp4_weight"):
        ops.grouped_linear_mxfp4(rows, torch.zeros(2, 8, 64), tpe)
    with pytest.raises(ValueError, match="swiglu"):
        ops.grouped_swiglu_mxfp4(rows, w, tpe)
    with pytest.raises(ValueError, match="mismatch"):
        ops.grouped_linear_mxfp4(ops.Mxfp4Rows(torch.zeros((4, 32), dtype=torch.uint8), 32), w, tpe)
    with pytest.raises(ValueError, match="mismatch"):
        ops.grouped_linear_mxfp4(x[:, :32], w, tpe)
    with pytest.raises(ValueError, match="tokens_per_expert"):
        ops.grouped_linear_mxfp4(rows, w, tpe[:1])
    with pytest.raises(RuntimeError, match="inference"):
        ops.grouped_linear_mxfp4(x.clone().requires_grad_(), w, tpe)
    sel = torch.zeros((4, 1), dtype=torch.int32)
    rw = torch.ones((4, 1), dtype=torch.bfloat16)
    up = ops.Mxfp4Weight(torch.zeros(16, dtype=torch.uint8), 2, 32, 64, True)
    down = ops.Mxfp4Weight(torch.zeros(16, dtype=torch.uint8), 2, 64, 32, False)
    with pytest.raises(TypeError, match="bf16"):
        ops.experts_forward_mxfp4(x.float(), sel, rw, up, down)
    with pytest.raises(ValueError, match="do not match"):
        ops.experts_forward_mxfp4(x, sel, rw, up, w)
    with pytest.raises(ValueError, match="do not match"):
        ops.experts_forward_mxfp4(x[:, :32], sel, rw, up, down)
    with pytest.raises(TypeError, match="pack_mxfp4_weight"):
        ops.ffn_forward_mxfp4(x, torch.zeros(2, 64), torch.zeros(2, 64, 64), down, 1, True)
    with pytest.raises(RuntimeError, match="inference"):
        ops.ffn_forward_mxfp4(x, torch.zeros(2, 64, requires_grad=True), up, down, 1, True)


def test_modules_refuse_stale_and_unserved_quantised_experts(ops):
    """What the modules refuse before any kernel; the packed weights stand in as strings."""
    layers = importlib.import_module("hrm-moe_b200.layers")
    ep = importlib.import_module("hrm-moe_b200.ep")

    def quantised(experts):
        experts._mxfp4 = ("gate_up", "down", experts._weights_state(),
                          (experts.gate_up_weight, experts.down_weight))
        return experts

    m = layers.SparseMoESwiGLU(32, 16, 4, 2, True, dtype=torch.bfloat16).requires_grad_(False)
    assert quantised(m.experts).quantized() == ("gate_up", "down")
    with pytest.raises(RuntimeError, match="no aux loss"):
        m(torch.zeros(3, 32, dtype=torch.bfloat16), moe_context={})
    w = m.experts.down_weight
    w.data = w.data.clone()  # leaves the version as it was
    with pytest.raises(RuntimeError, match="changed"):
        m(torch.zeros(3, 32, dtype=torch.bfloat16))
    quantised(m.experts).gate_up_weight = torch.nn.Parameter(m.experts.gate_up_weight.clone())
    with pytest.raises(RuntimeError, match="changed"):
        m.experts.quantized()
    m.drop_quantized_experts()
    assert m.experts.quantized() is None

    e = ep.SparseMoEExpertParallelSwiGLU(32, 16, 4, 2, True, dtype=torch.bfloat16)
    quantised(e.experts.local_experts)
    with pytest.raises(RuntimeError, match="no MXFP4 form"):
        e(torch.zeros(3, 32, dtype=torch.bfloat16))
