"""Refusals of the MXFP4 products on a dense input, and of their error word; no GPU needed."""
import ctypes
import errno
import importlib

import pytest
import torch

from _helpers import package


@pytest.fixture(scope="module")
def lib():
    package()
    return importlib.import_module("hrm-moe_b200._lib")


def _packed(ops, groups, n, k, swiglu):
    return ops.Mxfp4Weight(torch.zeros(ops._lib.load().hmoe_mxfp4_weight_bytes(groups, n, k, int(swiglu)),
                                       dtype=torch.uint8), groups, n, k, swiglu)


def test_c_abi_refusals_of_the_dense_products(lib):
    so = lib.load()
    p = ctypes.c_void_p(4096)       # never followed: the call fails before it touches memory
    odd = ctypes.c_void_p(4096 + 8)
    lin, glu = so.hmoe_grouped_linear_mxfp4_dense, so.hmoe_grouped_swiglu_mxfp4_dense
    #        x, stride, dtype, weight, counts, M, N, K, groups, [quantized,] output, scratch, ws, bytes, stream
    cases = [
        (lin, (p, 32, 0, p, p, 4, 12, 32, 2, p, p, None, 0, None), b"N must"),
        (lin, (p, 32, 0, p, p, -1, 8, 32, 2, p, p, None, 0, None), b"M must"),
        (lin, (p, 32, 2, p, p, 4, 8, 32, 2, p, p, None, 0, None), b"dtype"),
        (lin, (None, 32, 0, p, p, 4, 8, 32, 2, p, p, None, 0, None), b"required"),
        (lin, (p, 32, 0, p, p, 4, 8, 32, 2, p, None, None, 0, None), b"required"),
        (lin, (p, 33, 0, p, p, 4, 8, 32, 2, p, p, None, 0, None), b"aligned"),
        (lin, (p, 34, 1, p, p, 4, 8, 32, 2, p, p, None, 0, None), b"aligned"),
        (lin, (odd, 32, 0, p, p, 4, 8, 32, 2, p, p, None, 0, None), b"aligned"),
        (lin, (p, 32, 0, None, p, 4, 8, 32, 2, p, p, None, 0, None), b"NULL"),
        (lin, (p, 32, 0, p, p, 4, 8, 32, 2, odd, p, None, 0, None), b"aligned"),
        (lin, (p, 32, 0, p, p, 4, 8, 32, 2, p, p, ctypes.c_void_p(4098), 64, None), b"workspace"),
        (glu, (p, 32, 0, p, None, 4, 8, 32, 2, 1, p, p, None, 0, None), b"NULL"),
        (glu, (p, 32, 0, p, p, 4, 8, 32, 2, 0, p, p, ctypes.c_void_p(4098), 64, None), b"workspace"),
        (so.hmoe_grouped_linear_mxfp4, (p, p, p, 4, 8, 32, 2, p, ctypes.c_void_p(4097), 64, None),
         b"workspace"),
    ]
    for fn, args, word in cases:
        assert fn(*args) == errno.EINVAL, (fn.__name__, args)
        assert word in so.hmoe_last_error(), (fn.__name__, args, so.hmoe_last_error())
    assert lin(None, 32, 0, None, None, 0, 8, 32, 2, None, None, None, 0, None) == 0


def test_python_refuses_a_workspace_without_room_for_the_word(lib):
    ops = importlib.import_module("hrm-moe_b200.ops")
    w = _packed(ops, 2, 8, 64, False)
    rows = ops.Mxfp4Rows(torch.zeros((4, 48), dtype=torch.uint8), 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.grouped_linear_mxfp4(rows, w, torch.tensor([2, 2]), workspace=torch.zeros(64, dtype=torch.uint8))


def test_router_operands_of_other_sizes_are_refused(lib):
    """A short bias or a narrow router weight would be read past its end: refused before any kernel."""
    ops = importlib.import_module("hrm-moe_b200.ops")
    E, d, I = 4, 64, 32
    bf16 = dict(dtype=torch.bfloat16)
    x, wr = torch.zeros((3, d), **bf16), torch.zeros((E, d), **bf16)
    up, down = _packed(ops, E, I, d, True), _packed(ops, E, d, I, False)
    dense = torch.zeros((E, 2 * I, d), **bf16), torch.zeros((E, d, I), **bf16)
    calls = [lambda r, b: ops.ffn_forward_mxfp4(x, r, up, down, 2, True, router_bias=b),
             lambda r, b: ops.CapturedFfn(x, r, up, down, 2, True, b),
             lambda r, b: ops.CapturedFfn(x, r, *dense, 2, True, b),
             lambda r, b: ops.ffn_forward(x, r, *dense, 2, True, b)]
    for f in calls:
        for n in (1, E - 1, E + 1):
            with pytest.raises(ValueError, match="router bias"):
                f(wr, torch.zeros(n, **bf16))
        with pytest.raises(ValueError, match="router weight"):
            f(wr[:, :32], None)
        with pytest.raises(RuntimeError, match="CUDA"):
            f(wr, torch.zeros(E, **bf16))


def test_packed_weights_of_another_size_are_refused(lib):
    """Fewer bytes than the fields say would be read past their end: refused before any kernel."""
    ops = importlib.import_module("hrm-moe_b200.ops")
    E, d, I = 4, 64, 32
    bf16 = dict(dtype=torch.bfloat16)
    x, wr, tpe = torch.zeros((3, d), **bf16), torch.zeros((E, d), **bf16), torch.tensor([3, 0, 0, 0])
    sel, rw = torch.zeros((3, 2), dtype=torch.int32), torch.zeros((3, 2), **bf16)

    def calls(up, down):
        return [lambda: ops.grouped_swiglu_mxfp4(x, up, tpe), lambda: ops.grouped_linear_mxfp4(x[:, :I], down, tpe),
                lambda: ops.experts_forward_mxfp4(x, sel, rw, up, down),
                lambda: ops.ffn_forward_mxfp4(x, wr, up, down, 2, True),
                lambda: ops.CapturedFfn(x, wr, up, down, 2, True)]

    good = _packed(ops, E, I, d, True), _packed(ops, E, d, I, False)
    for f in calls(*good):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
    cuts = [lambda t: t[:-16], lambda t: t[:16], lambda t: torch.cat((t, t)), lambda t: torch.cat((t, t))[::2],
            lambda t: t.float()]
    for cut in cuts:
        bad = [ops.Mxfp4Weight(cut(w.data), w.groups, w.n, w.k, w.swiglu) for w in good]
        for f in calls(*bad):
            with pytest.raises(ValueError, match="packed weight"):
                f()
    with pytest.raises(ValueError, match="N must"):
        ops.grouped_linear_mxfp4(x, ops.Mxfp4Weight(good[1].data, E, 12, d, False), tpe)


def test_row_counts_whose_blocks_pass_int32_are_refused(lib):
    """The kernels count rows in 32 bits, up to the end of a row's block of 256."""
    so = lib.load()
    p = ctypes.c_void_p(4096)       # never followed
    for M in (2 ** 31 - 255, 2 ** 31 - 1, 2 ** 31, 2 ** 40):
        for fn, args in [(so.hmoe_grouped_linear_mxfp4, (p, p, p, M, 8, 8, 1, p, None, 0, None)),
                         (so.hmoe_grouped_swiglu_mxfp4, (p, p, p, M, 8, 8, 1, 1, p, None, 0, None)),
                         (so.hmoe_grouped_linear_mxfp4_dense, (p, 8, 0, p, p, M, 8, 8, 1, p, p, None, 0, None))]:
            assert fn(*args) == errno.EINVAL and b"M must" in so.hmoe_last_error(), (fn.__name__, M)
