"""MXFP4 products: the error word of a call, and the forms and sizes at the edges of what they take.

Tolerances as in test_gpu_11_mxfp4: fp32 sums of exact products, in any order
and with truncating adders, are within K * 2^-23 of the sum of magnitudes; a
bf16 output adds half a step, 2^-8 of the value.
"""
import pytest
import torch

from gpu_util import get_ops, ragged_counts

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8


def _rand(shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


# ---------------------------------------------------------------- error word --
@pytest.mark.parametrize("M", [0, 5, 300, 1500])
def test_the_calls_clear_their_error_word(M):
    ops = get_ops()
    N, K = 72, 96
    x = _rand((M, K), 1)
    w = ops.pack_mxfp4_weight(_rand((3, N, K), 2, 0.02))
    wg = ops.pack_mxfp4_weight(_rand((3, 2 * N, K), 3, 0.02), swiglu=True)
    tpe = torch.tensor([M // 3, M // 4, 0], device="cuda")
    ws = torch.empty(16, dtype=torch.uint8, device="cuda")
    rows = ops.quantize_mxfp4(x)
    done = M // 3 + M // 4
    for f in (lambda **a: ops.grouped_linear_mxfp4(x, w, tpe, **a),
              lambda **a: ops.grouped_linear_mxfp4(rows, w, tpe, **a),
              lambda **a: ops.grouped_swiglu_mxfp4(x, wg, tpe, **a),
              lambda **a: ops.grouped_swiglu_mxfp4(rows, wg, tpe, quantized=True, **a).data):
        want = f()
        ws.fill_(9)
        with pytest.raises(Exception, match="error word"):
            ops.workspace_status(ws)
        got = f(workspace=ws)
        ops.workspace_status(ws)
        assert torch.equal(got[:done], want[:done])
        assert not ws[:4].any() and (ws[4:] == 9).all()
    with pytest.raises(ValueError, match="workspace"):
        ops.grouped_linear_mxfp4(x, w, tpe, workspace=ws[:3])
    with pytest.raises(ValueError, match="workspace"):
        ops.grouped_linear_mxfp4(rows, w, tpe, workspace=ws.view(torch.int32))
    if M:
        with pytest.raises(ValueError, match="workspace"):
            ops.grouped_linear_mxfp4(x, w, tpe, workspace=ws[1:])
