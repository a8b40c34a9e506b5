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


# -------------------------------------------------------------------- silu --
@pytest.mark.parametrize("copies", [1, 12])  # single CTAs, CTA pairs
def test_swiglu_over_the_whole_range_of_the_gate(copies):
    """silu(g) * u for known g from -127 to 55, where 2^(|g| log2 e) leaves the range of fp32, and u up to 2^100.

    g is a sum of three operands and u one, all exact in MXFP4.  Relative
    error: |g| log2 e <= 184 carries two roundings (2^-23 of it, 2^-15.9 of its
    power of two after the factor ln 2), the rest is within 2^-18; half a step
    of bf16 on top.  Absolute: the exponential's subnormals are off by up to
    two of their steps, times g and u, and a result below 2^-126 by half a
    step of bf16's subnormals, 2^-134.
    """
    ops = get_ops()
    parts = torch.tensor([(a, b, c) for a in (-96.0, -64.0, -48.0, 0.0, 32.0) for b in (-24.0, -16.0, 0.0, 16.0)
                          for c in (-6.0, -1.5, -1.0, 0.0, 0.25, 3.0, 6.0)], device="cuda")
    M = parts.shape[0]
    x = torch.zeros((M, 128), device="cuda")
    x[:, 0], x[:, 32], x[:, 64], x[:, 96] = parts[:, 0], parts[:, 1], parts[:, 2], 1.0
    u = torch.tensor([1.0, -1.5, 2.0 ** -20, 1.5 * 2.0 ** 40, 2.0 ** 100, -(2.0 ** 60), 3.0, 2.0 ** -60],
                     device="cuda")
    w = torch.zeros((1, 16, 128), device="cuda")
    w[0, :8, [0, 32, 64]] = 1.0
    w[0, 8:, 96] = u
    tpe = torch.tensor([M * copies], device="cuda")
    out = ops.grouped_swiglu_mxfp4(x.repeat(copies, 1), ops.pack_mxfp4_weight(w, swiglu=True), tpe)
    g = parts.double().sum(1, keepdim=True)
    h = (g * torch.special.expit(g) * u.double()).repeat(copies, 1)
    tol = h.abs() * (BF16 + 2.0 ** -15) + (2.0 ** -148 * (g.abs() + 1) * u.double().abs()).repeat(copies, 1) + 2.0 ** -134
    err = (out.double() - h).abs()
    assert (err <= tol).all(), (err / tol).max()
