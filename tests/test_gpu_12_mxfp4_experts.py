"""MXFP4 expert path: its sums stay in fp32 whatever the size of the call.

Tolerances.  Given the quantised h, an expert's output is a sum of exact
products in fp32: in any order, with truncating adders, |error| <=
I * 2^-23 * sum|a b|.  The weighted sum over k experts adds at most
k * 2^-23 of the sum of magnitudes, and the one rounding to bf16 half a step,
2^-8 of the value.
"""
import pytest
import torch

from gpu_util import get_ops, random_topk

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8


def _rand(shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _layer(T, d, I, E, k, seed):
    x = _rand((T, d), seed)
    wgu, wd = _rand((E, 2 * I, d), seed + 1, 1.0 / d ** 0.5), _rand((E, d, I), seed + 2, 1.0 / I ** 0.5)
    idx = torch.from_numpy(random_topk(T, E, k, seed)).cuda()
    rw = torch.softmax(_rand((T, k), seed + 3).float(), -1).to(torch.bfloat16)
    return x, idx, rw, wgu, wd


# T, d, I, E, k: outputs of a few KB to 50 MB, groups of few and of many rows,
# more than 8 experts a token (the combine takes four at a time), up to the most there may be
LARGE = [(1025, 512, 96, 16, 8), (5000, 256, 96, 16, 4), (8000, 64, 40, 4, 2), (700, 1000, 64, 24, 13),
         (1500, 264, 72, 128, 32), (40, 96, 32, 128, 9), (3000, 8, 8, 4, 2), (90000, 24, 8, 4, 1),
         (129, 40, 16, 2, 1)]


@pytest.mark.parametrize("T,d,I,E,k", LARGE)
def test_experts_sum_in_fp32(T, d, I, E, k):
    ops = get_ops()
    x, idx, rw, wgu, wd = _layer(T, d, I, E, k, T + d)
    pgu, pd = ops.pack_mxfp4_weight(wgu, swiglu=True), ops.pack_mxfp4_weight(wd)
    y = ops.experts_forward_mxfp4(x, idx, rw, pgu, pd)
    base = _rand((T, d), 9)
    acc = ops.experts_forward_mxfp4(x, idx, rw, pgu, pd, base.clone())
    r = ops.dispatch(idx, E, x, rw)
    h = ops.grouped_swiglu_mxfp4(r["x_sorted"], pgu, r["counts"], quantized=True)
    hv = h.dequantize(torch.float32).double()
    w = ops.quantize_mxfp4(wd).dequantize(torch.float32).double()
    out, mag = (torch.zeros((T * k, d), dtype=torch.float64, device="cuda") for _ in range(2))
    start = 0
    for e, c in enumerate(r["counts"].tolist()):
        rows = r["sort_idx"][start:start + c].long()
        out[rows], mag[rows] = hv[start:start + c] @ w[e].T, hv[start:start + c].abs() @ w[e].abs().T
        start += c
    wt = rw.double()[:, :, None]
    y64, mag = (out.reshape(T, k, d) * wt).sum(1), (mag.reshape(T, k, d) * wt).sum(1)
    fp32 = (I + k) * 2.0 ** -23 * mag
    assert ((y.double() - y64).abs() <= BF16 * y64.abs() + fp32 * (1 + BF16)).all()
    a64 = y64 + base.double()
    fp32 += 2.0 ** -23 * (mag + base.double().abs())
    assert ((acc.double() - a64).abs() <= BF16 * a64.abs() + fp32 * (1 + BF16)).all()


@pytest.mark.parametrize("T,d,I,E,k", [(4100, 512, 96, 4, 2), (1200, 1536, 512, 64, 8)])
def test_a_tokens_bits_do_not_depend_on_its_batch(T, d, I, E, k):
    ops = get_ops()
    x, idx, rw, wgu, wd = _layer(T, d, I, E, k, T)
    pgu, pd = ops.pack_mxfp4_weight(wgu, swiglu=True), ops.pack_mxfp4_weight(wd)
    wr = _rand((E, d), 11, 0.05)
    y = ops.experts_forward_mxfp4(x, idx, rw, pgu, pd)
    f = ops.ffn_forward_mxfp4(x, wr, pgu, pd, k, True)
    for a, b in ((0, 1), (0, 37), (500, 671), (T - 3, T), (0, T // 2)):
        assert torch.equal(ops.experts_forward_mxfp4(x[a:b], idx[a:b], rw[a:b], pgu, pd), y[a:b])
        assert torch.equal(ops.ffn_forward_mxfp4(x[a:b], wr, pgu, pd, k, True), f[a:b])
