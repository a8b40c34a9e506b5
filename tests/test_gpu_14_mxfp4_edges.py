"""MXFP4 operators at the edges of what they take: offsets past 32 bits, the most groups, fp32 and
strided inputs, plain launches, streams, captured products."""
import importlib

import pytest
import torch

from gpu_util import get_ops, ragged_counts

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8


def _rand(shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


# ---------------------------------------------------- offsets past 32 bits --
def test_records_past_32_bits():
    """Records read and written whose byte offsets pass 2^32: rows in, rows out, quantised, dequantised."""
    ops = get_ops()
    M, N, K, last = 5_300_001, 1544, 1536, 257
    rows = ops.quantize_mxfp4(_rand((last, K), 1))
    data = torch.zeros((M, rows.data.shape[1]), dtype=torch.uint8, device="cuda")
    assert (M - last) * data.shape[1] > 2 ** 32
    data[M - last:] = rows.data
    big = ops.Mxfp4Rows(data, K)
    w = ops.pack_mxfp4_weight(_rand((2, 2 * N, K), 2, 0.02), swiglu=True)
    tpe, only = torch.tensor([M - last, last], device="cuda"), torch.tensor([0, last], device="cuda")
    out = ops.grouped_swiglu_mxfp4(big, w, tpe, quantized=True)
    assert (M - last) * out.data.shape[1] > 2 ** 32
    assert torch.equal(out.data[M - last:], ops.grouped_swiglu_mxfp4(rows, w, only, quantized=True).data)
    assert not out.data[:M - last].any()  # silu(0) * 0: zero codes and the smallest scale's byte, 0
    del out
    dense = big.dequantize()
    assert torch.equal(dense[M - last:], rows.dequantize())
    assert torch.equal(ops.quantize_mxfp4(dense).data, data)


def test_dispatched_records_past_32_bits():
    """The expert path's records (by expert, and of h) and fp32 outputs, past 2^32 bytes each."""
    ops = get_ops()
    T, d, I, E, k = 700_000, 1536, 1544, 64, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((T, d), generator=g, device="cuda", dtype=torch.bfloat16)
    idx = torch.rand((T, E), generator=g, device="cuda").topk(k, dim=-1).indices.to(torch.int32)
    rw = torch.rand((T, k), generator=g, device="cuda").to(torch.bfloat16)
    pgu = ops.pack_mxfp4_weight(_rand((E, 2 * I, d), 2, 0.02), swiglu=True)
    pd = ops.pack_mxfp4_weight(_rand((E, d, I), 3, 0.02))
    assert T * k * 816 > 2 ** 32  # the shorter of the two kinds of record
    y = ops.experts_forward_mxfp4(x, idx, rw, pgu, pd)
    for a, b in ((0, 7), (T // 2, T // 2 + 100), (T - 300, T)):
        assert torch.equal(y[a:b], ops.experts_forward_mxfp4(x[a:b], idx[a:b], rw[a:b], pgu, pd))


# ------------------------------------------------------------------- groups --
@pytest.mark.parametrize("M,N,K,G", [(3000, 72, 96, 200), (39000, 24, 64, 200), (5000, 8, 40, 1024),
                                     (200001, 8, 32, 1024)])  # single CTAs and CTA pairs
def test_more_than_128_groups(M, N, K, G):
    ops = get_ops()
    counts = torch.from_numpy(ragged_counts(M, G, seed=G, zeros=G // 5)).cuda()
    x, w, wg = _rand((M, K), 1), _rand((G, N, K), 2), _rand((G, 2 * N, K), 3)
    xq = ops.quantize_mxfp4(x)
    group = torch.repeat_interleave(torch.arange(G, device="cuda"), counts.long())
    xv = xq.dequantize(torch.float32).double()

    def product(weight):
        """(sums, sums of magnitudes), 64 bits, a few rows at a time."""
        wv = ops.quantize_mxfp4(weight).dequantize(torch.float32).double()
        parts = [(torch.einsum("mk,mnk->mn", a, wv[g]), torch.einsum("mk,mnk->mn", a.abs(), wv[g].abs()))
                 for a, g in zip(xv.split(4096), group.split(4096))]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])

    out = ops.grouped_linear_mxfp4(xq, ops.pack_mxfp4_weight(w), counts)
    ref, mag = product(w)
    assert ((out.double() - ref).abs() <= BF16 * ref.abs() + mag * K * 2.0 ** -23 * (1 + BF16)).all()
    out = ops.grouped_swiglu_mxfp4(xq, ops.pack_mxfp4_weight(wg, swiglu=True), counts)
    z, mag = product(wg)
    gate, up = z[:, :N], z[:, N:]
    dg, du = mag[:, :N] * K * 2.0 ** -23, mag[:, N:] * K * 2.0 ** -23
    silu = gate * torch.sigmoid(gate)
    h = silu * up
    # |d silu / dg| <= 1.1; the exponential's argument: two roundings of |g| log2 e, 2^-23 |g| after ln 2
    tol = 1.1 * dg * (up.abs() + du) + silu.abs() * du + h.abs() * (2.0 ** -18 + 2.0 ** -22 * gate.abs())
    assert ((out.double() - h).abs() <= BF16 * h.abs() + tol * (1 + BF16) + 2.0 ** -134).all()


# ------------------------------------------------------------- dense inputs --
@pytest.mark.parametrize("M", [1, 37, 900])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dense_inputs_of_any_layout(M, dtype):
    """fp32 inputs, rows with gaps, unaligned and transposed ones: as their records."""
    ops = get_ops()
    N, K, G = 72, 104, 3
    base = _rand((M + 3, 3 * K + 5), 1, dtype=dtype)
    w, wg = (ops.pack_mxfp4_weight(_rand((G, n, K), n, 0.1), swiglu=n > N) for n in (N, 2 * N))
    tpe = torch.tensor([M // 2, 0, M - M // 2], dtype=torch.int64, device="cuda")
    wide = _rand((M, 512), 2, dtype=dtype)
    for x in (base[:M, :K], base[1:M + 1, 3:K + 3], base[:M, :2 * K:2], wide[:, 8:8 + K], wide[:, 400:400 + K],
              _rand((K, M), 3, dtype=dtype).t(), _rand((1, K), 4, dtype=dtype).expand(M, K)):
        rows = ops.quantize_mxfp4(x.clone(memory_format=torch.contiguous_format))
        assert torch.equal(ops.grouped_linear_mxfp4(x, w, tpe), ops.grouped_linear_mxfp4(rows, w, tpe))
        assert torch.equal(ops.grouped_swiglu_mxfp4(x, wg, tpe), ops.grouped_swiglu_mxfp4(rows, wg, tpe))
        assert torch.equal(ops.grouped_swiglu_mxfp4(x, wg, tpe, quantized=True).data,
                           ops.grouped_swiglu_mxfp4(rows, wg, tpe, quantized=True).data)


# ------------------------------------------------- launches, streams, graphs --
def _calls(ops):
    """Small and large calls of every operator on fixed inputs."""
    d, I, E, k = 256, 96, 8, 2
    wr = _rand((E, d), 11, 0.05)
    pgu = ops.pack_mxfp4_weight(_rand((E, 2 * I, d), 1, 0.05), swiglu=True)
    pd = ops.pack_mxfp4_weight(_rand((E, d, I), 2, 0.05))
    out = []
    for T in (3, 2500):
        x = _rand((T, d), T)
        tpe = torch.from_numpy(ragged_counts(T, E, seed=T, zeros=5 if T == 3 else 1)).cuda()
        out += [lambda x=x: ops.quantize_mxfp4(x).dequantize(),
                lambda x=x, c=tpe: ops.grouped_linear_mxfp4(
                    ops.grouped_swiglu_mxfp4(x, pgu, c, quantized=True), pd, c),
                lambda x=x: ops.ffn_forward_mxfp4(x, wr, pgu, pd, k, True)]
    return out


def test_plain_launches_give_the_same_bits():
    """Without programmatic dependent launch."""
    ops, lib = get_ops(), importlib.import_module("hrm-moe_b200._lib").load()
    calls = _calls(ops)
    want = [f() for f in calls]
    before = lib.hmoe_set_pdl_mask(0)
    try:
        got = [f() for f in calls]
        torch.cuda.synchronize()
    finally:
        lib.hmoe_set_pdl_mask(before)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    ops = get_ops()
    calls = _calls(ops)
    want = [f() for f in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append([f() for f in (calls if i else calls[::-1])])
    torch.cuda.synchronize()
    for rounds, order in zip(got, (want[::-1], want)):
        for r in rounds:
            for a, b in zip(r, order):
                assert torch.equal(a, b)


def test_captured_products_take_new_inputs_and_counts():
    ops = get_ops()
    M, N, K, G = 700, 72, 96, 3
    x = _rand((M, K), 1)
    w, wg = ops.pack_mxfp4_weight(_rand((G, N, N), 2, 0.1)), \
        ops.pack_mxfp4_weight(_rand((G, 2 * N, K), 3, 0.1), swiglu=True)
    tpe = torch.tensor([300, 0, 400], dtype=torch.int32, device="cuda")
    ws = torch.empty(16, dtype=torch.uint8, device="cuda")

    def run(x, c):
        h = ops.grouped_swiglu_mxfp4(x, wg, c, quantized=True, workspace=ws)
        return ops.grouped_linear_mxfp4(h, w, c, workspace=ws)

    run(x, tpe)
    graphs, outs = [], []
    for _ in range(2):  # two graphs on the same inputs and error word
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(x, tpe))
        graphs.append(g)
    for i, counts in enumerate(([700, 0, 0], [1, 698, 1], [0, 0, 0], [200, 300, 200])):
        x.copy_(_rand((M, K), 10 + i))
        tpe.copy_(torch.tensor(counts, dtype=torch.int32))
        want, done = run(x, tpe), sum(counts)
        for g, out in zip(graphs, outs):
            g.replay()
            assert torch.equal(out[:done], want[:done])
        ops.workspace_status(ws)


# ------------------------------------------------------------------ modules --
def _module(dtype):
    L = importlib.import_module("hrm-moe_b200.layers")
    torch.manual_seed(0)
    return L.SparseMoESwiGLU(256, 96, 16, 4, True, device="cuda", dtype=dtype)


@torch.no_grad()
def test_a_module_serves_no_weights_that_were_written_over():
    m = _module(torch.bfloat16)
    x = _rand((40, 256), 1)
    m.quantize_experts()
    y = m(x)
    for write in (lambda: m.experts.down_weight.data.mul_(2), lambda: m.experts.down_weight.data.copy_(
            m.experts.down_weight.detach() * 0.5), lambda: m.experts.down_weight.mul_(2)):
        write()
        with pytest.raises(RuntimeError, match="changed"):
            m(x)
        m.quantize_experts()
        m(x)
    assert torch.equal(m(x).double(), 2 * y.double())  # a power of two moves every scale alike
    m.drop_quantized_experts()
    m.experts.down_weight.data.mul_(0.5)
    m.quantize_experts()
    assert torch.equal(m(x), y)


@torch.no_grad()
def test_fp32_parameters_serve_bf16_inputs():
    ops = get_ops()
    m = _module(torch.float32)
    x = _rand((40, 256), 1)
    m.quantize_experts()
    want = ops.ffn_forward_mxfp4(x, m.gate.weight, ops.pack_mxfp4_weight(m.experts.gate_up_weight, swiglu=True),
                                 ops.pack_mxfp4_weight(m.experts.down_weight), 4, True)
    assert torch.equal(m(x), want)
    with pytest.raises(TypeError, match="bf16"):
        m(x.float())
