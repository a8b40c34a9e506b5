"""MXFP4 quantiser, expert products and expert path vs the definition in 64 bits.

Tolerances.  Quantised values and codes are exact.  A product's sums of exact
products are fp32: in any order, with truncating adders, |error| <=
K * 2^-23 * sum|a b|.  A bf16 output adds half a step, 2^-8 of the value.
silu(g) * u in fp32: |d silu / dg| <= 1.1, and the exponential, the quotient
and the two products together stay within 2^-18 of the value (exp's argument
is reduced in fp32: an absolute error of 2^-22 |g| in it, |g| < 16 here).
"""
import ctypes
import importlib

import numpy as np
import pytest
import torch

import mxfp4_ref as R
from gpu_util import get_ops, ragged_counts, random_topk

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8


def _rand(shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _np(t):
    return t.double().cpu().numpy()


def _values64(x):
    """float64 tensor [..., K] of the MXFP4 values of x, on the GPU."""
    return torch.from_numpy(R.rounded(_np(x))).cuda()


def _grouped64(xv, wv, counts):
    """(sums, sums of magnitudes) per group, float64."""
    out = torch.zeros((xv.shape[0], wv.shape[1]), dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    start = 0
    for g, c in enumerate(counts.tolist()):
        if c:
            out[start:start + c] = xv[start:start + c] @ wv[g].T
            mag[start:start + c] = xv[start:start + c].abs() @ wv[g].abs().T
        start += c
    return out, mag


def _swiglu64(xv, wv, counts, K):
    """(h, bound on the fp32 error of h), float64."""
    z, mag = _grouped64(xv, wv, counts)
    I = z.shape[1] // 2
    g, u = z[:, :I], z[:, I:]
    dg, du = mag[:, :I] * K * 2.0 ** -23, mag[:, I:] * K * 2.0 ** -23
    silu = g * torch.sigmoid(g)
    h = silu * u
    return h, 1.1 * dg * (u.abs() + du) + silu.abs() * du + h.abs() * 2.0 ** -18


# ---------------------------------------------------------------- quantiser --
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 8), (1, 1536), (3, 32), (7, 40), (33, 72), (130, 448),
                                    (257, 1000), (64, 4104), (5000, 64)])
def test_quantize_is_the_definition(rows, k, dtype):
    x = _rand((rows, k), rows + k, dtype=torch.float32)
    # magnitudes over the whole range of the type, block by block
    x = x * torch.exp2(torch.randint(-130, 120, (rows, -(-k // 32)), device="cuda").float()
                       ).repeat_interleave(32, dim=1)[:, :k]
    x = x.to(dtype)
    q = get_ops().quantize_mxfp4(x)
    codes, s = R.quantize(_np(x))
    assert np.array_equal(q.scales.cpu().numpy(), s)
    assert np.array_equal(R.unpack_codes(q.codes.cpu().numpy()), codes)
    assert not q.data[:, 17 * (-(-k // 32)):].any()  # the record's padding
    want = torch.from_numpy(R.values(codes, s)[:, :k])
    for out in (torch.bfloat16, torch.float32):
        got = q.dequantize(out)
        assert got.dtype == out and torch.equal(got.double().cpu(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_special_values(dtype):
    big = torch.finfo(dtype).max
    rows = torch.zeros((12, 64), dtype=torch.float32)
    rows[1, 0], rows[1, 40] = -0.0, 2.0 ** -133
    rows[2, :32] = torch.linspace(-8, 8, 32)
    rows[3, :15] = torch.tensor([4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7, -.25, -.75, -5, -7, 6, -3.5])
    rows[4, 3], rows[4, 50] = big, -big
    rows[5, 7] = float("nan")
    rows[6, 31], rows[6, 32] = float("inf"), 1.0
    rows[7, 0] = -float("inf")
    rows[8, :] = 2.0 ** -126
    rows[9, :32], rows[9, 32:] = 2.0 ** -127, 1e-40
    rows[10, :] = torch.exp2(torch.arange(-32, 32).float())
    rows[11, 5] = 7.999
    x = rows.to(dtype).cuda()
    q = get_ops().quantize_mxfp4(x)
    codes, s = R.quantize(_np(x))
    assert np.array_equal(q.scales.cpu().numpy(), s)
    want = R.values(codes, s)
    got = _np(q.dequantize(torch.float32))
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])
    assert np.isnan(got[5, :32]).all() and not np.isnan(got[5, 32:]).any()


def test_quantize_strides_and_shapes():
    ops = get_ops()
    base = _rand((40, 200), 5)
    for x in (base[:, :64], base[::3, 8:136], base[:, 3:67], base.t()[:64, :40], base[:, ::2][:, :96],
              base[:0], base[0, :32], base.reshape(4, 10, 200)):
        q = ops.quantize_mxfp4(x)
        assert q.shape == x.shape
        want = ops.quantize_mxfp4(x.contiguous().clone())
        assert torch.equal(q.data, want.data)
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(base[:, :12])


# ----------------------------------------------------------------- products --
CASES = [
    # M, N, K, G, groups without rows
    (128, 128, 256, 1, 0),
    (1, 8, 8, 1, 0),
    (1, 512, 1536, 3, 2),
    (8, 512, 1536, 64, 56),
    (129, 136, 264, 2, 0),
    (300, 512, 448, 3, 1),
    (777, 64, 40, 7, 2),
    (513, 1280, 96, 16, 3),
    (2000, 24, 512, 16, 0),
    (4099, 200, 1000, 5, 1),
    (4096, 1536, 512, 64, 5),
    (9000, 328, 1536, 128, 30),
    # groups of many rows: CTA pairs
    (1000, 8, 8, 1, 0),
    (1025, 136, 264, 2, 0),
    (257, 64, 1536, 1, 0),
    (3000, 72, 2056, 3, 1),
    (1500, 320, 1800, 2, 0),
    (5001, 1536, 512, 8, 2),
    (30000, 512, 1536, 64, 3),
]


def _counts(M, G, zeros, seed):
    if M < G - zeros:
        zeros = G - M
    return ragged_counts(M, G, seed=seed, zeros=zeros)


@pytest.mark.parametrize("M,N,K,G,zeros", CASES)
def test_grouped_linear(M, N, K, G, zeros):
    ops = get_ops()
    counts = _counts(M, G, zeros, M + G)
    x, w = _rand((M, K), M), _rand((G, N, K), M + 1, 0.02)
    out = ops.grouped_linear_mxfp4(x, ops.pack_mxfp4_weight(w), torch.from_numpy(counts).cuda())
    ref, mag = _grouped64(_values64(x), _values64(w), counts)
    assert out.shape == (M, N) and out.dtype == torch.bfloat16
    tol = BF16 * ref.abs() + mag * K * 2.0 ** -23 * (1 + BF16)
    err = (out.double() - ref).abs()
    assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("M,N,K,G,zeros", CASES)
def test_grouped_swiglu(M, N, K, G, zeros):
    ops = get_ops()
    counts = _counts(M, G, zeros, M + 2 * G)
    x, w = _rand((M, K), M + 2), _rand((G, 2 * N, K), M + 3, 2.0 / K ** 0.5)
    pw = ops.pack_mxfp4_weight(w, swiglu=True)
    tpe = torch.from_numpy(counts).cuda()
    out = ops.grouped_swiglu_mxfp4(x, pw, tpe)
    h, tol = _swiglu64(_values64(x), _values64(w), counts, K)
    err = (out.double() - h).abs()
    lim = BF16 * h.abs() + tol * (1 + BF16)
    assert (err <= lim).all(), (err - lim).max()
    # the quantised form: each code within the room that the fp32 error leaves
    q = ops.grouped_swiglu_mxfp4(ops.quantize_mxfp4(x), pw, tpe, quantized=True)
    assert q.shape == (M, N) and not q.data[:, 17 * (-(-N // 32)):].any()
    h, tol = h.cpu().numpy(), tol.cpu().numpy()
    off = np.abs(_np(q.dequantize(torch.float32)) - R.rounded(h))
    room = R.flip_room(h, tol)
    assert (off <= room).all(), (off - room).max()
    assert np.mean(off > 0) < 1e-3 or off.size < 10000


def test_cta_pair_and_single_cta_kernels_agree(tmp_path):
    """The two kernels give the same bits (child processes that force one each:
    HMOE_GEMM_KERNEL is read once per process)."""
    import os
    import subprocess
    import sys

    import mxfp4_kernels_worker_gpu as W

    outs = {}
    for kern in ("pair", "single"):
        path = tmp_path / f"{kern}.pt"
        env = dict(os.environ, HMOE_GEMM_KERNEL=kern)
        subprocess.run([sys.executable, W.__file__, str(path)], env=env, check=True, timeout=600)
        outs[kern] = torch.load(path)
    assert outs["pair"].keys() == outs["single"].keys()
    for key in outs["pair"]:
        assert torch.equal(outs["pair"][key], outs["single"][key]), key


@pytest.mark.parametrize("M,N,K,G", [(30000, 512, 1536, 64), (20000, 320, 1800, 4),
                                     (4000, 512, 1536, 64), (3000, 200, 448, 100)])
def test_products_repeat_bit_for_bit(M, N, K, G):
    """Every run of a product gives the same bits, with cold and with warm caches
    (a race between its copies, MMAs and epilogue would show as a difference)."""
    ops = get_ops()
    x = _rand((M, K), 1, dtype=torch.float32)
    x *= torch.exp2((torch.arange(M, device="cuda") % 5).float())[:, None]  # scales by row
    x = ops.quantize_mxfp4(x.to(torch.bfloat16))
    w, wg = _rand((G, N, K), 2, 0.02), _rand((G, 2 * N, K), 3, 0.02)
    pw, pg = ops.pack_mxfp4_weight(w), ops.pack_mxfp4_weight(wg, swiglu=True)
    tpe = torch.from_numpy(ragged_counts(M, G, seed=M)).cuda()
    calls = [lambda: ops.grouped_linear_mxfp4(x, pw, tpe),
             lambda: ops.grouped_swiglu_mxfp4(x, pg, tpe),
             lambda: ops.grouped_swiglu_mxfp4(x, pg, tpe, quantized=True).data]
    want = [f() for f in calls]
    flush = torch.empty(200 << 20, dtype=torch.uint8, device="cuda")
    for i in range(40):
        if i % 2:
            flush.fill_(i)
        for f, r in zip(calls, want):
            assert torch.equal(f(), r)


def test_checkpoint_and_rows_pack_alike():
    ops = get_ops()
    w = _rand((3, 80, 104), 3, 0.02, torch.float32)
    rows = ops.quantize_mxfp4(w)
    for swiglu in (False, True):
        a = ops.pack_mxfp4_weight(w, swiglu=swiglu)
        b = ops.pack_mxfp4_weight(rows, swiglu=swiglu)
        c = ops.pack_mxfp4_weight((rows.codes.contiguous(), rows.scales.contiguous()), 104,
                                  swiglu=swiglu)
        assert (a.groups, a.n, a.k) == (3, 40 if swiglu else 80, 104)
        x = _rand((9, 104), 4)
        fn = ops.grouped_swiglu_mxfp4 if swiglu else ops.grouped_linear_mxfp4
        tpe = torch.tensor([4, 0, 5], device="cuda")
        want = fn(x, a, tpe)
        assert torch.equal(fn(x, b, tpe), want) and torch.equal(fn(x, c, tpe), want)


def test_nan_stays_in_its_row_and_column():
    ops = get_ops()
    M, N, K = 200, 96, 320
    x, w = _rand((M, K), 1), _rand((2, N, K), 2, 0.02)
    tpe = torch.tensor([130, 70], device="cuda")
    clean = ops.grouped_linear_mxfp4(x, ops.pack_mxfp4_weight(w), tpe)
    x2, w2 = x.clone(), w.clone()
    x2[17, 300], x2[140, 3] = float("nan"), float("inf")
    w2[1, 40, 100] = float("nan")
    out = ops.grouped_linear_mxfp4(x2, ops.pack_mxfp4_weight(w2), tpe)
    bad = torch.zeros((M, N), dtype=torch.bool, device="cuda")
    bad[17], bad[140], bad[130:, 40] = True, True, True
    assert torch.equal(out.isnan(), bad)
    assert torch.equal(out[~bad], clean[~bad])
    # a NaN that SwiGLU passes on becomes a NaN block of the quantised output
    wg = _rand((2, 2 * N, K), 3, 0.02)
    q = ops.grouped_swiglu_mxfp4(x2, ops.pack_mxfp4_weight(wg, swiglu=True), tpe, quantized=True)
    v = q.dequantize()
    assert v[17].isnan().all() and v[140].isnan().all()
    assert v.isnan().sum() == 2 * N


def _call_linear(lib, rows, w, tpe, M, out, swiglu=False, quantized=0):
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    args = (p(rows.data), p(w.data), p(tpe), M, w.n, w.k, w.groups)
    if swiglu:
        rc = lib.load().hmoe_grouped_swiglu_mxfp4(*args, quantized, p(out), None, 0, st)
    else:
        rc = lib.load().hmoe_grouped_linear_mxfp4(*args, p(out), None, 0, st)
    assert rc == 0, lib.last_error()


@pytest.mark.parametrize("M", [300, 1500])  # single CTAs, CTA pairs
def test_rows_past_the_groups_and_wrong_counts(M):
    ops, lib = get_ops(), importlib.import_module("hrm-moe_b200._lib")
    N, K = 72, 96
    x, w = ops.quantize_mxfp4(_rand((M, K), 1)), ops.pack_mxfp4_weight(_rand((3, N, K), 2, 0.02))
    wg = ops.pack_mxfp4_weight(_rand((3, 2 * N, K), 3, 0.02), swiglu=True)
    full = torch.tensor([100, 90, M - 190], dtype=torch.int32, device="cuda")
    want = ops.grouped_linear_mxfp4(x, w, full)
    for counts, done in [([100, 20, 0], 120), ([0, 0, 0], 0), ([100, 90, 2 ** 31 - 1], M),
                         ([100, -5, -(2 ** 31)], 100), ([2 ** 31 - 1] * 3, M)]:
        tpe = torch.tensor(counts, dtype=torch.int32, device="cuda")
        out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device="cuda")
        _call_linear(lib, x, w, tpe, M, out)
        assert (out[done:] == 7).all()
        same = min(done, 100)  # the first group's rows
        assert torch.equal(out[:same], want[:same])
        q = torch.full((M, lib.load().hmoe_mxfp4_row_bytes(N)), 9, dtype=torch.uint8, device="cuda")
        _call_linear(lib, x, wg, tpe, M, q, swiglu=True, quantized=1)
        assert (q[done:] == 9).all()
    assert ops.grouped_linear_mxfp4(x.dequantize()[:0], w, full).shape == (0, N)
    assert ops.grouped_swiglu_mxfp4(_rand((0, K), 1), wg, full, quantized=True).shape == (0, N)


def test_offsets_past_32_bits():
    """Records, outputs and quantised outputs whose byte offsets pass 2^31 and 2^32."""
    ops = get_ops()
    M, N, K, last = 2_200_001, 1024, 1536, 257
    x = _rand((last, K), 1)
    rows = ops.quantize_mxfp4(x)
    data = torch.zeros((M, rows.data.shape[1]), dtype=torch.uint8, device="cuda")
    data[M - last:] = rows.data
    big = ops.Mxfp4Rows(data, K)
    w = ops.pack_mxfp4_weight(_rand((2, N, K), 2, 0.02))
    tpe = torch.tensor([M - last, last], device="cuda")
    out = ops.grouped_linear_mxfp4(big, w, tpe)
    want = ops.grouped_linear_mxfp4(rows, w, torch.tensor([0, last], device="cuda"))
    assert torch.equal(out[M - last:], want)
    assert not out[:M - last].any()
    del out
    v = big.dequantize()
    assert torch.equal(v[M - last:], rows.dequantize())
    q = ops.quantize_mxfp4(v)
    assert torch.equal(q.data, data)


# -------------------------------------------------------------- expert path --
def _layer(T, d, I, E, k, seed):
    x = _rand((T, d), seed)
    wgu, wd = _rand((E, 2 * I, d), seed + 1, 1.0 / d ** 0.5), _rand((E, d, I), seed + 2, 1.0 / I ** 0.5)
    idx = torch.from_numpy(random_topk(T, E, k, seed)).cuda()
    rw = torch.softmax(_rand((T, k), seed + 3).float(), -1).to(torch.bfloat16)
    return x, idx, rw, wgu, wd


LAYERS = [(1, 64, 32, 4, 2), (3, 1536, 512, 64, 8), (65, 72, 40, 8, 1), (64, 1280, 448, 64, 8),
          (1025, 200, 328, 128, 8), (5000, 256, 96, 16, 4)]


@pytest.mark.parametrize("T,d,I,E,k", LAYERS)
def test_experts_forward(T, d, I, E, k):
    ops = get_ops()
    x, idx, rw, wgu, wd = _layer(T, d, I, E, k, T + d)
    pgu, pd = ops.pack_mxfp4_weight(wgu, swiglu=True), ops.pack_mxfp4_weight(wd)
    y = ops.experts_forward_mxfp4(x, idx, rw, pgu, pd)
    # the same steps through the public operators
    r = ops.dispatch(idx, E, x, rw)
    h = ops.grouped_swiglu_mxfp4(r["x_sorted"], pgu, r["counts"], quantized=True)
    eo = ops.grouped_linear_mxfp4(h, pd, r["counts"])
    prod = torch.empty((T * k, d), dtype=torch.float64, device="cuda")
    prod[r["sort_idx"].long()] = eo.double()
    prod = prod.reshape(T, k, d) * rw.double()[:, :, None]
    want, mag = prod.sum(1), prod.abs().sum(1)
    # small calls keep the experts' outputs in fp32: half a bf16 step from `eo`
    half = BF16 * mag if 4 * T * k * d <= 8 << 20 else torch.zeros_like(mag)
    err = (y.double() - want).abs()
    assert (err <= BF16 * want.abs() + (half + k * 2.0 ** -23 * mag) * (1 + BF16)).all()
    # added into final_hidden_states
    base = _rand((T, d), 9)
    acc = base.clone()
    assert ops.experts_forward_mxfp4(x, idx, rw, pgu, pd, acc) is acc
    want2 = want + base.double()
    err = (acc.double() - want2).abs()
    assert (err <= BF16 * want2.abs()
            + (half + (k + 1) * 2.0 ** -23 * (mag + base.double().abs())) * (1 + BF16)).all()
    # against 64 bits: two bf16 roundings, and the codes of h that the fp32 error may move
    xv, gv, dv = _values64(x), _values64(wgu), _values64(wd)
    xs = xv[r["sorted_token"].long()]
    counts = r["counts"].cpu().numpy()
    h64, tol = _swiglu64(xs, gv, counts, d)
    room = torch.from_numpy(R.flip_room(h64.cpu().numpy(), tol.cpu().numpy())).cuda()
    o64, omag = _grouped64(torch.from_numpy(R.rounded(h64.cpu().numpy())).cuda(), dv, counts)
    _, moved = _grouped64(room, dv, counts)
    otol = BF16 * o64.abs() + (omag * I * 2.0 ** -23 + moved) * (1 + BF16)
    full, lim = torch.empty_like(prod).reshape(T * k, d), torch.empty((T * k, d), dtype=torch.float64, device="cuda")
    full[r["sort_idx"].long()], lim[r["sort_idx"].long()] = o64, otol
    y64 = (full.reshape(T, k, d) * rw.double()[:, :, None]).sum(1)
    ytol = (lim.reshape(T, k, d) * rw.double()[:, :, None]).sum(1)
    ytol = (ytol + k * 2.0 ** -23 * mag) * (1 + BF16) + BF16 * y64.abs()
    assert ((y.double() - y64).abs() <= ytol).all()


def test_rows_aligned_to_16_bytes_only():
    """Inputs, accumulators and weights that start 16 bytes past a 32-byte boundary."""
    ops = get_ops()
    T, d, I, E, k = 70, 96, 64, 4, 2
    x, idx, rw, wgu, wd = _layer(T, d, I, E, k, 8)
    pgu, pd = ops.pack_mxfp4_weight(wgu, swiglu=True), ops.pack_mxfp4_weight(wd)
    want = ops.experts_forward_mxfp4(x, idx, rw, pgu, pd)

    def shifted(t):
        buf = torch.empty(t.numel() + 16, dtype=t.dtype, device="cuda")
        off = 16 // t.element_size()
        out = buf[off:off + t.numel()].view(t.shape)
        assert out.data_ptr() % 32 == 16
        return out.copy_(t)

    for dt in (torch.bfloat16, torch.float32):
        assert torch.equal(ops.quantize_mxfp4(shifted(x.to(dt))).data, ops.quantize_mxfp4(x.to(dt)).data)
    acc = shifted(torch.zeros_like(x))
    got = ops.experts_forward_mxfp4(shifted(x), idx, rw, ops.pack_mxfp4_weight(shifted(wgu), swiglu=True),
                                    pd, acc)
    assert torch.equal(got, want)


def test_error_word_of_the_expert_call():
    """Expert ids outside [0, E) are reported in the workspace's error word, and the next
    call on the workspace clears it (both dispatch forms)."""
    ops, lib = get_ops(), importlib.import_module("hrm-moe_b200._lib")
    d, I, E, k = 64, 32, 8, 2
    for T in (40, 900):
        x, idx, rw, wgu, wd = _layer(T, d, I, E, k, T)
        pgu, pd = ops.pack_mxfp4_weight(wgu, swiglu=True), ops.pack_mxfp4_weight(wd)
        so, shape = lib.load(), lib.HmoeShape(T, d, E, I, k, 0, 1)
        ws = torch.empty(so.hmoe_experts_mxfp4_workspace_bytes(ctypes.byref(shape)), dtype=torch.uint8,
                         device="cuda")
        y = torch.empty_like(x)
        p = lambda t: ctypes.c_void_p(t.data_ptr())
        for bad in (True, False):
            ids = idx.clone()
            if bad:
                ids[3, 1] = E
            rc = so.hmoe_experts_forward_mxfp4(
                ctypes.byref(shape), p(x), p(ids), p(rw), p(pgu.data), p(pd.data), None, p(y), None,
                None, p(ws), ws.numel(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
            assert rc == 0, lib.last_error()
            if bad:
                with pytest.raises(ValueError):
                    ops.workspace_status(ws)
            else:
                ops.workspace_status(ws)


def test_experts_forward_drops_and_empty():
    ops = get_ops()
    T, d, I, E, k = 40, 64, 32, 8, 2
    x, idx, rw, wgu, wd = _layer(T, d, I, E, k, 3)
    pgu, pd = ops.pack_mxfp4_weight(wgu, swiglu=True), ops.pack_mxfp4_weight(wd)
    idx2 = idx.clone()
    idx2[5], idx2[6, 0] = -1, E + 3          # token 5 loses both experts, token 6 one
    y, y2 = (ops.experts_forward_mxfp4(x, i, rw, pgu, pd) for i in (idx, idx2))
    keep = torch.ones(T, dtype=torch.bool)
    keep[5] = keep[6] = False
    assert torch.equal(y[keep], y2[keep]) and not y2[5].any()
    assert ops.experts_forward_mxfp4(x[:0], idx[:0], rw[:0], pgu, pd).shape == (0, d)
    # the same expert twice for one token: both assignments count
    idx3 = idx.clone()
    idx3[:, 1] = idx3[:, 0]
    half = torch.full_like(rw, 0.5)
    y3 = ops.experts_forward_mxfp4(x, idx3, half, pgu, pd)
    y4 = ops.experts_forward_mxfp4(x, idx3[:, :1], torch.ones_like(rw[:, :1]), pgu, pd)
    assert torch.equal(y3, y4)


@pytest.mark.parametrize("T", [1, 64, 1100])
def test_ffn_forward_routes_as_the_bf16_layer(T):
    ops = get_ops()
    d, I, E, k = 256, 96, 32, 4
    x, _, _, wgu, wd = _layer(T, d, I, E, k, T)
    wr = _rand((E, d), 11, 0.05)
    pgu, pd = ops.pack_mxfp4_weight(wgu, swiglu=True), ops.pack_mxfp4_weight(wd)
    y, r = ops.ffn_forward_mxfp4(x, wr, pgu, pd, k, True, return_routing=True)
    _, rb = ops.ffn_forward(x, wr, wgu, wd, k, True, return_routing=True)
    for key in r:
        assert torch.equal(r[key], rb[key]), key
    # the layer weights its rows in fp32, the expert call in bf16: half a step apart each
    again = ops.experts_forward_mxfp4(x, r["topk_idx"], r["topk_weight"], pgu, pd)
    rows = ops.dispatch(r["topk_idx"], E, x)
    eo = ops.grouped_linear_mxfp4(
        ops.grouped_swiglu_mxfp4(rows["x_sorted"], pgu, rows["counts"], quantized=True), pd,
        rows["counts"])
    mag = torch.zeros((T, d), dtype=torch.float64, device="cuda")
    mag.index_add_(0, rows["sorted_token"].long(),
                   eo.double().abs() * r["topk_weight"].reshape(-1)[rows["sort_idx"].long()].double()[:, None])
    assert ((y.double() - again.double()).abs() <= 3 * BF16 * mag).all()
    acc = y.clone()
    ops.ffn_forward_mxfp4(x, wr, pgu, pd, k, True, out=acc, accumulate=True)
    assert ((acc.double() - 2 * y.double()).abs() <= 2 * BF16 * (2 * y.double().abs()) + BF16 * mag).all()


def test_streams_graphs_and_replays():
    """Another stream than the inputs', captured graphs that run in turn, new inputs per replay."""
    ops = get_ops()
    d, I, E, k = 512, 160, 16, 4
    wr = _rand((E, d), 11, 0.05)
    _, _, _, wgu, wd = _layer(1, d, I, E, k, 5)
    pgu, pd = ops.pack_mxfp4_weight(wgu, swiglu=True), ops.pack_mxfp4_weight(wd)
    xs = {T: [_rand((T, d), 7 * T + i) for i in range(3)] for T in (1, 48, 700)}
    want = {T: [ops.ffn_forward_mxfp4(x, wr, pgu, pd, k, True) for x in v] for T, v in xs.items()}
    caps = {T: ops.CapturedFfn(v[0], wr, pgu, pd, k, True) for T, v in xs.items()}
    for i in range(3):
        for T in xs:
            assert torch.equal(caps[T](xs[T][i]), want[T][i])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.ffn_forward_mxfp4(x, wr, pgu, pd, k, True) for x in xs[700]]
    other = [ops.ffn_forward_mxfp4(x, wr, pgu, pd, k, True) for x in xs[48]]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[700]))
    assert all(torch.equal(a, b) for a, b in zip(other, want[48]))


def test_module_with_quantized_experts():
    ops, L = get_ops(), importlib.import_module("hrm-moe_b200.layers")
    torch.manual_seed(0)
    m = L.SparseMoESwiGLU(256, 96, 16, 4, True, router_bias=True, device="cuda", dtype=torch.bfloat16)
    x = _rand((2, 33, 256), 1)
    with torch.no_grad():
        plain = m(x)
        m.quantize_experts()
        y = m(x)
        want = ops.ffn_forward_mxfp4(x.reshape(-1, 256), m.gate.weight,
                                     ops.pack_mxfp4_weight(m.experts.gate_up_weight, swiglu=True),
                                     ops.pack_mxfp4_weight(m.experts.down_weight), 4, True,
                                     router_bias=m.gate.bias)
        assert y.shape == x.shape and torch.equal(y.reshape(-1, 256), want)
        # 4-bit operands: each element off by at most a quarter of itself, or an
        # eighth of the block's scale unit; the products of a layer of three
        # average that out, and the layers stay recognisably the same
        rel = (y.double() - plain.double()).norm() / plain.double().norm()
        assert 0.01 < rel < 0.5
        # the experts module alone, added into its accumulator
        idx, rw = ops.router_topk(x.reshape(-1, 256), m.gate.weight, 4, True, m.gate.bias)
        acc = torch.zeros((66, 256), dtype=torch.bfloat16, device="cuda")
        got = m.experts(x.reshape(-1, 256), idx, rw, acc)
        assert got is acc
        assert torch.equal(acc, ops.experts_forward_mxfp4(x.reshape(-1, 256), idx, rw, *m.experts.quantized()))
        cap = ops.CapturedFfn(x.reshape(-1, 256), m.gate.weight, *m.experts.quantized(), 4, True, m.gate.bias)
        assert torch.equal(cap(x.reshape(-1, 256)), want)
        assert "_mxfp4" not in "".join(m.state_dict())
        assert m(x[:0]).shape == x[:0].shape
    with pytest.raises(RuntimeError, match="no backward"):
        m(x)
    with torch.no_grad():
        m.experts.down_weight.mul_(2.0)
        with pytest.raises(RuntimeError, match="changed"):
            m(x)
        m.quantize_experts()
        assert torch.equal(m(x).double(), 2 * y.double())  # a power of two moves every scale alike
        m.drop_quantized_experts()
        assert torch.equal(m(x).double(), 2 * plain.double())
    m(x).sum().backward()
    assert m.experts.gate_up_weight.grad is not None


def test_refusals_on_the_device():
    ops = get_ops()
    x = _rand((8, 64), 1)
    w = ops.pack_mxfp4_weight(_rand((2, 16, 64), 2))
    tpe = torch.tensor([4, 4], device="cuda")
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(x[:, :20])
    with pytest.raises(TypeError):
        ops.grouped_linear_mxfp4(x.half(), w, tpe)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.grouped_linear_mxfp4(x, w, tpe.cpu())
    with pytest.raises(ValueError, match="even"):
        ops.pack_mxfp4_weight(_rand((2, 17, 64), 2), swiglu=True)
    with pytest.raises(ValueError):
        ops.pack_mxfp4_weight(_rand((2, 20, 64), 2))  # N not a multiple of 8
    with pytest.raises(ValueError, match="do not match"):
        ops.experts_forward_mxfp4(x, torch.zeros((8, 1), dtype=torch.int32, device="cuda"),
                                  torch.ones((8, 1), device="cuda"), w, w)
    with pytest.raises(TypeError):
        ops.quantize_mxfp4(x).dequantize(torch.float16)
    gu = ops.pack_mxfp4_weight(_rand((2, 16, 64), 3), swiglu=True)
    dn = ops.pack_mxfp4_weight(_rand((2, 64, 8), 4))
    idx, rw = torch.zeros((8, 1), dtype=torch.int32, device="cuda"), torch.ones((8, 1), device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    for bad in ({"counts_out": torch.zeros(1, **i32)}, {"counts_out": torch.zeros(2, device="cuda")},
                {"sort_idx_out": torch.zeros(7, **i32)}, {"sort_idx_out": torch.zeros(16, **i32)[::2]}):
        with pytest.raises(ValueError, match="contiguous int32"):
            ops.experts_forward_mxfp4(x, idx, rw, gu, dn, **bad)
    counts, order = torch.full((2,), -1, **i32), torch.full((8,), -1, **i32)
    ops.experts_forward_mxfp4(x, idx, rw, gu, dn, counts_out=counts, sort_idx_out=order)
    assert counts.tolist() == [8, 0] and order.tolist() == list(range(8))
    ops.experts_forward_mxfp4(x[:0], idx[:0], rw[:0], gu, dn, counts_out=counts)
    assert counts.tolist() == [0, 0]
