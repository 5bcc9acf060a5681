"""The grouped products' tiles on the GPU against 64-bit sums: enough rows and columns that the
kernels for few rows are not taken, both tile sizes, every height of a group's last tile, CTAs
that go on to further tiles, reductions that end inside a stage.  Whole numbers, exact in fp32."""
import numpy as np
import pytest

import grouped_testutil as G
from test_gpu_grouped import _dev, _equal, _ints, _mx_ints, _off, _stack, _t

pytestmark = pytest.mark.gpu

# rows of a group on both sides of 64, 128, 192 and 256, none, and one
HEIGHTS = [0, 1, 16, 40, 64, 65, 100, 128, 129, 160, 192, 193, 250, 256, 257, 300, 0, 5]
MANY = [(37 * i) % 50 for i in range(130)]
# rows of the groups, rows behind them, M, K.  Forward: many columns; few; more tiles than CTAs of either
# size; more groups than a wave has lanes
FORWARD = {
    "large": (HEIGHTS, 70, 4104, 200),
    "large_whole": ([256, 512], 0, 9472, 128),
    "small": ([0, 1, 64, 65, 130, 300], 3, 1032, 72),
    "small_whole": ([128, 256], 0, 1536, 64),
    "small_further": ([4100, 4300], 0, 1000, 72),
    "many_groups": (MANY, 9, 1032, 136),
}
# (dgrad's tiles are K wide, wgrad's M x K)
BACKWARD = {
    "dgrad_large": (HEIGHTS, 70, 200, 4104),
    "wgrad_further": (HEIGHTS, 0, 520, 1304),
    "wgrad_small_further": ([(11 * i) % 70 for i in range(36)], 2, 1000, 200),
    "whole": ([64, 512, 256], 0, 2560, 2560),
    "many_groups": (MANY, 9, 264, 264),
}


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("case", list(FORWARD))
def test_forward(gpu, case, dtype, out):
    from block_lut_amd import ops
    counts, pad, M, K = FORWARD[case]
    E, P = len(counts), sum(counts) + pad
    rng = np.random.default_rng(P + M)
    x, w = _ints(rng, (P, K)), _ints(rng, (E, M, K))
    y = ops.grouped_gemm(_dev(x, dtype, gpu), _dev(w, dtype, gpu), _off(counts, gpu), out_dtype=_t(out))
    _equal(y, G.forward(x, w, G.offsets_of(counts)), out)


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("case", list(BACKWARD))
def test_gradients(gpu, case, dtype, out):
    from block_lut_amd import ops
    counts, pad, M, K = BACKWARD[case]
    E, P = len(counts), sum(counts) + pad
    rng = np.random.default_rng(P + K)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    x, w, dy = _ints(rng, (P, K)), _ints(rng, (E, M, K)), _ints(rng, (P, M))
    dyd = _dev(dy, dtype, gpu)
    _equal(ops.grouped_gemm_dgrad(dyd, _dev(w, dtype, gpu), off, out_dtype=_t(out)), G.dgrad(dy, w, o), out)
    _equal(ops.grouped_gemm_wgrad(dyd, _dev(x, dtype, gpu), off, out_dtype=_t(out)), G.wgrad(dy, x, o, E), out)


MXFP4 = {
    "large": (HEIGHTS, 70, 1801, 160),
    "large_whole": ([256, 512], 0, 9472, 512),
    "large_dwords": (HEIGHTS, 0, 1808, 384),
    "small": ([0, 1, 64, 65, 130, 300], 3, 1850, 96),
    "small_long": ([70, 0, 129, 61], 0, 1030, 2336),
    "small_whole": ([128, 256], 0, 3584, 256),
    "small_further": ([4100, 4300], 0, 1001, 32),
    "many_groups": (MANY, 9, 1032, 288),
}


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("case", list(MXFP4))
def test_mxfp4(gpu, case, shift):
    """Both rows' types; scales that start at any byte."""
    import torch
    from block_lut_amd import ops
    from block_lut_amd.formats import MXFP4Stack
    counts, pad, M, K = MXFP4[case]
    E, P = len(counts), sum(counts) + pad
    rng = np.random.default_rng(P + M + K)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    (wc, ws), (xc, xs) = _mx_ints(rng, (E, M, K)), _mx_ints(rng, (P, K))
    w, x = G.mx_decode(wc, ws), _ints(rng, (P, K))

    def shifted(a):
        buf = torch.full((a.size + shift + 8,), 255, dtype=torch.uint8, device=gpu)   # (NaN around them)
        buf[shift:shift + a.size] = torch.from_numpy(a.reshape(-1)).to(gpu)
        return buf[shift:shift + a.size].view(a.shape)

    st = MXFP4Stack(torch.from_numpy(wc).to(gpu), shifted(ws))
    y = ops.grouped_gemm(torch.from_numpy(xc).to(gpu), st, off, x_scales=shifted(xs), out_dtype=torch.bfloat16)
    _equal(y, G.forward(G.mx_decode(xc, xs), w, o), "bf16")
    y = ops.grouped_gemm(_dev(x, "bf16", gpu), st, off, out_dtype=torch.bfloat16)
    _equal(y, G.forward(x, w, o), "bf16")


@pytest.mark.parametrize("M,K,counts", [(1032, 200, [100, 65, 300, 1]), (4104, 72, HEIGHTS)])
def test_neighbours_are_nan(gpu, M, K, counts):
    """Another group's rows and matrix never reach a result: the reduction's and the tiles' ends."""
    import torch
    from block_lut_amd import ops
    E, P = len(counts), sum(counts) + 40
    off, o = _off(counts, gpu), G.offsets_of(counts)
    rng = np.random.default_rng(M)
    x, w, dy = _ints(rng, (P, K)), _ints(rng, (E, M, K)), _ints(rng, (P, M))
    for e in range(0, E, 3):
        a, b = int(o[e]), int(o[e + 1])
        xn, wn, dyn = np.full_like(x, np.nan), np.full_like(w, np.nan), np.full_like(dy, np.nan)
        xn[a:b], wn[e], dyn[a:b] = x[a:b], w[e], dy[a:b]
        xd, wd, dyd = (_dev(v, "bf16", gpu) for v in (xn, wn, dyn))
        _equal(ops.grouped_gemm(xd, wd, off, out_dtype=torch.float32)[a:b], x[a:b] @ w[e].T, "f32")
        _equal(ops.grouped_gemm_dgrad(dyd, wd, off, out_dtype=torch.float32)[a:b], dy[a:b] @ w[e], "f32")
        _equal(ops.grouped_gemm_wgrad(dyd, xd, off, out_dtype=torch.float32)[e], dy[a:b].T @ x[a:b], "f32")


@pytest.mark.parametrize("K", [128, 160, 384, 512])
@pytest.mark.parametrize("M,counts", [(1850, [0, 1, 64, 65, 130, 300]), (1801, HEIGHTS)])
def test_mxfp4_rows_next_to_nan(gpu, M, counts, K):
    """Every second row and every second matrix row is NaN (scale bytes of 255), first of all behind the
    ends of the others: reductions that end in either half of a stage."""
    import torch
    from block_lut_amd import ops
    E, P = len(counts), sum(counts)
    rng = np.random.default_rng(M + K)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    (wc, ws), (xc, xs) = _mx_ints(rng, (E, M, K)), _mx_ints(rng, (P, K))
    ref = G.forward(G.mx_decode(xc, xs), G.mx_decode(wc, ws), o)
    ws[:, 1::2], xs[1::2] = 255, 255
    y = ops.grouped_gemm(torch.from_numpy(xc).to(gpu), _stack(wc, ws, gpu), off, x_scales=torch.from_numpy(xs).to(gpu),
                         out_dtype=torch.float32)
    _equal(y[::2, ::2], ref[::2, ::2], "f32")
    assert torch.isnan(y[1::2]).all() and torch.isnan(y[:, 1::2]).all()
    x = _ints(rng, (P, K))
    y = ops.grouped_gemm(_dev(x, "bf16", gpu), _stack(wc, ws, gpu), off, out_dtype=torch.float32)
    ws[:, 1::2] = 127
    _equal(y[:, ::2], G.forward(x, G.mx_decode(wc, ws), o)[:, ::2], "f32")
    assert torch.isnan(y[:, 1::2]).all()


@pytest.mark.parametrize("out,shift", [("bf16", 1), ("f16", 8), ("f32", 1)])
@pytest.mark.parametrize("M", [1032, 4104])
def test_element_alignment(gpu, M, out, shift):
    """Results that start between 16-byte boundaries; what lies around them stays."""
    import torch
    from block_lut_amd import ops
    counts, K = [100, 65, 300, 1], 72
    P = sum(counts)
    rng = np.random.default_rng(M + shift)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    x, w = _ints(rng, (P, K)), _ints(rng, (len(counts), M, K))
    buf = torch.full((P * M + 32,), 99.0, device=gpu, dtype=_t(out))
    y = buf[shift:shift + P * M].view(P, M)
    dtype = "f16" if out == "f16" else "bf16"
    ops.grouped_gemm(_dev(x, dtype, gpu), _dev(w, dtype, gpu), off, out=y)
    _equal(y, G.forward(x, w, o), out)
    assert torch.all(buf[:shift] == 99.0) and torch.all(buf[shift + P * M:] == 99.0)


@pytest.mark.parametrize("o", [[0, 900, 400, 1000], [700, 300, 1000, 1000], [0, 1000, 0, 1000]])
def test_decreasing_offsets_stay_in_bounds(gpu, o):
    """Groups that overlap or end before they start: whatever the results, nothing outside them is written."""
    import torch
    from block_lut_amd import ops
    P, M, K = 1000, 2056, 72
    rng = np.random.default_rng(sum(o))
    x, w = _ints(rng, (P, K)), _ints(rng, (3, M, K))
    off = torch.tensor(o, dtype=torch.int32, device=gpu)
    buf = torch.full((P * M + 64,), 99.0, device=gpu, dtype=torch.float32)
    ops.grouped_gemm(_dev(x, "bf16", gpu), _dev(w, "bf16", gpu), off, out=buf[32:32 + P * M].view(P, M))
    torch.cuda.synchronize()
    assert torch.all(buf[:32] == 99.0) and torch.all(buf[32 + P * M:] == 99.0)
