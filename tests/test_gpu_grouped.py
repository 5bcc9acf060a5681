"""The grouped products on the GPU against 64-bit sums.

Small whole numbers (products and sums exact in fp32) pin every index: the result has to be
the 64-bit one rounded once.  Gaussian values pin the rounding.  What a product must not
read -- rows of no group, other experts' matrices and rows -- holds NaN."""
import numpy as np
import pytest

import grouped_testutil as G

pytestmark = pytest.mark.gpu

# rows of each expert, rows behind the last group
GROUPS = {
    "one_row": ([1], 0),
    "empty_and_single": ([0, 1, 0, 0, 2, 0], 3),
    "edges": ([15, 16, 17, 31, 32, 33, 0, 63, 64, 65], 1),
    "tiles": ([127, 128, 129, 0, 255, 257], 70),
    "one_large": ([3, 700, 0, 1], 0),
    "nobody": ([0, 0, 0], 5),
    "many_experts": ([(7 * i) % 5 for i in range(130)], 2),
}
DENSE_SHAPES = [(8, 8), (72, 40), (136, 104), (264, 200), (128, 512), (256, 1000)]
MX_SHAPES = [(1, 32), (7, 64), (48, 96), (129, 160), (200, 544), (256, 1024), (260, 2336)]


def _t(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _dev(a, dtype, gpu):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(_t(dtype)).to(gpu)


def _ints(rng, shape):
    return rng.integers(-3, 4, shape).astype(np.float64)


def _off(counts, gpu):
    import torch
    return torch.from_numpy(G.offsets_of(counts)).to(gpu)


def _equal(got, ref, dtype):
    import torch
    r = G.round_to(ref, dtype)
    g = got.cpu()
    assert g.shape == r.shape and g.dtype == r.dtype
    if not torch.equal(g, r):
        bad = (g != r).nonzero()
        raise AssertionError(f"{len(bad)} of {g.numel()} differ, first at {bad[0].tolist()}: "
                             f"{g[tuple(bad[0])].item()} for {r[tuple(bad[0])].item()}")


def _within(got, ref, mags, n, dtype):
    g = got.double().cpu().numpy()
    tol = G.tolerance(ref, mags, n, dtype)
    off = np.abs(g - ref)
    assert np.all(off <= tol), f"off by {np.max(off / tol):.3g} times the tolerance"


def _mx_ints(rng, shape):
    """Random MXFP4 codes with scales of 1/2 to 2: multiples of 1/4 up to 12."""
    codes = rng.integers(0, 256, shape[:-1] + (shape[-1] // 2,), dtype=np.uint8)
    scales = rng.integers(126, 129, shape[:-1] + (shape[-1] // 32,), dtype=np.uint8)
    return codes, scales


def _stack(codes, scales, gpu):
    import torch
    from block_lut_amd.formats import MXFP4Stack
    return MXFP4Stack(torch.from_numpy(codes).to(gpu), torch.from_numpy(scales).to(gpu))


# ------------------------------------------------------------------- exact

@pytest.mark.parametrize("groups", list(GROUPS))
@pytest.mark.parametrize("M,K", DENSE_SHAPES)
def test_dense_products_exact(gpu, groups, M, K):
    """Forward, both gradients, both input types, results of the type and in fp32."""
    from block_lut_amd import ops
    counts, pad = GROUPS[groups]
    E, P = len(counts), sum(counts) + pad
    rng = np.random.default_rng(M * 7 + K + P)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    x, w, dy = _ints(rng, (P, K)), _ints(rng, (E, M, K)), _ints(rng, (P, M))
    y_ref, dx_ref, dw_ref = G.forward(x, w, o), G.dgrad(dy, w, o), G.wgrad(dy, x, o, E)
    for dtype, out in (("bf16", "bf16"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32")):
        xd, wd, dyd = (_dev(v, dtype, gpu) for v in (x, w, dy))
        _equal(ops.grouped_gemm(xd, wd, off, out_dtype=_t(out)), y_ref, out)
        _equal(ops.grouped_gemm_dgrad(dyd, wd, off, out_dtype=_t(out)), dx_ref, out)
        _equal(ops.grouped_gemm_wgrad(dyd, xd, off, out_dtype=_t(out)), dw_ref, out)


@pytest.mark.parametrize("groups", list(GROUPS))
@pytest.mark.parametrize("M,K", MX_SHAPES)
def test_mxfp4_products_exact(gpu, groups, M, K):
    import torch
    from block_lut_amd import ops
    counts, pad = GROUPS[groups]
    E, P = len(counts), sum(counts) + pad
    rng = np.random.default_rng(M * 5 + K + P)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    wc, ws = _mx_ints(rng, (E, M, K))
    w = G.mx_decode(wc, ws)
    st = _stack(wc, ws, gpu)
    x = _ints(rng, (P, K))
    xc, xs = _mx_ints(rng, (P, K))
    x4_ref = G.forward(G.mx_decode(xc, xs), w, o)
    ref = G.forward(x, w, o)
    for out in ("bf16", "f32"):
        _equal(ops.grouped_gemm(_dev(x, "bf16", gpu), st, off, out_dtype=_t(out)), ref, out)
        y4 = ops.grouped_gemm(torch.from_numpy(xc).to(gpu), st, off, x_scales=torch.from_numpy(xs).to(gpu),
                              out_dtype=_t(out))
        _equal(y4, x4_ref, out)


@pytest.mark.parametrize("M,K", [(1, 32), (129, 160), (256, 1024), (2816, 2048)])
@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 100])
def test_mxfp4_gemv_exact(gpu, T, M, K):
    from block_lut_amd import ops
    rng = np.random.default_rng(M + K + T)
    wc, ws = _mx_ints(rng, (3, M, K))
    st = _stack(wc, ws, gpu)
    x = _ints(rng, (T, K))
    ref = x @ G.mx_decode(wc[1], ws[1]).T
    for out in ("bf16", "f32"):
        _equal(ops.gemv(st, _dev(x, "bf16", gpu), expert=1, out_dtype=_t(out)), ref, out)
    _equal(ops.gemv(st, _dev(x[0], "bf16", gpu), expert=1), ref[0], "bf16")


# ----------------------------------------------------------------- rounding

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,K,counts", [(328, 1000, [40, 0, 300, 1]), (64, 4096, [9, 2])])
def test_dense_products_rounding(gpu, dtype, M, K, counts):
    from block_lut_amd import ops
    E, P = len(counts), sum(counts)
    rng = np.random.default_rng(M + K)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    x, w, dy = (_dev(rng.standard_normal(s) * f, dtype, gpu) for s, f in (((P, K), 1), ((E, M, K), 0.02), ((P, M), 1)))
    xn, wn, dyn = (v.double().cpu().numpy() for v in (x, w, dy))
    for out in (dtype, "f32"):
        _within(ops.grouped_gemm(x, w, off, out_dtype=_t(out)), G.forward(xn, wn, o),
                G.forward(np.abs(xn), np.abs(wn), o), K, out)
        _within(ops.grouped_gemm_dgrad(dy, w, off, out_dtype=_t(out)), G.dgrad(dyn, wn, o),
                G.dgrad(np.abs(dyn), np.abs(wn), o), M, out)
        _within(ops.grouped_gemm_wgrad(dy, x, off, out_dtype=_t(out)), G.wgrad(dyn, xn, o, E),
                G.wgrad(np.abs(dyn), np.abs(xn), o, E), max(counts), out)


@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("M,K,counts", [(328, 1056, [40, 0, 300, 1]), (64, 4096, [9, 2])])
def test_mxfp4_products_rounding(gpu, x4, M, K, counts):
    import torch
    from block_lut_amd import ops
    E, P = len(counts), sum(counts)
    rng = np.random.default_rng(M + K)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    wc, ws = G.mx_encode(rng.standard_normal((E, M, K)) * 0.02)
    x = _dev(rng.standard_normal((P, K)), "bf16", gpu)
    xn, wn = x.double().cpu().numpy(), G.mx_decode(wc, ws)
    kw = {}
    if x4:
        codes, scales = ops.mxfp4_encode(x)
        xn = G.mx_decode(*G.mx_encode(xn))
        x, kw = codes, dict(x_scales=scales)
    for out in ("bf16", "f32"):
        _within(ops.grouped_gemm(x, _stack(wc, ws, gpu), off, out_dtype=_t(out), **kw), G.forward(xn, wn, o),
                G.forward(np.abs(xn), np.abs(wn), o), K, out)


@pytest.mark.parametrize("x4", [False, True])
def test_mxfp4_scale_range(gpu, x4):
    """Scales over the whole range of the byte: each block's share is a power of two of its own."""
    import torch
    from block_lut_amd import ops
    M, K, P = 40, 256, 9
    rng = np.random.default_rng(11)
    wc = rng.integers(0, 256, (1, M, K // 2), dtype=np.uint8)
    ws = rng.choice([1, 20, 127, 150, 230, 250], (1, M, K // 32)).astype(np.uint8)
    xc = rng.integers(0, 256, (P, K // 2), dtype=np.uint8)
    xs = (np.full((P, K // 32), 127) - rng.integers(0, 3, (P, K // 32))).astype(np.uint8)
    off = _off([P], gpu)
    xn, wn = G.mx_decode(xc, xs), G.mx_decode(wc, ws)
    if x4:
        y = ops.grouped_gemm(torch.from_numpy(xc).to(gpu), _stack(wc, ws, gpu), off,
                             x_scales=torch.from_numpy(xs).to(gpu), out_dtype=torch.float32)
    else:
        y = ops.grouped_gemm(_dev(xn, "bf16", gpu), _stack(wc, ws, gpu), off, out_dtype=torch.float32)
    o = G.offsets_of([P])
    mags = G.forward(np.abs(xn), np.abs(wn), o)
    # a block at 2^123 times 32 x 6 x 6 x 2^0 passes fp32's largest value (2^128): where the sum of
    # magnitudes does, a partial sum may be infinite and the result is not compared
    fits = mags < 2.0 ** 127
    assert fits.mean() > 0.1
    _within(torch.where(torch.from_numpy(fits).to(gpu), y, 0.0), np.where(fits, G.forward(xn, wn, o), 0.0),
            np.where(fits, mags, 0.0), K, "f32")


# ------------------------------------------------- what must not be touched

@pytest.mark.parametrize("M,K", [(72, 40), (264, 200), (128, 512)])
def test_dense_reads_nothing_of_the_neighbours(gpu, M, K):
    """Rows of no group, and the matrices and rows of every other expert, are NaN."""
    import torch
    from block_lut_amd import ops
    counts, pad = [33, 5, 70, 1], 40
    E, P = len(counts), sum(counts) + pad
    off, o = _off(counts, gpu), G.offsets_of(counts)
    rng = np.random.default_rng(K)
    x, w, dy = _ints(rng, (P, K)), _ints(rng, (E, M, K)), _ints(rng, (P, M))
    for e in range(E):
        a, b = int(o[e]), int(o[e + 1])
        xn, wn, dyn = np.full_like(x, np.nan), np.full_like(w, np.nan), np.full_like(dy, np.nan)
        xn[a:b], wn[e], dyn[a:b] = x[a:b], w[e], dy[a:b]
        xd, wd, dyd = (_dev(v, "bf16", gpu) for v in (xn, wn, dyn))
        _equal(ops.grouped_gemm(xd, wd, off, out_dtype=torch.float32)[a:b], x[a:b] @ w[e].T, "f32")
        _equal(ops.grouped_gemm_dgrad(dyd, wd, off, out_dtype=torch.float32)[a:b], dy[a:b] @ w[e], "f32")
        _equal(ops.grouped_gemm_wgrad(dyd, xd, off, out_dtype=torch.float32)[e], dy[a:b].T @ x[a:b], "f32")


@pytest.mark.parametrize("M,K", [(7, 96), (129, 160), (256, 1024)])
def test_mxfp4_reads_nothing_of_the_neighbours(gpu, M, K):
    """Scale bytes of 255 (NaN) in every other expert's matrix and in the rows of other groups."""
    import torch
    from block_lut_amd import ops
    counts, pad = [33, 5, 70, 1], 9
    E, P = len(counts), sum(counts) + pad
    off, o = _off(counts, gpu), G.offsets_of(counts)
    rng = np.random.default_rng(K)
    wc, ws = _mx_ints(rng, (E, M, K))
    xc, xs = _mx_ints(rng, (P, K))
    x, w = G.mx_decode(xc, xs), G.mx_decode(wc, ws)
    for e in range(E):
        a, b = int(o[e]), int(o[e + 1])
        wse, xse, xne = np.full_like(ws, 255), np.full_like(xs, 255), np.full_like(x, np.nan)
        wse[e], xse[a:b], xne[a:b] = ws[e], xs[a:b], x[a:b]
        st = _stack(wc, wse, gpu)
        y = ops.grouped_gemm(_dev(xne, "bf16", gpu), st, off, out_dtype=torch.float32)
        _equal(y[a:b], x[a:b] @ w[e].T, "f32")
        y = ops.grouped_gemm(torch.from_numpy(xc).to(gpu), st, off, x_scales=torch.from_numpy(xse).to(gpu),
                             out_dtype=torch.float32)
        _equal(y[a:b], x[a:b] @ w[e].T, "f32")


def test_nan_and_infinity_reach_their_own_results_only(gpu):
    import torch
    from block_lut_amd import ops
    counts = [20, 30]
    off = _off(counts, gpu)
    x = torch.ones(50, 128, device=gpu, dtype=torch.bfloat16)
    w = torch.ones(2, 64, 128, device=gpu, dtype=torch.bfloat16)
    x[7, 100], x[31, 5], w[1, 9, 3] = float("nan"), float("inf"), float("nan")
    y = ops.grouped_gemm(x, w, off).float().cpu()
    want = torch.full((50, 64), 128.0)
    want[7], want[31], want[20:, 9] = float("nan"), float("inf"), float("nan")
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y[~y.isnan()], want[~want.isnan()])
    codes, scales = ops.mxfp4_encode(w)                       # a NaN block: 32 columns of row 9
    from block_lut_amd.formats import MXFP4Stack
    xc, xs = ops.mxfp4_encode(torch.ones(50, 128, device=gpu, dtype=torch.bfloat16))
    y = ops.grouped_gemm(xc, MXFP4Stack(codes, scales), off, x_scales=xs).float().cpu()
    want = torch.full((50, 64), 128.0)
    want[20:, 9] = float("nan")
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y[~y.isnan()], want[~want.isnan()])


@pytest.mark.parametrize("P", [16, 300])
def test_rows_behind_the_groups_stay_in_out(gpu, P):
    import torch
    from block_lut_amd import ops
    M, K, n = 136, 96, P - 7
    off = _off([n // 2, n - n // 2], gpu)
    rng = np.random.default_rng(P)
    x, w, dy = _ints(rng, (P, K)), _ints(rng, (2, M, K)), _ints(rng, (P, M))
    o = G.offsets_of([n // 2, n - n // 2])
    y, dx = torch.full((P, M), 77.0, device=gpu), torch.full((P, K), 55.0, device=gpu)
    xd, wd, dyd = (_dev(v, "bf16", gpu) for v in (x, w, dy))
    assert ops.grouped_gemm(xd, wd, off, out=y) is y
    assert ops.grouped_gemm_dgrad(dyd, wd, off, out=dx) is dx
    assert torch.all(y[n:] == 77.0) and torch.all(dx[n:] == 55.0)
    _equal(y[:n], G.forward(x, w, o)[:n], "f32")
    _equal(dx[:n], G.dgrad(dy, w, o)[:n], "f32")
    wc, ws = _mx_ints(rng, (2, M, K))
    y.fill_(77.0)
    ops.grouped_gemm(xd, _stack(wc, ws, gpu), off, out=y)
    assert torch.all(y[n:] == 77.0)
    _equal(y[:n], G.forward(x, G.mx_decode(wc, ws), o)[:n], "f32")


def test_results_at_element_alignment(gpu):
    """Results that start between 16-byte boundaries, rows of odd length, neighbours unwritten."""
    import torch
    from block_lut_amd import ops
    P, K = 21, 64
    rng = np.random.default_rng(4)
    off, o = _off([20, 1], gpu), G.offsets_of([20, 1])
    x = _ints(rng, (P, K))
    for M in (24, 13):
        wc, ws = _mx_ints(rng, (2, M, K))
        for dtype, shift in (("bf16", 1), ("f32", 1), ("bf16", 8)):
            buf = torch.full((P * M + 32,), 99.0, device=gpu, dtype=_t(dtype))
            y = buf[shift:shift + P * M].view(P, M)
            ops.grouped_gemm(_dev(x, "bf16", gpu), _stack(wc, ws, gpu), off, out=y)
            _equal(y, G.forward(x, G.mx_decode(wc, ws), o), dtype)
            assert torch.all(buf[:shift] == 99.0) and torch.all(buf[shift + P * M:] == 99.0)
    w, dy = _ints(rng, (2, 24, K)), _ints(rng, (P, 24))
    for shift in (1, 4):
        buf = torch.full((2 * 24 * K + 32,), 99.0, device=gpu)
        ops.grouped_gemm_wgrad(_dev(dy, "f16", gpu), _dev(x, "f16", gpu), off, out=buf[shift:shift + 2 * 24 * K].view(2, 24, K))
        _equal(buf[shift:shift + 2 * 24 * K].view(2, 24, K), G.wgrad(dy, x, o, 2), "f32")
        assert torch.all(buf[:shift] == 99.0) and torch.all(buf[shift + 2 * 24 * K:] == 99.0)


def test_offsets_outside_the_rows_are_clamped(gpu):
    import torch
    from block_lut_amd import ops
    P, M, K = 50, 64, 96
    rng = np.random.default_rng(9)
    x, w, dy = _ints(rng, (P, K)), _ints(rng, (3, M, K)), _ints(rng, (P, M))
    o = np.array([-5, 20, 60, 1000], np.int32)
    off = torch.from_numpy(o).to(gpu)
    xd, wd, dyd = (_dev(v, "bf16", gpu) for v in (x, w, dy))
    _equal(ops.grouped_gemm(xd, wd, off), G.forward(x, w, o), "bf16")
    _equal(ops.grouped_gemm_dgrad(dyd, wd, off), G.dgrad(dy, w, o), "bf16")
    _equal(ops.grouped_gemm_wgrad(dyd, xd, off, out_dtype=torch.float32), G.wgrad(dy, x, o, 3), "f32")


def test_no_rows(gpu):
    import torch
    from block_lut_amd import ops
    off = torch.zeros(4, dtype=torch.int32, device=gpu)
    w = torch.ones(3, 16, 32, device=gpu, dtype=torch.bfloat16)
    x, dy = w.new_ones(0, 32), w.new_ones(0, 16)
    assert tuple(ops.grouped_gemm(x, w, off).shape) == (0, 16)
    assert tuple(ops.grouped_gemm_dgrad(dy, w, off).shape) == (0, 32)
    dw = torch.full((3, 16, 32), 5.0, device=gpu)
    ops.grouped_gemm_wgrad(dy, x, off, out=dw)
    assert torch.all(dw == 0)


# ---------------------------------------------------------------- long sizes

def test_offsets_past_32_bits(gpu):
    """Matrices and rows of more than 2^32 bytes, results too: the last expert's and the last
    rows' against 64-bit sums over a sample."""
    import torch
    from block_lut_amd import ops
    E, M, K = 40, 4096, 16384                    # 5.4 GB of bf16
    counts = [0] * E
    counts[0], counts[E - 2], counts[E - 1] = 3, 2, 30
    off, P = _off(counts, gpu), 35
    gen = torch.Generator(device=gpu).manual_seed(1)
    w = torch.empty((E, M, K), dtype=torch.bfloat16, device=gpu)
    for e in range(E):
        w[e] = torch.randint(-3, 4, (M, K), generator=gen, device=gpu)
    x = torch.randint(-3, 4, (P, K), generator=gen, device=gpu).to(torch.bfloat16)
    dy = torch.randint(-3, 4, (P, M), generator=gen, device=gpu).to(torch.bfloat16)
    y = ops.grouped_gemm(x, w, off, out_dtype=torch.float32)
    dx = ops.grouped_gemm_dgrad(dy, w, off, out_dtype=torch.float32)
    for e, a, b in ((0, 0, 3), (E - 2, 3, 5), (E - 1, 5, 35)):
        assert torch.equal(y[a:b].double(), x[a:b].double() @ w[e].double().T)
        assert torch.equal(dx[a:b].double(), dy[a:b].double() @ w[e].double())
    del w
    dw = ops.grouped_gemm_wgrad(dy, x, off)
    assert torch.equal(dw[E - 1].double(), (dy[5:].double().T @ x[5:].double()))
    assert torch.count_nonzero(dw[5]) == 0
    del dw
    rows = (1 << 31) // 16384 + 77               # 4.3 GB of rows
    x = torch.zeros((rows, K), dtype=torch.bfloat16, device=gpu)
    x[-40:] = torch.randint(-3, 4, (40, K), generator=gen, device=gpu).to(torch.bfloat16)
    w = torch.randint(-3, 4, (2, 24, K), generator=gen, device=gpu).to(torch.bfloat16)
    off = torch.tensor([0, rows - 33, rows], dtype=torch.int32, device=gpu)
    y = ops.grouped_gemm(x, w, off, out_dtype=torch.float32)
    assert torch.equal(y[-33:].double(), x[-33:].double() @ w[1].double().T)
    assert torch.equal(y[-40:-33].double(), x[-40:-33].double() @ w[0].double().T)
    dy = torch.randint(-3, 4, (rows, 24), generator=gen, device=gpu).to(torch.bfloat16)
    dw = ops.grouped_gemm_wgrad(dy, x, off, out_dtype=torch.float32)
    assert torch.equal(dw[1].double(), dy[-33:].double().T @ x[-33:].double())
    assert torch.equal(dw[0].double(), dy[-40:-33].double().T @ x[-40:-33].double())
    dx = ops.grouped_gemm_dgrad(dy, w, off)
    assert torch.equal(dx[-33:].double(), (dy[-33:].double() @ w[1].double()).to(torch.bfloat16).double())


# --------------------------------------------------- streams, graphs, autograd

def _case(gpu, seed=0, P=300, M=136, K=200):
    rng = np.random.default_rng(seed)
    counts = [P // 3, 0, P - P // 3 - 5]
    return (counts, _ints(rng, (P, K)), _ints(rng, (3, M, K)), _ints(rng, (P, M)))


def test_two_streams_at_once(gpu):
    import torch
    from block_lut_amd import ops
    cases = [_case(gpu, s, P=900) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in cases]
    dev = [(_off(c, gpu), *(_dev(v, "bf16", gpu) for v in (x, w, dy))) for c, x, w, dy in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                off, x, w, dy = dev[i]
                got[i].append((ops.grouped_gemm(x, w, off), ops.grouped_gemm_dgrad(dy, w, off),
                               ops.grouped_gemm_wgrad(dy, x, off)))
    torch.cuda.synchronize()
    for (c, x, w, dy), all_ in zip(cases, got):
        o = G.offsets_of(c)
        for y, dx, dw in all_:
            _equal(y, G.forward(x, w, o), "bf16")
            _equal(dx, G.dgrad(dy, w, o), "bf16")
            _equal(dw, G.wgrad(dy, x, o, 3), "bf16")


@pytest.mark.parametrize("P", [12, 300])
def test_captured_and_replayed(gpu, P):
    """A graph of every product, replayed with new values and new group sizes in its buffers,
    the eager calls between the replays."""
    import torch
    from block_lut_amd import ops
    counts, x, w, dy = _case(gpu, P, P=P)
    off, xd, wd, dyd = _off(counts, gpu), *(_dev(v, "bf16", gpu) for v in (x, w, dy))
    rng = np.random.default_rng(3)
    st = _stack(*_mx_ints(rng, (3, 136, 224)), gpu)
    x2 = _dev(_ints(rng, (P, 224)), "bf16", gpu)

    def every():
        codes, scales = ops.mxfp4_encode(x2)
        return [ops.grouped_gemm(xd, wd, off), ops.grouped_gemm_dgrad(dyd, wd, off), ops.grouped_gemm_wgrad(dyd, xd, off),
                ops.grouped_gemm(x2, st, off), ops.grouped_gemm(codes, st, off, x_scales=scales), ops.gemv(st, x2, 1)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        every()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = every()
    for i in range(3):
        c = [i, P - 2 * i - 3, i + 1]
        off.copy_(_off(c, gpu))
        xd.copy_(_dev(_ints(rng, x.shape), "bf16", gpu))
        x2.copy_(_dev(_ints(rng, tuple(x2.shape)), "bf16", gpu))
        g.replay()
        eager = every()
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b)
        _equal(held[0], G.forward(xd.double().cpu().numpy(), w, G.offsets_of(c)), "bf16")


def test_same_results_every_time(gpu):
    import torch
    from block_lut_amd import ops
    gen = torch.Generator(device=gpu).manual_seed(5)
    x = torch.randn(700, 512, generator=gen, device=gpu).bfloat16()
    w = torch.randn(4, 264, 512, generator=gen, device=gpu).bfloat16()
    dy = torch.randn(700, 264, generator=gen, device=gpu).bfloat16()
    off = _off([300, 1, 0, 390], gpu)
    first = (ops.grouped_gemm(x, w, off), ops.grouped_gemm_dgrad(dy, w, off), ops.grouped_gemm_wgrad(dy, x, off))
    for _ in range(5):
        again = (ops.grouped_gemm(x, w, off), ops.grouped_gemm_dgrad(dy, w, off), ops.grouped_gemm_wgrad(dy, x, off))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_linear_gradients(gpu, dtype):
    """Against the formulas and against differences: the loss is linear in x and in w, so a
    whole-number step of one entry changes it by that entry's gradient exactly."""
    import torch
    from block_lut_amd import ops
    counts, x, w, dy = _case(gpu, 8, P=60, M=24, K=40)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    xd, wd, dyd = (_dev(v, dtype, gpu) for v in (x, w, dy))
    xd.requires_grad_()
    wd.requires_grad_()
    y = ops.grouped_linear(xd, wd, off)
    _equal(y.detach(), G.forward(x, w, o), dtype)
    y.backward(dyd)
    _equal(xd.grad, G.dgrad(dy, w, o), dtype)
    _equal(wd.grad, G.wgrad(dy, x, o, 3), dtype)

    def loss(xv, wv):
        out = ops.grouped_gemm(_dev(xv, dtype, gpu), _dev(wv, dtype, gpu), off, out_dtype=torch.float32)
        return float((out.double().cpu().numpy() * dy).sum())

    base = loss(x, w)
    for p, k in ((0, 0), (o[1] - 1, 39), (o[3] - 1, 17), (59, 3)):
        x1 = x.copy()
        x1[p, k] += 1
        assert loss(x1, w) - base == G.dgrad(dy, w, o)[p, k]
    for e, m, k in ((0, 0, 0), (1, 5, 5), (2, 23, 39)):
        w1 = w.copy()
        w1[e, m, k] += 1
        assert loss(x, w1) - base == G.wgrad(dy, x, o, 3)[e, m, k]


def test_linear_expanded_gradient_and_single_inputs(gpu):
    import torch
    from block_lut_amd import ops
    counts, x, w, dy = _case(gpu, 9, P=40, M=24, K=40)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    one = np.ones((40, 24))
    xd, wd = _dev(x, "bf16", gpu).requires_grad_(), _dev(w, "bf16", gpu)
    ops.grouped_linear(xd, wd, off).sum().backward()             # an expanded gradient
    _equal(xd.grad, G.dgrad(one, w, o), "bf16")
    assert wd.grad is None
    xd, wd = _dev(x, "bf16", gpu), _dev(w, "bf16", gpu).requires_grad_()
    ops.grouped_linear(xd, wd, off).sum().backward()
    _equal(wd.grad, G.wgrad(one, x, o, 3), "bf16")
    assert xd.grad is None
    # shared leaves: the same matrices in two calls add up
    xd = _dev(x, "bf16", gpu)
    wd.grad = None
    (ops.grouped_linear(xd, wd, off).sum() + ops.grouped_linear(xd, wd, off).sum()).backward()
    _equal(wd.grad, 2 * G.wgrad(one, x, o, 3), "bf16")


def test_linear_step_captured(gpu):
    """Forward and backward in one graph, replayed with new rows."""
    import torch
    from block_lut_amd import ops
    counts, x, w, dy = _case(gpu, 10, P=70, M=24, K=40)
    off, o = _off(counts, gpu), G.offsets_of(counts)
    xd, wd, dyd = (_dev(v, "bf16", gpu) for v in (x, w, dy))
    xd.requires_grad_()
    wd.requires_grad_()

    def step():
        return torch.autograd.grad(ops.grouped_linear(xd, wd, off), (xd, wd), dyd)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dx, dw = step()
    rng = np.random.default_rng(12)
    for _ in range(3):
        x1 = _ints(rng, x.shape)
        with torch.no_grad():
            xd.copy_(_dev(x1, "bf16", gpu))
        g.replay()
        torch.cuda.synchronize()
        _equal(dx, G.dgrad(dy, w, o), "bf16")
        _equal(dw, G.wgrad(dy, x1, o, 3), "bf16")


# ---------------------------------------------------------------- refusals

def test_shapes_and_types_are_refused(gpu):
    import torch
    from block_lut_amd import ops
    x = torch.zeros(10, 64, device=gpu, dtype=torch.bfloat16)
    w = torch.zeros(3, 16, 64, device=gpu, dtype=torch.bfloat16)
    dy = torch.zeros(10, 16, device=gpu, dtype=torch.bfloat16)
    off = torch.zeros(4, device=gpu, dtype=torch.int32)
    st = _stack(np.zeros((3, 16, 32), np.uint8), np.zeros((3, 16, 2), np.uint8), gpu)
    scales = torch.zeros(10, 2, device=gpu, dtype=torch.uint8)
    codes = torch.zeros(10, 32, device=gpu, dtype=torch.uint8)
    for bad in (lambda: ops.grouped_gemm(x[:, :32].contiguous(), w, off), lambda: ops.grouped_gemm(x.t(), w, off),
                lambda: ops.grouped_gemm(x, w.transpose(1, 2), off), lambda: ops.grouped_gemm(x, w, off[:3]),
                lambda: ops.grouped_gemm(x, w, off, x_scales=scales), lambda: ops.grouped_gemm(x[0], w, off),
                lambda: ops.grouped_gemm(x, w, off, out=torch.zeros(10, 8, device=gpu)),
                lambda: ops.grouped_gemm(codes, st, off, x_scales=scales[:5]),
                lambda: ops.grouped_gemm(codes[:, :16].contiguous(), st, off, x_scales=scales),
                lambda: ops.grouped_gemm_dgrad(x, w, off), lambda: ops.grouped_gemm_wgrad(dy, x[:5], off),
                lambda: ops.grouped_gemm_wgrad(dy, x, off[:1]), lambda: ops.grouped_gemm(x, w[0], off),
                lambda: ops.grouped_gemm(x, w, off.cpu())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.grouped_gemm(x.half(), w, off), lambda: ops.grouped_gemm(x, w, off.long()),
                lambda: ops.grouped_gemm(codes, st, off), lambda: ops.grouped_gemm(x, st, off, x_scales=scales),
                lambda: ops.grouped_gemm(x, w, off, out=torch.zeros(10, 16, device=gpu), out_dtype=torch.bfloat16),
                lambda: ops.grouped_gemm(x, w, off, out_dtype=torch.float64),
                lambda: ops.grouped_gemm_dgrad(dy.float(), w, off), lambda: ops.grouped_gemm_wgrad(dy, x.half(), off)):
        with pytest.raises(TypeError):
            bad()
    from block_lut_amd._native import LutMoeError
    for bad in (lambda: ops.grouped_gemm(x, w, off, out_dtype=torch.float16),
                lambda: ops.grouped_gemm(x, st, off, out_dtype=torch.float16),
                lambda: ops.grouped_gemm(x[:, :60].contiguous(), w[:, :, :60].contiguous(), off),
                lambda: ops.gemv(st, x.float())):
        with pytest.raises(LutMoeError):
            bad()


# --------------------------------------------------------------- as one run

def test_moe_block_of_mxfp4_experts(gpu):
    """Router, permutation, quantised rows, both products and the combine, against the same
    steps in 64 bits from the same quantised weights and rows."""
    import torch
    from block_lut_amd import ops
    from block_lut_amd.formats import MXFP4Stack
    T, H, I, E, k = 37, 256, 96, 6, 2
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(T, H, generator=gen).bfloat16().to(gpu)
    w13 = (torch.randn(E, 2 * I, H, generator=gen) * 0.05).bfloat16().to(gpu)
    w2 = (torch.randn(E, H, I, generator=gen) * 0.05).bfloat16().to(gpu)
    logits = torch.randn(T, E, generator=gen).to(gpu)
    s13, s2 = MXFP4Stack(*ops.mxfp4_encode(w13)), MXFP4Stack(*ops.mxfp4_encode(w2))
    topw, ids = ops.route_topk(logits, k)
    offsets, perm, inv, _ = ops.permute(ids, E)
    rows = x[(perm // k).long()]
    for x4 in (False, True):
        def product(r, st, out):
            if not x4:
                return ops.grouped_gemm(r, st, offsets, out_dtype=out)
            c, b = ops.mxfp4_encode(r)
            return ops.grouped_gemm(c, st, offsets, x_scales=b, out_dtype=out)

        h = product(rows, s13, torch.float32)
        act = (torch.nn.functional.silu(h[:, :I]) * h[:, I:]).bfloat16()
        y = product(act, s2, torch.float32)
        out = (y[inv.long()].view(T, k, H) * topw[..., None]).sum(1).double().cpu().numpy()

        o = offsets.cpu().numpy()
        d13, d2 = (G.mx_decode(s.codes.cpu().numpy(), s.scales.cpu().numpy()) for s in (s13, s2))
        q = (lambda v: G.mx_decode(*G.mx_encode(v))) if x4 else (lambda v: v)
        r64, a64 = q(rows.double().cpu().numpy()), q(act.double().cpu().numpy())
        h64 = G.forward(r64, d13, o)
        _within(h, h64, G.forward(np.abs(r64), np.abs(d13), o), H, "f32")
        y64 = G.forward(a64, d2, o)
        mags = G.forward(np.abs(a64), np.abs(d2), o)
        _within(y, y64, mags, I, "f32")
        w64, at = topw.double().cpu().numpy()[..., None], inv.cpu().numpy()
        ref = (y64[at].reshape(T, k, H) * w64).sum(1)
        tol = ((G.tolerance(y64, mags, I, "f32") + 4 * 2.0 ** -24 * np.abs(y64))[at].reshape(T, k, H) * w64).sum(1)
        assert np.all(np.abs(out - ref) <= tol)


def test_dense_experts_trained_then_quantised(gpu):
    """A gradient step of dense experts through two grouped layers, then the new matrices
    encoded and served: gradients against 64-bit ones of the same values."""
    import torch
    from block_lut_amd import ops
    from block_lut_amd.formats import MXFP4Stack
    counts = [40, 0, 25]
    off, o, P = _off(counts, gpu), G.offsets_of(counts), 65
    rng = np.random.default_rng(20)
    x, w1, w2, dy = _ints(rng, (P, 64)), _ints(rng, (3, 96, 64)), _ints(rng, (3, 32, 96)), _ints(rng, (P, 32))
    w1d, w2d = _dev(w1, "bf16", gpu).requires_grad_(), _dev(w2, "bf16", gpu).requires_grad_()
    h = ops.grouped_linear(_dev(x, "bf16", gpu), w1d, off)
    hr = torch.relu(h)
    ops.grouped_linear(hr, w2d, off).backward(_dev(dy, "bf16", gpu))
    h64 = G.round_to(G.forward(x, w1, o), "bf16").double().numpy()
    a64 = np.maximum(h64, 0)
    _equal(w2d.grad, G.wgrad(dy, a64, o, 3), "bf16")
    g64 = G.round_to(G.dgrad(dy, w2, o), "bf16").double().numpy() * (h64 > 0)
    dw1 = G.wgrad(g64, x, o, 3)
    mags = G.wgrad(np.abs(g64), np.abs(x), o, 3)
    _within(w1d.grad, dw1, mags, max(counts), "bf16")
    new = (w1d - w1d.grad * 2.0 ** -9).detach()
    codes, scales = ops.mxfp4_encode(new)
    c, s = G.mx_encode(new.double().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(scales.cpu().numpy(), s)
    y = ops.grouped_gemm(_dev(x, "bf16", gpu), MXFP4Stack(codes, scales), off, out_dtype=torch.float32)
    v = G.mx_decode(c, s)
    _within(y, G.forward(x, v, o), G.forward(np.abs(x), np.abs(v), o), 64, "f32")
