"""Refusals of the MXFP4 and grouped-product entry points: error codes of the C ABI before any
HIP call, exceptions of the Python layer before any library call (no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

import grouped_testutil as G

P = ctypes.c_void_p


@pytest.fixture(scope="module")
def N():
    from block_lut_amd import _native
    _native.lib()
    return _native


def _mx(N, E=2, M=48, K=96, codes=0x10000, tables=0x20001):
    w = N.lutmoe_weights()
    w.format, w.num_experts, w.rows, w.cols = N.FMT_MXFP4, E, M, K
    w.codes, w.tables, w.block_size = codes, tables, 32
    return w


def test_encode_refusals(N):
    f = N.lib().lutmoe_mxfp4_encode
    assert f(P(0x100), 0, -1, P(0x200), P(0x301), None) == N.LUTMOE_EINVAL
    assert f(P(0x100), 3, 4, P(0x200), P(0x301), None) == N.LUTMOE_EINVAL       # dtype
    assert f(None, 0, 4, P(0x200), P(0x301), None) == N.LUTMOE_EINVAL
    assert f(P(0x100), 0, 4, None, P(0x301), None) == N.LUTMOE_EINVAL
    assert f(P(0x100), 0, 4, P(0x200), None, None) == N.LUTMOE_EINVAL
    assert f(P(0x108), 0, 4, P(0x200), P(0x301), None) == N.LUTMOE_EALIGN
    assert f(P(0x100), 0, 4, P(0x204), P(0x301), None) == N.LUTMOE_EALIGN
    assert f(None, 2, 0, None, None, None) == N.LUTMOE_OK


def test_mxfp4_weights_in_the_general_entry_points(N):
    lib = N.lib()
    w = _mx(N, K=80)                                                            # K % 32
    assert lib.lutmoe_dequant(ctypes.byref(w), 0, 1, P(0x100), None) == N.LUTMOE_EINVAL
    w = _mx(N, codes=0x10008)
    assert lib.lutmoe_dequant(ctypes.byref(w), 0, 1, P(0x100), None) == N.LUTMOE_EALIGN
    w = _mx(N)
    assert lib.lutmoe_dequant(ctypes.byref(w), 1, 2, P(0x100), None) == N.LUTMOE_EINVAL
    assert lib.lutmoe_dequant(ctypes.byref(w), 0, 1, P(0x108), None) == N.LUTMOE_EALIGN
    assert lib.lutmoe_gemv(ctypes.byref(w), 2, P(0x100), 1, P(0x200), 0, None) == N.LUTMOE_EINVAL
    assert lib.lutmoe_gemv_ex(ctypes.byref(w), 0, P(0x100), 1, 1, P(0x200), 0, None) == N.LUTMOE_EUNSUPPORTED
    assert lib.lutmoe_gemv(ctypes.byref(w), 0, P(0x100), 1, P(0x201), 0, None) == N.LUTMOE_EALIGN
    assert lib.lutmoe_gemv(ctypes.byref(w), 0, P(0x100), 0, P(0x200), 0, None) == N.LUTMOE_OK
    # the fused layer does not take the format
    d = N.lutmoe_moe_desc()
    d.w13, d.w2 = _mx(N, 4, 256, 256), _mx(N, 4, 256, 128)
    d.hidden, d.inter, d.num_routed = 256, 128, 4
    rc = lib.lutmoe_moe_forward(ctypes.byref(d), P(0x1000), P(0x2000), P(0x3000), 4, 2, P(0x4000), 0, P(0x100000),
                                1 << 30, 0, None)
    assert rc == N.LUTMOE_EUNSUPPORTED


def test_grouped_dense_refusals(N):
    lib = N.lib()

    def fwd(x=0x100, dt=0, w=0x200, off=0x304, E=4, rows=16, M=64, K=64, y=0x400, ydt=0):
        return lib.lutmoe_grouped_gemm(P(x), dt, P(w), P(off), E, rows, M, K, P(y), ydt, 0, None)

    def dg(x=0x100, dt=0, w=0x200, off=0x304, E=4, rows=16, M=64, K=64, y=0x400, ydt=0):
        return lib.lutmoe_grouped_gemm_dgrad(P(x), dt, P(w), P(off), E, rows, M, K, P(y), ydt, 0, None)

    def wg(x=0x100, dt=0, w=0x200, off=0x304, E=4, rows=16, M=64, K=64, y=0x400, ydt=0):
        return lib.lutmoe_grouped_gemm_wgrad(P(x), dt, P(w), P(off), E, rows, M, K, P(y), ydt, None)

    for f in (fwd, dg, wg):
        for bad in (dict(E=0), dict(rows=-1), dict(M=0), dict(K=-8), dict(dt=1), dict(dt=3), dict(ydt=2), dict(ydt=7),
                    dict(dt=2, ydt=0), dict(x=0), dict(w=0), dict(off=0), dict(y=0)):
            assert f(**bad) == N.LUTMOE_EINVAL, (f, bad)
        for bad in (dict(E=4097), dict(M=(1 << 20) + 8), dict(K=(1 << 20) + 8), dict(M=60), dict(K=12)):
            assert f(**bad) == N.LUTMOE_EUNSUPPORTED, (f, bad)
        for bad in (dict(x=0x108), dict(w=0x204), dict(off=0x302), dict(y=0x401), dict(y=0x402, ydt=1)):
            assert f(**bad) == N.LUTMOE_EALIGN, (f, bad)
    assert fwd(rows=0, x=0, y=0, off=0) == N.LUTMOE_OK
    assert dg(rows=0, x=0, y=0, off=0) == N.LUTMOE_OK


def test_grouped_mxfp4_refusals(N):
    lib = N.lib()

    def f(w=None, x=0x100, dt=0, xs=0, off=0x304, rows=16, y=0x400, ydt=0):
        w = _mx(N) if w is None else w
        return lib.lutmoe_grouped_gemm_mxfp4(ctypes.byref(w), P(x), dt, P(xs), P(off), rows, P(y), ydt, 0, None)

    bl4 = _mx(N, K=128, tables=0x20000)
    bl4.format = N.FMT_BL4
    assert f(w=bl4) == N.LUTMOE_EUNSUPPORTED
    assert f(w=_mx(N, E=5000)) == N.LUTMOE_EUNSUPPORTED
    assert f(w=_mx(N, K=48)) == N.LUTMOE_EINVAL
    for bad in (dict(dt=1), dict(dt=2), dict(ydt=2), dict(ydt=3), dict(dt=3), dict(xs=0x501), dict(x=0), dict(y=0),
                dict(off=0), dict(rows=-1)):
        assert f(**bad) == N.LUTMOE_EINVAL, bad
    for bad in (dict(x=0x108), dict(y=0x401), dict(y=0x402, ydt=1), dict(off=0x301)):
        assert f(**bad) == N.LUTMOE_EALIGN, bad
    assert f(rows=0, x=0, y=0, off=0) == N.LUTMOE_OK
    assert lib.lutmoe_grouped_gemm_mxfp4(None, P(0x100), 0, None, P(0x304), 4, P(0x400), 0, 0, None) == N.LUTMOE_EINVAL


def test_host_tensors_and_types_are_refused():
    from block_lut_amd import ops
    from block_lut_amd.formats import MXFP4Stack
    x, w, off = torch.zeros(4, 64).bfloat16(), torch.zeros(2, 8, 64).bfloat16(), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.grouped_gemm(x, w, off)
    with pytest.raises(ValueError):
        ops.grouped_gemm_dgrad(torch.zeros(4, 8).bfloat16(), w, off)
    with pytest.raises(ValueError):
        ops.grouped_gemm_wgrad(torch.zeros(4, 8).bfloat16(), x, off)
    with pytest.raises(ValueError):
        ops.grouped_linear(x, w, off)
    with pytest.raises(TypeError):
        ops.grouped_gemm(x, w.float(), off)
    with pytest.raises(TypeError):
        ops.grouped_gemm(x, object(), off)
    with pytest.raises(TypeError):
        ops.grouped_gemm_dgrad(torch.zeros(4, 8), w, off)
    with pytest.raises(ValueError):
        ops.mxfp4_encode(x)
    with pytest.raises(TypeError):
        ops.mxfp4_encode(torch.zeros(4, 64, dtype=torch.float64))
    with pytest.raises(ValueError):
        MXFP4Stack(torch.zeros(2, 8, 32, dtype=torch.uint8), torch.zeros(2, 8, 2, dtype=torch.uint8))


def test_plain_encoder_against_the_definition():
    """The plain form the GPU tests compare with: hand-worked values."""
    x = np.zeros((3, 32))
    x[0, :8] = [6.0, 0.25, 0.75, -1.25, 1.75, 2.5, -3.5, 5.0]     # scale 1, every tie
    x[1, 0] = -7.9 * 2.0 ** -10                                   # past 6 in its block's scale
    c, s = G.mx_encode(x)
    assert s.tolist() == [[127], [117], [0]]
    nib = np.stack([c & 15, c >> 4], -1).reshape(3, 32)
    assert nib[0, :8].tolist() == [7, 0, 2, 10, 4, 4, 14, 6]
    assert nib[1, 0] == 15
    assert np.array_equal(G.mx_decode(c, s)[0, :8], [6, 0, 1, -1, 2, 2, -4, 4])
