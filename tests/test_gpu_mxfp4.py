"""The MXFP4 encoder and its dequantisation on the GPU against the 64-bit definition: codes,
scale bytes and bf16 values exactly."""
import numpy as np
import pytest

import grouped_testutil as G

pytestmark = pytest.mark.gpu
SHAPES = [(1, 32), (1, 2048), (3, 96), (17, 1056), (130, 64), (2, 5, 160), (4099, 32)]


def _dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _check(x):
    import torch
    from block_lut_amd import ops
    codes, scales = ops.mxfp4_encode(x)
    assert codes.dtype == scales.dtype == torch.uint8
    assert tuple(codes.shape) == tuple(x.shape[:-1]) + (x.shape[-1] // 2,)
    assert tuple(scales.shape) == tuple(x.shape[:-1]) + (x.shape[-1] // 32,)
    c, s = G.mx_encode(x.double().cpu().numpy())
    assert np.array_equal(scales.cpu().numpy(), s)
    assert np.array_equal(codes.cpu().numpy(), c)
    return codes, scales


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_encode_matches_the_definition(gpu, shape, dtype):
    import torch
    gen = torch.Generator().manual_seed(len(shape) + shape[-1])
    x = torch.randn(shape, generator=gen) * torch.exp2(torch.randint(-12, 8, shape[:-1] + (1,), generator=gen).float())
    _check(x.to(_dtype(dtype)).to(gpu))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_encode_ties_limits_and_special_values(gpu, dtype):
    """Every halfway value and its neighbours at several scales, zeros of both signs, the
    smallest and largest magnitudes of the type (subnormals too), blocks with infinity and NaN."""
    import torch
    t = _dtype(dtype)
    info = torch.finfo(t)
    mids = np.array([0.0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 6.5, 7, 7.9375])
    rows = []
    top = 14 if dtype == "f16" else 126
    low = -22 if dtype == "f16" else -131
    for e in [low, low + 3, -14, -9, -2, 0, 3, top - 3]:
        for first in (4.0, 7.9375, 6.0):
            r = np.zeros(32)
            r[0] = first
            v = np.concatenate([mids * (1 + d) for d in (0.0, 2.0 ** -7)])[:31]
            r[1:1 + len(v)] = np.minimum(v, first) * np.where(np.arange(len(v)) % 3 == 1, -1, 1)
            rows.append(r * 2.0 ** e)
    special = np.zeros((9, 32))
    special[1] = -0.0
    special[2, 5] = info.max
    special[3, 31] = -info.max
    special[3, 0] = 1.0
    special[4, 7] = info.tiny                     # the smallest normal value
    special[5, 9] = info.smallest_normal * info.eps   # the smallest subnormal one
    special[6, 2], special[6, 3] = np.inf, 1.0
    special[7, 30] = np.nan
    special[8, 0], special[8, 1] = -np.inf, np.nan
    x = torch.from_numpy(np.concatenate([np.array(rows), special])).to(t).to(gpu)
    codes, scales = _check(x)
    assert scales[-3:].flatten().tolist() == [255] * 3 and int(codes[-3:].sum()) == 0
    assert scales[-9:-7].flatten().tolist() == [0, 0]


def test_encode_strided_and_misaligned_inputs_are_refused(gpu):
    import torch
    from block_lut_amd import ops
    from block_lut_amd._native import LutMoeError
    x = torch.zeros(64, 64, device=gpu, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.mxfp4_encode(x.t())
    with pytest.raises(ValueError):
        ops.mxfp4_encode(x[:, :48].contiguous())
    with pytest.raises(LutMoeError):
        ops.mxfp4_encode(x.view(-1)[4:36])         # 8 bytes past an aligned address
    c, s = ops.mxfp4_encode(x[:0])
    assert tuple(c.shape) == (0, 32) and tuple(s.shape) == (0, 2)


def test_dequant_every_byte_at_every_scale(gpu):
    import torch
    from block_lut_amd import ops
    from block_lut_amd.formats import MXFP4Stack
    codes = torch.arange(256, dtype=torch.int32).repeat(256, 1).to(torch.uint8).to(gpu)       # [256, 256]
    scales = torch.arange(256, dtype=torch.int32).view(256, 1).repeat(1, 16).to(torch.uint8).to(gpu)
    v = ops.dequant(MXFP4Stack(codes, scales))[0]
    ref = torch.from_numpy(G.mx_decode(codes.cpu().numpy(), scales.cpu().numpy())).to(torch.bfloat16)
    got = v.cpu()
    assert torch.equal(got.isnan(), ref.isnan())
    ok = ~ref.isnan()
    assert torch.equal(got[ok].view(torch.int16), ref[ok].view(torch.int16))


def test_dequant_of_some_experts_and_the_round_trip(gpu):
    """Values that the format holds come back as they were; experts by range."""
    import torch
    from block_lut_amd import ops
    from block_lut_amd.formats import MXFP4Stack
    rng = np.random.default_rng(3)
    codes = rng.integers(0, 256, (5, 7, 48), dtype=np.uint8)
    codes[..., 0::16] = (codes[..., 0::16] & 0xf0) | 6        # a 4 in every block: the scale is the encoder's
    scales = rng.integers(90, 160, (5, 7, 3), dtype=np.uint8)
    st = MXFP4Stack(torch.from_numpy(codes).to(gpu), torch.from_numpy(scales).to(gpu))
    v = ops.dequant(st)
    assert np.array_equal(v.double().cpu().numpy(), G.mx_decode(codes, scales))
    assert torch.equal(ops.dequant(st, 2, 2), v[2:4])
    c, s = ops.mxfp4_encode(v)
    assert np.array_equal(c.cpu().numpy(), codes) and np.array_equal(s.cpu().numpy(), scales)
    assert st.hbm_bytes_per_expert() == 7 * 48 + 7 * 3


def test_encode_captured(gpu):
    import torch
    from block_lut_amd import ops
    x = torch.randn(37, 320, device=gpu).bfloat16()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.mxfp4_encode(x)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        codes, scales = ops.mxfp4_encode(x)
    for i in range(3):
        x.copy_(torch.randn(37, 320, device=gpu) * 2.0 ** i)
        g.replay()
        c, b = ops.mxfp4_encode(x)
        torch.cuda.synchronize()
        assert torch.equal(codes, c) and torch.equal(scales, b)
