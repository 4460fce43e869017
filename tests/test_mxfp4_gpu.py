"""MXFP4 quantisation against its definition in 64 bits, on the B200.

The scale is a power of two taken from the largest magnitude's exponent, so the codes have one
right value each: every comparison is exact.
"""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA device required"),
]

from loraforge_b200.ops.mxfp4 import MxTensor, mxfp4_dequantize, mxfp4_quantize  # noqa: E402

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantized64(x):
    """(codes, scales, values) of a float64 array [..., K] by the distance to each level."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    ok = np.isfinite(b).all(-1)
    top = np.abs(np.where(ok[..., None], b, 0.0)).max(-1)
    exponent = np.where(top > 0, np.maximum(np.frexp(top)[1] - 1 - 2, -127), -127)
    v = np.where(ok[..., None], b, 0.0) / np.ldexp(1.0, exponent)[..., None]
    far = np.abs(np.abs(v)[..., None] - LEVELS)
    near = far == far.min(-1, keepdims=True)  # one level, or two on a tie: then the even code
    code = np.where(near.sum(-1) > 1, (near * (np.arange(8) % 2 == 0)).argmax(-1), near.argmax(-1))
    values = np.where(ok[..., None], np.sign(v) * LEVELS[code] * np.ldexp(1.0, exponent)[..., None], np.nan)
    return code, np.where(ok, exponent + 127, 255), values.reshape(x.shape)


def check(x, q):
    code, scales, values = quantized64(x.double().cpu().numpy())
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    pairs = q.codes.cpu().numpy()
    got = np.stack((pairs & 15, pairs >> 4), -1).reshape(x.shape)
    assert np.array_equal(got & 7, code.reshape(x.shape))
    for dtype in (torch.float32, torch.bfloat16):
        np.testing.assert_array_equal(mxfp4_dequantize(q, dtype).double().cpu().numpy(), values)
    half = torch.from_numpy(values).to(torch.float16)
    assert torch.equal(mxfp4_dequantize(q, torch.float16).cpu().nan_to_num(1.0), half.nan_to_num(1.0))


@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (64, 4096), (1003, 96), (5, 7, 160), (32,), (2, 2, 2, 32), (0, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_random_values(shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(len(shape) + shape[-1])
    x = torch.randn(shape, generator=g, device="cuda")
    x = (x * torch.exp2(torch.randint(-6, 7, shape, generator=g, device="cuda").float())).to(dtype)
    check(x, mxfp4_quantize(x))


def test_ties_edges_and_special_blocks():
    inf = math.inf
    rows = [
        [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0],          # every tie
        [-0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -7.9],  # and over 6
        [0.0] * 8,
        [2.0**-149, 2.0**-130, 2.0**-127, 0.0, -(2.0**-126), 2.0**-128, 0.0, 0.0],  # subnormal
        [3.4028234663852886e38, 1e38, -2e38, 0.0, 1.0, 1e37, 2.0**127, 2.0**125],   # the largest
        [inf, 1.0, 2.0, 3.0, 0.0, 0.0, 0.0, 0.0],
        [math.nan, 1.0, 2.0, 3.0, 0.0, 0.0, 0.0, 0.0],
        [-0.0, -1e-30, 1.0, -1.0, 1.9999999, 2.0, 3.9999998, 4.0],
    ]
    x = torch.zeros(len(rows), 64, device="cuda")  # the second block of each row is zero
    x[:, 5:13] = torch.tensor(rows, dtype=torch.float64).float().cuda()
    q = mxfp4_quantize(x)
    check(x, q)
    assert q.scales[5:7, 0].tolist() == [255, 255] and not q.scales[:, 1].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_a_wider_buffer(dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    wide = torch.randn(37, 203, generator=g, device="cuda").to(dtype)
    for view in (wide[:, :96], wide[:, 1:97], wide[:, 8:200], wide[3:4, 5:69]):
        check(view.contiguous(), mxfp4_quantize(view))


def test_more_values_than_one_pass_of_the_grid():
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(3000, 1024, generator=g, device="cuda").bfloat16()
    check(x, mxfp4_quantize(x))


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    with pytest.raises(TypeError, match="torch.Tensor"):
        mxfp4_quantize([1.0])
    with pytest.raises(ValueError, match="dtype"):
        mxfp4_quantize(x.double())
    with pytest.raises(ValueError, match="multiple of 32"):
        mxfp4_quantize(x[:, :40])
    with pytest.raises(ValueError, match="CUDA"):
        mxfp4_quantize(x.cpu())
    with pytest.raises(ValueError, match="unit column stride"):
        mxfp4_quantize(x.T.contiguous().T)
    with pytest.raises(ValueError, match="contiguous"):
        mxfp4_quantize(torch.randn(4, 4, 64, device="cuda")[:, ::2])
    q = mxfp4_quantize(x)
    with pytest.raises(TypeError, match="MxTensor"):
        mxfp4_dequantize(tuple(q))
    with pytest.raises(ValueError, match="dtype"):
        mxfp4_dequantize(q, torch.float64)
    with pytest.raises(ValueError, match="scales"):
        mxfp4_dequantize(MxTensor(q.codes, q.scales[:, :1]))
    with pytest.raises(ValueError, match="codes"):
        mxfp4_dequantize(MxTensor(q.codes[:, 1:], q.scales))


def test_every_scale_byte_and_code():
    # Scales of other programs' tensors: the quantiser itself ends at 252.  What passes a type's range is infinite in it.
    codes = torch.arange(16, device="cuda", dtype=torch.uint8).repeat(256, 2)
    packed = (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous()
    q = MxTensor(packed, torch.arange(256, device="cuda", dtype=torch.int32).to(torch.uint8)[:, None].contiguous())
    levels = torch.tensor([*LEVELS, *(-LEVELS)], dtype=torch.float64, device="cuda").repeat(2)
    powers = torch.tensor([math.ldexp(1.0, i - 127) for i in range(255)] + [math.nan], dtype=torch.float64, device="cuda")
    want = levels * powers[:, None]
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = mxfp4_dequantize(q, dtype)
        assert torch.equal(got.nan_to_num(7.5), want.to(dtype).nan_to_num(7.5)) and torch.equal(got.isnan(), want.isnan())
    assert torch.equal(mxfp4_dequantize(q)[:253].double(), want[:253])  # BF16 holds these exactly
    assert mxfp4_dequantize(q)[253:255].isinf().any(1).all()
