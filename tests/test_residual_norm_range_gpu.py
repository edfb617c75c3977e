"""Residual addition and RMS norm over the whole range of FP32, and codes that are exact in every form, against 64 bits."""
import numpy as np
import pytest
import torch

from raftinfer_b200 import kernels as K
from kv_util import codes_for, normal, scale_for

pytestmark = pytest.mark.gpu

TYPES = {K.DTYPE_F32: torch.float32, K.DTYPE_BF16: torch.bfloat16, K.DTYPE_F16: torch.float16}
HALF_STEP = {K.DTYPE_F32: 2.0 ** -24, K.DTYPE_BF16: 2.0 ** -8, K.DTYPE_F16: 2.0 ** -11}


def reference(x, r, w, epsilon):
    """h is an FP32 sum; what follows is 64-bit arithmetic."""
    h = (x.float() + r.float() if r is not None else x.float()).double()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + epsilon) * w.double()


def run_codes(x, r, w, group, epsilon, dtype, weight_dtype):
    rows, columns = x.shape
    codes = torch.empty(rows, columns, device="cuda", dtype=torch.uint8)
    scales = torch.empty(rows, columns // group if group else 1, device="cuda")
    K.residual_rms_norm(x, r, w, codes, scales, None, rows, columns, group, epsilon, dtype, weight_dtype, K.DTYPE_E4M3,
                        torch.cuda.current_stream())
    torch.cuda.synchronize()
    return codes.cpu().numpy(), scales.cpu().numpy()


def check_exact(x, r, w, group, epsilon, dtype, weight_dtype):
    """Every scale and every code is the 64-bit value's, rounded once."""
    rows, columns = x.shape
    codes, scales = run_codes(x, r, w, group, epsilon, dtype, weight_dtype)
    y = reference(x, r, w, epsilon).cpu().numpy().reshape(rows, scales.shape[1], -1)
    want = np.vectorize(scale_for)(np.abs(y).max(-1))
    assert np.array_equal(scales, want)
    # (a zero keeps its sign)
    assert np.array_equal(codes.reshape(y.shape), codes_for(y / want[..., None]))


def check_plain(x, r, w, epsilon, dtype, weight_dtype):
    """Three roundings of 32 bits (two products and the row's factor) and one to the output's type.  Under the smallest normal
    number a product is off by half of FP32's smallest step, 2^-150, whatever its size: h times the power of two that brings the row
    to about one, that times the weight, and that times the factor, which is then between 0.7 and 1.5.  The first two
    are multiplied by what follows: 2^-150 (1.5 |w| + 1.5 + 1); the output's own half step of the smallest is beside it."""
    rows, columns = x.shape
    out = torch.empty_like(x)
    K.residual_rms_norm(x, r, w, out, None, None, rows, columns, 0, epsilon, dtype, weight_dtype, dtype,
                        torch.cuda.current_stream())
    torch.cuda.synchronize()
    y = reference(x, r, w, epsilon)
    smallest = {K.DTYPE_F32: 0.0, K.DTYPE_BF16: 2.0 ** -134, K.DTYPE_F16: 2.0 ** -25}[dtype]
    smallest = smallest + 2.0 ** -150 * (1.5 * w.double().abs() + 2.5)
    assert ((out.double() - y).abs() <= y.abs() * (HALF_STEP[dtype] + 2.0 ** -22) + smallest).all()


@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("value,weight", [(2.0 ** 127, 2.0), (2.0 ** 126, 4.0), (2.5e38, 1.5), (3.0e38, 1.9375),
                                          (2.0 ** -126, 0.75), (2.0 ** -140, 1.5), (2.0 ** -149, 1.0), (1e-20, 1e-25),
                                          (1e20, 1e-30)])
def test_equal_columns_of_any_magnitude(group, value, weight):
    """y is the weight: the products of value and weight leave FP32's range on either side."""
    x = torch.full((3, 512), value, device="cuda")
    w = torch.full((512,), weight, device="cuda")
    check_exact(x, None, w, group, 0.0, K.DTYPE_F32, K.DTYPE_F32)
    check_plain(x, None, w, 0.0, K.DTYPE_F32, K.DTYPE_F32)


@pytest.mark.parametrize("dtype", [K.DTYPE_F32, K.DTYPE_BF16])
@pytest.mark.parametrize("weight_dtype", [K.DTYPE_F32, K.DTYPE_BF16])
@pytest.mark.parametrize("magnitude", [1e38, 1e30, 1e16, 1e-16, 1e-30, 1e-37, 2.0 ** -130])
def test_rows_at_both_ends_of_the_range(dtype, weight_dtype, magnitude):
    x = (normal(11, 6, 520).clamp(-3, 3) * magnitude).to(TYPES[dtype]).cuda()
    r = (normal(12, 6, 520).clamp(-3, 3) * 0.1 * magnitude).to(TYPES[dtype]).cuda()
    w = (1.5 + 0.5 * normal(13, 520)).to(TYPES[weight_dtype]).cuda()
    check_exact(x, r, w, 0, 0.0, dtype, weight_dtype)
    check_plain(x, r, w, 0.0, dtype, weight_dtype)


@pytest.mark.parametrize("columns", [512, 4096, 16384])
def test_zeros_beside_a_large_value(columns):
    """Zeros, and values that the large one leaves near nothing, beside 3e38 with a weight above one."""
    x = torch.zeros(4, columns, device="cuda")
    x[0, 5] = 3e38
    x[1, columns - 1] = -2.9e38
    x[2, 8], x[2, 9] = 1.7e38, 1e-3
    x[3, 0::2] = 1e30
    w = torch.full((columns,), 1.5, device="cuda")
    for group in (0, 32, 128):
        check_exact(x, None, w, group, 1e-6, K.DTYPE_F32, K.DTYPE_F32)
    check_plain(x, None, w, 1e-6, K.DTYPE_F32, K.DTYPE_F32)


@pytest.mark.parametrize("group", [0, 32, 128])
def test_weights_of_any_magnitude(group):
    """Values far under the row's mean under weights far over one, and the reverse."""
    x = normal(21, 8, 640)
    w = torch.ones(640)
    x[:, 32:64] *= 2.0 ** -100
    w[32:64] = 2.0 ** 100
    x[:, 64:96] *= 2.0 ** -140
    w[64:96] = 2.0 ** 120
    w[96:128] = 2.0 ** -90
    x, w = x.cuda(), (w * (1.0 + 0.1 * normal(22, 640))).cuda()
    check_exact(x, None, w, group, 1e-6, K.DTYPE_F32, K.DTYPE_F32)


def test_values_that_lie_in_the_middle_of_two_codes():
    """Rows of one magnitude with no epsilon: y is plus or minus the weight, and the weights are middles and largest values of a
    scale: ties go to the even code, and a scale does not grow for a value that it just holds."""
    columns = 256
    w = torch.tensor([1.0625, 1.1875, 1.3125, 1.4375, 1.5625, 1.6875, 1.75, 1.0] * 32)
    for i in range(8):
        w[32 * i:32 * i + 32] *= 2.0 ** -i
    for value in (1.0, 3.0, 1e4, 7e-5, 0.1, 5e37, 3e-39):
        sign = torch.where(normal(31, 5, columns) > 0, 1.0, -1.0)
        x = (value * sign).cuda()
        for group in (0, 32, 128):
            check_exact(x, None, w.cuda(), group, 0.0, K.DTYPE_F32, K.DTYPE_F32)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("weight_dtype", [K.DTYPE_F32, K.DTYPE_BF16])
@pytest.mark.parametrize("rows,columns", [(180, 640), (200, 1920), (160, 4096), (40, 16384)])
def test_codes_are_the_value_rounded_once_in_every_form(dtype, weight_dtype, rows, columns):
    """One, two and four pieces a thread, more rows than CTAs and fewer, every type and every kind of scale."""
    x = normal(41, rows, columns).to(TYPES[dtype]).cuda()
    r = (3.0 * normal(42, rows, columns)).to(TYPES[dtype]).cuda()
    w = (1.0 + 0.2 * normal(43, columns)).to(TYPES[weight_dtype]).cuda()
    for group in (0, 32, 128):
        check_exact(x, r, w, group, 1e-6, dtype, weight_dtype)
    check_plain(x, r, w, 1e-6, dtype, weight_dtype)
