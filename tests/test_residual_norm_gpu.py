"""Residual addition and RMS norm of hidden rows, with outputs in 8 bits and in the input's type, against 64 bits."""
import numpy as np
import pytest
import torch

from raftinfer_b200 import kernels as K
from kv_util import E4M3_VALUES, codes_for, normal, scale_for

pytestmark = pytest.mark.gpu

TYPES = {K.DTYPE_F32: torch.float32, K.DTYPE_BF16: torch.bfloat16, K.DTYPE_F16: torch.float16}
HALF_STEP = {K.DTYPE_F32: 2.0 ** -24, K.DTYPE_BF16: 2.0 ** -8, K.DTYPE_F16: 2.0 ** -11}
EPSILON = 1.0e-6


def reference(x, r, w):
    h = x.double() + (r.double() if r is not None else 0.0)
    return h, h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPSILON) * w.double()


def make(rows, columns, dtype, weight_dtype=K.DTYPE_F32, seed=1):
    t = TYPES[dtype]
    x, r = normal(seed, rows, columns).to(t), (normal(seed + 1, rows, columns) * 3.0).to(t)
    w = (1.0 + 0.2 * normal(seed + 2, columns)).to(TYPES[weight_dtype])
    return x.cuda(), r.cuda(), w.cuda()


# FP32 sums of up to 16384 squares: pieces of a thread in turn, then a tree; the relative error of the sum is below
# (64 + 16) half steps, of the root below half of that, and five more operations follow: 2^-17 in all.
FP32_WORK = 2.0 ** -17


def check_plain(y, dtype, got):
    assert ((got.double() - y).abs() <= y.abs() * (HALF_STEP[dtype] + FP32_WORK) + 2.0 ** -25).all()


def check_codes(y, group, codes, scales):
    """The scale is that of some value within FP32_WORK of the largest; a code is its value rounded to nearest."""
    rows, columns = y.shape
    groups = columns // group if group else 1
    y = y.cpu().numpy().reshape(rows, groups, -1)
    got = codes.view(torch.uint8).cpu().numpy().reshape(y.shape)
    s = scales.cpu().numpy().astype(np.float64)
    largest = np.abs(y).max(-1)
    low = np.vectorize(scale_for)(largest * (1 - FP32_WORK))
    high = np.vectorize(scale_for)(largest * (1 + FP32_WORK))
    assert ((s == low) | (s == high)).all()
    scaled = y / s[..., None]
    off = np.abs(E4M3_VALUES[got] - scaled)
    # half a step of an e4m3 value (2^-4 of it, 2^-10 below its smallest normal), and the FP32 work in front
    assert (off <= np.maximum(np.abs(scaled) * 2.0 ** -4, 2.0 ** -10) + np.abs(scaled) * FP32_WORK).all()
    exact = got == codes_for(scaled)
    assert exact.mean() > 0.999


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,columns", [(1, 8), (1, 4096), (3, 24), (7, 1000), (130, 2056), (5, 16384), (1000, 512)])
def test_output_in_the_input_type(dtype, rows, columns):
    x, r, w = make(rows, columns, dtype)
    h, y = reference(x, r, w)
    out, back = torch.full((rows + 1, columns), 7.0, device="cuda", dtype=x.dtype), torch.empty_like(x)
    K.residual_rms_norm(x, r, w, out, None, back, rows, columns, 0, EPSILON, dtype, K.DTYPE_F32, dtype,
                        torch.cuda.current_stream())
    torch.cuda.synchronize()
    check_plain(y, dtype, out[:rows])
    assert (out[rows] == 7.0).all()
    assert torch.equal(back, (x.float() + r.float()).to(x.dtype))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,columns,group", [(1, 4096, 0), (1, 128, 128), (3, 32, 32), (9, 1024, 32), (5, 16384, 128),
                                                (2, 1000, 0), (64, 4096, 128), (3, 8, 0), (300, 640, 32), (1, 16384, 0)])
def test_output_in_8_bits(dtype, rows, columns, group):
    x, r, w = make(rows, columns, dtype, K.DTYPE_BF16)
    h, y = reference(x, r, w)
    codes = torch.full((rows + 1, columns), 0x55, device="cuda", dtype=torch.uint8)
    groups = columns // group if group else 1
    scales = torch.full((rows + 1, groups), 7.0, device="cuda")
    back = torch.empty_like(x)
    K.residual_rms_norm(x, r, w, codes, scales, back, rows, columns, group, EPSILON, dtype, K.DTYPE_BF16, K.DTYPE_E4M3,
                        torch.cuda.current_stream())
    torch.cuda.synchronize()
    check_codes(y, group, codes[:rows], scales[:rows])
    assert (codes[rows] == 0x55).all() and (scales[rows] == 7.0).all()
    assert torch.equal(back, (x.float() + r.float()).to(x.dtype))


def test_without_a_residual_and_without_its_output():
    x, r, w = make(33, 768, K.DTYPE_BF16)
    out, back = torch.empty_like(x), torch.empty_like(x)
    stream = torch.cuda.current_stream()
    for residual, residual_out in ((None, None), (None, back), (r, None)):
        K.residual_rms_norm(x, residual, w, out, None, residual_out, 33, 768, 0, EPSILON, K.DTYPE_BF16, K.DTYPE_F32,
                            K.DTYPE_BF16, stream)
        torch.cuda.synchronize()
        check_plain(reference(x, residual, w)[1], K.DTYPE_BF16, out)
    assert torch.equal(back, x)


@pytest.mark.parametrize("columns", [256, 4096, 16384])
def test_in_place(columns):
    """residual_out is the residual or the input itself, and the output replaces the input."""
    x, r, w = make(70, columns, K.DTYPE_BF16)
    h, y = reference(x, r, w)
    stream = torch.cuda.current_stream()
    x1, r1 = x.clone(), r.clone()
    K.residual_rms_norm(x1, r1, w, x1, None, r1, 70, columns, 0, EPSILON, K.DTYPE_BF16, K.DTYPE_F32, K.DTYPE_BF16, stream)
    torch.cuda.synchronize()
    check_plain(y, K.DTYPE_BF16, x1)
    assert torch.equal(r1, (x.float() + r.float()).bfloat16())


def test_rows_of_zeros_and_of_extremes():
    columns = 512
    x = torch.zeros(4, columns, device="cuda")
    x[1] = 1e-25
    x[2] = 1e15
    x[3, 7] = 1e18
    w = torch.ones(columns, device="cuda")
    codes, scales = torch.empty(4, columns, device="cuda", dtype=torch.uint8), torch.empty(4, 4, device="cuda")
    K.residual_rms_norm(x, None, w, codes, scales, None, 4, columns, 128, EPSILON, K.DTYPE_F32, K.DTYPE_F32, K.DTYPE_E4M3,
                        torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert (codes[0] == 0).all() and (scales[0] == 2.0 ** -100).all()
    check_codes(reference(x[1:], None, w)[1], 128, codes[1:], scales[1:])


@pytest.mark.parametrize("dtype", [K.DTYPE_F32, K.DTYPE_BF16])
def test_magnitudes_whose_squares_leave_32_bits(dtype):
    """Rows around 1e25 and 1e-25 (with no epsilon), and one with an infinity: its finite columns become zeros."""
    columns, stream = 520, torch.cuda.current_stream()
    x = normal(3, 3, columns)
    x[0] *= 1e25
    x[1] *= 1e-25
    x[2, 9] = float("inf")
    x = x.to(TYPES[dtype]).cuda()
    w = (1.0 + 0.2 * normal(4, columns)).cuda()
    out, codes = torch.empty_like(x), torch.empty(3, columns, device="cuda", dtype=torch.uint8)
    scales = torch.empty(3, 1, device="cuda")
    K.residual_rms_norm(x, None, w, out, None, None, 3, columns, 0, 0.0, dtype, K.DTYPE_F32, dtype, stream)
    K.residual_rms_norm(x, None, w, codes, scales, None, 3, columns, 0, 0.0, dtype, K.DTYPE_F32, K.DTYPE_E4M3, stream)
    torch.cuda.synchronize()
    h = x[:2].double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True)) * w.double()
    check_plain(y, dtype, out[:2])
    check_codes(y, 0, codes[:2], scales[:2])
    assert torch.isnan(out[2]).nonzero().flatten().tolist() == [9]
    assert (out[2, :9] == 0).all() and (out[2, 10:] == 0).all()


def test_codes_are_the_value_rounded_once():
    """Half a million values, outlier columns among them: every code is that of the 64-bit value, and so is every scale."""
    rows, columns, stream = 256, 2048, torch.cuda.current_stream()
    spread = torch.exp(0.5 * normal(5, columns)) * torch.where(normal(6, columns) > 3.0, 30.0, 1.0)
    x, r = (normal(7, rows, columns) * spread).bfloat16().cuda(), (normal(8, rows, columns) * spread).bfloat16().cuda()
    w = (1.0 + 0.2 * normal(9, columns)).cuda()
    h = x.double() + r.double()
    y = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPSILON) * w.double()).cpu().numpy().reshape(rows, -1, 128)
    codes, scales = torch.empty(rows, columns, device="cuda", dtype=torch.uint8), torch.empty(rows, columns // 128, device="cuda")
    K.residual_rms_norm(x, r, w, codes, scales, None, rows, columns, 128, EPSILON, K.DTYPE_BF16, K.DTYPE_F32, K.DTYPE_E4M3,
                        stream)
    torch.cuda.synchronize()
    want = np.vectorize(scale_for)(np.abs(y).max(-1))
    assert np.array_equal(scales.cpu().numpy(), want)
    assert np.array_equal(codes.cpu().numpy().reshape(y.shape), codes_for(y / want[..., None]))


def test_a_not_a_number_stays_in_its_row():
    x, r, w = make(4, 256, K.DTYPE_F32)
    x[2, 5] = float("nan")
    out = torch.empty_like(x)
    K.residual_rms_norm(x, r, w, out, None, None, 4, 256, 0, EPSILON, K.DTYPE_F32, K.DTYPE_F32, K.DTYPE_F32,
                        torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert torch.isnan(out[2]).all() and torch.isfinite(out[[0, 1, 3]]).all()


def test_captured_and_replayed():
    x, r, w = make(16, 4096, K.DTYPE_BF16)
    out, stream, graph = torch.zeros_like(x), torch.cuda.current_stream(), torch.cuda.CUDAGraph()
    call = lambda: K.residual_rms_norm(x, r, w, out, None, None, 16, 4096, 0, EPSILON, K.DTYPE_BF16, K.DTYPE_F32,
                                       K.DTYPE_BF16, stream)
    call()
    torch.cuda.synchronize()
    eager = out.clone()
    with torch.cuda.graph(graph, stream=stream):
        call()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
