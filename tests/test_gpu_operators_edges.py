"""The operators on feature rows where their first tests did not look: infinities in the backward direction, buffers that
the C interface allows to be one, sizes past one launch, and what torch's autograd sees.

u = 2^-24 is float32's unit roundoff.  Results that two calls compute from the same numbers in the same order are
compared bit by bit."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mdescriptor_amd as mdx
from mdescriptor_amd import _hip

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
KINDS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


def randn(seed: int, *shape: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def call(name: str, args: ctypes.Structure) -> None:
    """An entry point of the C interface on the current stream."""

    lib = _hip.load_library()
    status = getattr(lib, "mdx_hip_" + name)(0, ctypes.byref(args), torch.cuda.current_stream().cuda_stream)
    assert status == _hip.MDX_OK, lib.mdx_hip_last_error(None).decode()


# --------------------------------------------------- gradients of the norm

# columns that take 16, 32 and 64 lanes a row, and 128: 16, 8, 4, 4 and 2 rows side by side
WIDTHS = [100, 200, 500, 1000, 1500]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [1, 5, 67])
def test_norm_backward_of_an_infinite_gradient_in_the_last_row(dtype, width, rows):
    """Rows that do not fill a workgroup: the gain's gradient is infinite in that column, as its sum is, and the other
    columns and rows are what they are without it."""

    t, grad = randn(1, rows, width, dtype=dtype), randn(2, rows, width, dtype=dtype)
    t[-1, 3] = 0.5
    gain = randn(3, width)
    rstd = (1.0 / torch.sqrt(t.double().square().mean(dim=1) + 1e-5)).float()
    plain_rows, plain_gain = mdx.rms_norm_backward(grad, t, gain, rstd)
    for sign in (1.0, -1.0):
        grad[-1, 3] = sign * math.inf
        got, got_gain = mdx.rms_norm_backward(grad, t, gain, rstd)
        assert float(got_gain[3]) == sign * math.inf
        others = torch.arange(width, device="cuda") != 3
        assert torch.equal(got_gain[others], plain_gain[others])
        assert torch.equal(got[:-1], plain_rows[:-1]) and not torch.isfinite(got[-1, 3])


def backward_into(grad, t, gain, rstd, grad_total, grad_x):
    rows, width = t.shape
    lib = _hip.load_library()
    size = lib.mdx_hip_rms_norm_backward_workspace(rows, width)
    workspace = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    grad_gain = torch.empty(width, device="cuda")
    call("rms_norm_backward", _hip.NormBackwardArgs(
        rows=rows, width=width, grad=grad.data_ptr(), grad_pitch=grad.stride(0), t=t.data_ptr(), t_pitch=t.stride(0),
        grad_total=None if grad_total is None else grad_total.data_ptr(),
        grad_total_pitch=0 if grad_total is None else grad_total.stride(0), gain=gain.data_ptr(), rstd=rstd.data_ptr(),
        grad_x=grad_x.data_ptr(), grad_x_pitch=grad_x.stride(0), grad_gain=grad_gain.data_ptr(),
        workspace=workspace.data_ptr(), workspace_bytes=size, dtype=KINDS[t.dtype]))
    return grad_gain


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [*WIDTHS, 3696, 20000])
@pytest.mark.parametrize("rows", [5, 131])
def test_norm_backward_into_its_own_inputs(dtype, width, rows):
    """grad_x may be grad or grad_total: the same bits as into a buffer of its own.  The last row's rstd is so large that
    its float16 result overflows, which must not reach the gain's gradient."""

    t, grad, other = (randn(s, rows, width, dtype=dtype) for s in (4, 5, 6))
    t[-1] = 0.0  # a gain's gradient of zero, whatever the gradient
    gain = 1.0 + 0.1 * randn(7, width)
    rstd = (1.0 / torch.sqrt(t.double().square().mean(dim=1) + 1e-10)).float()
    want = torch.empty_like(t)
    want_gain = backward_into(grad, t, gain, rstd, other, want)
    assert torch.all(torch.isfinite(want_gain)) and (dtype != torch.float16 or torch.isinf(want[-1]).any())
    for name in ("grad", "grad_total"):
        inputs = {"grad": grad.clone(), "grad_total": other.clone()}
        got_gain = backward_into(inputs["grad"], t, gain, rstd, inputs["grad_total"], inputs[name])
        assert torch.equal(inputs[name], want) and torch.equal(got_gain, want_gain)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(37, 100), (1030, 1000), (5, 3696), (3, 20000), (2, 40000)])
@pytest.mark.parametrize("to_codes", [False, True])
def test_norm_whose_total_is_an_input(dtype, shape, to_codes):
    """total may be x or residual: the same bits as into a buffer of its own."""

    rows, width = shape
    x, r, gain = randn(8, rows, width, dtype=dtype), randn(9, rows, width, dtype=dtype), randn(10, width)
    want = mdx.rms_norm(x, gain, residual=r, dtype=CODES if to_codes else None)
    for name in ("x", "residual"):
        inputs = {"x": x.clone(), "residual": r.clone()}
        values, rstd = torch.empty_like(want.values), torch.empty_like(want.rstd)
        scales = torch.empty(rows, -(-width // 128), dtype=torch.uint8, device="cuda")
        values_pitch = width
        if to_codes:
            values_pitch = -(-width // 128) * 128
            values = torch.empty(rows, values_pitch, dtype=torch.uint8, device="cuda").view(CODES)[:, :width]
        call("rms_norm", _hip.NormArgs(
            rows=rows, width=width, x=inputs["x"].data_ptr(), x_pitch=width, residual=inputs["residual"].data_ptr(),
            residual_pitch=width, gain=gain.data_ptr(), values=values.data_ptr(), values_pitch=values_pitch,
            scales=scales.data_ptr(), scales_pitch=scales.stride(0), total=inputs[name].data_ptr(), total_pitch=width,
            rstd=rstd.data_ptr(), eps=1e-6, dtype=KINDS[dtype], out_dtype=3 if to_codes else KINDS[dtype]))
        assert torch.equal(inputs[name], want.total) and torch.equal(rstd, want.rstd)
        assert torch.equal(values.float(), want.values.float())
        if to_codes:
            assert torch.equal(scales, want.scales.contiguous().view(torch.uint8))
