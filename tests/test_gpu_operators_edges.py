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


# ------------------------------------------ sizes past one launch's lanes

# A launch takes 2^28 lanes: what needs more goes in several.  The whole has to be what calls on its parts give.


@pytest.fixture
def freed():
    yield
    torch.cuda.empty_cache()


def by_parts(x, at, call):
    return torch.cat([call(x[:at]), call(x[at:])])


def raw(x: torch.Tensor) -> torch.Tensor:
    return x.contiguous().view(torch.uint8) if x.element_size() == 1 else x


def test_norm_of_more_rows_than_a_launch_takes(freed):
    rows = (1 << 24) + 37  # sixteen lanes each
    x, r, gain = randn(20, rows, 1, dtype=torch.bfloat16), randn(21, rows, 1, dtype=torch.bfloat16), randn(22, 1)
    got = mdx.rms_norm(x, gain, residual=r)
    at = 1 << 23
    parts = [mdx.rms_norm(x[part], gain, residual=r[part]) for part in (slice(0, at), slice(at, None))]
    for name in ("values", "total", "rstd"):
        assert torch.equal(getattr(got, name), torch.cat([getattr(p, name) for p in parts]))
    codes = mdx.rms_norm(x, gain, dtype=CODES)
    for name in ("values", "scales"):
        assert torch.equal(raw(getattr(codes, name)),
                           by_parts(x, at, lambda p: raw(getattr(mdx.rms_norm(p, gain, dtype=CODES), name))))


def test_gradients_of_more_wide_rows_than_a_launch_takes(freed):
    rows, width = (1 << 18) + 3, 16385  # a workgroup of 1,024 lanes each
    g = torch.Generator(device="cuda").manual_seed(23)
    t, grad = (torch.randn(rows, width, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    gain, rstd = randn(24, width), randn(25, rows).abs()
    last = mdx.rms_norm_backward(grad[-5:], t[-5:], gain, rstd[-5:], grad_total=grad[-5:])[0]
    grad_gain = backward_into(grad, t, gain, rstd, grad, grad)
    assert torch.equal(grad[-5:], last) and torch.isfinite(grad_gain).all()


def test_gradient_of_a_gain_of_more_columns_than_a_launch_takes(freed):
    width = (1 << 23) + 77  # 1,024 lanes for 32 columns
    t, grad, gain, rstd = randn(26, 2, width), randn(27, 2, width), randn(28, width), randn(29, 2).abs()
    got = mdx.rms_norm_backward(grad, t, gain, rstd)[1]
    terms = grad.double() * (t.double() * rstd.double()[:, None])
    assert torch.all((got.double() - terms.sum(dim=0)).abs() <= 10 * U * terms.abs().sum(dim=0))
    assert not mdx.rms_norm_backward(grad[:0], t[:0], gain, rstd[:0])[1].any()


def test_quantize_of_more_blocks_than_a_launch_takes(freed):
    x = randn(30, (1 << 24) + 37, 1, dtype=torch.float16)  # sixteen lanes a block
    codes, scales = mdx.quantize_fp8(x)
    for which, whole in enumerate((codes, scales)):
        assert torch.equal(raw(whole), by_parts(x, 1 << 23, lambda p: raw(mdx.quantize_fp8(p)[which])))


@pytest.mark.parametrize("tile, transpose", [(128, False), (128, True), (1, True)])
@pytest.mark.parametrize("shape", [(3, (1 << 25) + 130), ((1 << 22) + 1, 1)])
def test_quantize_of_more_tiles_than_a_launch_takes(freed, tile, transpose, shape):
    """Across (2^18 tiles a launch) and down (32,768)."""

    x = randn(31, *shape, dtype=torch.bfloat16)
    wide = shape[1] > shape[0]
    at = 1 << (24 if wide else 21)
    parts = [mdx.quantize_fp8(p, block=(tile, 128), transpose=transpose)
             for p in ((x[:, :at], x[:, at:]) if wide else (x[:at], x[at:]))]
    whole = mdx.quantize_fp8(x, block=(tile, 128), transpose=transpose)
    for which in range(2):
        assert torch.equal(raw(whole[which]), torch.cat([raw(p[which]) for p in parts], dim=int(wide != transpose)))


def test_product_of_more_columns_than_a_launch_takes(freed):
    n = (1 << 23) + 40  # 512 lanes for 16 x 16 results
    g = torch.Generator(device="cuda").manual_seed(32)
    b, sb = mdx.quantize_fp8(torch.randn(n, 128, generator=g, device="cuda", dtype=torch.bfloat16))
    a, sa = mdx.quantize_fp8(randn(33, 3, 128))
    got = mdx.matmul_fp8(a, sa, b, sb)
    at = 1 << 22
    assert torch.equal(got, torch.cat([mdx.matmul_fp8(a, sa, b[:at], sb[:at]), mdx.matmul_fp8(a, sa, b[at:], sb[at:])], 1))
    none = torch.empty(20, 0, dtype=torch.uint8, device="cuda")
    zeros = mdx.matmul_fp8(none.view(CODES), none.view(SCALES), b[:, :0], sb[:, :0])
    assert zeros.shape == (20, n) and not zeros.any()


def test_product_of_more_unaligned_rows_than_a_launch_packs(freed):
    n, k = (1 << 25) + 3, 100  # eight pieces of 16 bytes a row
    g = torch.Generator(device="cuda").manual_seed(34)
    b = torch.empty(n, k, dtype=torch.uint8, device="cuda")
    for part in b.split(1 << 22):
        part.copy_(torch.randint(0, 256, part.shape, generator=g, device="cuda", dtype=torch.uint8) & 0xF7)  # no NaN
    b, sb = b.view(CODES), torch.randint(120, 130, (n, 1), generator=g, device="cuda", dtype=torch.uint8).view(SCALES)
    a, sa = mdx.quantize_fp8(randn(35, 1, k))
    got = mdx.matmul_fp8(a, sa, b, sb)
    at = 1 << 24
    assert torch.equal(got, torch.cat([mdx.matmul_fp8(a, sa, b[:at], sb[:at]), mdx.matmul_fp8(a, sa, b[at:], sb[at:])], 1))
    assert torch.isfinite(got).all() and got.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_product_of_rows_far_apart(freed, dtype):
    """Rows of 2^22 bytes and more take the kernel for few rows, at any number of them.  Whole numbers: exact."""

    m, n, k, pitch = 40, 24, 200, 1 << 22
    g = torch.Generator(device="cuda").manual_seed(36)
    a, b = (torch.randint(-15, 16, (rows, k), generator=g, device="cuda").float() for rows in (m, n))
    far = torch.empty(m, pitch, dtype=torch.uint8, device="cuda").view(CODES)[:, :k]
    far.copy_(a.to(CODES))
    ones = [torch.full((rows, 2), 127, dtype=torch.uint8, device="cuda").view(SCALES) for rows in (m, n)]
    got = mdx.matmul_fp8(far, ones[0], b.to(CODES), ones[1], dtype=dtype)
    assert torch.equal(got, (a.double() @ b.double().T.contiguous()).to(dtype))


# --------------------------------------------------------------- autograd

@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_is_seen_by_graphs_that_saved_what_it_writes(bits):
    """A backward pass through a weight that has moved since must not give gradients of the new weight."""

    weight = randn(40, 300).requires_grad_()
    loss = weight.square().sum()
    state = mdx.adamw_state([weight], bits=bits)
    before = [t._version for part in state if part is not None for t in part]
    mdx.adamw_step([weight.detach()], [torch.ones(300, device="cuda")], *state, step=1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    assert all(t._version > v for t, v in zip((t for part in state if part is not None for t in part), before))
    weight.square().sum().backward()  # a new graph is whole again
    assert torch.equal(weight.grad, 2 * weight.detach())


def test_a_product_into_a_buffer_is_seen_by_graphs_that_saved_it():
    codes, scales = mdx.quantize_fp8(randn(41, 20, 256))
    out, factor = torch.ones(20, 24, device="cuda"), randn(42, 20, 20).requires_grad_()
    loss = (out[:, :20] * factor).sum()
    mdx.matmul_fp8(codes, scales, codes, scales, out=out[:, :20])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_of_inference_mode_are_written_too():
    with torch.inference_mode():
        codes, scales = mdx.quantize_fp8(randn(43, 20, 256))
        out = torch.zeros(20, 20, device="cuda")
        mdx.matmul_fp8(codes, scales, codes, scales, out=out)
        p = torch.zeros(100, device="cuda")
        mdx.adamw_step([p], [torch.ones(100, device="cuda")], *mdx.adamw_state([p], bits=8), step=1, lr=0.5)
    assert torch.equal(out, mdx.matmul_fp8(codes, scales, codes, scales, dtype=torch.float32)) and torch.all(p < -0.49)


def recorded_calls():
    """Each call with one input that requires gradients, and the input."""

    x, gain = randn(50, 20, 256), randn(51, 256)
    rstd = torch.ones(20, device="cuda")
    codes, scales = mdx.quantize_fp8(x)

    def leaf(t):
        return t.clone().requires_grad_()

    for v in (leaf(x),):
        yield "norm of rows", v, lambda v=v: mdx.rms_norm(v, gain).values
        yield "norm's total", v, lambda v=v: mdx.rms_norm(x, gain, residual=v).total
        yield "norm's rstd", v, lambda v=v: mdx.rms_norm(v, gain).rstd
        yield "norm to codes", v, lambda v=v: mdx.rms_norm(v, gain, dtype=CODES).values
        yield "codes", v, lambda v=v: mdx.quantize_fp8(v)[0]
        yield "product of codes", v, lambda v=v: mdx.matmul_fp8(*mdx.quantize_fp8(v), codes, scales)
        yield "gradients", v, lambda v=v: mdx.rms_norm_backward(v, x, gain, rstd)[0]
        yield "gradients' total", v, lambda v=v: mdx.rms_norm_backward(x, x, gain, rstd, grad_total=v)[1]
    w = leaf(gain)
    yield "norm's gain", w, lambda: mdx.rms_norm(x, w, dtype=CODES).values


def test_gradients_are_not_lost_in_silence():
    """A sum of a call's result and another way: the backward pass raises, it does not leave the call's part out."""

    for name, v, run in recorded_calls():
        out = run()
        assert out.requires_grad, name
        with pytest.raises(RuntimeError, match="records no gradients"):
            (out.float().sum() + v.sum()).backward()
        with torch.no_grad():
            assert not run().requires_grad, name


def test_out_and_forward_gradients_are_refused_where_gradients_are_recorded():
    x, gain = randn(52, 20, 256), randn(53, 256)
    v = x.clone().requires_grad_()
    codes, scales = mdx.quantize_fp8(x)
    out = torch.zeros(20, 20, device="cuda")
    with pytest.raises(mdx.DescriptorInputError, match="out records no gradients"):
        mdx.matmul_fp8(*mdx.quantize_fp8(v), codes, scales, out=out)
    with pytest.raises(mdx.DescriptorInputError, match="out requires gradients"):
        mdx.matmul_fp8(codes, scales, codes, scales, out=out.clone().requires_grad_())
    with torch.no_grad():
        mdx.matmul_fp8(*mdx.quantize_fp8(v), codes, scales, out=out)
    assert torch.equal(out, mdx.matmul_fp8(codes, scales, codes, scales, dtype=torch.float32))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(mdx.DescriptorInputError, match="forward gradient"):
            mdx.rms_norm(dual, gain)


# ------------------------------------------------ steps in a replayed graph

def number(value: int) -> torch.Tensor:
    return torch.tensor([value], dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [8, 32])
def test_replays_of_a_captured_step_are_successive_steps(dtype, bits):
    """One captured step that moves its own step and seed on, replayed, against eager steps with numbers.  The moments do not
    depend on the bias corrections: the same bits.  The corrections are rounded from float64, so the update is the
    same to a unit in the last place, 2 u, of either factor, and its difference to the roundings that follow."""

    sizes = (1, 130, 5000)
    start = [randn(60 + i, n) for i, n in enumerate(sizes)]
    grads = [0.01 * randn(70 + i, n) for i, n in enumerate(sizes)]
    grads = [g.to(dtype) for g in grads]
    lr = 1e-2
    eager, replayed = ([p.clone() for p in start] for _ in range(2))
    states = [mdx.adamw_state(eager, bits=bits) for _ in range(2)]
    step = number(0)

    def move():
        step.add_(1)
        mdx.adamw_step(replayed, grads, *states[1], step=step, seed=step, lr=lr)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # once before the capture: the first step
        move()
    torch.cuda.current_stream().wait_stream(side)
    mdx.adamw_step(eager, grads, *states[0], step=1, seed=1, lr=lr)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        move()
    for turn in range(2, 8):
        graph.replay()
        mdx.adamw_step(eager, grads, *states[0], step=turn, seed=turn, lr=lr)
        torch.cuda.synchronize()
        assert int(step) == turn
        for parts in zip(*states):
            for want, got in zip(*parts) if parts[0] is not None else ():
                assert torch.equal(raw(got), raw(want))
        for want, got in zip(eager, replayed):
            # an update is at most lr sqrt(1 / (1 - beta2)) = 32 lr
            assert torch.all((got - want).abs() <= turn * (8 * U * 32 * lr + 2 * U * want.abs()))


@pytest.mark.parametrize("step", [1, 2, 1000, 10 ** 6, 2 ** 40])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.0, 0.0), (0.5, 0.9999999)])
def test_a_step_in_device_memory_is_the_step(step, betas):
    grad, lr = randn(80, 700), 1e-2
    results = []
    for at in (step, number(step), torch.tensor(step), torch.tensor([step], dtype=torch.int64)):  # the latter are numbers
        p = randn(81, 700)
        state = mdx.adamw_state([p])
        mdx.adamw_step([p], [grad], *state, step=at, lr=lr, betas=betas)
        results.append((p, state.first[0], state.second[0]))
    want = results[0]
    for got in results[1:]:
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        # the update m / (1 - beta1^step) / sqrt(v / (1 - beta2^step)) is at most 1 / sqrt(1 - beta2) here
        moved = lr / math.sqrt(1.0 - betas[1])
        assert torch.all((got[0] - want[0]).abs() <= 8 * U * moved + 2 * U * want[0].abs())
    for got in results[2:]:
        assert torch.equal(got[0], want[0])


def test_a_seed_in_device_memory_is_the_seed():
    grad = randn(82, 5000)
    for seed in (0, 7, -3, 2 ** 32 - 1, 2 ** 33 + 5):
        codes = []
        for at in (seed, number(seed)):
            p = randn(83, 5000)
            state = mdx.adamw_state([p], bits=8)
            mdx.adamw_step([p], [grad], *state, step=2, seed=at)
            codes.append((p, raw(state.first[0]), raw(state.second[0])))
        assert all(torch.equal(a, b) for a, b in zip(*codes))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_below_one_in_device_memory_changes_nothing(bits):
    p, grad = randn(84, 300), randn(85, 300)
    state = mdx.adamw_state([p], bits=bits)
    mdx.adamw_step([p], [grad], *state, step=1)
    before = [t.clone() for t in (p, *(part[0] for part in state if part is not None))]
    for at in (0, -1):
        mdx.adamw_step([p], [grad], *state, step=number(at))
    after = (p, *(part[0] for part in state if part is not None))
    assert all(torch.equal(raw(a), raw(b)) for a, b in zip(before, after))


def test_numbers_in_device_memory_are_refused_where_they_are_not_one():
    p = randn(86, 30)
    state = mdx.adamw_state([p])
    for name in ("step", "seed"):
        with pytest.raises(mdx.DescriptorInputError, match=f"{name} must be a whole number or an int64 tensor"):
            mdx.adamw_step([p], [p.clone()], *state, **{"step": 1, name: torch.ones(2, dtype=torch.int64, device="cuda")})


def test_a_step_over_tensors_that_overlap_is_refused():
    flat, grad = randn(87, 1000), randn(88, 300)
    for first in (flat[200:500], flat[299:599]):
        with pytest.raises(mdx.DescriptorInputError, match="overlaps"):
            mdx.adamw_step([flat[:300]], [grad], [first], [torch.zeros_like(grad)], step=1)
    with pytest.raises(mdx.DescriptorInputError, match="gradient overlaps"):
        mdx.adamw_step([flat[:300]], [flat[1:301]], [grad], [torch.zeros_like(grad)], step=1)
    # side by side, and with the gradient in its parameter's own place
    p = [flat[:300], flat[300:600]]
    g = [flat[:300], grad]
    want = [x.clone() for x in p]
    mdx.adamw_step(want, [x.clone() for x in g], *mdx.adamw_state(want), step=1)
    mdx.adamw_step(p, g, *mdx.adamw_state(p), step=1)
    assert all(torch.equal(a, b) for a, b in zip(p, want))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_of_zero_gradients_with_the_smallest_eps(bits):
    """0 / (0 + eps) is zero: the parameters decay and nothing else."""

    p, g = randn(89, 300), torch.zeros(300, device="cuda")
    for eps in (2.0 ** -126, 1e-30, 1e-8):
        q = p.clone()
        mdx.adamw_step([q], [g], *mdx.adamw_state([q], bits=bits), step=1, eps=eps, lr=0.5, weight_decay=0.5)
        assert torch.equal(q, 0.75 * p)
    with pytest.raises(mdx.DescriptorInputError, match="eps"):
        mdx.adamw_step([p], [g], *mdx.adamw_state([p], bits=bits), step=1, eps=1e-39)


# -------------------------------------------------- precision of products

SHAPES = [(5, 24, 200), (70, 90, 300), (300, 300, 1000)]  # the kernel for few rows, and tiles


def whole_codes(seed: int, rows: int, k: int) -> torch.Tensor:
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-15, 16, (rows, k), generator=g, device="cuda").float()


def one_scale(rows: int, k: int, byte: int) -> torch.Tensor:
    return torch.full((rows, -(-k // 128)), byte, dtype=torch.uint8, device="cuda").view(SCALES)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_product_at_every_scale(dtype, shape):
    """Scales 2^e and 2^-e of whole numbers: exact.  16-bit results take every scale there is, float32 ones those whose
    elements bfloat16 holds: 15 * 2^124 is below 2^128, 15 * 2^-124 a multiple of 2^-133."""

    m, n, k = shape
    a, b = whole_codes(90, m, k), whole_codes(91, n, k)
    want = (a.double() @ b.double().T.contiguous()).to(dtype)
    for byte in range(3, 252) if dtype == torch.float32 else range(255):
        got = mdx.matmul_fp8(a.to(CODES), one_scale(m, k, byte), b.to(CODES), one_scale(n, k, 254 - byte), dtype=dtype)
        assert torch.equal(got, want), byte


@pytest.mark.parametrize("shape", SHAPES)
def test_float32_product_of_the_largest_and_smallest_elements(shape):
    """Every code at the ends of the documented scales: 448 * 2^119 with multiples of 2^-9 * 2^-124.  Exact: products are
    whole multiples of 7 * 2^-8, below 2^24 of them."""

    m, n, k = shape
    a, b = 448.0 * whole_codes(92, m, k).sign(), whole_codes(93, n, k) * 2.0 ** -9
    want = a.double() @ b.double().T.contiguous() * 2.0 ** -5
    for first, second in (((a, 246), (b, 3)), ((b, 3), (a, 246))):
        (x, xs), (y, ys) = first, second
        got = mdx.matmul_fp8(x.to(CODES), one_scale(len(x), k, xs), y.to(CODES), one_scale(len(y), k, ys), dtype=torch.float32)
        assert torch.equal(got, (want if x is a else want.T).float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_product_of_blocks_of_zeros_at_any_scale(dtype, shape):
    """Zero codes stand for zeros whatever their scale's byte, NaN apart."""

    m, n, k = shape
    a, b = whole_codes(94, m, k), whole_codes(95, n, k)
    a[:, :128] = 0.0
    want = (a.double() @ b.double().T.contiguous()).to(dtype)
    for byte in (0, 1, 253, 254):
        scales = one_scale(m, k, 127).clone()
        scales.view(torch.uint8)[:, 0] = byte
        got = mdx.matmul_fp8(a.to(CODES), scales, b.to(CODES), one_scale(n, k, 127), dtype=dtype)
        assert torch.equal(got, want), byte


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(70, 90, 300), (130, 200, 8000)])
def test_product_of_equal_signs(dtype, shape):
    """Operands without a sign, as features often are: nothing cancels what the groups of eight lose, at most 7 * 2^-13 of
    their largest products' sum; then one rounding to the result's type."""

    m, n, k = shape
    (a, sa), (b, sb) = (mdx.quantize_fp8(randn(96 + i, rows, k).abs()) for i, rows in enumerate((m, n)))
    x, y = (c.double() * torch.exp2(s.contiguous().view(torch.uint8).double() - 127).repeat_interleave(128, 1)[:, :k]
            for c, s in ((a, sa), (b, sb)))
    want = x @ y.T.contiguous()
    error = (2 * k + 16) * U * want
    if dtype != torch.float32:
        largest = [torch.nn.functional.pad(v, (0, -k % 8)).view(v.shape[0], -1, 8).amax(2) for v in (x, y)]
        error = error + 7 * 2.0 ** -13 * (largest[0] @ largest[1].T.contiguous())
    got = mdx.matmul_fp8(a, sa, b, sb, dtype=dtype).double()
    assert torch.all(((want - error).to(dtype).double() <= got) & (got <= (want + error).to(dtype).double()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_of_rows_whose_squares_pass_the_range(dtype):
    """2^64 squared is past float32: rstd and the row are zero, the rows beside it are not touched."""

    x, gain = randn(100, 6, 200, dtype=dtype), randn(101, 200)
    want = mdx.rms_norm(x, gain)
    x[2, 7] = 2.0 ** 64
    got = mdx.rms_norm(x, gain)
    assert float(got.rstd[2]) == 0.0 and not got.values[2].any()
    rest = torch.arange(6, device="cuda") != 2
    assert torch.equal(got.values[rest], want.values[rest]) and torch.equal(got.rstd[rest], want.rstd[rest])
