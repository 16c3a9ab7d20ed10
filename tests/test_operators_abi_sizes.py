"""Sizes at the limits of the operators' C entry points, without a GPU: every call here is refused, or has nothing to do,
before a device is touched."""

from __future__ import annotations

import ctypes
import subprocess
import sys

import pytest

from conftest import ROOT

pytest.importorskip("torch")

P = 4096  # an address that nothing here reads


@pytest.fixture(scope="module")
def hip():
    from mdescriptor_amd import _hip

    if not _hip.LIBRARY_PATH.is_file():
        subprocess.run([sys.executable, "-m", "mdescriptor_amd.build"], check=True, cwd=ROOT)
    return _hip


def matmul(hip, **changes):
    values = dict(m=40, n=8, k=200, a=P, a_pitch=256, a_scales=P, a_scales_pitch=4, b=P, b_pitch=256, b_scales=P,
                  b_scales_pitch=4, out=P, out_pitch=8, b_tile=1, out_dtype=1, a_packed=1, b_packed=1)
    return hip.MatmulArgs(**{**values, **changes})


WORKSPACES = """
import ctypes, sys
sys.path.insert(0, {root!r})
from mdescriptor_amd import _hip
lib = _hip.load_library()
for sizes in ({{"k": -1}}, {{"k": -63}}, {{"k": -64}}, {{"k": -200}}, {{"m": -40}}, {{"n": -8}}, {{"k": 1 << 31}},
              {{"k": 1 << 62}}, {{"m": 1 << 62, "n": 1 << 62}}, {{"m": (1 << 31) - 1, "n": (1 << 31) - 1}}):
    args = _hip.MatmulArgs(**{{**dict(m=40, n=8, k=200, out_dtype=1, b_tile=1), **sizes}})
    assert lib.mdx_hip_matmul_fp8_workspace(ctypes.byref(args)) == 0, sizes
for rows, width in ((-1, 5), (5, -1), (1 << 31, 5), (5, 1 << 31), (1 << 62, 1 << 62)):
    assert lib.mdx_hip_rms_norm_backward_workspace(rows, width) == 0, (rows, width)
"""


def test_workspaces_of_refused_sizes_are_empty():
    """In a process of its own: sizes that a workspace's arithmetic does not expect must not end the caller."""

    done = subprocess.run([sys.executable, "-c", WORKSPACES.format(root=str(ROOT))], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


def test_workspaces_of_taken_sizes_hold_their_parts(hip):
    lib = hip.load_library()
    size = lib.mdx_hip_matmul_fp8_workspace(ctypes.byref(matmul(hip, a_packed=0)))
    assert size >= 40 * 256 + 40 * 2 and size % 16 == 0
    assert lib.mdx_hip_rms_norm_backward_workspace(1000, 256) >= 256 * 4


def test_adamw_refuses_tensors_of_more_than_one_launch(hip):
    """256 lanes for 2,048 elements, fewer than 2^32 lanes: the count is checked before anything is queued."""

    lib = hip.load_library()
    for n in ((1 << 35) - 2047, 1 << 35, 1 << 41):
        table = (hip.AdamwTensor * 1)(hip.AdamwTensor(n, P, P, P, P, P, P))
        args = hip.AdamwArgs(tensors=ctypes.addressof(table), count=1, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8,
                             weight_decay=0.0, step=1, seed=0, grad_dtype=1, bits=8)
        assert lib.mdx_hip_adamw_step(0, ctypes.byref(args), None) == hip.MDX_INVALID_ARGUMENT
        assert "size" in lib.mdx_hip_last_error(None).decode()


def test_adamw_takes_a_step_from_device_memory_in_place_of_the_number(hip):
    lib = hip.load_library()
    values = dict(tensors=None, count=0, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, step=0, seed=0,
                  grad_dtype=0, bits=32)

    def call(step, step_at, seed_at):
        args = hip.AdamwArgs(**{**values, "step": step})
        return lib.mdx_hip_adamw_step_at(0, ctypes.byref(args), step_at, seed_at, None), lib.mdx_hip_last_error(None).decode()

    status, message = call(0, None, None)
    assert status == hip.MDX_INVALID_ARGUMENT and "step must" in message
    for places in ((P + 4, None), (None, P + 4)):
        status, message = call(1, *places)
        assert status == hip.MDX_INVALID_ARGUMENT and "aligned" in message
    assert lib.mdx_hip_adamw_step_at(0, None, None, None, None) == hip.MDX_INVALID_ARGUMENT


M = 1 << 20  # addresses far apart that nothing here reads


@pytest.mark.parametrize("bits, places, apart", [
    # (params, grads, first, second, first_scales, second_scales) of tensors of 200 elements
    (32, [(M, 2 * M, 3 * M, 4 * M)], True),
    (32, [(M, M, 3 * M, 4 * M)], True),                      # the gradient in its parameter's place
    (32, [(M, 3 * M, 3 * M, 4 * M)], True),                  # or in a float32 moment's
    (32, [(M, 2 * M, M, 4 * M)], False),
    (32, [(M, 2 * M, M + 796, 4 * M)], False),               # the last element of one is the first of the other
    (32, [(M, 2 * M, M + 800, 4 * M)], True),
    (32, [(M, M + 4, 3 * M, 4 * M)], False),                 # a gradient one element off
    (32, [(M, 3 * M - 796, 3 * M, 4 * M)], False),
    (32, [(M, 3 * M - 800, 3 * M, 4 * M)], True),
    (32, [(M, 2 * M, 3 * M, 4 * M), (M + 400, 2 * M, 5 * M, 6 * M)], False),
    (32, [(M, 2 * M, 3 * M, 4 * M), (7 * M, 2 * M + 4, 5 * M, 6 * M)], True),  # gradients may share
    (32, [(M, 2 * M, 3 * M, 4 * M), (7 * M, M, 5 * M, 6 * M)], False),         # another tensor's parameter
    (8, [(M, 2 * M, 3 * M, 4 * M, 5 * M, 6 * M)], True),
    (8, [(M, 2 * M, 3 * M, 3 * M + 199, 5 * M, 6 * M)], False),
    (8, [(M, 2 * M, 3 * M, 3 * M + 200, 5 * M, 6 * M)], True),
    (8, [(M, 2 * M, 3 * M, 4 * M, 5 * M, 5 * M + 1)], False),
    (8, [(M, 2 * M, 3 * M, 4 * M, 5 * M, 5 * M + 2)], True),
    (8, [(M, 3 * M, 3 * M, 4 * M, 5 * M, 6 * M)], False),    # codes are not where a float32 gradient is read
])
def test_adamw_refuses_tensors_that_overlap(hip, bits, places, apart):
    """On a device that is not there, so that what is not refused for this goes no further."""

    lib = hip.load_library()
    table = (hip.AdamwTensor * len(places))(*(hip.AdamwTensor(200, *place) for place in places))
    args = hip.AdamwArgs(tensors=ctypes.addressof(table), count=len(places), lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8,
                         weight_decay=0.0, step=1, seed=0, grad_dtype=0, bits=bits)
    status = lib.mdx_hip_adamw_step(12345, ctypes.byref(args), None)
    message = lib.mdx_hip_last_error(None).decode()
    assert status != hip.MDX_OK and ("overlaps" not in message) == apart, message


@pytest.mark.parametrize("eps", [1e-45, 1e-39, 1.1754942e-38])
def test_adamw_refuses_an_eps_whose_quotient_is_infinite(hip, eps):
    """1 / eps is infinite below float32's normal numbers, and the zero moment of a zero gradient times it NaN."""

    lib = hip.load_library()
    table = (hip.AdamwTensor * 1)(hip.AdamwTensor(200, M, 2 * M, 3 * M, 4 * M))
    args = hip.AdamwArgs(tensors=ctypes.addressof(table), count=1, lr=1e-3, beta1=0.9, beta2=0.99, eps=eps,
                         weight_decay=0.0, step=1, seed=0, grad_dtype=0, bits=32)
    assert lib.mdx_hip_adamw_step(12345, ctypes.byref(args), None) == hip.MDX_INVALID_ARGUMENT
    assert "eps" in lib.mdx_hip_last_error(None).decode()
