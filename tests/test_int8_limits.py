"""The limits that include/tandem_w4.h states for the operators on 8-bit integers, on both of their sides: what is refused, without a GPU, and the
largest call that is taken."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tandem_amd.layers import w4_hip

P = ctypes.c_void_p(4096)


def _product(m, n, k, rows, x=P, xs=P, w=P, ws=P, y=P):
    """tw4_gemm_int8's streaming kernel with so many rows of w a workgroup."""
    return w4_hip.library().tw4_gemm_int8(x, k, xs, w, k, ws, y, None, 0, None, 0, m, n, k, 0, 0, 0, rows, None)


def _refused(status, code, needle):
    message = w4_hip.library().tw4_last_error().decode()
    assert status == code and needle in message, (status, message)


# ------------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("m", [(1 << 20) - 15, (1 << 20) - 1, 1 << 20])
def test_tokens_of_the_streaming_kernel(m):
    _refused(_product(m, 1, 16, 4), w4_hip.TW4_ECONFIG, "M <= 2^20 - 16")


@pytest.mark.parametrize("n,rows", [(1 << 22, 1), (1 << 24, 1), (1 << 24, 4)])
def test_workgroups_of_the_streaming_kernel(n, rows):
    """2^22 workgroups of 1024 threads are past what a launch holds."""
    _refused(_product(1, n, 16, rows), w4_hip.TW4_ECONFIG, "too many rows")


# ------------------------------------------------------------------------------------------- GPU
def _ones(*shape):
    return torch.ones(*shape, device="cuda")


@pytest.mark.gpu
def test_most_tokens_of_the_streaming_kernel():
    m, n, k = (1 << 20) - 16, 3, 16
    x = (torch.arange(m * k, device="cuda") % 251 - 125).to(torch.int8).view(m, k)
    w = (torch.arange(n * k, device="cuda") % 7 - 3).to(torch.int8).view(n, k)
    xs, ws, y = _ones(m), _ones(n), torch.empty(m, n, dtype=torch.float16, device="cuda")
    w4_hip.check(_product(m, n, k, 4, *(t.data_ptr() for t in (x, xs, w, ws, y))))
    torch.cuda.synchronize()
    assert torch.equal(y.float(), torch.matmul(x.float(), w.float().t()).half().float())


@pytest.mark.gpu
def test_most_workgroups_of_the_streaming_kernel():
    m, n, k = 1, (1 << 22) - 1, 16
    x = (torch.arange(m * k, device="cuda") % 7 - 3).to(torch.int8).view(m, k)
    w = (torch.arange(n * k, device="cuda") % 251 - 125).to(torch.int8).view(n, k)
    xs, ws, y = _ones(m), _ones(n), torch.empty(m, n, dtype=torch.float16, device="cuda")
    w4_hip.check(_product(m, n, k, 1, *(t.data_ptr() for t in (x, xs, w, ws, y))))
    torch.cuda.synchronize()
    assert torch.equal(y.float(), torch.matmul(x.float(), w.float().t()).half().float())
