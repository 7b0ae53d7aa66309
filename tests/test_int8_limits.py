"""The limits that include/tandem_w4.h states for the operators on 8-bit integers, on both of their sides: what is refused, without a GPU, and the
largest call that is taken."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from tandem_amd.layers import norm, w4_hip, w8

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


def _at(address):
    return ctypes.c_void_p(address)


@pytest.mark.parametrize("residual,x_stride,r_stride,rows", [
    (4096, 64, 64, 3), (4096 + 16, 64, 64, 3), (4096 - 16, 64, 64, 3), (4096 + 128, 64, 64, 3), (4096 + 2 * 128 + 112, 64, 64, 3),
    (4096 + 112, 128, 128, 3), (4096 + 144, 128, 128, 3), (4096 + 128, 128, 136, 3), (4096, 64, 64, 1), (4096 + 112, 64, 64, 1)])
def test_residual_in_the_rows_memory(residual, x_stride, r_stride, rows):
    status = w4_hip.library().tw4_rms_norm_int8(P, x_stride, _at(residual), r_stride, _at(1 << 20), 1e-6, _at(1 << 21), _at(1 << 22), rows, 64, 0, None)
    _refused(status, w4_hip.TW4_EINVAL, "the residual needs memory of its own")


TOKEN = {"x": 4096, "residual": 8192, "residual_out": 12288, "norm_weight": 16384, "y": 20480}  # 128 bytes each, y 12


@pytest.mark.parametrize("moved,to,what", [
    (name, TOKEN[other] + shift, what)
    for name, others, shifts, what in (("residual_out", ("x", "residual", "norm_weight"), (-112, 0, 16, 112), "the new residual"),
                                       ("y", ("x", "residual", "norm_weight", "residual_out"), (-10, 0, 2, 126), "y needs"))
    for other in others for shift in shifts])
def test_one_token_outputs_in_the_inputs_memory(moved, to, what):
    at = {name: _at(to if name == moved else address) for name, address in TOKEN.items()}
    status = w4_hip.library().tw4_token_int8(at["x"], at["residual"], at["residual_out"], at["norm_weight"], 1e-6, _at(1 << 20), 64, _at(1 << 21), at["y"],
                                             6, 64, 0, 0, 256, None)
    _refused(status, w4_hip.TW4_EINVAL, what)


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


@pytest.mark.gpu
def test_memory_side_by_side():
    """Rows of x and of the residual between each other's, and a token's operands end to end, are taken."""
    lib, m, k, n = w4_hip.library(), 5, 64, 6
    both = torch.randn(m, 2 * k, device="cuda").half()
    x, r = both[:, :k].clone(), both[:, k:].clone()
    weight = torch.rand(k, device="cuda").half() + 0.5
    want = norm.fused_add_rms_norm_int8(x, r, weight, 1e-6)
    codes, scales = torch.empty_like(want[0]), torch.empty_like(want[1])
    before = both.clone()
    w4_hip.check(lib.tw4_rms_norm_int8(both.data_ptr(), 2 * k, both.data_ptr() + 2 * k, 2 * k, weight.data_ptr(), 1e-6, codes.data_ptr(), scales.data_ptr(),
                                       m, k, 0, w4_hip.raw_stream(0)))
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1]) and torch.equal(both[:, k:], want[2]) and torch.equal(both[:, :k], x)

    w, ws = torch.randint(-127, 128, (n, k), device="cuda", dtype=torch.int8), torch.rand(n, device="cuda")
    row = torch.cat([before[0], weight, torch.zeros(k + n, device="cuda", dtype=torch.float16)])  # x, residual, weight, new residual, y
    at = [row.data_ptr() + 2 * k * i for i in range(5)]
    w4_hip.check(lib.tw4_token_int8(at[0], at[1], at[3], at[2], 1e-6, w.data_ptr(), k, ws.data_ptr(), at[4], n, k, 0, 0, 256, w4_hip.raw_stream(0)))
    assert torch.equal(row[3 * k:4 * k], want[2][0]) and torch.equal(row[4 * k:], w8.linear_int8(codes[:1], scales[:1], w, ws)[0])
    assert torch.equal(row[:2 * k], before[0]) and torch.equal(row[2 * k:3 * k], weight)


class Own(torch.Tensor):
    pass


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 3])
def test_norm_weights_that_are_followed(m):
    """A norm's weight that a gradient, a tangent, a transform or a type of its own follows is refused, for one token and for more, as every other operand
    is; where no gradient is asked for it is a value."""
    k = 64
    layer = w8.W8Linear(k, 32).cuda()
    layer.weight.random_(-127, 128)
    layer.weight_scale.fill_(0.01)
    x, r = torch.randn(m, k, device="cuda").half(), torch.randn(m, k, device="cuda").half()
    plain = torch.rand(k, device="cuda").half() + 0.5
    calls = (lambda w: norm.rms_norm_int8(x, w, 1e-6), lambda w: norm.fused_add_rms_norm_int8(x, r.clone(), w, 1e-6),
             lambda w: layer.forward_norm(x, None, w, 1e-6), lambda w: layer.forward_norm(x, r.clone(), w, 1e-6))
    weight = torch.nn.Parameter(plain.clone())
    for call in calls:
        want = call(plain)
        with pytest.raises(RuntimeError, match="inference only"):
            call(weight)
        with pytest.raises(RuntimeError, match="inference only"):
            call(plain.as_subclass(Own))
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="inference only"):
            call(forward_ad.make_dual(plain, torch.ones_like(plain)))
        with pytest.raises(RuntimeError, match="inference only"):
            torch.func.vmap(lambda w: call(w)[0])(plain[None])
        with torch.no_grad():
            got = call(weight)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(call(torch.nn.Parameter(plain, requires_grad=False)), want))
