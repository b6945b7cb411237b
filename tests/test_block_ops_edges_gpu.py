"""Calls of the transformer-block operators at the edges of what they take:
infinities, NaNs and far scales in the data, overlapping views, widths next
to 2^31.  Tolerances count roundings as in test_block_ops_gpu."""
import pytest
import torch

import ppdl

pytestmark = pytest.mark.gpu

WIDEST = 2 ** 31 - 1


def guarded(n, t, fill):
    """n values with 4096 of `fill` in front and behind, all of that value."""
    room = torch.full((n + 8192,), fill, device="cuda", dtype=t)
    return room, room[4096:4096 + n]


def test_widest_row_quantised(cuda):
    """The last step over a row of 2^31 - 1 values passes 2^31."""
    x = torch.ones(WIDEST, device="cuda", dtype=torch.bfloat16)
    x[1::2] = -1
    x[-1] = 0.5
    room, q = guarded(2 ** 31, torch.int8, 55)
    scale = torch.zeros(1, device="cuda")
    ppdl.check(ppdl.lib().ppdl_quantize_rows_i8(x.data_ptr(), WIDEST, 1, 1, WIDEST, q.data_ptr(), 2 ** 31,
                                                scale.data_ptr(), torch.cuda.current_stream().cuda_stream))
    step = (torch.ones((), dtype=torch.float64) / 127).float()
    assert scale[0] == step
    assert (q[0:WIDEST - 1:2] == 127).all() and (q[1:WIDEST:2] == -127).all()
    assert q[WIDEST - 1] == round(0.5 / step.item())
    assert (room[:4096] == 55).all() and (room[4096 + WIDEST:] == 55).all()


def test_widest_row_normalised(cuda):
    """Values +-1 in turn: 512 threads add one sign each, 2^22 times, which is
    exact; the mean is 2^-31, the variance 1."""
    x = torch.ones(WIDEST, device="cuda", dtype=torch.bfloat16)
    x[1::2] = -1
    room, y = guarded(WIDEST, torch.bfloat16, 7.0)
    ppdl.check(ppdl.lib().ppdl_layernorm(x.data_ptr(), WIDEST, None, 0, None, None, 1, 1, 1, WIDEST, 1e-5, y.data_ptr(),
                                         WIDEST, None, 0, None, None, torch.cuda.current_stream().cuda_stream))
    want = torch.tensor((1 + 1e-5) ** -0.5, dtype=torch.bfloat16).item()
    assert (y[::2] == want).all() and (y[1::2] == -want).all()
    assert (room[:4096] == 7).all() and (room[4096 + WIDEST:] == 7).all()


def test_widest_row_backward(cuda):
    """x = + - + - and dy = + + - - in turn: exact sums of 0 and 1 over the row,
    so that dx is dy to within 2^-31, at mean 0 and rstd 1."""
    x = torch.ones(WIDEST, device="cuda", dtype=torch.bfloat16)
    x[1::2] = -1
    dy = torch.ones(WIDEST, device="cuda", dtype=torch.bfloat16)
    dy[2::4] = -1
    dy[3::4] = -1
    room, dx = guarded(WIDEST, torch.bfloat16, 7.0)
    mean, rstd = torch.zeros(1, device="cuda"), torch.ones(1, device="cuda")
    ppdl.check(ppdl.lib().ppdl_layernorm_backward(
        dy.data_ptr(), WIDEST, x.data_ptr(), WIDEST, None, mean.data_ptr(), rstd.data_ptr(), None, 0, 1, 1, 1, WIDEST,
        dx.data_ptr(), WIDEST, None, None, None, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(dx, dy)
    assert (room[:4096] == 7).all() and (room[4096 + WIDEST:] == 7).all()

