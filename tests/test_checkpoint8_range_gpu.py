"""The bound of the 8-bit format over the whole range of each type."""
import pytest
import torch

import fpscan_b200 as fp
from fpscan_b200 import _lib
from delta_ref import half_step

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SMALLEST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


@pytest.fixture(autouse=True)
def _healthy():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def _bound(x, most):
    """Half a step; the step's rounding (2^-24 of itself, 127 times; 2^-150 where it is subnormal) and the
    quotient's in fp32; the product's and the result's."""
    return (most / 254 + most * 2.0 ** -22 + (half_step(x.dtype) + 2.0 ** -24) * x.double().abs()
            + 127 * 2.0 ** -150 + SMALLEST[x.dtype])


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_of_every_magnitude(dtype):
    # a block for each power of two, with its largest magnitude first; and blocks of the very largest numbers
    lo, hi = {torch.bfloat16: (-133, 127), torch.float16: (-24, 15), torch.float32: (-149, 127)}[dtype]
    gen = torch.Generator().manual_seed(1)
    power = torch.arange(lo, hi + 1, dtype=torch.float64)
    x = torch.rand(len(power), 64, generator=gen, dtype=torch.float64) * 2 - 1
    x[:, 0] = 1
    x = (x * 2.0 ** power[:, None]).to(dtype)
    big = torch.finfo(dtype).max
    top = torch.tensor([big, -big, big / 2, big / 3, -big / 127, 0.0, 1.0, big * 0.99] * 8, dtype=torch.float64).to(dtype)
    below = (top.view(torch.int32 if dtype == torch.float32 else torch.int16) - 1).view(dtype)  # next towards zero
    below[top == 0] = 0
    x = torch.cat([x, top[None], below[None], -top[None]]).cuda()
    codes, steps = fp.quantize8(x)
    back = fp.dequantize8(codes, steps, dtype)
    most = x.double().abs().amax(1, keepdim=True)
    assert torch.isfinite(steps).all() and torch.isfinite(back).all()
    assert ((back.double() - x.double()).abs() <= _bound(x, most)).all()


def test_scan_keeps_the_largest_number():
    # y[0] is the largest fp32 number; the gradient of the next gate is that times an output's gradient
    g, x = torch.zeros(1, 16, 4, device="cuda"), torch.zeros(1, 16, 4, device="cuda")
    x[0, 0] = torch.finfo(torch.float32).max
    g.requires_grad_()
    y = fp.pscan_channels_last(g, x, checkpoint8=True)
    go = torch.full_like(y, 2.0 ** -100)
    dg, = torch.autograd.grad(y, g, go)
    assert torch.isfinite(dg).all()
    want = x[0, 0].double() * 2.0 ** -100
    assert ((dg[0, 1].double() - want).abs() <= want * 2.0 ** -21).all()  # 127 steps, rounded
