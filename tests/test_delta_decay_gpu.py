"""Gradients of the gated delta rule where decays are strong, resets cut sequences apart and writes are idle: the
gradient kernels of 16-bit and of 32-bit results, token by token against the recurrence in 64 bits."""
import math

import pytest
import torch

import fpscan_b200 as fp
from fpscan_b200 import _lib
from delta_ref import decay_gradient_sizes, delta64, half_step, make, off, tolerance

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
BACKWARD = 14  # products one after another, as in test_delta_gpu.py
# seqlen, key heads, heads per key head, dk, dv: chunks of one head; shared key heads; more chunks than CTAs, 64
# values a CTA in the sequential kernels
SHAPES = [(150, 2, 1, 128, 128), (130, 2, 2, 24, 40), (200, 80, 2, 16, 16)]


@pytest.fixture(autouse=True)
def _healthy():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def _gradients(x, s0, scale=0.5, seed=1, size=None):
    """Gradients, those in 64 bits, and the sizes of the terms of dlog_decay.  size: of each output's gradient."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    go = 8 * torch.randn(x[2].shape, generator=gen, device="cuda")
    go = (go if size is None else go * size).to(x[2].dtype)
    leaves = [t.clone().requires_grad_() for t in x] + ([] if s0 is None else [s0.clone().requires_grad_()])
    ref = [t.detach().double().requires_grad_() for t in leaves]
    want, last = delta64(*ref[:5], None if s0 is None else ref[5], scale)
    if s0 is None:
        gs = None
        got = torch.autograd.grad(fp.gated_delta(*leaves, scale=scale), leaves, go)
        wanted = torch.autograd.grad(want, ref, go.double())
    else:
        gs = torch.randn(s0.shape, generator=gen, device="cuda")
        o, s1 = fp.gated_delta(*leaves[:5], initial_state=leaves[5], scale=scale, return_state=True)
        got = torch.autograd.grad((o, s1), leaves, (go, gs))
        wanted = torch.autograd.grad((want, last), ref, (go.double(), gs.double()))
    return got, [torch.nan_to_num(w) for w in wanted], decay_gradient_sizes(x, s0, go, gs, scale)


def _check_decays(got, want, sizes, dtype, wide):
    """Each token by itself: rounded once (fp16: to multiples of 2^-24 at the least), after `BACKWARD` products
    whose operands are no larger than `sizes`."""
    unit = tolerance(dtype, wide, 1) - half_step(dtype)
    tol = half_step(dtype) * want.abs() + BACKWARD * unit * sizes + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    # the nearest fp16 number of what is half a step past 65504, 65520, or more is infinity: where the gradient in
    # 64 bits comes that near, an infinity of its sign is as right as 65504
    past = torch.isinf(got) & (want.abs() + tol >= 65520) & (got.sign() == want.sign()) & (dtype == torch.float16)
    worst = torch.where(past, 0.0, (got.double() - want).abs() / tol).max()
    assert worst <= 1, float(worst)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("level", [-4.0, -6.0, -10.0, -14.0])
def test_decays_of_a_head_that_forgets(level, state, shape, dtype):
    x, s0 = make(1, *shape, dtype, seed=21, state=state)
    x[3].fill_(level)
    x[3][:, ::3] *= 0.75
    got, want, sizes = _gradients(x, s0)
    _check_decays(got[3], want[3], sizes, dtype, state)
    for i in (0, 1, 2, 4):
        tol = tolerance(dtype, state, BACKWARD) + (7 if i == 4 else 0) * (tolerance(dtype, state, BACKWARD) - half_step(dtype))
        assert off(got[i], want[i]) <= tol, i


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("at", [32, 64, 79])
def test_nothing_behind_a_reset_counts_before_it(at, state, shape, dtype):
    # what follows is 100 times larger (fp32: 10000 times), in values and in the outputs' gradients
    much = 1e4 if dtype == torch.float32 else 100.0
    x, s0 = make(1, *shape, dtype, seed=22, state=state)
    x[3].fill_(-1.0)
    x[3][:, at] = -math.inf
    x[2][:, at:] *= much
    size = torch.ones(1, shape[0], 1, 1, device="cuda")
    size[:, at:] = much
    got, want, sizes = _gradients(x, s0, size=size)
    assert (got[3][:, at] == 0).all()
    sizes[:, at] = 1.0  # 0, as it has to be
    _check_decays(got[3], want[3], sizes, dtype, state)
    for i in range(5):  # and by itself what lies before it
        assert off(got[i][:, :at], want[i][:, :at]) <= 8 * tolerance(dtype, state, BACKWARD), i


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("state", [False, True])
def test_resets_strong_decays_and_idle_writes(state, shape, dtype):
    x, s0 = make(1, *shape, dtype, seed=23, resets=0.05, zero_beta=0.3, state=state)
    for t in (0, 63, 64, 127, 128, 129):
        x[3][:, t, 0] = -math.inf
    x[3][:, 20:24] = torch.finfo(dtype).min
    x[3][:, 30:34] = -80.0
    x[3][:, 40:46] = -9.0
    x[3][:, 50:52] = 0.0
    got, want, sizes = _gradients(x, s0)
    assert (got[3][x[3] < -10000] == 0).all()
    sizes[x[3] < -10000] = 1.0
    _check_decays(got[3], want[3], sizes, dtype, state)
    for i in (0, 1, 2, 4):
        assert torch.isfinite(got[i]).all()
        tol = half_step(dtype) + (8 if i == 4 else 1) * (tolerance(dtype, state, BACKWARD) - half_step(dtype))
        assert off(got[i], want[i]) <= tol, i
    if state:
        assert off(got[5], want[5]) <= tolerance(torch.float32, True, BACKWARD)
