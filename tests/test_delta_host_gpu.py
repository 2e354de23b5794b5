"""Gated delta rule and 8-bit checkpoints on the GPU: slices of larger tensors, and what the host keeps or refuses."""
import pytest
import torch

import fpscan_b200 as fp
from fpscan_b200 import _lib, checkpoint8, delta, ops
from delta_ref import make

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _healthy():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


@pytest.fixture(params=["binding", "ctypes"])
def path(request, monkeypatch):
    if request.param == "ctypes":
        for m in (ops, delta, checkpoint8):
            monkeypatch.setattr(m, "_EXT", None)
    return request.param


def _shifted(t, by=1):
    """The same values in memory that starts `by` elements behind a 16-byte boundary."""
    s = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)[by:].view(t.shape)
    return s.copy_(t)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [1, 3, 6])
def test_slices_along_time_and_batch(heads, dtype, path):
    # a server steps through a packed (1, L, heads) tensor; a batch's sequences one by one
    x, s0 = make(1, 7, heads, 1, 16, 24, dtype, seed=1, state=True)
    whole, state = s0.clone(), s0.clone()
    want = fp.gated_delta_step(*x, whole)
    got = torch.cat([fp.gated_delta_step(*(t[:, i:i + 1] for t in x), state) for i in range(7)], 1)
    assert torch.equal(got, want) and torch.equal(state, whole)
    y, t0 = make(3, 33, heads, 1, 16, 24, dtype, seed=2, state=True)
    o, last = fp.gated_delta_forward(*y, initial_state=t0, return_state=True)
    for i in range(3):
        p, one = fp.gated_delta_forward(*(t[i:i + 1] for t in y), initial_state=t0[i:i + 1], return_state=True)
        assert torch.equal(p, o[i:i + 1]) and torch.equal(one, last[i:i + 1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_takes_values_from_anywhere(dtype, path):
    x, s0 = make(2, 2, 1, 3, 16, 24, dtype, seed=3, state=True)
    want = fp.gated_delta_step(*x, s0.clone())
    out = _shifted(torch.zeros_like(x[2]), 3)
    got = fp.gated_delta_step(*x[:2], *(_shifted(t) for t in x[2:]), s0.clone(), out=out)
    assert got is out and torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_that_are_slices(dtype, path):
    # the outputs are part of a flat vector whose gradient is cut up again
    x, s0 = make(2, 70, 1, 2, 16, 24, dtype, seed=4, state=True)
    go, gs = torch.randn_like(x[2]), torch.randn_like(s0)
    decays = [_shifted(t) for t in x[3:]]
    want = delta.gated_delta_backward(*x, go, s0, gs, need_initial=True)
    for a, b in zip(delta.gated_delta_backward(*x[:3], *decays, _shifted(go), s0, _shifted(gs), need_initial=True), want):
        assert torch.equal(a, b)
    for eight in (False, True):
        leaves = [t.clone().requires_grad_() for t in x]
        o = fp.gated_delta(*leaves, checkpoint8=eight)
        want = torch.autograd.grad(o, leaves, go, retain_graph=True)
        flat = torch.cat([torch.zeros(1, dtype=dtype, device="cuda"), o.flatten()])
        got = torch.autograd.grad(flat[1:], leaves, go.flatten(), retain_graph=True)
        some = torch.autograd.grad(flat, leaves, torch.cat([go.new_zeros(1), go.flatten()]))
        for a, b, c in zip(got, some, want):
            assert torch.equal(a, c) and torch.equal(b, c)
    g, t = (torch.rand(2, 50, 24, device="cuda").to(dtype).requires_grad_() for _ in range(2))
    y = fp.pscan_channels_last(g, t, checkpoint8=True)
    go = torch.randn_like(y)
    want = torch.autograd.grad(y, (g, t), go, retain_graph=True)
    flat = torch.cat([go.new_zeros(1), y.flatten()])
    for a, b in zip(torch.autograd.grad(flat, (g, t), torch.cat([go.new_zeros(1), go.flatten()])), want):
        assert torch.equal(a, b)


def test_operands_that_stay_refused(path):
    x, s0 = make(1, 4, 2, 1, 16, 16, torch.float32, seed=5, state=True)
    for i in (0, 1, 2):
        y = list(x)
        y[i] = _shifted(x[i])
        with pytest.raises(RuntimeError, match="aligned"):
            fp.gated_delta_forward(*y)
        if i < 2:
            with pytest.raises(RuntimeError, match="aligned"):
                fp.gated_delta_step(*y, s0.clone())
    with pytest.raises(RuntimeError, match="aligned"):
        fp.gated_delta_step(*x, _shifted(s0))


@pytest.mark.parametrize("mode", ["no_grad", "inference", "no leaf"])
def test_no_checkpoint_without_a_backward_pass(mode, path):
    # what the call leaves allocated besides its results, at most and in the end, is what it needs without one
    x, s0 = make(2, 200, 2, 1, 64, 64, torch.bfloat16, seed=6, state=True)
    g, t = (torch.rand(2, 600, 2048, device="cuda").to(torch.bfloat16) for _ in range(2))
    want = fp.gated_delta_forward(*x, initial_state=s0, return_state=True), fp.scan_forward_channels_last(g, t)
    if mode != "no leaf":
        for y in (*x, s0, g, t):
            y.requires_grad_()
    guard = {"no_grad": torch.no_grad, "inference": torch.inference_mode, "no leaf": torch.enable_grad}[mode]

    def peak(call):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        res = call()
        return res, torch.cuda.max_memory_allocated() - before

    with guard():
        for eight in (False, True):
            fp.gated_delta(*x, initial_state=s0, return_state=True, checkpoint8=eight)
            fp.pscan_channels_last(g, t, checkpoint8=eight)
        (o, s1), most = peak(lambda: fp.gated_delta(*x, initial_state=s0, return_state=True, checkpoint8=True))
        _, plain = peak(lambda: fp.gated_delta(*x, initial_state=s0, return_state=True))
        assert most == plain
        y, most = peak(lambda: fp.pscan_channels_last(g, t, checkpoint8=True))
        _, plain = peak(lambda: fp.pscan_channels_last(g, t))
        # a workspace of its own, as every call with checkpoint8 has; the codes would be half of the output
        assert most <= plain + _lib.load().fpscan_cl_workspace_bytes(2, 600, 2048, 2, 0) + 1024 < plain + y.numel()
    assert not o.requires_grad and not y.requires_grad
    assert torch.equal(o, want[0][0]) and torch.equal(s1, want[0][1]) and torch.equal(y, want[1])


def test_a_checkpoint_where_one_input_asks_for_it(path):
    x, s0 = make(1, 70, 1, 1, 16, 16, torch.bfloat16, seed=7, state=True)
    go = torch.randn_like(x[2])
    kept = [fp.dequantize8(*fp.quantize8(t), torch.bfloat16) for t in x[:3]]
    want = delta.gated_delta_backward(*kept, *x[3:], go, s0, need_initial=True)
    for i, t in enumerate((*x, s0)):
        leaves = [y.clone() for y in (*x, s0)]
        leaves[i].requires_grad_()
        o = fp.gated_delta(*leaves[:5], initial_state=leaves[5], checkpoint8=True)
        assert torch.equal(torch.autograd.grad(o, leaves[i], go)[0], want[i])
    g, t = (torch.rand(1, 40, 8, device="cuda") for _ in range(2))
    for a, b in ((g.clone().requires_grad_(), t), (g, t.clone().requires_grad_())):
        y = fp.pscan_channels_last(a, b, checkpoint8=True)
        leaf = a if a.requires_grad else b
        assert torch.isfinite(torch.autograd.grad(y.sum(), leaf)[0]).all()


def test_a_step_does_not_overwrite_a_state_that_has_a_gradient(path):
    x, s0 = make(1, 66, 1, 1, 16, 16, torch.float32, seed=8, state=True)
    one = [t[:, :1].contiguous() for t in x]
    leaf = s0.clone().requires_grad_()
    _, last = fp.gated_delta(*x, initial_state=leaf, return_state=True)
    for state in (leaf, last):
        held = state.detach().clone()
        with pytest.raises(RuntimeError, match="gradient"):
            fp.gated_delta_step(*one, state)
        assert torch.equal(state, held)
    state = last.detach().clone()
    want = fp.gated_delta_step(*one, state)
    with torch.no_grad():  # as torch's own operations in place
        assert torch.equal(fp.gated_delta_step(*one, last), want)
    assert torch.equal(fp.gated_delta_step(*one, last.detach()), fp.gated_delta_step(*one, state))


def test_an_output_written_over_a_saved_tensor_is_noticed(path):
    x, s0 = make(1, 66, 1, 1, 16, 16, torch.float32, seed=9, state=True)
    one = [t[:, :1].contiguous() for t in x]
    for y, call in ((x, lambda out: fp.gated_delta_forward(*x, out=out)),
                    (one, lambda out: fp.gated_delta_step(*one, s0.clone(), out=out))):
        leaf = torch.ones_like(y[2]).requires_grad_()
        held = torch.zeros_like(y[2])
        product = (leaf * held).sum()
        assert call(held) is held
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()
        with pytest.raises(RuntimeError, match="gradient"):
            call(leaf)
        with torch.no_grad():
            assert torch.equal(call(leaf), held)
        with torch.inference_mode():
            made = torch.zeros_like(y[2])
            call(made)
        assert torch.equal(call(made), held)
