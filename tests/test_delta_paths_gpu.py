"""Gated delta rule and 8-bit checkpoints on the GPU: every launch variant and every host path."""
import math

import pytest
import torch

import fpscan_b200 as fp
from fpscan_b200 import _lib, checkpoint8, delta, ops
from delta_ref import delta64, make, off, tolerance

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
FORWARD, BACKWARD = 6, 14  # as in test_delta_gpu.py


@pytest.fixture(autouse=True)
def _healthy():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


# 160 heads: more than any SM count of 32-value slices, so the kernels that take 64 values, and more chunks
# than CTAs, so that one takes several; dv ends inside the first or second half of such a slice
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dv", [8, 24, 40, 72])
@pytest.mark.parametrize("state", [False, True])
def test_many_heads(dv, dtype, state):
    x, s0 = make(1, 130, 80, 2, 24, dv, dtype, seed=dv, state=state)
    gen = torch.Generator(device="cuda").manual_seed(1)
    go = torch.randn(x[2].shape, generator=gen, device="cuda").to(dtype)
    leaves = [t.clone().requires_grad_() for t in x]
    ref = [t.double().requires_grad_() for t in x]
    want, last = delta64(*ref, s0, 24 ** -0.5)
    o = fp.gated_delta(*leaves, initial_state=s0, return_state=state)
    if state:
        o, s1 = o
        assert off(s1, last) <= tolerance(torch.float32, True, FORWARD)
    assert off(o, want) <= tolerance(dtype, state, FORWARD)
    got = torch.autograd.grad(o, leaves, go)
    for name, g, w in zip("q k v log_decay beta".split(), got, torch.autograd.grad(want, ref, go.double())):
        assert off(g, w) <= tolerance(dtype, state, BACKWARD), name


@pytest.mark.parametrize("heads", [1, 160])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_value_spoils_what_follows_it_alone(bad, dtype, heads):
    x, s0 = make(1, 140, heads, 1, 32, 48, dtype, seed=3, state=True)
    clean, last = fp.gated_delta_forward(*x, initial_state=s0, return_state=True)
    x[2][0, 69, 0, 37] = bad
    o, s1 = fp.gated_delta_forward(*x, initial_state=s0, return_state=True)
    assert torch.isnan(o[0, 70:, 0, 37]).all() and not torch.isfinite(o[0, 69, 0, 37])
    assert not torch.isfinite(s1[0, 0, 37]).any()
    o[0, 69:, 0, 37] = clean[0, 69:, 0, 37]
    s1[0, 0, 37] = last[0, 0, 37]
    assert torch.equal(o, clean) and torch.equal(s1, last)


def _everything(x, s0, go, tokens):
    """Results of every entry point, as one list."""
    res = []
    for state in (None, s0):
        o, s1 = fp.gated_delta_forward(*x, initial_state=state, return_state=True)
        res += [o, s1, fp.gated_delta_forward(*x, initial_state=state, scale=0.5)]
        for eight in (False, True):
            leaves = [t.clone().requires_grad_() for t in x]
            held = None if state is None else state.clone().requires_grad_()
            o, s1 = fp.gated_delta(*leaves, initial_state=held, return_state=True, checkpoint8=eight)
            res += torch.autograd.grad((o, s1), leaves + ([] if held is None else [held]), (go, s0))
            o = fp.gated_delta(*leaves, checkpoint8=eight)
            res += [o.detach(), *torch.autograd.grad(o, leaves[2:4], go)]
    held = s0.clone()
    res += [fp.gated_delta_step(*(t[:, :1].contiguous() for t in x), held), held]
    codes, steps = fp.quantize8(x[2])
    res += [codes, steps, fp.dequantize8(codes, steps, x[2].dtype)]
    g, t = torch.sigmoid(tokens).requires_grad_(), tokens.clone().requires_grad_()
    y = fp.pscan_channels_last(g, t, checkpoint8=True)
    res += [y.detach(), *torch.autograd.grad(y, (g, t), torch.ones_like(y))]
    return res


@pytest.mark.parametrize("dtype", DTYPES)
def test_host_paths_agree(dtype, monkeypatch):
    # the compiled binding, the same with ranges for a profiler, and ctypes: the same bits
    x, s0 = make(2, 100, 2, 2, 40, 24, dtype, seed=4, state=True)
    gen = torch.Generator(device="cuda").manual_seed(2)
    go = torch.randn(x[2].shape, generator=gen, device="cuda").to(dtype)
    tokens = torch.randn(2, 100, 48, generator=gen, device="cuda").to(dtype)
    assert ops._EXT is not None
    want = _everything(x, s0, go, tokens)
    for m in (ops, delta):
        monkeypatch.setattr(m, "NVTX", True)
    ranges = _everything(x, s0, go, tokens)
    for m in (ops, delta, checkpoint8):
        monkeypatch.setattr(m, "_EXT", None)
    plain = _everything(x, s0, go, tokens)
    assert len(want) == len(ranges) == len(plain)
    for i, (a, b, c) in enumerate(zip(want, ranges, plain)):
        assert a.dtype == b.dtype == c.dtype
        assert torch.equal(a, b) and torch.equal(a, c), i


def test_captured_training_step_beside_an_eager_one():
    # an eager graph of the same leaves lives on while forward and backward are captured and replayed, on the
    # capturing stream (autograd refuses to capture for leaves whose live graph belongs to another stream)
    x, _ = make(2, 150, 1, 2, 64, 64, torch.bfloat16, seed=5)
    y, _ = make(2, 150, 1, 2, 64, 64, torch.bfloat16, seed=6)
    leaves = [t.clone().requires_grad_() for t in x]
    go = torch.randn_like(x[2])

    def step(eight):
        return torch.autograd.grad(fp.gated_delta(*leaves, checkpoint8=eight), leaves, go)

    side = torch.cuda.Stream()
    for eight in (False, True):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = fp.gated_delta(*leaves, checkpoint8=eight)
            step(eight)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(eight)
        with torch.cuda.stream(side):
            old = torch.autograd.grad(eager, leaves, go)
        torch.cuda.synchronize()
        with torch.no_grad():
            for a, b in zip(leaves, y):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step(eight)
        for a, w in zip(got, want):
            assert torch.equal(a, w)
        with torch.no_grad():
            for a, b in zip(leaves, x):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, w in zip(got, old):
            assert torch.equal(a, w)


def test_two_captured_calls_at_once():
    # graphs of two calls replayed on two streams together share nothing
    calls = []
    for seed, shape in ((7, (2, 500, 2, 1, 128, 128)), (8, (1, 900, 3, 1, 64, 64))):
        x, s0 = make(*shape, torch.bfloat16, seed=seed, state=True)
        go = torch.randn_like(x[2])
        work = lambda x=x, s0=s0, go=go: delta.gated_delta_backward(*x, go, s0, need_initial=True)  # noqa: E731
        want = [t.clone() for t in work()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = work()
        calls.append((graph, got, want, torch.cuda.Stream(), work))  # and the inputs, which the graph reads
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, _, _, stream, _ in calls:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _ in calls:
        for a, w in zip(got, want):
            assert torch.equal(a, w)


def test_a_state_changed_by_a_step_is_noticed():
    x, s0 = make(1, 66, 1, 1, 16, 16, torch.float32, seed=9, state=True)
    v = x[2].clone().requires_grad_()
    for binding in (True, False):
        with pytest.MonkeyPatch.context() as m:
            if not binding:
                for mod in (ops, delta):
                    m.setattr(mod, "_EXT", None)
            o = fp.gated_delta(x[0], x[1], v, x[3], x[4], initial_state=s0)
            fp.gated_delta_step(*(t[:, :1].contiguous() for t in x), s0)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                o.sum().backward()
    with torch.inference_mode():
        s1 = s0.clone()
        fp.gated_delta_step(*(t[:, :1].contiguous() for t in x), s1)
    fp.gated_delta_step(*(t[:, :1].contiguous() for t in x), s1)  # made there, used here



@pytest.mark.parametrize("heads", [2, 160])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "log_decay", "beta"])
def test_a_bad_value_reaches_no_earlier_token(which, dtype, heads):
    x, s0 = make(1, 140, heads, 1, 40, 24, dtype, seed=11, state=True)
    clean = fp.gated_delta_forward(*x, initial_state=s0)
    i = "q k v log_decay beta".split().index(which)
    x[i].view(1, 140, heads, -1)[0, 70, 1, -1] = math.nan
    o = fp.gated_delta_forward(*x, initial_state=s0)
    assert torch.equal(o[:, :70], clean[:, :70])
    assert torch.equal(o[:, :, 0], clean[:, :, 0]) and torch.equal(o[:, :, 2:], clean[:, :, 2:])
    assert torch.isnan(o[0, 70, 1]).all()
    if which == "q":
        assert torch.equal(o[:, 71:], clean[:, 71:])
    else:
        assert torch.isnan(o[0, 71:, 1]).all()


@pytest.mark.parametrize("binding", [True, False])
def test_second_derivatives_are_refused(binding, monkeypatch):
    if not binding:
        for m in (ops, delta, checkpoint8):
            monkeypatch.setattr(m, "_EXT", None)
    x, s0 = make(1, 66, 1, 1, 16, 16, torch.float32, seed=12, state=True)
    leaves = [t.requires_grad_() for t in (*x, s0)]
    o = fp.gated_delta(*leaves[:5], initial_state=leaves[5])
    plain = torch.autograd.grad(o.square().sum(), leaves, retain_graph=True)
    grads = torch.autograd.grad(o.square().sum(), leaves, create_graph=True)
    for a, b in zip(plain, grads):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="gated_delta is differentiable once"):
        sum(t.sum() for t in grads).backward()  # (grad() finds the inputs unused, and says so)
    g = torch.rand(1, 40, 8, device="cuda").requires_grad_()
    y = fp.pscan_channels_last(g, torch.ones_like(g), checkpoint8=True)
    d, = torch.autograd.grad(y.sum(), g, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()
