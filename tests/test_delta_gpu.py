"""Gated delta rule on the GPU against the recurrence in 64 bits."""
import math

import pytest
import torch

import fpscan_b200 as fp
from fpscan_b200 import _lib, delta, ops
from delta_ref import delta64, half_step, make, off, tolerance
from guard import guarded

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# batch, seqlen, key heads, heads per key head, dk, dv: one token, a chunk's ends and its neighbours, odd
# counts of everything, channels off the padded sizes, several slices of values
SHAPES = [(1, 1, 1, 1, 8, 8), (2, 2, 1, 1, 128, 128), (2, 63, 2, 1, 16, 24), (1, 64, 1, 2, 64, 64),
          (1, 65, 1, 3, 72, 136), (3, 130, 2, 2, 40, 72), (1, 200, 1, 1, 128, 264), (2, 257, 3, 1, 128, 16)]
FORWARD, BACKWARD = 6, 14  # products one after another: K S, N, P / the state, and into the next chunk; twice more


@pytest.fixture(autouse=True)
def _healthy():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("state", [False, True])
def test_forward(shape, dtype, state):
    x, s0 = make(*shape, dtype, seed=sum(shape), state=state)
    scale = 0.37
    want, last = delta64(*x, s0, scale)
    if state:
        o, s1 = fp.gated_delta_forward(*x, initial_state=s0, scale=scale, return_state=True)
        assert s1.dtype == torch.float32
        assert off(s1, last) <= tolerance(torch.float32, True, FORWARD)
    else:
        o = fp.gated_delta_forward(*x, scale=scale)
    assert o.dtype == dtype and o.shape == x[2].shape
    assert off(o, want) <= tolerance(dtype, state, FORWARD)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("state", [False, True])
def test_gradients(shape, dtype, state):
    x, s0 = make(*shape, dtype, seed=1 + sum(shape), state=state)
    b, l, h, dv = x[2].shape
    gen = torch.Generator(device="cuda").manual_seed(5)
    go = torch.randn(x[2].shape, generator=gen, device="cuda").to(dtype)
    leaves = [t.clone().requires_grad_() for t in x] + ([s0.clone().requires_grad_()] if state else [])
    ref = [t.double().detach().clone().requires_grad_() for t in leaves]
    want, last = delta64(*ref, scale=0.5) if not state else delta64(*ref[:5], ref[5], 0.5)
    if state:
        gs = 0.2 * torch.randn(b, h, dv, x[0].shape[3], generator=gen, device="cuda")
        o, s1 = fp.gated_delta(*leaves[:5], initial_state=leaves[5], scale=0.5, return_state=True)
        got = torch.autograd.grad((o, s1), leaves, (go, gs))
        wanted = torch.autograd.grad((want, last), ref, (go.double(), gs.double()))
    else:
        got = torch.autograd.grad(fp.gated_delta(*leaves, scale=0.5), leaves, go)
        wanted = torch.autograd.grad(want, ref, go.double())
    for name, a, w, leaf in zip(("q", "k", "v", "log_decay", "beta", "state"), got, wanted, leaves):
        assert a.dtype == leaf.dtype and a.shape == leaf.shape
        # dlog_decay is a sum of up to 64 terms of either sign that may cancel: its terms' size counts
        slack = 8 if name in ("log_decay", "beta") else 1
        tol = half_step(a.dtype) + slack * (tolerance(dtype, state, BACKWARD) - half_step(dtype))
        if w.norm() == 0:  # nothing reaches log_decay of a lone first token
            assert a.double().norm() <= tol * go.double().norm(), name
        else:
            assert off(a, w) <= tol, name


@pytest.mark.parametrize("dtype", DTYPES)
def test_resets_and_idle_writes(dtype):
    # resets at a chunk's first, last and inner tokens, several in a row; beta of exactly 0; strong decays
    x, s0 = make(2, 200, 2, 2, 64, 64, dtype, seed=3, resets=0.05, zero_beta=0.3, state=True)
    for t in (0, 63, 64, 127, 130, 131):
        x[3][:, t, 0] = -math.inf
    x[3][:, 20:24] = torch.finfo(dtype).min
    x[3][:, 30:34] = -80.0
    leaves = [t.clone().requires_grad_() for t in x] + [s0.clone().requires_grad_()]
    ref = [t.detach().double().requires_grad_() for t in leaves]
    want, last = delta64(*ref[:5], ref[5], 0.2)
    o, s1 = fp.gated_delta(*leaves[:5], initial_state=leaves[5], scale=0.2, return_state=True)
    go = torch.randn_like(o)
    gs = torch.randn_like(s1)
    got = torch.autograd.grad((o, s1), leaves, (go, gs))
    wanted = torch.autograd.grad((want, last), ref, (go.double(), gs.double()))
    assert off(o, want) <= tolerance(dtype, True, FORWARD)
    assert off(s1, last) <= tolerance(torch.float32, True, FORWARD)
    for name, a, w in zip(("q", "k", "v", "log_decay", "beta", "state"), got, wanted):
        assert torch.isfinite(a).all(), name
        slack = 8 if name in ("log_decay", "beta") else 1
        tol = half_step(a.dtype) + slack * (tolerance(dtype, True, BACKWARD) - half_step(dtype))
        assert off(a, torch.nan_to_num(w)) <= tol, name
    assert (got[3][torch.isinf(x[3])] == 0).all()


def test_reset_is_a_new_sequence():
    # a sequence packed behind another gives, bit for bit when chunk-aligned, what it gives alone
    x, _ = make(1, 192, 2, 1, 64, 64, torch.bfloat16, seed=4)
    x[3][:, 128] = -math.inf
    packed = fp.gated_delta_forward(*x)
    alone = fp.gated_delta_forward(*(t[:, 128:].contiguous() for t in x))
    assert torch.equal(packed[:, 128:], alone)


def test_all_reset_and_all_idle():
    x, _ = make(1, 70, 1, 1, 32, 32, torch.float32, seed=5)
    x[3].fill_(-math.inf)
    o = fp.gated_delta_forward(*x, scale=1.0)
    want, _ = delta64(*x)
    assert off(o, want) <= tolerance(torch.float32, True, FORWARD)
    x[4].zero_()
    o, s = fp.gated_delta_forward(*x, return_state=True)
    assert (o == 0).all() and (s == 0).all()


def test_zero_keys_and_zero_gradient():
    x, s0 = make(1, 100, 1, 2, 32, 40, torch.float32, seed=6, state=True)
    x[1].zero_()
    leaves = [t.clone().requires_grad_() for t in x]
    o = fp.gated_delta(*leaves, initial_state=s0)
    want, _ = delta64(*x, s0, 32 ** -0.5)
    assert off(o, want) <= tolerance(torch.float32, True, FORWARD)
    for g in torch.autograd.grad(o, leaves, torch.zeros_like(o)):
        assert (g == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_differences(dtype):
    # the slope along a random direction, by central differences of the 64-bit rule at the kernel's inputs
    x, _ = make(1, 90, 2, 1, 32, 32, dtype, seed=7)
    gen = torch.Generator(device="cuda").manual_seed(8)
    go = torch.randn(x[2].shape, generator=gen, device="cuda").to(dtype)
    leaves = [t.clone().requires_grad_() for t in x]
    got = torch.autograd.grad(fp.gated_delta(*leaves, scale=1.0), leaves, go)
    for i in range(5):
        d = torch.randn(x[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-4
        f = []
        for sign in (1, -1):
            y = [t.double() for t in x]
            y[i] = y[i] + sign * h * d
            f.append((delta64(*y)[0] * go.double()).sum())
        slope = (f[0] - f[1]) / (2 * h)
        size = got[i].double().norm() * d.norm()  # differences are off by h^2: far below
        assert abs(slope - (got[i].double() * d).sum()) <= 8 * tolerance(dtype, False, BACKWARD) * size + 1e-6 * size


def test_shared_key_heads_are_a_sum():
    x, _ = make(2, 100, 2, 3, 64, 32, torch.float32, seed=9)
    go = torch.randn_like(x[2])
    leaves = [t.clone().requires_grad_() for t in x]
    got = torch.autograd.grad(fp.gated_delta(*leaves), leaves, go)
    wide = [x[0].repeat_interleave(3, 2), x[1].repeat_interleave(3, 2), *x[2:]]
    wide = [t.contiguous().requires_grad_() for t in wide]
    one = torch.autograd.grad(fp.gated_delta(*wide), wide, go)
    for a, w in zip(got[:2], one[:2]):
        w = w.view(2, 100, 2, 3, 64)
        assert torch.equal(a, (w[:, :, :, 0] + w[:, :, :, 1]) + w[:, :, :, 2])  # in this order
    for a, w in zip(got[2:], one[2:]):
        assert torch.equal(a, w)


def test_same_bits_twice():
    x, s0 = make(2, 300, 2, 2, 128, 128, torch.bfloat16, seed=10, state=True)
    go = torch.randn_like(x[2])

    def once():
        leaves = [t.clone().requires_grad_() for t in x] + [s0.clone().requires_grad_()]
        o, s1 = fp.gated_delta(*leaves[:5], initial_state=leaves[5], return_state=True)
        return [o, s1, *torch.autograd.grad((o, s1), leaves, (go, torch.ones_like(s1)))]

    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES[:4] + [(3, 5, 2, 3, 96, 40), (65, 1, 1, 2, 120, 104)])
def test_step(shape, dtype):
    x, s0 = make(*shape, dtype, seed=11, state=True)
    want, last = delta64(*x, s0, 0.7)
    state = s0.clone()
    at = state.data_ptr()
    o = fp.gated_delta_step(*x, state, scale=0.7)
    assert state.data_ptr() == at
    # plain fp32 sums of dk terms, l tokens one after another
    fp32 = (shape[4] + shape[1]) * 2 ** -24
    assert off(state, last) <= fp32
    assert off(o, want) <= half_step(dtype) + 2 * fp32
    out = torch.empty_like(x[2])
    again = s0.clone()
    assert fp.gated_delta_step(*x, again, scale=0.7, out=out) is out
    assert torch.equal(out, o) and torch.equal(again, state)


def test_step_resets_and_strong_decay():
    x, s0 = make(4, 3, 1, 2, 64, 64, torch.float32, seed=12, state=True)
    x[3][0] = -math.inf
    x[3][1, 1] = -200.0
    want, last = delta64(*x, s0, 1.0)
    o = fp.gated_delta_step(*x, s0, scale=1.0)
    assert off(o, want) <= 80 * 2 ** -24 and off(s0, last) <= 80 * 2 ** -24


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_then_tokens(dtype):
    # a server's run: prompts of a ragged length, then tokens one and three at a time
    x, s0 = make(3, 150, 2, 2, 64, 72, dtype, seed=13, state=True)
    want, last = delta64(*x, s0, 64 ** -0.5)
    cut = lambda i, j: [t[:, i:j].contiguous() for t in x]  # noqa: E731
    o, state = fp.gated_delta_forward(*cut(0, 131), initial_state=s0, return_state=True)
    parts = [o]
    for i in range(131, 141):
        parts.append(fp.gated_delta_step(*cut(i, i + 1), state))
    for i in range(141, 150, 3):
        parts.append(fp.gated_delta_step(*cut(i, i + 3), state))
    assert off(torch.cat(parts, 1), want) <= tolerance(dtype, True, 2 * FORWARD)
    assert off(state, last) <= tolerance(torch.float32, True, 2 * FORWARD)


def test_heads_and_sequences_do_not_mix():
    x, s0 = make(2, 80, 2, 1, 64, 64, torch.bfloat16, seed=14, state=True)
    clean = fp.gated_delta_forward(*x, initial_state=s0)
    x[2][0, 3, 1, 5] = math.nan
    x[1][1, 70, 0, 0] = math.inf
    o = fp.gated_delta_forward(*x, initial_state=s0)
    assert torch.equal(o[0, :, 0], clean[0, :, 0]) and torch.equal(o[1, :, 1], clean[1, :, 1])
    assert torch.equal(o[0, :3, 1], clean[0, :3, 1])  # nor tokens before it
    assert torch.isnan(o[0, 3:, 1, 5]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_written_outside(dtype):
    b, l, hk, h, dk, dv = 2, 67, 1, 3, 40, 24
    x, s0 = make(b, l, hk, h // hk, dk, dv, dtype, seed=15, state=True)
    go = torch.randn_like(x[2])
    sizes = (b, l, hk, h, dk, dv)
    code = ops.DTYPE_CODES[dtype]
    ptr = [t.data_ptr() for t in x]
    shapes = [x[0].shape, x[1].shape, x[2].shape, x[3].shape, x[4].shape]
    for wide in (0, 1):
        o, fin = guarded(x[2].shape, dtype), guarded((b, h, dv, dk), torch.float32)
        ws = guarded((_lib.load().fpscan_delta_workspace_bytes(*sizes, code, wide, 0) // 4,), torch.float32)
        ops._launch(0, "fpscan_delta_fwd", *ptr, s0.data_ptr(), o.out.data_ptr(), fin.out.data_ptr(), *sizes,
                    0.5, code, wide, ws.out.data_ptr(), ws.out.numel() * 4)
        for g in (o, fin, ws):
            g.check("forward")
        assert torch.isfinite(o.out).all() and torch.isfinite(fin.out).all()
        grads = [guarded(s, dtype) for s in shapes]
        di = guarded((b, h, dv, dk), torch.float32)
        ws = guarded((_lib.load().fpscan_delta_workspace_bytes(*sizes, code, wide, 1) // 4,), torch.float32)
        ops._launch(0, "fpscan_delta_bwd", *ptr, s0.data_ptr(), go.data_ptr(), s0.data_ptr(),
                    *(g.out.data_ptr() for g in grads), di.out.data_ptr(), *sizes, 0.5, code, wide,
                    ws.out.data_ptr(), ws.out.numel() * 4)
        for g in (*grads, di, ws):
            g.check("backward")
        for g in (*grads, di):
            assert torch.isfinite(g.out).all()
    o, fin = guarded(x[2].shape, dtype), guarded((b, h, dv, dk), torch.float32)
    ops._launch(0, "fpscan_delta_step", *ptr, s0.data_ptr(), o.out.data_ptr(), fin.out.data_ptr(), *sizes, 0.5,
                code)
    o.check("step")
    fin.check("step")
    assert torch.isfinite(o.out).all() and torch.isfinite(fin.out).all()


def test_long_batch_in_passes():
    # more sequences than the workspace's bound takes at once: same bits as each by itself
    x, _ = make(36, 1100, 1, 16, 128, 128, torch.bfloat16, seed=16)
    go = torch.randn_like(x[2])
    grads = delta.gated_delta_backward(*x, go)[:5]
    for i in (0, 17, 35):
        one = [t[i:i + 1].contiguous() for t in x]
        for a, w in zip(grads, delta.gated_delta_backward(*one, go[i:i + 1].contiguous())[:5]):
            assert torch.equal(a[i:i + 1], w)


def test_offsets_past_32_bits():
    # 2^31 values of v and more: the last sequence must be its own
    b, l, h, dv = 33, 4096, 128, 128
    assert b * l * h * dv > 2 ** 31
    x, _ = make(1, l, 1, h, 16, dv, torch.bfloat16, seed=17)
    big = [t.expand(b, *t.shape[1:]).contiguous() for t in x]
    o = fp.gated_delta_forward(*big)
    one = fp.gated_delta_forward(*x)
    assert torch.equal(o[-1:], one) and torch.equal(o[16:17], one)


def test_other_stream_and_two_at_once():
    x, s0 = make(2, 500, 2, 1, 128, 128, torch.bfloat16, seed=18, state=True)
    y, t0 = make(1, 700, 4, 1, 64, 64, torch.float16, seed=19, state=True)
    want = fp.gated_delta_forward(*x, initial_state=s0), fp.gated_delta_forward(*y, initial_state=t0)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(a):
            o = fp.gated_delta_forward(*x, initial_state=s0)
        with torch.cuda.stream(b):
            p = fp.gated_delta_forward(*y, initial_state=t0)
    torch.cuda.synchronize()
    assert torch.equal(o, want[0]) and torch.equal(p, want[1])


def test_graph_replay():
    # a training step and a serving step, captured once and replayed on new inputs
    x, s0 = make(2, 150, 2, 2, 64, 64, torch.bfloat16, seed=20, state=True)
    y, t0 = make(2, 150, 2, 2, 64, 64, torch.bfloat16, seed=21, state=True)
    go = torch.randn_like(x[2])

    def work(x, s0):
        o, s1 = fp.gated_delta_forward(*x, initial_state=s0, return_state=True)
        grads = delta.gated_delta_backward(*x, go, s0, need_initial=True)
        p = fp.gated_delta_step(*(t[:, :1].contiguous() for t in x), s1)
        return [o, s1, p, *grads]

    want = [t.clone() for t in work(y, t0)]
    held, h0 = [t.clone() for t in x], s0.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work(held, h0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(held, h0)
    for a, b in zip(held + [h0], y + [t0]):
        a.copy_(b)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for a, w in zip(got, want):
            assert torch.equal(a, w)


def test_backward_of_parts():
    # one of the two results used, or only some inputs' gradients wanted; a broadcast gradient
    x, s0 = make(1, 70, 1, 2, 32, 32, torch.float32, seed=22, state=True)
    v = x[2].clone().requires_grad_()
    o, s1 = fp.gated_delta(x[0], x[1], v, x[3], x[4], initial_state=s0, return_state=True)
    ref = x[2].double().requires_grad_()
    want, last = delta64(x[0], x[1], ref, x[3], x[4], s0, 32 ** -0.5)
    tol = tolerance(torch.float32, True, BACKWARD)
    g, = torch.autograd.grad(s1.sum(), v, retain_graph=True)
    assert off(g, torch.autograd.grad(last.sum(), ref, retain_graph=True)[0]) <= tol
    g, = torch.autograd.grad(o.sum(), v)
    assert off(g, torch.autograd.grad(want.sum(), ref)[0]) <= tol


def test_state_of_another_type():
    x, s0 = make(1, 66, 1, 1, 16, 16, torch.float32, seed=23, state=True)
    s = s0.bfloat16().requires_grad_()
    o = fp.gated_delta(*x, initial_state=s)
    assert torch.equal(o, fp.gated_delta_forward(*x, initial_state=s.detach().float()))
    g, = torch.autograd.grad(o.sum(), s)
    assert g.dtype == torch.bfloat16


def test_empty_batch():
    x, _ = make(1, 5, 1, 1, 16, 16, torch.float32)
    none = [t[:0].contiguous().requires_grad_() for t in x]
    o = fp.gated_delta(*none)
    assert o.shape == (0, 5, 1, 16)
    assert torch.autograd.grad(o.sum(), none[2])[0].shape == none[2].shape
    assert fp.gated_delta_step(*(t.detach() for t in none), torch.empty(0, 1, 16, 16, device="cuda")).numel() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_checkpoint8_gradients_are_those_at_the_kept_values(dtype):
    x, s0 = make(2, 140, 2, 2, 64, 72, dtype, seed=24, state=True)
    go = torch.randn_like(x[2])
    leaves = [t.clone().requires_grad_() for t in x]
    o = fp.gated_delta(*leaves, initial_state=s0, checkpoint8=True)
    assert torch.equal(o, fp.gated_delta(*x, initial_state=s0))
    got = torch.autograd.grad(o, leaves, go)
    kept = [fp.dequantize8(*fp.quantize8(t), dtype) for t in x[:3]]
    want = delta.gated_delta_backward(*kept, *x[3:], go, s0)
    for a, w in zip(got, want):
        assert torch.equal(a, w)


def test_refusals():
    x, s0 = make(1, 4, 2, 1, 16, 16, torch.float32, state=True)
    for change, match in ((lambda y: y.__setitem__(0, y[0][..., :12].contiguous()), "same shape"),
                          (lambda y: y.__setitem__(3, y[3][:, :, :1].contiguous()), "log_decay"),
                          (lambda y: y.__setitem__(4, y[4].half()), "dtype"),
                          (lambda y: y.__setitem__(2, y[2].transpose(1, 2)), "contiguous|agree"),
                          (lambda y: y.__setitem__(2, y[2].cpu()), "CUDA")):
        y = list(x)
        change(y)
        with pytest.raises(RuntimeError, match=match):
            fp.gated_delta(*y)
    with pytest.raises(RuntimeError, match="state"):
        fp.gated_delta_forward(*x, initial_state=s0[:, :1])
    with pytest.raises(RuntimeError, match="state"):
        fp.gated_delta_step(*x, s0.half())
    with pytest.raises(RuntimeError, match="state"):
        fp.gated_delta_step(*x, s0.transpose(2, 3))
    with pytest.raises(RuntimeError, match="overlaps"):
        fp.gated_delta_forward(*x, out=x[2])
    big = torch.zeros(4 * 2 * 16 + 1, device="cuda")
    odd = big[1:].view(1, 4, 2, 16)
    with pytest.raises(RuntimeError, match="aligned"):
        fp.gated_delta_forward(*x[:2], odd, *x[3:])
