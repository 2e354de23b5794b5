"""8-bit activation checkpoints on the GPU: the format, and their use in the channel-last scan's backward."""
import math

import numpy as np
import pytest
import torch

import fpscan_b200 as fp
from fpscan_b200 import _lib, ops
from delta_ref import delta64, half_step, off, tolerance
from guard import guarded

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _healthy():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def codes64(x, most):
    """Nearest multiple of most / 127, ties to even, in 64 bits; 0 where most is 0 or not finite."""
    fine = (most > 0) & np.isfinite(most)
    return np.where(fine, np.rint(np.where(fine, x, 0.0) * 127.0 / np.where(fine, most, 1.0)), 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 63, 64, 65, 127, 1000, 4097, 300001])
def test_quantize8(n, dtype):
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, generator=gen, device="cuda") * torch.exp(3 * torch.randn(n, generator=gen, device="cuda"))
    x = x.to(dtype)
    codes, steps = fp.quantize8(x)
    assert codes.dtype == torch.int8 and codes.shape == x.shape and steps.shape == ((n + 63) // 64,)
    x64 = np.zeros((n + 63) // 64 * 64)
    x64[:n] = x.double().cpu().numpy()
    x64 = x64.reshape(-1, 64)
    most = np.abs(x64).max(1, keepdims=True)
    want = codes64(x64, most).reshape(-1)[:n]
    got = codes.cpu().numpy().astype(np.float64)
    if dtype == torch.float32:  # product and quotient are rounded: a value next to a tie may go either way
        r = (x64 * 127.0 / np.where(most > 0, most, 1.0)).reshape(-1)[:n]
        far = np.abs(np.abs(r - np.floor(r)) - 0.5) > 127 * 2.0 ** -22
        assert (got[far] == want[far]).all() and np.abs(got - want).max() <= 1
    else:
        assert (got == want).all()
    step = most[:, 0] / 127
    assert np.allclose(steps.cpu().numpy(), step, rtol=2.0 ** -23, atol=2.0 ** -149)
    for to in DTYPES:
        back = fp.dequantize8(codes, steps, to)
        assert back.dtype == to
        stands = (codes.double() * steps.double().repeat_interleave(64)[:n])
        # the same draws in fp16 hold infinities themselves: their blocks read back as NaN
        assert torch.equal(torch.isnan(back), torch.isnan(stands))
        back, stands = back[~torch.isnan(back)], stands[~torch.isnan(stands)]
        eps = half_step(to) + 2.0 ** -24
        # fp16 ends at 65504: half a step past it (65520) and beyond, as exp(3 x 4.5) of the largest of 300001
        # draws is, the nearest value is infinity
        past = stands.abs() >= torch.finfo(to).max * (1 + half_step(to))
        assert torch.equal(torch.isinf(back), past) and (back.sign() == stands.sign())[past].all()
        back, stands = back[~past], stands[~past]
        assert ((back.double() - stands).abs() <= eps * stands.abs() + 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize8_odd_blocks(dtype):
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = torch.zeros(8, 64, dtype=dtype, device="cuda")
    x[1, 5], x[1, 6] = big, -big / 2
    x[2, 0], x[2, 1] = tiny, -tiny
    x[3] = 1.0
    x[4, 3] = math.inf
    x[5, 9] = math.nan
    x[6, 0], x[6, 1] = 2.0, 1.0  # half of the largest: 63.5, a tie
    x[7, 63] = -3.0
    codes, steps = fp.quantize8(x)
    back = fp.dequantize8(codes, steps, dtype).cpu()
    c = codes.cpu()
    assert (c[0] == 0).all() and (back[0] == 0).all()
    assert c[1, 5] == 127 and c[1, 6] in (-63, -64) and (c[1, :5] == 0).all()
    assert c[2, 0] == 127 and c[2, 1] == -127
    assert (c[3] == 127).all()
    assert torch.isnan(back[4]).all() and torch.isnan(back[5]).all()
    assert c[6, 0] == 127 and c[6, 1] == 64
    assert c[7, 63] == -127 and (c[7, :63] == 0).all()
    for i in (0, 3, 6, 7):
        assert ((back[i].double() - x[i].double().cpu()).abs()
                <= steps[i].double().cpu() / 2 + half_step(dtype) * 3).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_written_outside(dtype):
    for n in (1, 65, 1001):
        x = torch.randn(n, device="cuda").to(dtype)
        code, steps = guarded(((n + 3) // 4,), torch.float32), guarded(((n + 63) // 64,), torch.float32)
        ops._launch(0, "fpscan_quantize8", x.data_ptr(), code.out.data_ptr(), steps.out.data_ptr(), n,
                    ops.DTYPE_CODES[dtype])
        code.check("codes")
        steps.check("steps")
        out = guarded((n,), dtype)
        ops._launch(0, "fpscan_dequantize8", code.out.data_ptr(), steps.out.data_ptr(), out.out.data_ptr(), n,
                    ops.DTYPE_CODES[dtype])
        out.check("values")
        assert torch.isfinite(out.out).all()


def _scan_inputs(b, l, d, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda: torch.randn(b, l, d, generator=gen, device="cuda")  # noqa: E731
    return torch.sigmoid(r() + 2).to(dtype), r().to(dtype), r().to(dtype)


def _kept(y):
    """What the 8-bit checkpoint of y stands for, in 64 bits: blocks of 8 timesteps x 16 bytes of channels."""
    b, l, d = y.shape
    vec = 16 // y.element_size()
    z = torch.zeros(b, (l + 7) // 8 * 8, d, dtype=torch.float64, device=y.device)
    z[:, :l] = y.double()
    z = z.view(b, -1, 8, d // vec, vec)
    most = z.abs().amax((2, 4), keepdim=True)
    c = torch.where(most > 0, torch.round(z * 127 / most), 0.0)
    return (c * (most / 127)).view(b, -1, d)[:, :l]


# few columns (cut along the time axis: several segments, and too short to cut) and many; ragged in both
SCANS = [(1, 1, 8), (2, 7, 24), (1, 8, 64), (1, 9, 72), (1, 255, 136), (1, 257, 64), (2, 1030, 72), (1, 5000, 136),
         (3, 300, 3080), (130, 20, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SCANS)
def test_scan_checkpoint8(shape, dtype):
    g, x, go = _scan_inputs(*shape, dtype, seed=sum(shape))
    a, b = (t.clone().requires_grad_() for t in (g, x))
    y = fp.pscan_channels_last(a, b, checkpoint8=True)
    dg, dx = torch.autograd.grad(y, (a, b), go)
    c, d = (t.clone().requires_grad_() for t in (g, x))
    plain = fp.pscan_channels_last(c, d)
    _, dx0 = torch.autograd.grad(plain, (c, d), go)
    assert torch.equal(y, plain) and torch.equal(dx, dx0)
    # dgates[t] = dtokens[t] (before its rounding) x kept y[t-1]: dtokens in 64 bits
    h, d64 = torch.zeros_like(go[:, 0], dtype=torch.float64), torch.zeros(shape, dtype=torch.float64, device="cuda")
    for t in range(shape[1] - 1, -1, -1):
        h = go[:, t].double() + (g[:, t + 1].double() * h if t + 1 < shape[1] else 0)
        d64[:, t] = h
    want = torch.zeros_like(d64)
    want[:, 1:] = d64[:, 1:] * _kept(y)[:, :-1]
    if dtype == torch.float32:  # codes next to a tie may go either way: one step in about 10^4 values
        assert off(dg, want) <= 2.0 ** -12
    else:
        assert off(dg, want) <= half_step(dtype) + 2.0 ** -16
    assert (dg[:, 0] == 0).all()


def test_scan_checkpoint8_nothing_written_outside():
    for dtype in DTYPES:
        for b, l, d in ((1, 300, 72), (130, 13, 72), (2, 1100, 72)):
            g, x, go = _scan_inputs(b, l, d, dtype)
            code = ops.DTYPE_CODES[dtype]
            y = guarded((b, l, d), dtype)
            codes = guarded((b * l * 80 // 4,), torch.float32)
            steps = guarded((b, (l + 7) // 8, d * x.element_size() // 16), torch.float32)
            ws = guarded((_lib.load().fpscan_cl_workspace_bytes(b, l, d, code, 0) // 4,), torch.float32)
            ops._launch(0, "fpscan_scan_fwd_cl8", g.data_ptr(), x.data_ptr(), y.out.data_ptr(),
                        codes.out.data_ptr(), steps.out.data_ptr(), b, l, d, code, ws.out.data_ptr(),
                        ws.out.numel() * 4)
            dg, dx = guarded((b, l, d), dtype), guarded((b, l, d), dtype)
            ops._launch(0, "fpscan_scan_bwd_cl8", g.data_ptr(), codes.out.data_ptr(), steps.out.data_ptr(),
                        go.data_ptr(), dg.out.data_ptr(), dx.out.data_ptr(), b, l, d, code, ws.out.data_ptr(),
                        ws.out.numel() * 4)
            for t in (y, codes, steps, ws, dg, dx):
                t.check(f"{dtype} {b} {l} {d}")
            assert torch.isfinite(steps.out).all() and torch.isfinite(dg.out).all()


def test_scan_checkpoint8_infinities_stay_in_their_blocks():
    g, x, go = _scan_inputs(1, 64, 64, torch.float32)
    x[0, 20, 3] = math.inf
    a, b = g.clone().requires_grad_(), x.clone().requires_grad_()
    dg, _ = torch.autograd.grad(fp.pscan_channels_last(a, b, checkpoint8=True), (a, b), go)
    assert torch.isfinite(dg[0, :, 4:]).all() and torch.isfinite(dg[0, :17]).all()
    assert torch.isnan(dg[0, 21:, 3]).all()


def test_scan_checkpoint8_graphs_share_nothing():
    # two graphs captured on one stream, replayed at once on two
    sets = [_scan_inputs(1, 4000, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    want, graphs, got = [], [], []
    for g, x, go in sets:
        a, b = g.clone().requires_grad_(), x.clone().requires_grad_()
        y = fp.pscan_channels_last(a, b, checkpoint8=True)
        want.append([y.detach().clone(), *(t.clone() for t in torch.autograd.grad(y, (a, b), go))])
    torch.cuda.synchronize()
    for g, x, go in sets:
        a, b = g.clone().requires_grad_(), x.clone().requires_grad_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp.pscan_channels_last(a, b, checkpoint8=True)
            got.append([y, *torch.autograd.grad(y, (a, b), go)])
        graphs.append(graph)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for graph, stream in zip(graphs, s):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for p, w in zip(got, want):
        for a, b in zip(p, w):
            assert torch.equal(a, b)


def test_a_layer_of_both():
    # values mixed along time by the channel-last scan, then the delta rule, both with 8-bit checkpoints;
    # gradients against the same layer in 64 bits.  Off by the checkpoints' half steps: 2^-8 of a block's
    # largest magnitude, about three times its rms, in each factor of a product, and the layer's bf16 values
    b, l, h, dk, dv, dtype = 2, 190, 4, 32, 32, torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)  # noqa: E731
    leaves = [t.to(dtype).requires_grad_() for t in (
        torch.sigmoid(r(b, l, h * dv) + 1), r(b, l, h * dv), unit(r(b, l, h, dk)), unit(r(b, l, h, dk)),
        -torch.nn.functional.softplus(r(b, l, h)), torch.sigmoid(r(b, l, h)))]
    gates, tokens, q, k, g, beta = leaves
    v = fp.pscan_channels_last(gates, tokens, checkpoint8=True).view(b, l, h, dv)
    o = fp.gated_delta(q, k, v, g, beta, checkpoint8=True)
    go = r(b, l, h, dv).to(dtype)
    got = torch.autograd.grad(o, leaves, go)
    ref = [t.detach().double().requires_grad_() for t in leaves]
    y, ys = torch.zeros(b, h * dv, dtype=torch.float64, device="cuda"), []
    for t in range(l):
        y = ref[1][:, t] + (ref[0][:, t] * y if t else 0)
        ys.append(y)
    want, _ = delta64(ref[2], ref[3], torch.stack(ys, 1).view(b, l, h, dv), ref[4], ref[5], None, dk ** -0.5)
    assert off(o, want) <= 2 * half_step(dtype) + tolerance(dtype, False, 6)
    for a, w in zip(got, torch.autograd.grad(want, ref, go.double())):
        assert off(a, w) <= 4 * 3 * 2.0 ** -8 + tolerance(dtype, False, 14)


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    with pytest.raises(RuntimeError, match="contiguous"):
        fp.quantize8(x.t())
    with pytest.raises(RuntimeError, match="float"):
        fp.quantize8(x.int())
    codes, steps = fp.quantize8(x)
    with pytest.raises(RuntimeError, match="steps"):
        fp.dequantize8(codes, steps[:-1])
    with pytest.raises(RuntimeError, match="codes"):
        fp.dequantize8(codes.int(), steps)
    with pytest.raises(RuntimeError, match="dtype"):
        fp.dequantize8(codes, steps, torch.float64)
    with pytest.raises(RuntimeError, match="dim"):
        fp.pscan_channels_last(x.view(1, 4, 64)[..., :3].contiguous(), x.view(1, 4, 64)[..., :3].contiguous(),
                               checkpoint8=True)
    assert fp.quantize8(x[:0].contiguous())[0].shape == (0, 64)
