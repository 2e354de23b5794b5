"""The bounds-checking build (libfpscan_b200_debug.so) over the gated delta rule, the 8-bit scan and the 8-bit
format: at edge shapes, a clean status and the release build's bits."""
import ctypes
import os

import pytest
import torch

from fpscan_b200 import _lib, build
from delta_ref import make

pytestmark = pytest.mark.gpu
CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


@pytest.fixture(scope="module")
def dbg():
    if not os.path.exists(build.DEBUG_LIB_PATH):
        pytest.skip("bounds-checking build not present (fpscan_b200.build.build_debug)")
    return _lib.open_library(build.DEBUG_LIB_PATH)


def _status(lib):
    v = ctypes.c_uint(0)
    torch.cuda.synchronize()
    _lib.check(lib.fpscan_device_status(ctypes.byref(v), 1), "fpscan_device_status")
    return int(v.value)


def _s():
    return torch.cuda.current_stream().cuda_stream


def _ptrs(ts):
    return [0 if t is None else t.data_ptr() for t in ts]


def _same(a, b):
    for x, y in zip(a, b):
        assert torch.equal(x, y)


# batch, seqlen, key heads, heads per key head, dk, dv: one token; odd sizes of everything; a chunk's end; 64 values
# a CTA and several chunks to one
@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 8, 8), (2, 67, 1, 3, 40, 24), (1, 128, 2, 1, 128, 136),
                                   (1, 130, 80, 2, 24, 40)])
def test_delta_rule(dbg, shape, dtype):
    b, l, hk, group, dk, dv = shape
    h, code = hk * group, CODES[dtype]
    sizes = (b, l, hk, h, dk, dv)
    x, s0 = make(*shape, dtype, seed=sum(shape), state=True)
    go = torch.randn_like(x[2])

    def run(lib, wide):
        state = s0 if wide else None
        o, fin = torch.zeros_like(x[2]), torch.zeros_like(s0)
        n = lib.fpscan_delta_workspace_bytes(*sizes, code, wide, 0)
        ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
        _lib.check(lib.fpscan_delta_fwd(*_ptrs([*x, state, o, fin if wide else None]), *sizes, 0.5, code, wide,
                                        ws.data_ptr(), n, _s()), "delta_fwd")
        grads, di = [torch.zeros_like(t) for t in x], torch.zeros_like(s0)
        n = lib.fpscan_delta_workspace_bytes(*sizes, code, wide, 1)
        ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
        _lib.check(lib.fpscan_delta_bwd(*_ptrs([*x, state, go, state, *grads, di if wide else None]), *sizes, 0.5,
                                        code, wide, ws.data_ptr(), n, _s()), "delta_bwd")
        p, held = torch.zeros_like(x[2]), s0.clone()
        _lib.check(lib.fpscan_delta_step(*_ptrs([*x, held, p, held]), *sizes, 0.5, code, _s()), "delta_step")
        torch.cuda.synchronize()
        return [o, fin, *grads, di, p, held]

    _status(dbg)
    for wide in (0, 1):
        _same(run(dbg, wide), run(_lib.load(), wide))
        assert _status(dbg) == 0


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("shape", [(1, 1, 8), (1, 300, 72), (130, 13, 72), (2, 1100, 72)])
def test_scan_in_8_bits(dbg, shape, dtype):
    b, l, d = shape
    code = CODES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(l)
    g, x, go = (torch.rand(shape, generator=gen, device="cuda").to(dtype) for _ in range(3))

    def run(lib):
        y, dg, dx = (torch.zeros_like(x) for _ in range(3))
        codes = torch.zeros(b, l, (d + 15) // 16 * 16, dtype=torch.int8, device="cuda")
        steps = torch.zeros(b, (l + 7) // 8, d * x.element_size() // 16, device="cuda")
        for back in (0, 1):
            n = lib.fpscan_cl_workspace_bytes(b, l, d, code, back)
            ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
            if back:
                _lib.check(lib.fpscan_scan_bwd_cl8(*_ptrs([g, codes, steps, go, dg, dx]), b, l, d, code,
                                                   ws.data_ptr(), n, _s()), "bwd_cl8")
            else:
                _lib.check(lib.fpscan_scan_fwd_cl8(*_ptrs([g, x, y, codes, steps]), b, l, d, code, ws.data_ptr(), n,
                                                   _s()), "fwd_cl8")
        torch.cuda.synchronize()
        return [y, codes, steps, dg, dx]

    _status(dbg)
    _same(run(dbg), run(_lib.load()))
    assert _status(dbg) == 0


@pytest.mark.parametrize("dtype", list(CODES))
def test_8_bit_format(dbg, dtype):
    _status(dbg)
    for n in (1, 15, 16, 65, 1001, 4096):
        x = torch.randn(n, device="cuda").to(dtype)

        def run(lib):
            codes = torch.zeros(n, dtype=torch.int8, device="cuda")
            steps, back = torch.zeros((n + 63) // 64, device="cuda"), torch.zeros_like(x)
            _lib.check(lib.fpscan_quantize8(*_ptrs([x, codes, steps]), n, CODES[dtype], _s()), "quantize8")
            _lib.check(lib.fpscan_dequantize8(*_ptrs([codes, steps, back]), n, CODES[dtype], _s()), "dequantize8")
            torch.cuda.synchronize()
            return [codes, steps, back]

        _same(run(dbg), run(_lib.load()))
    assert _status(dbg) == 0
