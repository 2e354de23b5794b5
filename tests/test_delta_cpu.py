"""Gated delta rule and 8-bit checkpoints: what the host refuses, without a GPU."""
import pytest
import torch

import fpscan_b200 as fp
from fpscan_b200 import _lib
from fpscan_b200.delta import validate_delta_layout
from delta_ref import make


def _layout(**change):
    x, _ = make(2, 3, 2, 2, 16, 24, torch.float32, device="cpu")
    d = dict(zip(("q", "k", "v", "log_decay", "beta"), x), **change)
    validate_delta_layout(**d)


def test_valid_layout():
    _layout()
    _layout(state=torch.zeros(2, 4, 24, 16), out=torch.zeros(2, 3, 4, 24))


@pytest.mark.parametrize("change, match", [
    (dict(q=torch.zeros(2, 3, 2)), "4-D"),
    (dict(q=torch.zeros(2, 3, 2, 8)), "same shape"),
    (dict(q=torch.zeros(2, 4, 2, 16), k=torch.zeros(2, 4, 2, 16)), "agree"),
    (dict(q=torch.zeros(2, 3, 3, 16), k=torch.zeros(2, 3, 3, 16)), "multiple"),
    (dict(q=torch.zeros(2, 3, 2, 12), k=torch.zeros(2, 3, 2, 12)), "dk"),
    (dict(q=torch.zeros(2, 3, 2, 136), k=torch.zeros(2, 3, 2, 136)), "dk"),
    (dict(v=torch.zeros(2, 3, 4, 20)), "dv"),
    (dict(beta=torch.zeros(2, 3, 2)), "beta"),
    (dict(log_decay=torch.zeros(2, 3, 4, dtype=torch.float64)), "dtype"),
    (dict(state=torch.zeros(2, 4, 16, 24)), "state"),
    (dict(state=1.0), "state"),
    (dict(out=torch.zeros(2, 3, 4, 16)), "out"),
])
def test_refused_layouts(change, match):
    with pytest.raises(RuntimeError, match=match):
        _layout(**change)


def test_empty_sequences_are_refused():
    x, _ = make(1, 1, 1, 1, 16, 16, torch.float32, device="cpu")
    with pytest.raises(RuntimeError, match="seqlen"):
        validate_delta_layout(*(t[:, :0] for t in x))


def test_cpu_tensors_are_refused():
    x, s = make(1, 4, 1, 1, 16, 16, torch.float32, device="cpu", state=True)
    for call in (lambda: fp.gated_delta(*x), lambda: fp.gated_delta_forward(*x),
                 lambda: fp.gated_delta_step(*x, s), lambda: fp.quantize8(x[0]),
                 lambda: fp.dequantize8(torch.zeros(4, dtype=torch.int8), torch.zeros(1)),
                 lambda: fp.pscan_channels_last(x[0][0], x[1][0], checkpoint8=True)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


GOOD = dict(batch=2, seqlen=3, key_heads=2, heads=4, dk=16, dv=24)


def _addresses(n, step=1 << 20):
    return [(i + 1) * step for i in range(n)]


def _fwd(ptr=None, ws=1 << 24, dtype=0, wide=0, **change):
    d = dict(GOOD, **change)
    p = _addresses(9) if ptr is None else ptr
    lib = _lib.load()
    rc = lib.fpscan_delta_fwd(*p[:8], *d.values(), 1.0, dtype, wide, p[8], ws, None)
    return rc, lib.fpscan_last_error()


@pytest.mark.parametrize("change, match", [
    (dict(batch=-1), b"batch"), (dict(seqlen=0), b"seqlen"), (dict(heads=3), b"multiple"),
    (dict(key_heads=0), b"multiple"), (dict(dk=4), b"dk"), (dict(dk=132), b"dk"), (dict(dk=136), b"dk"),
    (dict(dv=0), b"dv"), (dict(dv=12), b"dv"), (dict(dtype=5), b"dtype"), (dict(ws=100), b"workspace"),
    (dict(batch=1 << 30, heads=4, seqlen=64 * 16), b"grid"), (dict(seqlen=1 << 40), b"2^31"),
])
def test_c_abi_refuses(change, match):
    rc, msg = _fwd(**change)
    assert rc == 1 and match in msg


def test_c_abi_refuses_bad_pointers():
    for i, name in ((0, b"q"), (4, b"beta"), (6, b"out"), (8, b"workspace")):
        p = _addresses(9)
        p[i] = 0
        rc, msg = _fwd(p)
        assert rc == 1 and name in msg and b"NULL" in msg
        p[i] = 8 + (1 << 20) * 20
        rc, msg = _fwd(p)
        assert rc == 1 and name in msg and b"aligned" in msg
    p = _addresses(9)
    p[6] = p[2] + 16
    rc, msg = _fwd(p)
    assert rc == 1 and b"overlaps" in msg
    p = _addresses(9)
    p[7] = p[5]  # the final state over the initial one
    rc, msg = _fwd(p)
    assert rc == 1 and b"overlaps" in msg


def test_c_abi_backward_and_step_refuse():
    lib = _lib.load()
    p = _addresses(15)
    p[10] = p[2]  # dv over v
    need = lib.fpscan_delta_workspace_bytes(*GOOD.values(), 0, 0, 1)
    assert lib.fpscan_delta_bwd(*p[:14], *GOOD.values(), 1.0, 0, 0, p[14], need, None) == 1
    assert b"overlaps" in lib.fpscan_last_error()
    assert lib.fpscan_delta_bwd(*_addresses(14), *GOOD.values(), 1.0, 0, 0, 0, 0, None) == 1
    p = _addresses(8)
    p[7] = p[5] + 64  # a state shifted against itself
    assert lib.fpscan_delta_step(*p, *GOOD.values(), 1.0, 0, None) == 1
    assert b"overlaps" in lib.fpscan_last_error()


def test_c_abi_empty_batch_is_noop():
    lib = _lib.load()
    d = dict(GOOD, batch=0)
    assert lib.fpscan_delta_fwd(*[0] * 8, *d.values(), 1.0, 0, 0, 0, 0, None) == 0
    assert lib.fpscan_delta_bwd(*[0] * 14, *d.values(), 1.0, 0, 0, 0, 0, None) == 0
    assert lib.fpscan_delta_step(*[0] * 8, *d.values(), 1.0, 0, None) == 0
    assert lib.fpscan_delta_workspace_bytes(*d.values(), 0, 0, 0) == 0


def test_workspace_is_bounded_by_a_sequence():
    lib = _lib.load()
    need = [lib.fpscan_delta_workspace_bytes(b, 4096, 16, 16, 128, 128, 2, 0, 1) for b in (1, 2, 8, 64, 512)]
    assert need == sorted(need) and need[-1] <= max(1 << 31, need[0])
    assert lib.fpscan_delta_workspace_bytes(1, 1 << 20, 16, 16, 128, 128, 2, 0, 1) > 1 << 31


def test_c_abi_checkpoints_refuse():
    lib = _lib.load()
    a = _addresses(8)
    assert lib.fpscan_quantize8(0, a[0], a[1], 64, 0, None) == 1 and b"NULL" in lib.fpscan_last_error()
    assert lib.fpscan_quantize8(a[0], a[0] + 16, a[1], 64, 0, None) == 1 and b"overlaps" in lib.fpscan_last_error()
    assert lib.fpscan_quantize8(a[0], a[1], a[2], -1, 0, None) == 1
    assert lib.fpscan_quantize8(a[0], a[1], a[2], 64, 9, None) == 1 and b"dtype" in lib.fpscan_last_error()
    assert lib.fpscan_dequantize8(a[0], a[1] + 4, a[2], 64, 0, None) == 1 and b"aligned" in lib.fpscan_last_error()
    assert lib.fpscan_quantize8(0, 0, 0, 0, 0, None) == 0
    assert lib.fpscan_scan_fwd_cl8(*a[:5], 1, 4, 6, 2, a[5], 1 << 20, None) == 1 and b"dim" in lib.fpscan_last_error()
    assert lib.fpscan_scan_fwd_cl8(a[0], a[1], a[1], *a[3:5], 1, 4, 16, 2, a[5], 1 << 20, None) == 1
    assert b"overlaps" in lib.fpscan_last_error()
    assert lib.fpscan_scan_bwd_cl8(*a[:6], 1, 4, 16, 2, a[6], 1, None) == 1 and b"workspace" in lib.fpscan_last_error()
