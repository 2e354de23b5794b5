"""Nothing is written outside by the delta rule's kernels of 64 values a CTA, which take many heads."""
import pytest
import torch

from fpscan_b200 import _lib, ops
from delta_ref import make
from guard import guarded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dv", [8, 40, 72])
def test_nothing_written_outside(dv, dtype):
    b, l, hk, group, dk = 1, 130, 80, 2, 24
    h, code = hk * group, ops.DTYPE_CODES[dtype]
    assert h * ((dv + 31) // 32) > torch.cuda.get_device_properties(0).multi_processor_count
    x, s0 = make(b, l, hk, group, dk, dv, dtype, seed=dv, state=True)
    go, sizes = torch.randn_like(x[2]), (b, l, hk, h, dk, dv)
    ptr = [t.data_ptr() for t in x]

    def room(wide, backward):
        return guarded((_lib.load().fpscan_delta_workspace_bytes(*sizes, code, wide, backward) // 4,), torch.float32)

    for wide in (0, 1):
        o, fin, ws = guarded(x[2].shape, dtype), guarded(s0.shape, torch.float32), room(wide, 0)
        ops._launch(0, "fpscan_delta_fwd", *ptr, s0.data_ptr(), o.out.data_ptr(), fin.out.data_ptr(), *sizes,
                    0.5, code, wide, ws.out.data_ptr(), ws.out.numel() * 4)
        grads, di, back = [guarded(t.shape, dtype) for t in x], guarded(s0.shape, torch.float32), room(wide, 1)
        ops._launch(0, "fpscan_delta_bwd", *ptr, s0.data_ptr(), go.data_ptr(), s0.data_ptr(),
                    *(g.out.data_ptr() for g in grads), di.out.data_ptr(), *sizes, 0.5, code, wide,
                    back.out.data_ptr(), back.out.numel() * 4)
        for g in (o, fin, ws, *grads, di, back):
            g.check(f"wide {wide}")
        for g in (o, fin, *grads, di):
            assert torch.isfinite(g.out).all()
    assert _lib.device_status() == 0
