"""Layer calls of several widths from several host threads, each on its own
stream.  A kernel's limit on dynamic shared memory belongs to the process: no
call may lower it between another call's setting and its launch."""
import threading

import pytest
import torch

from mhc_ascend_b200 import _C, ops

pytestmark = pytest.mark.gpu


def static_call(cuda, n, C):
    gen = torch.Generator(device=cuda).manual_seed(C)
    x = torch.randn(300, n, C, device=cuda, generator=gen)
    w, hp, hq = torch.ones(C, device=cuda), torch.zeros(n, device=cuda), torch.zeros(n, device=cuda)
    hr = torch.randn(n, n, device=cuda, generator=gen)
    want, _ = ops.mhc_layer_fwd_static(x, w, hp, hq, hr, save_rms=False)
    out, stream = torch.empty_like(x), torch.cuda.Stream()
    ws = torch.empty(_C.load().mhc_layer_static_workspace_bytes(300, n, C), dtype=torch.uint8, device=cuda)
    args = (x.data_ptr(), w.data_ptr(), hp.data_ptr(), hq.data_ptr(), hr.data_ptr(), out.data_ptr(), None, 300, n, C,
            20, 1e-8, 1e-5, ws.data_ptr(), ws.numel(), stream.cuda_stream)
    return _C.load().mhc_layer_fwd_static_f32, args, out, want, (x, w, hp, hq, hr, ws, stream)


def wide_call(cuda, n, C):
    gen = torch.Generator(device=cuda).manual_seed(C)
    x = torch.randn(2, n, C, device=cuda, generator=gen)
    w = torch.ones(C, device=cuda)
    pp, pq, pr = (torch.randn(k, n * C, device=cuda, generator=gen) * 0.02 for k in (n, n, n * n))
    a, b, br = torch.full((1,), 0.1, device=cuda), torch.zeros(n, device=cuda), torch.zeros(n, n, device=cuda)
    want, _ = ops.mhc_layer_fwd_dynamic(x, w, pp, pq, pr, a, a, a, b, b, br, save_state=False)
    out, stream = torch.empty_like(x), torch.cuda.Stream()
    ws = torch.empty(_C.load().mhc_layer_fwd_dynamic_workspace_bytes(2, n, C), dtype=torch.uint8, device=cuda)
    args = (x.data_ptr(), w.data_ptr(), pp.data_ptr(), pq.data_ptr(), pr.data_ptr(), a.data_ptr(), a.data_ptr(),
            a.data_ptr(), b.data_ptr(), b.data_ptr(), br.data_ptr(), out.data_ptr(), None, 2, n, C, 20, 1e-8, 1e-5,
            ws.data_ptr(), ws.numel(), stream.cuda_stream)
    return _C.load().mhc_layer_fwd_dynamic, args, out, want, (x, w, pp, pq, pr, a, b, br, ws, stream)


@pytest.mark.parametrize("call,n,widths,turns", [(static_call, 4, (512, 2048, 4096), 2000),
                                                 (wide_call, 12, (64, 2048, 8192), 500)])
def test_widths_side_by_side(cuda, call, n, widths, turns):
    calls = [call(cuda, n, C) for C in widths]
    torch.cuda.synchronize()
    errors = []

    def work(fn, args):
        for _ in range(turns):
            if fn(*args):
                errors.append(_C.last_error())
                return

    threads = [threading.Thread(target=work, args=c[:2]) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for _, _, out, want, _ in calls:
        assert torch.equal(out, want)
