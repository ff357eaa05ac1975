"""ms_class_ce, _fwd and _bwd with a workspace of the caller's own: whatever it holds beforehand, exactly the size that is asked for, nothing behind it written."""
import pytest
import torch

from maxstyle_amd import ops
from maxstyle_amd._lib import check, lib

pytestmark = pytest.mark.gpu
F, B = torch.float32, torch.bfloat16
GUARD = 4096


def make(shape, V, hdt, wdt):
    g = torch.Generator().manual_seed(V)
    C = shape[1]
    lab = torch.randint(0, V, (shape[0],) + tuple(shape[2:]), generator=g)
    lab = torch.where(torch.rand(lab.shape, generator=g) < 0.1, torch.full_like(lab, -100), lab)
    return (torch.randn(*shape, generator=g).to(hdt).cuda(), (torch.randn(V, C, generator=g) / C ** 0.5).to(wdt).cuda(), (0.3 * torch.randn(V, generator=g)).cuda(), lab.cuda())


@pytest.mark.parametrize("hdt,wdt", [(F, F), (B, F), (F, B), (B, B)])
@pytest.mark.parametrize("shape,V", [((1, 512), 700), ((2, 512, 16, 17), 900), ((130, 640), 9000), ((300, 136), 33), ((2, 64, 18, 20), 300), ((40, 16), 9)])
def test_what_the_workspace_holds(shape, V, hdt, wdt):
    h, w, b, lab = make(shape, V, hdt, wdt)
    N, C = shape[:2]
    P = lab.numel()
    HW, types, st = P // N, int(hdt == B) | 2 * int(wdt == B), torch.cuda.current_stream().cuda_stream
    want = ops.class_ce(h, w, b, lab, mean_over="valid")
    grad = torch.randn(lab.shape, generator=torch.Generator().manual_seed(1)).cuda()
    nll, lse = ops.class_ce_fwd(h, w, b, lab)
    wantb = ops.class_ce_bwd(h, w, b, lab, lse, grad)
    sizes = [lib.ms_class_ce_ws_bytes(N, C, V, HW, types, k) for k in (0, 1)]
    for fill in (0, 255, 127):           # 255: every float and half a NaN; 127: large numbers
        ws = [torch.full((n + GUARD,), fill, dtype=torch.uint8, device="cuda") for n in (sizes[1], sizes[0], sizes[1])]
        out = [torch.full_like(t, float("nan")) for t in (want[0].reshape(1), h, w, b, nll, nll, h, w, b)]
        p = [t.data_ptr() for t in out]
        check(lib.ms_class_ce(h.data_ptr(), w.data_ptr(), b.data_ptr(), lab.data_ptr(), p[0], p[1], p[2], p[3], N, C, V, HW, types, 1.0, 1, 0, ws[0].data_ptr(), sizes[1], st), "ms_class_ce")
        check(lib.ms_class_ce_fwd(h.data_ptr(), w.data_ptr(), b.data_ptr(), lab.data_ptr(), p[4], p[5], N, C, V, HW, types, ws[1].data_ptr(), sizes[0], st), "ms_class_ce_fwd")
        check(lib.ms_class_ce_bwd(h.data_ptr(), w.data_ptr(), b.data_ptr(), lab.data_ptr(), lse.data_ptr(), grad.data_ptr(), p[6], p[7], p[8], N, C, V, HW, types, ws[2].data_ptr(), sizes[1], st),
              "ms_class_ce_bwd")
        for a, c in zip(out, (want[0].reshape(1),) + want[1:] + (nll, lse) + wantb):
            assert torch.equal(a, c)
        for t, n in zip(ws, (sizes[1], sizes[0], sizes[1])):
            assert (t[n:] == fill).all()
