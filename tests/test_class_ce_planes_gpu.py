"""The two fp16 planes of a value add up to it, for every single element."""
import pytest
import torch

from maxstyle_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("C,V,bf", [(512, 32768, False), (130, 30001, False), (512, 32768, True)])
def test_every_class_of_one_row(C, V, bf):
    """One row, an upstream gradient that is no power of two: dw[v] = G[v] h, so that each class shows its own element of G.  Held to 2^-22, as h and (twice, in the logit and in the exponent's argument) the logit of at most
    max|z| log2(e): 3 2^-22 + 4 2^-24 max|z| log2(e) of the class's norm; fp32 sums of C products in the logit, 3 C 2^-24 of sum |w h|.  Planes that belong to different roundings are 2^-11 off,
    in some of these classes."""
    g = torch.Generator().manual_seed(C)
    h, w = torch.randn(1, C, generator=g), torch.randn(V, C, generator=g) / C ** 0.5
    b, lab = 0.3 * torch.randn(V, generator=g), torch.zeros(1, dtype=torch.int64)
    h, w, b, lab = h.to(torch.bfloat16 if bf else torch.float32).cuda(), w.cuda(), b.cuda(), lab.cuda()
    _, _, dw, _ = ops.class_ce(h, w, b, lab, need_dh=False, grad_scale=torch.tensor([0.7], device="cuda"))
    z = (w.double() @ h[0].double()) + b.double()
    p = torch.softmax(z, 0)
    p[0] -= 1
    want = float(torch.tensor(0.7)) * p.unsqueeze(1) * h.double()
    A = float((w.double().abs() @ h[0].double().abs()).max())
    tol = 3 * 2.0 ** -22 + 4 * 2.0 ** -24 * 1.4427 * float(z.abs().max() + torch.logsumexp(z, 0)) + 2 * 3 * C * 2.0 ** -24 * A / C ** 0.5
    err = (dw.double() - want).norm(dim=1) / want.norm(dim=1)
    assert float(err.max()) <= tol, (float(err.max()), tol, int((err > tol).sum()))
