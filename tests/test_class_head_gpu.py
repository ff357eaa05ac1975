"""class_cross_entropy: reductions inside a captured graph, gradients of the bias alone, rows whose every class is switched off."""
import pytest
import torch

import maxstyle_amd
from maxstyle_amd import ops

pytestmark = pytest.mark.gpu


def make(shape, V, seed):
    g = torch.Generator().manual_seed(seed)
    C = shape[1]
    lab = torch.randint(0, V, (shape[0],) + tuple(shape[2:]), generator=g)
    lab = torch.where(torch.rand(lab.shape, generator=g) < 0.1, torch.full_like(lab, -100), lab)
    return torch.randn(*shape, generator=g).cuda(), (torch.randn(V, C, generator=g) / C ** 0.5).cuda(), (0.3 * torch.randn(V, generator=g)).cuda(), lab.cuda()


@pytest.mark.parametrize("reduction", ["mean", "valid", "sum", "none"])
@pytest.mark.parametrize("shape,V", [((4, 16, 256, 256), 9), ((3000, 136), 300)])
def test_captured_without_gradients(reduction, shape, V):
    """Every replay gives what the eager call gives, with eager work between the replays; the value is the reduction of the rows' losses (each side sums in its own order: fp32 once at the
    end, so half a step of the result and 2^-24 of the sum's factor)."""
    h, w, b, lab = make(shape, V, 1)
    h2, _, _, lab2 = make(shape, V, 2)
    hs, ls = h.clone(), lab.clone()
    call = lambda x, y: maxstyle_amd.class_cross_entropy(x, w, b, y, reduction=reduction)
    want = [call(h, lab).clone(), call(h2, lab2).clone()]
    nll = ops.class_ce_fwd(h, w, b, lab)[0].double()
    n = {"mean": nll.numel(), "valid": max(int(((lab >= 0) & (lab < V)).sum()), 1), "sum": 1}
    if reduction != "none":
        assert abs(float(want[0]) - float(nll.sum()) / n[reduction]) <= 4 * 2.0 ** -24 * float(want[0])
    else:
        assert torch.equal(want[0].double(), nll)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(hs, ls)
    for it in range(6):
        hs.copy_(h if it % 2 == 0 else h2)
        ls.copy_(lab if it % 2 == 0 else lab2)
        g.replay()
        junk = torch.randn(1 << 20, device="cuda").sum()          # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out, want[it % 2]), it
    del junk


def test_no_sum_of_the_library_is_captured(monkeypatch):
    """A reduction without gradients runs the package's own kernels only: a library sum over many blocks clears its counters with a memset node, which a replay may not repeat."""
    h, w, b, lab = make((4, 16, 64, 64), 9, 1)
    used = []
    monkeypatch.setattr(torch.Tensor, "sum", lambda self, *a, **k: used.append(1))
    for reduction in ("mean", "valid", "sum"):
        with torch.no_grad():
            maxstyle_amd.class_cross_entropy(h, w, b, lab, reduction=reduction)
    assert not used


@pytest.mark.parametrize("shape,V", [((2, 64, 20, 20), 50), ((300, 136), 700)])
def test_only_what_is_asked_for(shape, V, monkeypatch):
    """Every subset of the gradients has the bits of the whole call, and nothing else is computed or returned."""
    h, w, b, lab = make(shape, V, 3)
    gr = torch.randn(lab.shape, generator=torch.Generator().manual_seed(1)).cuda()
    lse = ops.class_ce_fwd(h, w, b, lab)[1]
    whole = ops.class_ce_bwd(h, w, b, lab, lse, gr)
    for k in range(1, 8):
        need = [bool(k & 1), bool(k & 2), bool(k & 4)]
        got = ops.class_ce_bwd(h, w, b, lab, lse, gr, *need)
        for a, c, n in zip(got, whole, need):
            assert (a is None) if not n else torch.equal(a, c)
        seen = []
        inner = ops.class_ce_bwd
        monkeypatch.setattr(ops, "class_ce_bwd", lambda *a, **kw: seen.append(inner(*a, **kw)) or seen[-1])
        leaves = [t.clone().requires_grad_(n) for t, n in zip((h, w, b), need)]
        (maxstyle_amd.class_cross_entropy(*leaves, lab, reduction="none") * gr).sum().backward()
        monkeypatch.setattr(ops, "class_ce_bwd", inner)
        for t, c, n, made in zip(leaves, whole, need, seen[0]):
            assert (t.grad is None and made is None) if not n else torch.equal(t.grad, c)


@pytest.mark.parametrize("shape,V", [((1, 16, 8, 8), 70), ((40, 136), 300)])
def test_every_class_switched_off(shape, V):
    """There is no softmax then: loss and gradients are NaN, as the definition's, whichever entry makes them; rows without a class still get exactly 0."""
    h, w, b, lab = make(shape, V, 4)
    b = torch.full_like(b, float("-inf"))
    ok = (lab >= 0).reshape(-1)
    rows = lambda t: t.movedim(1, -1).reshape(-1, t.shape[1])
    nll, lse = ops.class_ce_fwd(h, w, b, lab)
    assert torch.isnan(nll.reshape(-1)[ok]).all() and (nll.reshape(-1)[~ok] == 0).all()
    for loss, dh, dw, db in (ops.class_ce(h, w, b, lab), (nll.sum(),) + ops.class_ce_bwd(h, w, b, lab, lse, torch.ones_like(nll))):
        assert torch.isnan(loss) and torch.isnan(rows(dh)[ok]).all() and (rows(dh)[~ok] == 0).all() and torch.isnan(dw).all() and torch.isnan(db).all()
