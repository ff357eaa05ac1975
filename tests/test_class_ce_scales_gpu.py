"""Gradients of the many-class loss where rows or classes are zero or of very different size (a padded vocabulary, a dead pixel, one outlier, a fresh class).

Every row of dh and every class of dw is judged by itself, against its own terms m = |g| (p + hot) times the other operand's magnitudes: the error's norm over m's, its median, 99 % quantile
and maximum over rows (classes).  An element of G is held to 2^-41 g_p at least, so m takes every p as 2^-20 more than it is.  The bar is what the plain form leaves in fp32 on the same input: 4 times its quantile, plus 3 2^-22 (both operands of a product are held to 2^-22, and the
product of their low planes is left out), plus 2 2^-24 max|z| log2(e) (z - lse, both rounded at that size, is an exponent).  A bf16 result adds half a step, 2^-8 of the value; where h and w
are both bf16, G has 11 bits: 2^-11."""
import pytest
import torch

from maxstyle_amd import ops

pytestmark = pytest.mark.gpu
F, B = torch.float32, torch.bfloat16
CASES = ["plain", "zero row", "zero class", "both", "both, small", "padded", "spread rows", "spread classes", "spread gradients", "large row", "switched off", "near classes", "near rows", "all classes zero", "all rows zero"]


def rows_of(t):
    return t.movedim(1, -1).reshape(-1, t.shape[1])


def make(name, shape, V, hdt, wdt, narrow):
    gen = torch.Generator().manual_seed(5)
    C, P = shape[1], torch.Size(shape).numel() // shape[1]
    h, w, b = torch.randn(*shape, generator=gen), torch.randn(V, C, generator=gen) * (2.0 / C ** 0.5), 0.3 * torch.randn(V, generator=gen)
    lab = torch.randint(0, max(V // 2, 1), (shape[0],) + tuple(shape[2:]), generator=gen)          # (half of the classes are never a label)
    gr = torch.full((P,), 1.0 / P)
    hr = rows_of(h).clone()
    spread = lambda n, bits: 2.0 ** (-bits * torch.rand(n, generator=gen))
    if "small" in name:
        hr, w = hr * 0.01, w * 0.1
    if name.startswith("both") or name == "zero row":
        hr[3] = 0
    if name.startswith("both") or name == "zero class":
        w[min(5, V - 1)] = 0
    if name == "padded":
        w[V - V // 8:], b[V - V // 8:] = 0, -1e30
    if name == "spread rows":
        hr = hr * spread(P, 30).unsqueeze(1)
    if name == "spread classes":          # (the narrow form keeps 64 classes below one scale: their weights to 2^-39 of the largest)
        w = w * spread(V, 15 if narrow else 30).unsqueeze(1)
    if name == "spread gradients":
        gr = gr * spread(P, 30)
    if name == "switched off":          # ... classes whose weights are anything finite
        off = torch.arange(V) % 7 == 3
        w[off], b[off] = 1e30, float("-inf")
        lab[off[lab]] += 1
    if name == "near classes":          # weights that differ little: dh is a difference
        w = 3 + 0.02 * w
    if name == "near rows":          # ... features: dw is one
        hr = 3 + 0.02 * hr
    if name == "large row":
        hr[7] *= 1e6 if narrow else 1e4
    if name == "all classes zero":
        w = w * 0
    if name == "all rows zero":
        hr = hr * 0
    h = hr.reshape((shape[0],) + tuple(shape[2:]) + (C,)).movedim(-1, 1).contiguous()
    return h.to(hdt).cuda(), w.to(wdt).cuda(), b.cuda(), lab.cuda(), gr.cuda()


def definition(h, w, b, lab, gr, dt):
    x, wd, y = rows_of(h).to(dt), w.to(dt), lab.reshape(-1, 1)
    z = x @ wd.t().contiguous() + b.to(dt)
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    G = e / e.sum(1, keepdim=True)
    mag = (G + 2.0 ** -20).scatter_add_(1, y, torch.ones_like(y, dtype=dt)) * gr.to(dt).unsqueeze(1)
    G = G.scatter_add(1, y, -torch.ones_like(y, dtype=dt)) * gr.to(dt).unsqueeze(1)
    return dict(dh=G @ wd, dw=G.t().contiguous() @ x, db=G.sum(0), mdh=mag @ wd.abs(), mdw=mag.t().contiguous() @ x.abs(), mdb=mag.sum(0), zmax=float(z[e > 0].abs().max()))


def quantiles(a, e, k, bf):
    d = (a.double() - e[k]).abs()
    if bf:
        d = (d - 2.0 ** -8 * (1 + 2.0 ** -7) * e[k].abs()).clamp_min(0)
    m = e["m" + k].norm(dim=1)
    q = (d.norm(dim=1)[m > 0] / m[m > 0])
    return torch.quantile(q, torch.tensor([0.5, 0.99, 1.0], dtype=torch.float64, device=q.device)) if q.numel() else torch.zeros(3, dtype=torch.float64, device=m.device)


def check(name, shape, V, hdt, wdt, narrow):
    h, w, b, lab, gr = make(name, shape, V, hdt, wdt, narrow)
    _, lse = ops.class_ce_fwd(h, w, b, lab)
    dh, dw, db = ops.class_ce_bwd(h, w, b, lab, lse, gr.view(lab.shape))
    e, plain = definition(h, w, b, lab, gr, torch.float64), definition(h, w, b, lab, gr, F)
    bar = 3 * 2.0 ** -22 + 2.0 ** -23 * 1.4427 * e["zmax"] + (2.0 ** -11 if hdt == B and wdt == B else 0)
    for k, own, dt in (("dh", rows_of(dh), hdt), ("dw", dw, wdt)):
        a, c = quantiles(own, e, k, dt == B), quantiles(plain[k], e, k, False)
        assert torch.isfinite(own.double()).all() and (a <= 4 * c + bar).all(), (k, a.tolist(), c.tolist(), bar)
    # db: fp32 sums of at most P terms, each G off by the argument's rounding
    assert ((db.double() - e["db"]).abs() <= (2.0 ** -22 + 2.0 ** -23 * 1.4427 * e["zmax"] + gr.numel() * 2.0 ** -24) * e["mdb"]).all()


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("hdt,wdt", [(F, F), (B, F), (F, B), (B, B)])
@pytest.mark.parametrize("shape,V", [((256, 512), 8192), ((2, 136, 12, 13), 1000), ((40, 130), 33)])
def test_wide_form(name, hdt, wdt, shape, V):
    check(name, shape, V, hdt, wdt, False)


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("hdt,wdt", [(F, F), (B, F), (F, B), (B, B)])
@pytest.mark.parametrize("shape,V", [((2, 64, 40, 40), 151), ((1, 16, 50, 37), 104), ((3000, 100), 40)])
def test_narrow_form(name, hdt, wdt, shape, V):
    check(name, shape, V, hdt, wdt, True)


@pytest.mark.parametrize("name", ["plain", "confident", "near classes"])
@pytest.mark.parametrize("hdt,wdt", [(F, F), (B, F), (B, B)])
@pytest.mark.parametrize("shape,V", [((256, 136), 700), ((2, 512, 16, 17), 900), ((2, 64, 40, 40), 151), ((1, 16, 50, 37), 104)])
def test_loss_and_gradients_in_one_call(name, hdt, wdt, shape, V):
    """No log-sum is stored in between, so the size of the logits does not enter: 4 times plain fp32's own error, plus 4 2^-22 of the terms (both operands, the product of the low planes, G)."""
    h, w, b, lab, gr = make(name, shape, V, hdt, wdt, True)
    if name == "confident":
        hr = rows_of(h).float() + 6 * w.float()[lab.reshape(-1)]
        h = hr.reshape((shape[0],) + tuple(shape[2:]) + (shape[1],)).movedim(-1, 1).contiguous().to(hdt)
    _, dh, dw, _ = ops.class_ce(h, w, b, lab)
    e, plain = definition(h, w, b, lab, gr, torch.float64), definition(h, w, b, lab, gr, F)
    for k, own, dt in (("dh", rows_of(dh), hdt), ("dw", dw, wdt)):
        a, c = quantiles(own, e, k, dt == B), quantiles(plain[k], e, k, False)
        assert (a <= 4 * c + 4 * 2.0 ** -22 + (2.0 ** -11 if hdt == B and wdt == B else 0)).all(), (k, a.tolist(), c.tolist())
