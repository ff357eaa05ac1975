"""Head + cross entropy over many classes (ops.class_ce, class_ce_fwd / class_ce_bwd, class_cross_entropy) against the operator's definition in 64 bits.

Tolerances (u16 = 2^-11, u32 = 2^-24: half a step of fp16 / fp32), from the kernels' arithmetic:
  logits     each operand is held to 2^-22 (two fp16 planes; exactly if it came as bf16), the product of the two low planes (2^-22) is left out, and the C products are
             summed in fp32 with at most three terms each: |dz| <= A (3 2^-22 + (3 C + 8) u32) with A = sum_c |w h| + |b|
  nll, lse   |dz| twice (label's logit and the log-sum) + 8 u32 of the values joined + C classes' sum
  gradients  G = g (p - hot): p carries a relative 2 |dz| + 2^-21 (exp2 and its argument); G and w are held to 2^-22 or, for a bf16 result, to u16 each;
             the sum over the long axis has at most three terms each in fp32.  On top half a step of the result's type."""
import pytest
import torch

import maxstyle_amd
from maxstyle_amd import ops

pytestmark = pytest.mark.gpu
U16, U32 = 2.0 ** -11, 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def make(shape, V, hdt=torch.float32, wdt=torch.float32, bias=True, void=0.1, seed=0, wscale=1.0):
    g = torch.Generator().manual_seed(seed)
    C = shape[1]
    h = torch.randn(*shape, generator=g)
    w = torch.randn(V, C, generator=g) * (wscale / C ** 0.5)
    b = torch.randn(V, generator=g) * 0.3 if bias else None
    lab = torch.randint(0, V, (shape[0],) + tuple(shape[2:]), generator=g)
    lab = torch.where(torch.rand(lab.shape, generator=g) < void, torch.full_like(lab, -100), lab)
    to = lambda t: None if t is None else t.cuda()
    return to(h.to(hdt)), to(w.to(wdt)), to(b), to(lab)


def rows_of(t, C):
    return t.movedim(1, -1).reshape(-1, C)


def reference(h, w, b, lab, grad):
    """nll, lse, dh (as rows), dw, db in 64 bits, and the tolerances' sums; grad: upstream gradient of every row (flat, fp64)."""
    C, V = h.shape[1], w.shape[0]
    x, wd = rows_of(h.double(), C), w.double().reshape(V, C)
    bd = torch.zeros(V, dtype=torch.float64, device=h.device) if b is None else b.double()
    y = lab.reshape(-1)
    ok = (y >= 0) & (y < V)
    x = torch.where(ok.unsqueeze(1), x, torch.zeros_like(x))
    z = x @ wd.T + bd
    A = (x.abs() @ wd.abs().T + bd.abs()).amax(1)
    dz = A * (3 * 2.0 ** -22 + (3 * C + 8) * U32)
    lse = torch.logsumexp(z, 1)
    yy = torch.where(ok, y, torch.zeros_like(y))
    nll = torch.where(ok, lse - z.gather(1, yy.unsqueeze(1)).squeeze(1), torch.zeros_like(lse))
    gr = torch.where(ok, grad, torch.zeros_like(grad)).unsqueeze(1)
    p = torch.exp(z - lse.unsqueeze(1))
    hot = torch.zeros_like(p).scatter_(1, yy.unsqueeze(1), 1.0)
    G = gr * (p - hot)
    relp = (2 * dz + 2.0 ** -21).unsqueeze(1)
    mag = gr.abs() * (p + hot)                       # what is rounded
    err = gr.abs() * p * relp + mag * 2 * U32        # error of G before it is split
    return dict(x=x, w=wd, ok=ok, lse=lse, nll=nll, dz=dz, G=G, mag=mag, err=err, dh=G @ wd, dw=G.T @ x, db=G.sum(0))


def tolerances(r, hdt, wdt):
    P, V = r["G"].shape
    gx = 2 * U16 if hdt == torch.bfloat16 else 3 * 2.0 ** -22
    gw = 2 * U16 if wdt == torch.bfloat16 else 3 * 2.0 ** -22
    # a gradient element far below the largest is held to 2^-38 of it (the lowest fp16 step)
    ex = r["x"].abs().amax(1, keepdim=True).clamp_min(1e-30)
    lowest = (r["mag"] * ex).max() * 2.0 ** -36
    wm = r["w"].abs().amax(0)
    tdh = r["err"] @ r["w"].abs() + r["mag"] @ r["w"].abs() * (gx + (3 * V + 8) * U32) + lowest / ex * V * wm + HALF[hdt] * r["dh"].abs()
    tdw = r["err"].T @ r["x"].abs() + r["mag"].T @ r["x"].abs() * (gw + (3 * P + 8) * U32) + lowest * P + HALF[wdt] * r["dw"].abs()
    tdb = r["err"].sum(0) + r["mag"].sum(0) * (P * U32 + 2.0 ** -22)
    return tdh, tdw, tdb


def close(a, b, tol, what):
    if a.numel() == 0:                   # (no row takes part)
        return
    d = (a.double() - b).abs()
    assert torch.isfinite(a.double()).all(), what
    worst = (d / tol.clamp_min(1e-300)).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} of the tolerance, off by {d.max().item():.3e}"


F, B = torch.float32, torch.bfloat16
CASES = [  # shape, V, h, w, bias
    ((1, 16, 33, 31), 9, F, F, True),
    ((2, 16, 7, 5), 5, F, F, False),
    ((3, 64, 20, 21), 151, F, F, True),
    ((1, 8, 1, 1), 2, F, F, True),
    ((1, 1, 3, 3), 1, F, F, True),
    ((2, 65, 9, 16), 257, F, F, True),
    ((2, 24, 16, 16), 1000, B, F, True),
    ((2, 64, 18, 20), 300, F, B, True),
    ((4, 130, 6, 6), 513, B, B, True),
    ((1, 512), 700, F, F, True),
    ((257, 512), 1025, B, B, False),
    ((300, 100), 70, F, F, True),
    ((2, 512, 16, 17), 900, F, F, True),
    ((130, 640), 9000, B, F, True),
    ((2, 33, 5), 40, F, F, True),
    ((1, 16, 4, 5, 6), 12, F, F, True),
]


@pytest.mark.parametrize("shape,V,hdt,wdt,bias", CASES)
@pytest.mark.parametrize("mean", ["all", "valid"])
def test_loss_and_gradients(shape, V, hdt, wdt, bias, mean):
    h, w, b, lab = make(shape, V, hdt, wdt, bias, seed=V)
    P = lab.numel()
    ok = (lab >= 0) & (lab < V)
    n = max(int(ok.sum()), 1) if mean == "valid" else P
    r = reference(h, w, b, lab, torch.full((P,), 1.0 / n, dtype=torch.float64, device="cuda"))
    loss, dh, dw, db = ops.class_ce(h, w, b, lab, mean_over=mean)
    assert dh.dtype == hdt and dh.shape == h.shape and dw.dtype == wdt and dw.shape == w.shape and (db is None) == (b is None)
    tn = 2 * r["dz"] + 16 * U32 * (r["lse"].abs() + r["nll"] + 1)
    close(loss, r["nll"].sum() / n, tn.sum() / n + 2 * U32 * r["nll"].sum() / n, "loss")
    tdh, tdw, tdb = tolerances(r, hdt, wdt)
    close(rows_of(dh, shape[1]), r["dh"], tdh, "dh")
    close(dw, r["dw"], tdw, "dw")
    if b is not None:
        close(db, r["db"], tdb, "db")
    assert (rows_of(dh, shape[1])[~ok.reshape(-1)] == 0).all()
    again = ops.class_ce(h, w, b, lab, mean_over=mean)
    for a, c in zip((loss, dh, dw, db), again):
        assert a is None or torch.equal(a, c)


@pytest.mark.parametrize("shape,V,hdt,wdt,bias", CASES)
def test_rows_and_autograd(shape, V, hdt, wdt, bias):
    h, w, b, lab = make(shape, V, hdt, wdt, bias, seed=V + 1)
    P = lab.numel()
    gr = torch.randn(P, generator=torch.Generator().manual_seed(3)).cuda()
    r = reference(h, w, b, lab, gr.double())
    nll, lse = ops.class_ce_fwd(h, w, b, lab)
    tn = 2 * r["dz"] + 16 * U32 * (r["lse"].abs() + r["nll"] + 1)
    close(nll.reshape(-1), r["nll"], tn, "nll")
    close(lse.reshape(-1)[r["ok"]], r["lse"][r["ok"]], tn[r["ok"]], "lse")
    leaves = [t.clone().requires_grad_(True) if t is not None else None for t in (h, w, b)]
    out = maxstyle_amd.class_cross_entropy(*leaves, lab, reduction="none")
    assert torch.equal(out, nll)
    (out * gr.view(out.shape)).sum().backward()
    tdh, tdw, tdb = tolerances(r, hdt, wdt)
    close(rows_of(leaves[0].grad, shape[1]), r["dh"], tdh, "dh")
    close(leaves[1].grad, r["dw"], tdw, "dw")
    if b is not None:
        close(leaves[2].grad, r["db"], tdb, "db")


def test_reductions_and_scale():
    h, w, b, lab = make((2, 16, 12, 12), 20, seed=5)
    nll = ops.class_ce_fwd(h, w, b, lab)[0].double()
    nv = int(((lab >= 0) & (lab < 20)).sum())
    for red, want in (("mean", nll.mean()), ("sum", nll.sum()), ("valid", nll.sum() / nv)):
        got = maxstyle_amd.class_cross_entropy(h, w, b, lab, reduction=red).double()
        assert abs(got - want) <= 400 * U32 * want.abs()
    base = ops.class_ce(h, w, b, lab)
    half = ops.class_ce(h, w, b, lab, grad_scale=torch.tensor([0.5], device="cuda"))
    assert torch.equal(half[0], base[0])
    for a, c in zip(base[1:], half[1:]):
        assert torch.equal(c, 0.5 * a)               # a power of two: the same bits
    # The matrix instruction's additions do not round a sum and its negative alike: both are the same sum of 3 K terms (K = 20 classes, 288 rows), each addition off by
    # at most one unit, 2 u32, of the sum of magnitudes.
    neg = ops.class_ce(h, w, b, lab, loss_sign=-1.0)
    assert torch.equal(neg[0], -base[0]) and torch.equal(neg[3], -base[3])
    mag = reference(h, w, b, lab, torch.full((288,), 1.0 / 288, dtype=torch.float64, device="cuda"))
    for a, c, m, K in ((rows_of(base[1], 16), rows_of(neg[1], 16), mag["mag"] @ mag["w"].abs(), 20), (base[2], neg[2], mag["mag"].T @ mag["x"].abs(), 288)):
        assert ((a.double() + c.double()).abs() <= 2 * 3 * K * 2 * U32 * m).all()
    only = ops.class_ce(h, w, b, lab, need_dh=False, need_dw=False)
    assert torch.equal(only[0], base[0]) and only[1] is only[2] is only[3] is None
    assert torch.equal(ops.class_ce(h, w, b, lab, need_dw=False)[1], base[1])
    assert torch.equal(ops.class_ce(h, w, b, lab, need_dh=False)[2], base[2])


def test_agrees_with_the_small_head():
    h, w, b, lab = make((2, 16, 24, 24), 4, seed=9)
    loss, dh, _ = ops.head_ce(h, w, b, lab)
    l2, dh2, _, _ = ops.class_ce(h, w, b, lab)
    assert abs(float(loss[0] - l2)) < 1e-6 * float(l2)
    assert (dh - dh2).abs().max() < 1e-6 * dh.abs().max()


@pytest.mark.parametrize("c", [4, 5, 21, 150])
def test_cross_entropy_2D_of_any_number_of_classes(c):
    g = torch.Generator().manual_seed(c)
    z = torch.randn(2, c, 17, 19, generator=g).cuda() * 3
    lab = torch.randint(0, c, (2, 17, 19), generator=g).cuda()
    zd = z.double()
    want = (torch.logsumexp(zd, 1) - zd.gather(1, lab.unsqueeze(1)).squeeze(1)).mean()
    # each pixel within 2 |z| 3 2^-22 (the planes) + 16 u32 of its log-sum and loss
    tol = (6 * 2.0 ** -22 + 32 * U32) * float(zd.abs().max() + want + 6)
    assert abs(float(maxstyle_amd.cross_entropy_2D(z, lab)) - float(want)) <= tol


def test_no_row_takes_part():
    h, w, b, lab = make((2, 16, 9, 9), 11)
    lab.fill_(11)
    for mean in ("all", "valid"):
        loss, dh, dw, db = ops.class_ce(h, w, b, lab, mean_over=mean)
        assert float(loss) == 0 and not dh.any() and not dw.any() and not db.any()
    assert float(maxstyle_amd.class_cross_entropy(h, w, b, lab, reduction="valid")) == 0


def test_void_rows_may_hold_anything():
    for shape in ((2, 64, 9, 9), (90, 512)):
        h, w, b, lab = make(shape, 77, seed=2)
        want = ops.class_ce(h, w, b, lab)
        bad = (lab < 0).reshape(lab.shape[0], 1, *lab.shape[1:]).expand(h.shape)
        for v in (float("nan"), float("inf"), -3e38):
            got = ops.class_ce(torch.where(bad, torch.full_like(h, v), h), w, b, lab)
            for a, c in zip(want, got):
                assert torch.equal(a, c)


def test_classes_switched_off_and_wide_ranges():
    h, w, b, lab = make((1, 32, 10, 10), 50, seed=4)
    off = torch.arange(50, device="cuda") % 3 == 0
    lab = torch.where((lab >= 0) & (lab % 3 == 0), lab + 1, lab)
    b = torch.where(off, torch.full_like(b, float("-inf")), b)
    loss, dh, dw, db = ops.class_ce(h, w, b, lab)
    keep = (~off).nonzero()[:, 0]
    remap = torch.full((51,), -1, device="cuda"); remap[keep] = torch.arange(len(keep), device="cuda")
    l2, dh2, dw2, db2 = ops.class_ce(h, w[keep].contiguous(), b[keep].contiguous(), torch.where(lab >= 0, remap[lab.clamp(0)], lab))
    assert abs(float(loss - l2)) < 1e-6 * float(l2) and (dh - dh2).abs().max() <= 1e-5 * dh.abs().max()
    assert not dw[off].any() and not db[off].any() and (dw[keep] - dw2).abs().max() <= 1e-5 * dw.abs().max()
    # rows of very different magnitude: each is scaled by itself
    h, w, b, lab = make((40, 64), 30, void=0.0, seed=6)
    sc = 10.0 ** torch.linspace(-18, 1.5, 40, device="cuda").unsqueeze(1)
    r = reference(h * sc, w, b, lab, torch.full((40,), 1.0, dtype=torch.float64, device="cuda"))
    nll, lse = ops.class_ce_fwd(h * sc, w, b, lab)
    close(nll, r["nll"], 2 * r["dz"] + 16 * U32 * (r["lse"].abs() + r["nll"] + 1), "nll")
    # a NaN stays in its row
    h2 = h.clone(); h2[7, 3] = float("nan")
    n2 = ops.class_ce_fwd(h2, w, b, lab)[0]
    n1 = ops.class_ce_fwd(h, w, b, lab)[0]
    assert torch.isnan(n2[7]) and torch.equal(torch.cat([n1[:7], n1[8:]]), torch.cat([n2[:7], n2[8:]]))


def test_gradient_against_differences():
    h, w, b, lab = make((1, 16, 6, 6), 13, seed=8, void=0.2)
    _, dh, dw, db = ops.class_ce(h, w, b, lab)
    g = torch.Generator().manual_seed(1)
    for t, d in ((h, dh), (w, dw), (b, db)):
        dirn = torch.randn(t.shape, generator=g).cuda()
        eps = 2.0 ** -6
        args = lambda s: [x + s * eps * dirn if x is t else x for x in (h, w, b)]
        # 64-bit differences of the definition; third derivatives of a log-sum-exp of these sizes leave less than eps^2 = 2.4e-4 of the slope's scale
        f = lambda s: reference(*[a.double() for a in args(s)], lab, torch.ones(36, dtype=torch.float64, device="cuda"))["nll"].sum() / 36
        want = (f(1) - f(-1)) / (2 * eps)
        scale = d.double().norm() * dirn.double().norm()
        assert abs((d.double() * dirn.double()).sum() - want) <= 2e-3 * scale


def test_captured_replayed_and_on_another_stream():
    h, w, b, lab = make((2, 64, 16, 16), 300, B, F, seed=11)
    want = ops.class_ce(h, w, b, lab, mean_over="valid")
    h2, _, _, lab2 = make((2, 64, 16, 16), 300, B, F, seed=12)
    want2 = ops.class_ce(h2, w, b, lab2, mean_over="valid")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.class_ce(h, w, b, lab, mean_over="valid")
        other = ops.class_ce(h2, w, b, lab2, mean_over="valid")
    torch.cuda.current_stream().wait_stream(s)
    for a, c in zip(want + want2, got + other):
        assert torch.equal(a, c)
    hs, ls = h.clone(), lab.clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = ops.class_ce(hs, w, b, ls, mean_over="valid")
    with torch.cuda.graph(g2):
        o2 = ops.class_ce(h2, w, b, lab2, mean_over="valid")
    for it in range(4):
        src = (h, lab, want) if it % 2 == 0 else (h2, lab2, want2)
        hs.copy_(src[0]); ls.copy_(src[1])
        g1.replay(); g2.replay()
        ops.class_ce(h, w, b, lab)                    # eager work between the replays
        torch.cuda.synchronize()
        for a, c in zip(src[2] + want2, o1 + o2):
            assert torch.equal(a, c)
    with pytest.raises(RuntimeError, match="capture"):
        leaf = w.clone().requires_grad_(True)
        g3 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g3):
            maxstyle_amd.class_cross_entropy(h, leaf, b, lab)


def test_several_pieces():
    """More rows and more classes than one piece of G holds: the running sums of dh and dw, and db's."""
    for shape, V, hdt, wdt in (((9001, 64), 8300, B, B), ((4500, 64), 8300, F, F), ((14000, 64), 17000, B, B), ((7100, 48), 17000, F, F), ((28, 64, 16, 16), 17000, B, F)):
        h, w, b, lab = make(shape, V, hdt, wdt, seed=1, wscale=2.0)
        P = lab.numel()
        r = reference(h, w, b, lab, torch.full((P,), 1.0 / P, dtype=torch.float64, device="cuda"))
        loss, dh, dw, db = ops.class_ce(h, w, b, lab)
        tdh, tdw, tdb = tolerances(r, hdt, wdt)
        close(rows_of(dh, shape[1]), r["dh"], tdh, "dh")
        close(dw, r["dw"], tdw, "dw")
        close(db, r["db"], tdb, "db")


def test_the_most_classes():
    """2^20 classes: the statistics of all rows no longer fit beside one another and are formed 2048 rows at a time.  Checked on rows around the cut and at the end."""
    V, C, P = 1 << 20, 136, 2100
    h, w, b, lab = make((P, C), 64, B, B, seed=3, void=0.0)
    g = torch.Generator(device="cuda").manual_seed(0)
    w = (torch.randn(V, C, generator=g, device="cuda") / C ** 0.5).to(B)
    b = torch.randn(V, generator=g, device="cuda") * 0.3
    lab = torch.randint(0, V, (P,), generator=g, device="cuda")
    nll, lse = ops.class_ce_fwd(h, w, b, lab)
    for i in (0, 1, 1023, 1024, 2047, 2048, 2049, 2098, 2099):
        z = (w.double() @ h[i].double()) + b.double()
        A = float((w.double().abs() @ h[i].double().abs()).max() + b.abs().max())
        want = torch.logsumexp(z, 0)
        # classes are summed 64 fp32 terms a thread, then in a tree of 16384 / 16 + 16 parts: (64 + 1040) u32 of the sum
        tol = 2 * A * (3 * 2.0 ** -22 + (3 * C + 8) * U32) + (16 + 1104) * U32 * (abs(float(want)) + 1)
        assert abs(float(lse[i]) - float(want)) <= tol and abs(float(nll[i]) - float(want - z[lab[i]])) <= tol


def test_unaligned_views():
    h, w, b, lab = make((2, 16, 9, 7), 21, seed=3)
    want = ops.class_ce(h, w, b, lab)
    shift = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
    got = ops.class_ce(shift(h), shift(w), shift(b), shift(lab))
    for a, c in zip(want, got):
        assert torch.equal(a, c)


@pytest.mark.parametrize("shape,V", [((1, 512), 700), ((2, 512, 16, 17), 900), ((130, 640), 9000), ((2, 64, 18, 20), 300), ((40, 16), 9)])
def test_whatever_the_workspace_held(shape, V):
    h, w, b, lab = make(shape, V, seed=21)
    N, C = shape[:2]
    nbytes = ops.lib.ms_class_ce_ws_bytes(N, C, V, lab.numel() // N, 0, 1)
    got = []
    for fill in (0, 255):                # 255: every float and half of it a NaN
        block = torch.full((nbytes,), fill, dtype=torch.uint8, device="cuda")
        del block                        # the caching allocator hands the block to the call
        got.append(ops.class_ce(h, w, b, lab, mean_over="valid"))
    for a, c in zip(*got):
        assert torch.equal(a, c) and torch.isfinite(a).all()


@pytest.mark.parametrize("images", [17, 33])
def test_features_of_more_than_two_and_four_gigabytes(images):
    g = torch.Generator(device="cuda").manual_seed(images)
    shape, V = (images, 64, 1024, 1024), 7
    h = torch.randn(shape, generator=g, device="cuda", dtype=B)
    w = (torch.randn(V, 64, generator=g, device="cuda") / 8)
    lab = torch.randint(0, V, (images, 1024, 1024), generator=g, device="cuda")
    gr = torch.randn(lab.shape, generator=g, device="cuda")
    nll, lse = ops.class_ce_fwd(h, w, None, lab)
    dh = ops.class_ce_bwd(h, w, None, lab, lse, gr, need_dw=False)[0]
    for i in (0, 15, 16, images - 1):
        cut = (slice(i, i + 1), slice(None), slice(1016, 1024))
        hc, lc, gc = h[cut].contiguous(), lab[i:i + 1, 1016:].contiguous(), gr[i:i + 1, 1016:].contiguous()
        r = reference(hc, w, None, lc, gc.double().reshape(-1))
        close(nll[i, 1016:].reshape(-1), r["nll"], 2 * r["dz"] + 16 * U32 * (r["lse"].abs() + r["nll"] + 1), "nll")
        close(rows_of(dh[cut], 64), r["dh"], tolerances(r, B, F)[0], "dh")


def test_more_rows_than_one_axis_of_a_launch_holds():
    P, C, V = (1 << 26) + 300, 130, 5
    g = torch.Generator(device="cuda").manual_seed(2)
    h = torch.randn(P, C, generator=g, device="cuda", dtype=B)
    w = (torch.randn(V, C, generator=g, device="cuda") / C ** 0.5).to(B)
    b = torch.randn(V, generator=g, device="cuda") * 0.3
    lab = torch.randint(0, V, (P,), generator=g, device="cuda")
    gr = torch.randn(P, generator=g, device="cuda")
    nll, lse = ops.class_ce_fwd(h, w, b, lab)
    dh = ops.class_ce_bwd(h, w, b, lab, lse, gr, need_dw=False)[0]
    for a in (0, (1 << 25) - 50, (1 << 26) - 50, P - 100):
        s = slice(a, a + 100)
        r = reference(h[s], w, b, lab[s], gr[s].double())
        close(nll[s], r["nll"], 2 * r["dz"] + 16 * U32 * (r["lse"].abs() + r["nll"] + 1), "nll")
        # the lowest step of G is that of the largest upstream gradient of all rows (at most 7 of a normal draw, times the largest feature, below 8)
        low = 7 * 8 * 2.0 ** -36 / r["x"].abs().amax(1, keepdim=True).clamp_min(1e-30) * V * r["w"].abs().amax(0)
        close(dh[s], r["dh"], tolerances(r, B, B)[0] + low, "dh")


@pytest.mark.parametrize("shape,V", [((1, 16, 60, 60), 5), ((4, 64, 30, 30), 700), ((4000, 136), 400)])
def test_errors_of_rows_do_not_add_up(shape, V):
    """The log-sums are off by single roundings that lie on both sides: their mean stays below what the exponential's and the logarithm's cut results leave (half a step of
    [0, 1) each, 2 u32) and four standard deviations of the roundings (uniform, at most one step, 16 u32, of values in [8, 16), P of them)."""
    h, w, b, lab = make(shape, V, seed=31, void=0.0)
    lse = ops.class_ce_fwd(h, w, b, lab)[1].double().reshape(-1)
    want = torch.logsumexp(rows_of(h.double(), shape[1]) @ w.double().T + b.double(), 1)
    assert abs(float((lse - want).mean())) <= 2 * U32 + 4 * 16 * U32 / 12 ** 0.5 / lab.numel() ** 0.5


def test_both_forms_over_many_rows_and_classes():
    """Several pieces of rows and classes in the wide form (more than 128 channels), as rows and as planes, and the narrow form's long class loop."""
    for shape, V, hdt, wdt in (((9001, 136), 8300, B, B), ((14000, 136), 17000, B, B), ((7100, 136), 17000, F, F), ((28, 136, 16, 16), 17000, B, F), ((12000, 64), 9001, F, F),
                               ((8, 16, 32, 33), 7000, B, F)):
        h, w, b, lab = make(shape, V, hdt, wdt, seed=1, wscale=2.0)
        P = lab.numel()
        r = reference(h, w, b, lab, torch.full((P,), 1.0 / P, dtype=torch.float64, device="cuda"))
        loss, dh, dw, db = ops.class_ce(h, w, b, lab)
        tdh, tdw, tdb = tolerances(r, hdt, wdt)
        close(rows_of(dh, shape[1]), r["dh"], tdh, "dh")
        close(dw, r["dw"], tdw, "dw")
        close(db, r["db"], tdb, "db")
