"""Random calls of the kernels' host build, every buffer between unmapped pages: python sweep.py class_ce|class_ce_pieces|logit_ce|act8 SEED COUNT.

A read or write outside a buffer ends the process; margins that a page cannot guard are checked; results are compared with the definition in 64 bits.  The case is
printed before it runs.  class_ce_pieces: the limits of a piece and of the larger tiles lowered, so that small inputs take several pieces and every tile size.

Tolerances of class_ce (u = 2^-24): logits |dz| <= A (3 2^-22 + (3 C + 8) u), A = sum_c |w h| + |b|; G relative 2 |dz| + 2^-21 and 2 u; its planes and the other operand's 3 2^-22, or
G's 2^-11 where h and w are both bf16; sums of 3 terms a step; half a step of the result's type."""
import random
import sys

import numpy as np

import build
import guarded as g

U = 2.0 ** -24
PIECES = {"kCePieceBytes = (size_t)224 << 20, kCeStatsBytes = (size_t)256 << 20": "kCePieceBytes = (size_t)1 << 20, kCeStatsBytes = (size_t)1 << 17",
          "even(k.Vp, 16384)": "even(k.Vp, 512)", "* split >= 200": "* split >= 4", "* split >= 128": "* split >= 2"}


def log(r, a, b):
    return int(round(np.exp(r.uniform(np.log(a), np.log(b)))))


def class_ce_bounds(e, h, w, b, hb, wb):
    """Elementwise tolerances of dh, dw, db for exact_ce's result."""
    h = g.from_bf16(g.to_bf16(h)) if hb else h
    w = g.from_bf16(g.to_bf16(w)) if wb else w
    x, wd = np.where(e["ok"][:, None], g.rows(h), 0).astype(np.float64), w.astype(np.float64)
    (P, C), V = x.shape, wd.shape[0]
    A = (np.abs(x) @ np.abs(wd).T + (0 if b is None else np.abs(b))).max(1)
    dz = A * (3 * 2.0 ** -22 + (3 * C + 8) * U)
    mag = e["rounded"]
    err = mag * ((2 * dz + 2.0 ** -21)[:, None] + 2 * U)
    gx = gw = 2.0 ** -11 if hb and wb else 3 * 2.0 ** -22
    half = {0: U, 1: 2.0 ** -8}
    planes = lambda a: np.moveaxis(a.reshape((h.shape[0],) + h.shape[2:] + (C,)), -1, 1)
    tdh = planes(err @ np.abs(wd) + mag @ np.abs(wd) * (gx + (3 * V + 8) * U)) + half[hb] * np.abs(e["dh"])
    tdw = err.T @ np.abs(x) + mag.T @ np.abs(x) * (gw + (3 * P + 8) * U) + half[wb] * np.abs(e["dw"])
    tdb = err.sum(0) + mag.sum(0) * (P * U + 2.0 ** -22)
    tn = 2 * dz + 16 * U * (np.abs(e["lse"]) + e["nll"] + 1)
    return dict(dh=tdh, dw=tdw, db=tdb, nll=tn)


def class_ce(r, lib, show):
    while True:
        C = r.choice([16, 32, 64, 96, 128, log(r, 1, 128), log(r, 1, 128), log(r, 129, 700), r.choice([136, 192, 256, 512, 130])])
        V = log(r, 1, 3000)
        shape = (log(r, 1, 3000), C) if r.random() < 0.4 else (log(r, 1, 5), C, log(r, 1, 40), log(r, 1, 40))
        P = int(np.prod(shape)) // C
        if P * V * C <= 3e7:
            break
    hb, wb = r.choice([(0, 0), (0, 0), (1, 0), (0, 1), (1, 1)])
    mode, align, bias, valid, fill = r.choice(["end", "start"]), r.choice([16, 4]), r.random() < 0.8, r.random() < 0.5, r.choice([255, 0])
    need = r.choice(["hwb", "hwb", "hwb", "h", "w", "b", "hw", ""])
    bwd = need != "" and (need != "b" or bias) and r.random() < 0.3
    rng = np.random.default_rng(r.randrange(1 << 30))
    h = rng.standard_normal(shape).astype(np.float32)
    w = (rng.standard_normal((V, C)) / C ** 0.5).astype(np.float32)
    b = (0.3 * rng.standard_normal(V)).astype(np.float32) if bias else None
    lab = rng.integers(0, V, (shape[0],) + shape[2:])
    lab[rng.random(lab.shape) < 0.1] = r.choice([-100, V, 255 + V])
    grad = rng.standard_normal(P) if bwd else None
    show(shape, V, hb, wb, mode, align, bias, valid, fill, need, bwd)
    o = g.class_ce(lib, h, w, b, lab, hb, wb, valid, mode, align, need, grad, fill=fill)
    assert o["inside"]
    e = g.exact_ce(h, w, b, lab, hb, wb, valid, grad)
    t = class_ce_bounds(e, h, w, b, hb, wb)
    if bwd:
        assert (np.abs(o["nll"] - e["nll"]) <= t["nll"]).all()
        assert (np.abs(o["lse"] - e["lse"]) <= t["nll"])[e["ok"]].all()
    else:
        assert abs(o["loss"] - e["loss"]) <= t["nll"].sum() / max(int(e["ok"].sum()) if valid else P, 1) + 2 * U * e["loss"]
    for k in ("dh", "dw", "db"):
        if k in o:
            assert (np.abs(o[k] - e[k]) <= t[k]).all(), k


def logit_ce(r, lib, show):
    while True:
        N, K, HW = log(r, 1, 6), log(r, 1, 3000), log(r, 1, 3000)
        if N * K * HW <= 400000:
            break
    HW = HW // 4 * 4 if r.random() < 0.5 and HW >= 4 else HW
    mode, align, mask = r.choice(["end", "start"]), r.choice([16, 4]), r.choice([None, -1e4, -1e12, -3.4028234663852886e38, -np.inf])
    rng = np.random.default_rng(r.randrange(1 << 30))
    z = (3 * rng.standard_normal((N, K, HW))).astype(np.float32)
    lab = rng.integers(0, K, (N, HW))
    if mask is not None:
        keep = rng.random((N, K, HW)) < 0.5
        np.put_along_axis(keep, lab[:, None], True, 1)
        z = np.where(keep, z, np.float32(mask))
    lab[rng.random(lab.shape) < 0.1] = r.choice([-1, K, -100])
    show(N, K, HW, mode, align, mask)
    c = g.Call(mode)
    Z, L, out = c.put(z, align), c.put(lab.astype(np.int64), 8), c.block(4, 4)
    lib.ms_logit_ce_ws_bytes.restype = g.ctypes.c_size_t
    ws = c.block(lib.ms_logit_ce_ws_bytes(), 8)
    assert lib.ms_logit_ce(g.p(Z), g.p(L), g.p(out), N, K, HW, g.ctypes.c_float(1.0), g.p(ws), g.ctypes.c_size_t(ws.nbytes), None) == 0
    got = float(out.array(np.float32, (1,))[0])
    assert c.done()
    zd = z.astype(np.float64)
    m = zd.max(1)
    with np.errstate(all="ignore"):
        lse = m + np.log(np.exp(zd - m[:, None]).sum(1))
    ok = (lab >= 0) & (lab < K)
    nll = np.where(ok, lse - np.take_along_axis(zd, np.where(ok, lab, 0)[:, None], 1)[:, 0], 0)
    # exponents to 2 u |z - max| log2(e), of at most 30 where a term counts; K fp32 additions; the difference and the logarithm 4 u of their size
    assert abs(got - nll.sum() / nll.size) <= (K + 100) * U + 8 * U * (np.abs(nll).sum() / nll.size + 1), (got, nll.sum() / nll.size)


def act8(r, lib, show):
    while True:
        shape = (log(r, 1, 40), log(r, 1, 300), log(r, 1, 400), log(r, 1, 400)) if r.random() < 0.7 else (1, log(r, 1, 3), log(r, 100, 700), log(r, 100, 700))
        if np.prod(shape) <= 400000:
            break
    bf, mode, align, kind = r.random() < 0.4, r.choice(["end", "start"]), r.choice([16, 1]), r.choice([None, "near", "far"])
    ref, slope = r.random() < 0.4, r.choice([0.0, 0.2, 1.0])
    rng = np.random.default_rng(r.randrange(1 << 30))
    C = shape[1]
    x = rng.standard_normal(shape) * 1.7 + rng.standard_normal((1, C, 1, 1)) * 2
    x = (g.from_bf16(g.to_bf16(x)) if bf else x.astype(np.float32)).astype(np.float64)
    coef = None
    if kind:
        m, inv = x.mean((0, 2, 3)), 1 / np.sqrt(x.var((0, 2, 3)) + 1e-5)
        gamma = (0.5 + rng.random(C)) * np.where(np.arange(C) % 3 == 1, -1, 1)
        beta = 0.3 * rng.standard_normal(C) + (9 * gamma if kind == "far" else 0)
        coef = np.stack([gamma * inv, beta - m * gamma * inv, m, inv], 1).astype(np.float32)
    gr = rng.standard_normal(shape)
    rq = rng.integers(-3, 4, shape) if ref else None
    show(shape, bf, mode, align, kind, ref, slope)
    o, e = g.act8(lib, x, coef, gr, rq, slope, bf, mode, align), g.exact_act8(x, coef, gr, rq, slope, bf)
    half = 2.0 ** -8 if bf else U
    assert o["inside"] and (o["q"] == e["q"]).all() and (o["s"] == e["s"]).all()
    assert (np.abs(o["x"] - e["x"]) <= half * (1 + 2.0 ** -20) * np.abs(e["x"])).all()
    if coef is None:
        return
    assert (o["x2"] == o["x"]).all() and (np.abs(o["g"] - e["g"]) <= (half + U) * (1 + 2.0 ** -20) * np.abs(e["g"])).all()
    # x' - mean: 3 u of its two parts; four (16 in the one-launch kernel) fp32 terms, their products, then 64 bits: 20 u of the sum of magnitudes
    col = lambda a: a.astype(np.float64)[None, :, None, None]
    xm, ge = e["x"] - col(coef[:, 2]), np.abs(e["g"])
    xe = 3 * U * (np.abs(e["x"] - col(e["centre"])) + np.abs(col(e["centre"]) - col(coef[:, 2])))
    e1, e2 = 20 * U * ge.sum((0, 2, 3)), 20 * U * (ge * np.abs(xm)).sum((0, 2, 3)) + (ge * xe).sum((0, 2, 3))
    assert (np.abs(o["part"] - np.stack([e["s1"], e["s2"]], 1)) <= np.stack([e1, e2], 1) + U * np.abs(np.stack([e["s1"], e["s2"]], 1))).all()
    assert (np.abs(o["dbeta"] - e["s1"]) <= e1 + U * np.abs(e["s1"])).all()
    assert (np.abs(o["dgamma"] - e["dgamma"]) <= e2 * coef[:, 3] + 2 * U * np.abs(e["dgamma"])).all()
    M, k = x.size // C, coef.astype(np.float64)
    w = k[:, 3] ** 2 / M
    t1, t2 = col(e["s1"] / M), xm * col(e["s2"] * w)
    tol = col(np.abs(k[:, 0])) * (4 * U * (ge + np.abs(t1) + 2 * np.abs(t2)) + col(e1 / M) + np.abs(xm) * col(e2 * w) + xe * col(np.abs(e["s2"]) * w))
    assert (np.abs(o["du"] - e["du"]) <= tol + half * np.abs(e["du"]) * (1 + 2.0 ** -20)).all()


def main(which, seed, count):
    run, lib = {"class_ce": class_ce, "class_ce_pieces": class_ce, "act8": act8, "logit_ce": logit_ce}[which], build.load(PIECES if which == "class_ce_pieces" else None)
    r = random.Random(seed)
    for i in range(count):
        run(r, lib, lambda *case: print(which, seed, i, *case, flush=True))
    print("done", flush=True)


if __name__ == "__main__":
    main(sys.argv[1], int(sys.argv[2]), int(sys.argv[3]))
