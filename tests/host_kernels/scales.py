"""Gradients of the many-class loss where rows or classes are zero or of very different size, on the host build: python scales.py wide|narrow.

Every row of dh and every class of dw is judged by itself, against its own terms m = |G|-magnitudes times the other operand: the error's norm over |m|'s, its median, 99 % quantile
and maximum over rows (classes).  An element of G is held to 2^-41 g_p at least, so m takes every p as 2^-20 more than it is.  The bar is what the plain form leaves in fp32 on the same input: 4 times its quantile, plus 3 2^-22 (both operands of a product are held to 2^-22, and
the product of the two low planes is left out), plus 2 2^-24 max|z| log2(e) where the gradients come from
a stored lse (z - lse, both rounded at that size, is an exponent; one call for loss and gradients has 2^-22 in its place).  A bf16 result adds half a step, 2^-8 of the value;
where h and w are both bf16, G has 11 bits: 2^-11."""
import sys

import numpy as np

import build
import guarded as g
import sweep


def errors(a, e, bf):
    """Relative errors of dh's rows and dw's classes."""
    out = {}
    for k in ("dh", "dw"):
        r = g.rows if k == "dh" else (lambda t: t)
        d = np.maximum(np.abs(r(a[k]).astype(np.float64) - r(e[k])) - (2.0 ** -8 * (1 + 2.0 ** -7) * np.abs(r(e[k])) if bf[k] else 0), 0)
        m = np.linalg.norm(r(e["m" + k]) + 2.0 ** -20 * r(e["t" + k]), axis=1)
        q = np.linalg.norm(d, axis=1)[m > 0] / m[m > 0]
        out[k] = np.quantile(q, [0.5, 0.99, 1.0])
    return out


def cases(narrow):
    F, B = 0, 1
    shape, V = ((1, 64, 16, 16), 151) if narrow else ((128, 136), 400)
    for hb, wb in ((F, F), (B, F), (F, B), (B, B)):
        for name in ("plain", "zero row", "zero class", "both", "both, small", "padded", "spread rows", "spread classes", "spread gradients", "large row", "switched off", "near classes", "near rows", "confident", "one channel"):
            rng = np.random.default_rng(5)
            if name == "one channel":
                if narrow:
                    continue
                shape, V = (78, 1), 2682
            C = shape[1]
            h = rng.standard_normal(shape)
            w = rng.standard_normal((V, C)) * (2.0 / C ** 0.5)
            b = 0.3 * rng.standard_normal(V)
            lab = rng.integers(0, V // 2, (shape[0],) + shape[2:])          # (half of the classes are never a label)
            P = lab.size
            grad = np.full(P, 1.0 / P)
            hr = np.moveaxis(h, 1, -1).reshape(P, C)
            if name == "confident":
                hr = hr + 6.0 * w[lab.reshape(-1)]
            if "small" in name:
                hr, w = hr * 0.01, w * 0.1
            if name.startswith("both") or name == "zero row":
                hr[3] = 0
            if name.startswith("both") or name == "zero class":
                w[5] = w[V - 2] = 0
            if name == "padded":
                w[V - 60:], b[V - 60:] = 0, -1e30
            if name == "spread rows":
                hr = hr * 2.0 ** rng.uniform(-30, 0, (P, 1))
            if name == "spread classes":          # (the narrow form keeps 64 classes below one scale: their weights to 2^-39 of the largest)
                w *= 2.0 ** rng.uniform(-15 if narrow else -30, 0, (V, 1))
            if name == "spread gradients":
                grad = grad * 2.0 ** rng.uniform(-30, 0, P)
            if name == "switched off":          # ... classes whose weights are anything finite
                w[3::7], b[3::7] = 1e30, -np.inf
                lab[np.isin(lab, np.arange(3, V, 7))] += 1
            if name == "near classes":          # weights that differ little: dh is a difference
                w = 3 + 0.02 * w
            if name == "near rows":          # ... features: dw is one
                hr = 3 + 0.02 * hr
            if name == "large row":
                hr[7] *= 1e6 if narrow else 1e4
            h = np.moveaxis(hr.reshape((shape[0],) + shape[2:] + (C,)), -1, 1).astype(np.float32)
            yield name, hb, wb, np.ascontiguousarray(h), w.astype(np.float32), b.astype(np.float32), lab, grad.astype(np.float32)
        shape, V = ((1, 64, 16, 16), 151) if narrow else ((128, 136), 400)


def main(form):
    narrow, bad = form == "narrow", 0
    for lib, pieces in ((build.load(), False), (build.load(sweep.PIECES), True)):
        for name, hb, wb, h, w, b, lab, grad in cases(narrow):
            if pieces and (narrow or hb != wb):          # (the narrow form has no pieces)
                continue
            e = g.exact_ce(h, w, b, lab, hb, wb, False, grad)
            plain = g.exact_ce(h, w, b, lab, hb, wb, False, grad, dtype=np.float32)
            own = g.class_ce(lib, h, w, b, lab, hb, wb, grad=grad)
            bf = {"dh": hb, "dw": wb}
            a, c = errors(own, e, bf), errors(plain, e, {"dh": 0, "dw": 0})
            bar = 3 * 2.0 ** -22 + 2.0 ** -23 * 1.4427 * e["zmax"] + (2.0 ** -11 if hb and wb else 0)
            fail = [] if own["inside"] else ["inside"]
            for k in a:
                fail += [k] if not (a[k] <= 4 * c[k] + bar).all() else []
            if name in ("plain", "confident", "near classes"):          # loss and gradients in one call: no log-sum is rounded in between
                e1, p1 = (g.exact_ce(h, w, b, lab, hb, wb, False, dtype=t) for t in (np.float64, np.float32))
                a1, c1 = errors(g.class_ce(lib, h, w, b, lab, hb, wb), e1, bf), errors(p1, e1, {"dh": 0, "dw": 0})
                fail += ["one call: %s %s" % (k, a1[k]) for k in a1 if not (a1[k] <= 4 * c1[k] + 4 * 2.0 ** -22 + (2.0 ** -11 if hb and wb else 0)).all()]
            bad += len(fail)
            print(form, name, "bf16" if hb else "fp32", "bf16" if wb else "fp32", *("%s %.1e %.1e %.1e (plain %.1e %.1e %.1e)" % ((k,) + tuple(a[k]) + tuple(c[k])) for k in a), "FAIL %s" % fail if fail else "",
                  flush=True)
    print("done" if not bad else "%d outside" % bad, flush=True)
    return bad


if __name__ == "__main__":
    sys.exit(1 if main(sys.argv[1]) else 0)
