"""Arrays between unmapped pages, and the C entries of the host build called with them."""
import ctypes
import mmap
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import build  # noqa: E402

PAGE = 4096
_libc = ctypes.CDLL(None, use_errno=True)
_libc.mmap.restype = ctypes.c_void_p
_libc.mmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_long]
_libc.munmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t]
_libc.mprotect.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]


class Block:
    """`nbytes` that end (mode "end", but for what `align` leaves) or start ("start") at an unmapped page; filled with `fill`."""

    def __init__(self, nbytes, mode, align=16, fill=0xFF):
        self.body = (nbytes + 2 * PAGE - 1) // PAGE * PAGE
        self.total = self.body + 2 * PAGE
        self.base = _libc.mmap(None, self.total, mmap.PROT_READ | mmap.PROT_WRITE, mmap.MAP_PRIVATE | mmap.MAP_ANONYMOUS, -1, 0)
        if self.base in (None, ctypes.c_void_p(-1).value):
            raise MemoryError
        first, last = self.base + PAGE, self.base + PAGE + self.body
        self.ptr = first if mode == "start" else (last - nbytes) // align * align
        self.nbytes = nbytes
        ctypes.memset(first, fill, self.body)
        _libc.mprotect(self.base, PAGE, 0)
        _libc.mprotect(last, PAGE, 0)
        self.first, self.last, self.fill = first, last, fill

    def array(self, dtype, shape):
        return np.frombuffer((ctypes.c_char * self.nbytes).from_address(self.ptr), dtype=dtype).reshape(shape)

    def margins_untouched(self):
        """The bytes between the pages and the block still hold `fill`."""
        a = ctypes.string_at(self.first, self.ptr - self.first)
        b = ctypes.string_at(self.ptr + self.nbytes, self.last - self.ptr - self.nbytes)
        return a.count(bytes([self.fill])) == len(a) and b.count(bytes([self.fill])) == len(b)

    def free(self):
        _libc.munmap(self.base, self.total)


def to_bf16(x):
    """Nearest even, as uint16."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


class Call:
    """Blocks of one call."""

    def __init__(self, mode):
        self.mode, self.blocks = mode, []

    def block(self, nbytes, align=16, fill=0xFF):
        b = Block(max(int(nbytes), 1), self.mode, align, fill)
        self.blocks.append(b)
        return b

    def put(self, a, align=16):
        b = self.block(a.nbytes, align)
        b.array(a.dtype, a.shape)[...] = a
        return b

    def done(self):
        ok = all(b.margins_untouched() for b in self.blocks)
        for b in self.blocks:
            b.free()
        self.blocks = []
        return ok


def p(b):
    return ctypes.c_void_p(0 if b is None else b.ptr)


def class_ce(lib, h, w, b, lab, hb=False, wb=False, mean_valid=False, mode="end", align=16, need="hwb", grad=None, sign=1.0, fill=0xFF):
    """ms_class_ce (grad None) or ms_class_ce_fwd + ms_class_ce_bwd (grad: one value a row).  Returns dict of float64 arrays."""
    N, C = h.shape[:2]
    V = w.shape[0]
    HW = int(np.prod(h.shape[2:])) if h.ndim > 2 else 1
    types = int(hb) | 2 * int(wb)
    c = Call(mode)
    ha, wa = (2 if hb else 4) if align < 16 else 16, (2 if wb else 4) if align < 16 else 16
    H = c.put(to_bf16(h) if hb else h.astype(np.float32), ha)
    W = c.put(to_bf16(w) if wb else w.astype(np.float32), wa)
    B = None if b is None else c.put(b.astype(np.float32), 4)
    L = c.put(lab.astype(np.int64), 8)
    dh = c.block(H.nbytes, ha) if "h" in need else None
    dw = c.block(W.nbytes, wa) if "w" in need else None
    db = c.block(4 * V, 4) if "b" in need and b is not None else None
    lib.ms_class_ce_ws_bytes.restype = ctypes.c_size_t
    P = N * HW
    out = {}

    def check(rc):
        if rc:
            raise RuntimeError(f"{rc}: {lib.host_last_error().decode()}")

    grads = dh is not None or dw is not None or db is not None
    if grad is None:
        ws = c.block(lib.ms_class_ce_ws_bytes(N, C, V, HW, types, int(grads)), fill=fill)
        loss = c.block(4, 4)
        check(lib.ms_class_ce(p(H), p(W), p(B), p(L), p(loss), p(dh), p(dw), p(db), N, C, V, HW, types, ctypes.c_float(sign), int(mean_valid), None, p(ws), ctypes.c_size_t(ws.nbytes), None))
        out["loss"] = float(loss.array(np.float32, (1,))[0])
    else:
        ws = c.block(lib.ms_class_ce_ws_bytes(N, C, V, HW, types, 0), fill=fill)
        nll, lse = c.block(4 * P, 4), c.block(4 * P, 4)
        check(lib.ms_class_ce_fwd(p(H), p(W), p(B), p(L), p(nll), p(lse), N, C, V, HW, types, p(ws), ctypes.c_size_t(ws.nbytes), None))
        out["nll"], out["lse"] = (x.array(np.float32, (P,)).astype(np.float64) for x in (nll, lse))
        if grads:
            ws2 = c.block(lib.ms_class_ce_ws_bytes(N, C, V, HW, types, 1), fill=fill)
            G = c.put(np.asarray(grad, np.float32), 4)
            check(lib.ms_class_ce_bwd(p(H), p(W), p(B), p(L), p(lse), p(G), p(dh), p(dw), p(db), N, C, V, HW, types, p(ws2), ctypes.c_size_t(ws2.nbytes), None))
    val = lambda x, bf, shape: (from_bf16(x.array(np.uint16, shape)) if bf else x.array(np.float32, shape)).astype(np.float64)
    if dh is not None:
        out["dh"] = val(dh, hb, h.shape)
    if dw is not None:
        out["dw"] = val(dw, wb, w.shape)
    if db is not None:
        out["db"] = val(db, False, (V,))
    out["inside"] = c.done()
    return out


def rows(x):
    return np.moveaxis(x, 1, -1).reshape(-1, x.shape[1])


def exact_ce(h, w, b, lab, hb, wb, mean_valid, grad=None, sign=1.0, dtype=np.float64):
    """The definition in 64 bits (or, dtype=float32, the plain form: every product and sum rounded as numpy's), on the values as they are held."""
    h = from_bf16(to_bf16(h)) if hb else h.astype(np.float32)
    w = from_bf16(to_bf16(w)) if wb else w.astype(np.float32)
    x, wd = rows(h).astype(dtype), w.astype(dtype)
    V, y = w.shape[0], lab.reshape(-1)
    ok = (y >= 0) & (y < V)
    x = np.where(ok[:, None], x, 0).astype(dtype)          # (what a row without a class holds does not matter)
    z = x @ wd.T + (0 if b is None else b.astype(np.float32).astype(dtype))
    m = z.max(1, keepdims=True)
    e = np.exp(z - m)
    t = e.sum(1, keepdims=True)
    pos = np.nonzero(ok)[0]
    nll = np.zeros(len(y), dtype)
    nll[pos] = (m[pos, 0] - z[pos, y[pos]]) + np.log(t[pos, 0])
    n = max(int(ok.sum()), 1) if mean_valid else len(y)
    g = (np.full(len(y), dtype(sign) / dtype(n)) if grad is None else np.asarray(grad, np.float32)).astype(dtype)
    g = np.where(ok, g, 0).astype(dtype)
    G = e / t
    mag = G.copy()
    mag[pos, y[pos]] += 1
    mag = np.where(ok[:, None], mag * np.abs(g)[:, None], 0)          # what is rounded
    G[pos, y[pos]] -= 1
    G = np.where(ok[:, None], G * g[:, None], 0).astype(dtype)
    planes = lambda a: np.moveaxis(a.reshape((h.shape[0],) + h.shape[2:] + (h.shape[1],)), -1, 1)
    return dict(loss=sign * float(nll.astype(np.float64).sum()) / n, nll=nll, lse=(m + np.log(t))[:, 0], dh=planes(G @ wd), dw=G.T @ x, db=G.sum(0), G=G, ok=ok,
                rounded=mag, zmax=float(np.abs(z[e > 0]).max(initial=0)), mdh=planes(mag @ np.abs(wd)), mdw=mag.T @ np.abs(x),
                tdh=planes(np.repeat(np.abs(g)[:, None], V, 1) @ np.abs(wd)), tdw=np.repeat(np.abs(g)[None], V, 0) @ np.abs(x))


def act8(lib, x, coef, g, ref, slope, bf, mode="end", align=16):
    """pack, unpack, bwd_reduce (with x') and bn_act_bwd of one checkpoint; returns dict of arrays."""
    N, C = x.shape[:2]
    HW = int(np.prod(x.shape[2:]))
    c = Call(mode)
    al = 16 if align == 16 else (2 if bf else 4)
    act = (lambda a: c.put(to_bf16(a) if bf else a.astype(np.float32), al))
    nbytes = x.size * (2 if bf else 4)
    X, G = act(x), act(g)
    K = None if coef is None else c.put(coef.astype(np.float32), 16)
    nb = -(-HW // 256)
    q, s = c.block(x.size, 16 if align == 16 else 1), c.block(4 * N * C * nb, 4)
    sfx = "_bf16" if bf else ""

    def check(rc):
        if rc:
            raise RuntimeError(f"{rc}: {lib.host_last_error().decode()}")

    val = lambda b, shape=x.shape: from_bf16(b.array(np.uint16, shape)).copy() if bf else b.array(np.float32, shape).copy()
    check(getattr(lib, "ms_act8_pack" + sfx)(p(X), p(K), p(q), p(s), N, C, HW, None))
    U = c.block(nbytes, al)
    check(getattr(lib, "ms_act8_unpack" + sfx)(p(q), p(s), p(K), p(U), N, C, HW, None))
    out = dict(q=q.array(np.int8, x.shape).copy(), s=s.array(np.float32, (N, C, nb)).copy(), x=val(U))
    if K is not None:
        R = None if ref is None else c.put(ref.astype(np.int8), 16 if align == 16 else 1)
        parts = lib.ms_act8_bwd_parts(N, C, HW)
        part, go, uo = c.block(8 * C * parts, 8), c.block(nbytes, al), c.block(nbytes, al)
        sl = ctypes.c_float(slope)
        check(getattr(lib, "ms_act8_bwd_reduce" + sfx)(p(G), p(R), p(q), p(s), p(K), p(go), p(uo), p(part), N, C, HW, sl, None))
        lib.ms_act8_bwd_ws_bytes.restype = ctypes.c_size_t
        ws = c.block(lib.ms_act8_bwd_ws_bytes(N, C, HW), 8)
        du, dg, db = c.block(nbytes, al), c.block(4 * C, 4), c.block(4 * C, 4)
        check(getattr(lib, "ms_act8_bn_act_bwd" + sfx)(p(G), p(R), p(q), p(s), p(K), p(du), p(dg), p(db), N, C, HW, sl, p(ws), ctypes.c_size_t(ws.nbytes), None))
        out.update(g=val(go), x2=val(uo), part=part.array(np.float32, (C, parts, 2)).astype(np.float64).sum(1), du=val(du),
                   dgamma=dg.array(np.float32, (C,)).astype(np.float64), dbeta=db.array(np.float32, (C,)).astype(np.float64))
    out["inside"] = c.done()
    return out


def exact_act8(x, coef, g, ref, slope, bf):
    """The definition in 64 bits, on the values as they are held."""
    N, C = x.shape[:2]
    up = (lambda a: from_bf16(to_bf16(a))) if bf else (lambda a: a.astype(np.float32))
    X, g = (up(a).astype(np.float64).reshape(N, C, -1) for a in (x, g))
    cen, near = np.zeros(C), np.zeros(C, bool)
    if coef is not None:
        k = coef.astype(np.float32).astype(np.float64)
        with np.errstate(all="ignore"):
            t = -k[:, 1] / k[:, 0]
            near = np.abs(t - k[:, 2]) * k[:, 3] <= 4
        cen = np.where(near, t, k[:, 2])
    d = X - cen[None, :, None]
    q, s = np.zeros_like(d), []
    for i in range(0, d.shape[2], 256):
        b = d[:, :, i:i + 256]
        sc = (np.abs(b).max(2).astype(np.float32).astype(np.float64) / 127).astype(np.float32)
        r = np.rint(np.divide(b, sc[..., None].astype(np.float64), out=np.zeros_like(b), where=sc[..., None] > 0))
        q[:, :, i:i + 256] = np.where((r == 0) & (b != 0), np.sign(b), r)
        s.append(sc)
    s = np.stack(s, 2)
    off = q * np.repeat(s.astype(np.float64), 256, 2)[:, :, :d.shape[2]]
    kept = cen[None, :, None] + off
    out = dict(q=q.reshape(x.shape), s=s, x=kept.reshape(x.shape), centre=cen)
    if coef is not None:
        col = lambda a: a[None, :, None]
        z = np.where(col(near), col(k[:, 0]) * q, col(k[:, 0]) * kept + col(k[:, 1])) if ref is None else ref.reshape(N, C, -1)
        gm = g * np.where(z > 0, 1.0, slope)
        xm = kept - col(k[:, 2])
        M = N * d.shape[2]
        s1, s2 = gm.sum((0, 2)), (gm * xm).sum((0, 2))
        out.update(g=gm.reshape(x.shape), s1=s1, s2=s2, dbeta=s1, dgamma=s2 * k[:, 3],
                   du=(col(k[:, 0]) * (gm - col(s1) / M - xm * col(k[:, 3] ** 2 * s2) / M)).reshape(x.shape))
    return out
