"""8-bit activation checkpoints (ops.act8_*) against their definition in 64 bits.

The checkpoint's whole numbers and scales are decided in 64 bits by the kernel as well: they have to be equal.  What is read back carries one rounding of the output type
(2^-24 / 2^-8).  The backward: x' - mean carries 3 u32 of |centre - mean| + |q s|; du is four fp32 operations on terms g', S1/M and (x'-mean) invstd^2 S2/M, each within
4 u32 of its magnitude, times the scale; S1 and S2 are sums of at most 2^14/256 = 64 fp32 terms a thread, then 8 in a tree, then 64 bits: <= 80 u32 of the sum of magnitudes."""
import pytest
import torch

from maxstyle_amd import ops

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
SHAPES = [(1, 1, 1, 1), (2, 3, 1, 7), (1, 2, 15, 17), (2, 5, 16, 16), (1, 4, 16, 17), (3, 7, 33, 31), (2, 16, 64, 64), (4, 130, 12, 12), (2, 3, 129, 130), (1, 2, 300, 300), (2, 4, 257), (1, 3, 4, 5, 6)]


def record(u, seed, kind="near"):
    g = torch.Generator().manual_seed(seed)
    C = u.shape[1]
    x = u.double().transpose(0, 1).reshape(C, -1)
    mean, inv = x.mean(1), (x.var(1, unbiased=False) + 1e-5).rsqrt()
    gamma = (0.5 + torch.rand(C, generator=g).double()).cuda() * torch.where(torch.arange(C) % 3 == 1, -1.0, 1.0).double().cuda()
    beta = torch.randn(C, generator=g).double().cuda() * 0.3
    if kind == "far":
        beta = beta + 9 * gamma          # the BatchNorm's zero is 9 standard deviations away: centred on the mean
    if kind == "flat":
        gamma = gamma * 0                # a channel that is switched off
    sc = gamma * inv
    return torch.stack([sc, beta - mean * sc, mean, inv], 1).float().contiguous()


def centre(coef):
    c = coef.double()
    t = -c[:, 1] / c[:, 0]
    near = ((t - c[:, 2]).abs() * c[:, 3]) <= 4
    return torch.where(near, t, c[:, 2]), near


def pack(x, coef):
    N, C = x.shape[:2]
    d = x.double().reshape(N, C, -1)
    if coef is not None:
        d = d - centre(coef)[0].view(1, C, 1)
    q, s = torch.zeros_like(d), []
    for i in range(0, d.shape[2], 256):
        b = d[:, :, i:i + 256]
        sc = (b.abs().amax(2).float().double() / 127).float()
        r = torch.round(b / sc.double().unsqueeze(2))
        q[:, :, i:i + 256] = torch.where((r == 0) & (b != 0), torch.sign(b), r).nan_to_num(0.0)
        s.append(sc)
    return q.to(torch.int8).reshape(x.shape), torch.stack(s, 2)


def kept(q, s, coef):
    N, C = q.shape[:2]
    d = q.reshape(N, C, -1).double()
    d = d * s.double().repeat_interleave(256, 2)[:, :, :d.shape[2]]
    if coef is not None:
        d = d + centre(coef)[0].view(1, C, 1)
    return d.reshape(q.shape)


def act(shape, seed, dt):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(*shape, generator=g) * 1.7 + torch.randn(1, shape[1], *[1] * (len(shape) - 2), generator=g) * 2
    return u.to(dt).cuda()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", [None, "near", "far", "flat"])
def test_pack_and_read_back(shape, dt, kind):
    x = act(shape, 1, dt)
    coef = None if kind is None else record(x, 2, kind)
    q, s = ops.act8_pack(x, coef)
    wq, ws = pack(x, coef)
    assert torch.equal(s, ws) and torch.equal(q, wq)
    want = kept(q, s, coef)
    for odt in (torch.float32, torch.bfloat16):
        y = ops.act8_unpack(q, s, coef, dtype=odt)
        assert y.dtype == odt and ((y.double() - want).abs() <= HALF[odt] * want.abs() * (1 + 2 ** -20)).all()
    step = s.double().repeat_interleave(256, 2)[:, :, :x[0, 0].numel()].reshape(x.shape)
    d = x.double() if coef is None else x.double() - centre(coef)[0].view(1, -1, *[1] * (x.dim() - 2))
    assert ((want - x.double()).abs() <= torch.where(d.abs() < step / 2, step, step / 2 * (1 + 1e-6))).all()
    assert torch.equal(torch.sign(q.double()), torch.sign(d))                 # a sign is never lost


def test_ties_zeros_and_extremes():
    # steps of exactly 3: values on the border of two steps go to the even one
    x = torch.zeros(1, 1, 16, 16, device="cuda")
    v = torch.arange(-127, 127, device="cuda").float() * 3 + 1.5
    x.view(-1)[:254] = v
    x.view(-1)[254] = 381.0
    q, s = ops.act8_pack(x)
    wq, ws = pack(x, None)
    assert float(s) == 3.0 and torch.equal(q, wq) and torch.equal(s, ws)
    for scale in (1e-30, 1e-20, 1e30, 3e38):
        y = torch.randn(1, 2, 16, 16, generator=torch.Generator().manual_seed(0)).clamp(-1, 1).cuda() * scale
        q, s = ops.act8_pack(y)
        wq, ws = pack(y, None)
        assert torch.equal(q, wq) and torch.equal(s, ws)
    z = torch.zeros(2, 2, 5, 5, device="cuda")
    q, s = ops.act8_pack(z)
    assert not q.any() and not s.any() and not ops.act8_unpack(q, s).any()
    q, s = ops.act8_pack(z + 1e-38)                  # below 2^-120: kept as zeros
    assert not ops.act8_unpack(q, s).any()
    big = torch.ones(1, 2, 20, 20, device="cuda")
    big[0, 0, 3, 3] = float("inf"); big[0, 1, 19, 19] = float("nan")
    y = ops.act8_unpack(*ops.act8_pack(big)).view(2, 400)
    assert torch.isnan(y[0, :256]).all() and torch.equal(y[0, 256:], torch.ones(144, device="cuda"))
    assert torch.equal(y[1, :256], torch.ones(256, device="cuda")) and torch.isnan(y[1, 256:]).all()


def oracle(g, q, s, coef, slope, ref):
    N, C = q.shape[:2]
    flat = lambda t: t.double().reshape(N, C, -1)
    c = coef.double()
    col = lambda t: t.view(1, C, 1)
    ctr, near = centre(coef)
    x = flat(kept(q, s, coef))
    if ref is not None:
        on = flat(ref) > 0
    else:
        on = torch.where(col(near), flat(q) * col(torch.sign(c[:, 0])) > 0, (x - col(ctr)) * col(c[:, 0]) + col(c[:, 0] * ctr + c[:, 1]) > 0)
    gm = flat(g) * torch.where(on, 1.0, slope)
    xm = x - col(c[:, 2])
    M = N * x.shape[2]
    s1, s2 = gm.sum((0, 2)), (gm * xm).sum((0, 2))
    t1, t2 = col(s1 / M), xm * col(s2 * c[:, 3] ** 2 / M)
    du = col(c[:, 0]) * (gm - t1 - t2)
    xe = 3 * U32 * ((x - col(ctr)).abs() + col((ctr - c[:, 2]).abs()))
    e1 = gm.abs().sum((0, 2)) * 80 * U32
    e2 = ((gm * xm).abs().sum((0, 2)) * 80 * U32 + (gm.abs() * xe).sum((0, 2)))
    w = c[:, 3] ** 2 / M
    edu = col(c[:, 0].abs()) * (4 * U32 * (gm.abs() + t1.abs() + 2 * t2.abs()) + col(e1 / M) + xm.abs() * col(e2 * w) + xe * col(s2.abs() * w))
    return dict(gm=gm, x=x, s1=s1, s2=s2, du=du, edu=edu, e1=e1, e2=e2, inv=c[:, 3])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["near", "far", "flat", "ref"])
def test_backward(shape, dt, kind):
    u = act(shape, 3, dt)
    coef = record(u, 4, "near" if kind == "ref" else kind)
    q, s = ops.act8_pack(u, coef)
    ref = ops.act8_pack(act(shape, 5, dt))[0] if kind == "ref" else None
    g = act(shape, 6, dt)
    slope = 0.0 if kind == "ref" else 0.2
    o = oracle(g, q, s, coef, slope, ref)
    du, dg, db = ops.act8_bn_act_bwd(g, q, s, coef, slope, ref_q=ref)
    assert du.dtype == dt and du.shape == g.shape
    N, C = shape[:2]
    got = du.double().reshape(N, C, -1)
    assert ((got - o["du"]).abs() <= o["edu"] + HALF[dt] * o["du"].abs() + 1e-37).all()
    assert ((dg.double() - o["s2"] * o["inv"]).abs() <= o["e2"] * o["inv"] + 2 * U32 * (o["s2"] * o["inv"]).abs()).all()
    assert ((db.double() - o["s1"]).abs() <= o["e1"] + U32 * o["s1"].abs()).all()
    again = ops.act8_bn_act_bwd(g, q, s, coef, slope, ref_q=ref)
    assert torch.equal(du, again[0]) and torch.equal(dg, again[1]) and torch.equal(db, again[2])
    inplace = g.clone()
    ops.act8_bn_act_bwd(inplace, q, s, coef, slope, ref_q=ref, out=inplace)
    assert torch.equal(inplace, du)
    # the first pass alone, for the kernels behind it
    uo = torch.empty_like(g)
    gout, part, n = ops.act8_bwd_reduce(g, q, s, coef, slope, ref_q=ref, uout=uo)
    assert ((gout.double().reshape(N, C, -1) - o["gm"]).abs() <= (HALF[dt] + U32) * o["gm"].abs()).all()
    assert torch.equal(uo, ops.act8_unpack(q, s, coef, dtype=dt))
    p = part.double().sum(1)
    assert ((p[:, 0] - o["s1"]).abs() <= o["e1"]).all() and ((p[:, 1] - o["s2"]).abs() <= o["e2"]).all()


def test_close_to_the_unrounded_backward():
    """A whole layer: u -> BatchNorm -> LeakyReLU, its backward out of the checkpoint against autograd's on the unrounded u.  Each x' is off by at most a step, at random:
    du's difference stays within the relative step of the blocks' largest deviation (about 3.2 sigma / 127 = 2.5 %, uniform: / sqrt 12 = 0.7 %) of the terms it enters."""
    g = torch.Generator().manual_seed(0)
    u = torch.randn(4, 16, 40, 40, generator=g).cuda()
    coef = record(u, 1)
    gy = torch.randn(4, 16, 40, 40, generator=g).cuda()
    ud = u.double().requires_grad_(True)
    mean, var = ud.mean((0, 2, 3), keepdim=True), ud.var((0, 2, 3), unbiased=False, keepdim=True)
    c = coef.double()
    gamma = (c[:, 0] / c[:, 3]).view(1, -1, 1, 1)
    beta = (c[:, 1] + c[:, 0] * c[:, 2]).view(1, -1, 1, 1)
    y = torch.nn.functional.leaky_relu((ud - mean) * (var + 1e-5).rsqrt() * gamma + beta, 0.2)
    (want,) = torch.autograd.grad(y, ud, gy.double())
    du, _, _ = ops.act8_bn_act_bwd(gy, *ops.act8_pack(u, coef), coef, 0.2)
    assert (du.double() - want).norm() <= 0.01 * want.norm()


def test_unaligned_captured_streams():
    u = act((2, 8, 20, 20), 1, torch.float32)
    coef = record(u, 2)
    shift = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
    q, s = ops.act8_pack(u, coef)
    q2, s2 = ops.act8_pack(shift(u), coef)
    assert torch.equal(q, q2) and torch.equal(s, s2)
    assert torch.equal(ops.act8_unpack(q, s, coef), ops.act8_unpack(shift(q), shift(s), coef))
    g = act((2, 8, 20, 20), 3, torch.float32)
    want = ops.act8_bn_act_bwd(g, q, s, coef, 0.2)
    got = ops.act8_bn_act_bwd(shift(g), shift(q), shift(s), coef, 0.2)
    for a, c in zip(want, got):
        assert torch.allclose(a, c, rtol=1e-4, atol=1e-6 * float(a.abs().max()))      # another order of the same sums
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = ops.act8_bn_act_bwd(g, *ops.act8_pack(u, coef), coef, 0.2)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, c) for a, c in zip(want, other))
    gr = torch.cuda.CUDAGraph()
    gin, uin = g.clone(), u.clone()
    with torch.cuda.graph(gr):
        cq, cs = ops.act8_pack(uin, coef)
        out = ops.act8_bn_act_bwd(gin, cq, cs, coef, 0.2)
    for it in range(3):
        gin.copy_(g * (it + 1))
        gr.replay()
        eager = ops.act8_bn_act_bwd(g * (it + 1), q, s, coef, 0.2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(eager, out))


def test_refusals():
    x = torch.randn(2, 4, 6, 6, device="cuda")
    q, s = ops.act8_pack(x)
    coef = torch.zeros(4, 4, device="cuda")
    with pytest.raises(TypeError):
        ops.act8_pack(x.half())
    with pytest.raises(ValueError):
        ops.act8_pack(x.transpose(2, 3))
    with pytest.raises(ValueError):
        ops.act8_pack(x, coef[:3])
    with pytest.raises(ValueError):
        ops.act8_unpack(q, s[:, :, :0])
    with pytest.raises(TypeError):
        ops.act8_unpack(q.float(), s)
    with pytest.raises(ValueError):
        ops.act8_bn_act_bwd(x, q, s, None, 0.2)
    with pytest.raises(ValueError):
        ops.act8_bn_act_bwd(x[:1], q, s, coef, 0.2)
    with pytest.raises(ValueError):
        ops.act8_bn_act_bwd(x, q, s, coef, 1.5)
    with pytest.raises(ValueError):
        ops.act8_bn_act_bwd(x, q, s, coef, 0.2, ref_q=q[:, :2])
    h, w, b, lab = torch.randn(1, 8, 4, 4, device="cuda"), torch.randn(5, 8, device="cuda"), torch.zeros(5, device="cuda"), torch.zeros(1, 4, 4, dtype=torch.int64, device="cuda")
    for bad in ((h.half(), w, b, lab), (h, w[:, :7], b, lab), (h, w, b[:4], lab), (h, w, b, lab.int()), (h, w, b, lab[:, :3]), (h.transpose(2, 3), w, b, lab), (h, w.t().contiguous().t(), b, lab)):
        with pytest.raises((TypeError, ValueError)):
            ops.class_ce(*bad)
    with pytest.raises(ValueError):
        ops.class_ce(h, w, b, lab, mean_over="some")
    with pytest.raises(ValueError):
        ops.class_ce_bwd(h, w, b, lab, lab.float()[0], lab.float()[0])
