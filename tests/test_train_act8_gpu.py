"""Training passes that keep their activations in 8 bits (EngineOptions.train_act8).

The backward out of the checkpoints must be the backward of the plain engine run on the activations that the checkpoints stand for: the same kernels read the same fp32
values, and only the two sums of each BatchNorm's backward are cut into other parts (<= 80 u32 of the sum of magnitudes each, in up to 26 layers one behind the other; the
masks cannot differ: a checkpoint keeps signs).  26 x 2 x 80 u32 = 2.5e-4 of a tensor's norm where nothing cancels; weight gradients of these nets cancel by up to two
powers of ten (the reference's own fp32 noise on them is 1e-3), so tensors are compared at 5e-3 and the whole gradient at 2.5e-4."""
import pytest
import torch

from maxstyle_amd import ops, synthetic as syn
from maxstyle_amd.engine import NetSpec, PackedNets
from maxstyle_amd import train_engine as T
from test_solver_gpu import make_solver

pytestmark = pytest.mark.gpu


def solver(dev, reduce, image_ch, classes, act8, **kw):
    from oracle import maxstyle_oracle as orc
    S, _ = make_solver(dev, orc.NetSpec(reduce, image_ch, classes))
    S.train_options = dict(train_act8=act8, **kw)
    S.reset_all_optimizers()
    return S


def run(S, dev, B, size, ch, cls, between=None, track=True):
    img, lab = syn.synthetic_batch(B, size, ch, cls, 1234)
    img, lab = img.to(dev), lab.to(dev)
    noisy = img + 0.05 * torch.randn(img.shape, generator=torch.Generator().manual_seed(5)).to(dev)
    seg, rec, _, _ = S.standard_training(img, lab, perturbed_image=noisy, disable_track_bn_stats=not track)
    eng = [e for pool in S._train_engines.values() for e in pool if e.pending][0]
    if between is not None:
        between(eng)
    (seg + rec).backward()
    return float(seg.detach()), float(rec.detach()), S._param_bank().flat_g.clone(), eng


def emulate(eng):
    """The plain engine's saved activations replaced by what their checkpoints stand for."""
    b = eng.buf
    for name in list(b):
        m = T._ACT8_NAME.match(name)
        if m is None or name in ("s.u4.out", "d.u4.out", "e.d4.out"):
            continue
        coef = None
        last = name.rsplit(".", 1)[1]
        if last in ("u1", "ua"):
            coef = b[name.rsplit(".", 1)[0] + ".bn1.coef"]
        if last in ("u2", "ub"):
            coef = b[name.rsplit(".", 1)[0] + ".bn4.coef"]
        ops.act8_unpack(*ops.act8_pack(b[name], coef), coef, out=b[name])


@pytest.mark.parametrize("reduce,ch,cls,B,size,track", [(4, 1, 4, 3, 64, True), (4, 1, 4, 2, 80, False), (1, 3, 2, 2, 32, True)])
def test_backward_is_the_plain_one_on_the_kept_values(reduce, ch, cls, B, size, track):
    dev = torch.device("cuda:0")
    s0, r0, g0, e0 = run(solver(dev, reduce, ch, cls, False), dev, B, size, ch, cls, emulate, track)
    s1, r1, g1, e1 = run(solver(dev, reduce, ch, cls, True), dev, B, size, ch, cls, None, track)
    assert s0 == s1 and r0 == r1                       # the forward pass is the same bits
    assert (g1 - g0).norm() <= 2.5e-4 * g0.norm()
    S = e1.bank
    for key, (off, n, shape) in S.index.items():
        a, c = g0[off:off + n].double(), g1[off:off + n].double()
        assert (a - c).norm() <= 5e-3 * a.norm() + 1e-9, key
    # memory: everything the plain engine holds per activation element is 4 bytes; the shared buffers do not grow with the number of blocks
    kept = sum(t.numel() * t.element_size() for k, t in e1.buf.items() if k.endswith((".q8", ".s8")))
    full = sum(t.numel() * 4 for k, t in e0.buf.items() if T._ACT8_NAME.match(k) and k not in ("s.u4.out", "d.u4.out", "e.d4.out"))
    pool = sum(t.numel() * 4 for t in e1._act8_pool.values())
    largest = B * (64 // reduce) * size * size * 4
    assert pool <= 10 * largest
    extra = sum(e1.buf[k + ".out"].numel() for k in ("s.u4", "d.u4", "e.d4"))
    assert kept <= (full / 4 + extra) * 1.04 + 4096 * 40
    grads = sum(t.numel() * 4 for k, t in e0.buf.items() if T._ACT8_GRAD.match(k))
    own = sum(t.numel() * 4 for k, t in e1.buf.items() if (T._ACT8_GRAD.match(k) or T._ACT8_NAME.match(k)) and e1._act8_role(k) is None)
    print("saved and gradient bytes: plain %.1f MB, 8-bit %.1f MB" % ((full + extra * 4 + grads) / 1e6, (kept + pool + own) / 1e6))
    assert kept + pool + own < 0.75 * (full + extra * 4 + grads)


def test_close_to_the_unrounded_gradient_and_graph_replay():
    """Each kept value is off by at most half a step of a 3 - 4 sigma range / 127: 0.8 % rms of a standard deviation, independent from layer to layer; a weight gradient
    sees it twice in each of up to 26 layers: 0.8 % sqrt(52) = 6 %, for the whole gradient."""
    dev = torch.device("cuda:0")
    _, _, g0, _ = run(solver(dev, 4, 1, 4, False), dev, 4, 64, 1, 4)
    S = solver(dev, 4, 1, 4, True)
    _, _, g1, _ = run(S, dev, 4, 64, 1, 4)
    assert (g1 - g0).norm() <= 0.06 * g0.norm()
    Sg = solver(dev, 4, 1, 4, True, train_graph=True)
    for _ in range(4):                                  # eager, captured, replayed twice
        Sg._param_bank().zero_grad()
        _, _, g2, _ = run(Sg, dev, 4, 64, 1, 4, track=False)
        S._param_bank().zero_grad()
        _, _, g3, _ = run(S, dev, 4, 64, 1, 4, track=False)
        assert torch.equal(g2, g3)


def test_mixstyle_is_refused():
    dev = torch.device("cuda:0")
    S = solver(dev, 4, 1, 4, True)
    img, lab = syn.synthetic_batch(2, 64, 1, 4, 1234)
    with pytest.raises(NotImplementedError, match="train_act8"):
        S.mixstyle_training(img.to(dev), lab.to(dev), img.to(dev), layers_indexes=[1, 2], p=1.0)
