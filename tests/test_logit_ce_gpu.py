"""cross_entropy_2D above 4 classes and ops.logit_ce against the definition in 64 bits.

u = 2^-24.  A pixel's loss: exponents (z - max) log2(e) to 2 u of their size, of at most 30 where a term counts (60 u); K fp32 additions (K u); max - z and the logarithm to 4 u of their sizes."""
import pytest
import torch

import maxstyle_amd
from maxstyle_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def definition(z, lab):
    K = z.shape[1]
    zd = z.double()
    ok = (lab >= 0) & (lab < K)
    pick = zd.gather(1, torch.where(ok, lab, torch.zeros_like(lab)).unsqueeze(1)).squeeze(1)
    return torch.where(ok, torch.logsumexp(zd, 1) - pick, torch.zeros_like(pick))


def make(shape, seed, void=0.1):
    g = torch.Generator().manual_seed(seed)
    z = 3 * torch.randn(*shape, generator=g)
    lab = torch.randint(0, shape[1], (shape[0],) + tuple(shape[2:]), generator=g)
    lab = torch.where(torch.rand(lab.shape, generator=g) < void, torch.full_like(lab, -100), lab)
    return z.cuda(), lab.cuda()


def tol(K, nll):
    return (K + 100) * U + 8 * U * (float(nll.abs().mean()) + 1)


SHAPES = [(1, 5, 1, 1), (2, 5, 17, 19), (2, 21, 64, 64), (3, 150, 33, 30), (1, 1000, 64, 64), (1, 3000, 5, 7), (16, 9, 256, 256), (4, 7, 200, 100), (2, 6, 2, 2)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("mask", [None, -1e4, -1e12, torch.finfo(torch.float32).min, float("-inf")])
def test_masked_logits(shape, mask):
    """Half of the classes masked: neither the lowest value of the type nor -infinity disturbs the others."""
    z, lab = make(shape, shape[1])
    if mask is not None:
        keep = torch.rand(z.shape, generator=torch.Generator().manual_seed(1)).cuda() < 0.5
        keep = keep.scatter(1, lab.clamp(0).unsqueeze(1), True)
        z = torch.where(keep, z, torch.full_like(z, mask))
    nll = definition(z, lab)
    want = float(nll.mean())
    got = maxstyle_amd.cross_entropy_2D(z, lab)
    assert got.dim() == 0 and abs(float(got) - want) <= tol(shape[1], nll)
    assert torch.equal(got, ops.logit_ce(z, lab)) and torch.equal(-got, ops.logit_ce(z, lab, loss_sign=-1.0))


def test_special_values():
    z, lab = make((1, 8, 6, 6), 3, void=0.0)
    inf = float("inf")
    y = z.clone(); y[0, :, 2, 2] = -inf                       # nothing is left of a pixel
    assert torch.isnan(ops.logit_ce(y, lab)) and torch.isnan(definition(y, lab).mean())
    off = lab.clone(); off[0, 2, 2] = -1                      # ... but it takes no part
    assert abs(float(ops.logit_ce(y, off)) - float(definition(y, off).mean())) <= tol(8, definition(z, lab))
    y = z.clone(); y[0, lab[0, 1, 1], 1, 1] = -inf            # the label itself is masked
    assert float(ops.logit_ce(y, lab)) == inf
    y = z.clone(); y[0, 3, 4, 4] = float("nan")
    assert torch.isnan(ops.logit_ce(y, lab))
    assert float(ops.logit_ce(z, torch.full_like(lab, 8))) == 0
    big = z * 1e37
    nll = definition(big, lab)
    assert abs(float(ops.logit_ce(big, lab)) - float(nll.mean())) <= 8 * U * float(nll.abs().mean())


def test_layouts_streams_and_graphs():
    z, lab = make((2, 12, 20, 24), 4)
    want = ops.logit_ce(z, lab)
    nll = definition(z, lab)
    shift = torch.cat([z.new_zeros(1), z.reshape(-1)])[1:].view(z.shape)          # no whole vectors
    assert abs(float(ops.logit_ce(shift, lab)) - float(nll.mean())) <= tol(12, nll)
    assert abs(float(maxstyle_amd.cross_entropy_2D(z.to(memory_format=torch.channels_last), lab)) - float(nll.mean())) <= tol(12, nll)
    assert torch.equal(maxstyle_amd.cross_entropy_2D(z.to(torch.bfloat16), lab), ops.logit_ce(z.to(torch.bfloat16).float(), lab))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.logit_ce(z, lab)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    zs = z.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.logit_ce(zs, lab)
    for it in range(4):
        zs.copy_(z * (it + 1))
        graph.replay()
        eager = ops.logit_ce(z * (it + 1), lab)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_many_pixels_and_refusals():
    g = torch.Generator(device="cuda").manual_seed(0)
    z = torch.randn(9, 5, 8192, 8192, generator=g, device="cuda")          # 12 GB, more pixels than a round of workgroups, offsets past 32 bits
    lab = torch.randint(0, 5, (9, 8192, 8192), generator=g, device="cuda")
    got = float(ops.logit_ce(z, lab))
    want = sum(float(definition(z[i:i + 1, :, j:j + 1024], lab[i:i + 1, j:j + 1024]).sum()) for i in range(9) for j in range(0, 8192, 1024)) / lab.numel()
    assert abs(got - want) <= 105 * U + 8 * U * 3
    for bad in ((z[0, :, :4, :4].half(), lab[0, :4, :4]), (z[:1, :, :4, :4].contiguous(), lab[:1, :4, :3].contiguous()), (z[:1, :, :4, :4].contiguous(), lab[:1, :4, :4].int())):
        with pytest.raises((TypeError, ValueError)):
            ops.logit_ce(*bad)
