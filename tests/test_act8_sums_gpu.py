"""The sums of the 8-bit backward, held to what its arithmetic leaves: up to four fp32 terms a thread and step (16 in the one-launch kernel) and their products, everything behind in 64 bits.

u = 2^-24.  sum g': 16 u of the sum of magnitudes; sum g'(x' - mean): 16 + 4 u, and 3 u of the two parts of x' - mean.  64 terms summed in fp32 would leave up to 80 u, and a third of that
on average: the larger cases below are 1 M elements a channel."""
import pytest
import torch

from maxstyle_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("shape", [(4, 5, 512, 512), (3, 4, 129, 130), (2, 7, 33, 31), (4, 130, 12, 12)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0.0, 3.0])
def test_sums(shape, dt, offset):
    g = torch.Generator().manual_seed(1)
    N, C = shape[:2]
    u = (1.7 * torch.randn(*shape, generator=g) + torch.randn(1, C, 1, 1, generator=g)).to(dt).cuda()
    gr = (offset + torch.randn(*shape, generator=g)).to(dt).cuda()          # (an offset: the sum of equal signs, where fp32 sums drift)
    mean, inv = u.double().mean((0, 2, 3)), (u.double().var((0, 2, 3), unbiased=False) + 1e-5).rsqrt()
    gamma = (0.5 + torch.rand(C, generator=g)).double().cuda()
    coef = torch.stack([gamma * inv, 0.2 - mean * gamma * inv, mean, inv], 1).float().contiguous()
    q, s = ops.act8_pack(u, coef)
    c = coef.double()
    centre = -c[:, 1] / c[:, 0]
    per = lambda t: t.view(1, C, 1)
    d = q.reshape(N, C, -1).double() * s.double().repeat_interleave(256, 2)[:, :, :q[0, 0].numel()]
    gm = gr.reshape(N, C, -1).double() * torch.where(q.reshape(N, C, -1).double() * per(c[:, 0]) > 0, 1.0, 0.2)
    off = per(centre - c[:, 2])
    xm = d + off
    s1, s2 = gm.sum((0, 2)), (gm * xm).sum((0, 2))
    e1 = 16 * U * gm.abs().sum((0, 2))
    e2 = 20 * U * (gm * xm).abs().sum((0, 2)) + 3 * U * (gm.abs() * (d.abs() + off.abs())).sum((0, 2))
    _, dgamma, dbeta = ops.act8_bn_act_bwd(gr, q, s, coef, 0.2)
    assert ((dbeta.double() - s1).abs() <= e1 + U * s1.abs()).all()
    assert ((dgamma.double() - s2 * c[:, 3]).abs() <= e2 * c[:, 3] + 2 * U * (s2 * c[:, 3]).abs()).all()
    part = ops.act8_bwd_reduce(gr, q, s, coef, 0.2)[1].double().sum(1)
    assert ((part[:, 0] - s1).abs() <= e1 + U * gm.abs().sum((0, 2))).all() and ((part[:, 1] - s2).abs() <= e2 + U * (gm * xm).abs().sum((0, 2))).all()
    # the mean error of the channels' sums of equal signs: 64-bit sums leave no drift
    if offset and shape[2] == 512:
        assert float(((dbeta.double() - s1).abs() / gm.abs().sum((0, 2))).max()) <= 2 * U
