"""Scaled embedding and clipping by a common norm on the CPU."""
import numpy as np
import pytest
import torch

import anand_mxnet_amd as mx
from anand_mxnet_amd import gluon, nd
from anand_mxnet_amd.base import MXNetError


@pytest.mark.parametrize("dt", [torch.float32, torch.float64,
                                torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 2.5])
def test_embedding(dt, scale):
    w = torch.randn(11, 6).to(dt)
    idx = torch.tensor([[3, 3, 0], [10, 3, 1]])
    dy = torch.randn(2, 3, 6).to(dt)
    a = nd.from_torch(w)
    a.attach_grad()
    with mx.autograd.record():
        out = nd.Embedding(nd.from_torch(idx), a, input_dim=11, output_dim=6,
                           scale=scale)
    out.backward(nd.from_torch(dy))
    g = torch.zeros(11, 6, dtype=torch.float64)
    g.index_add_(0, idx.flatten(), dy.double().reshape(-1, 6))
    # two 16-bit roundings at most, and three terms in the type's own sums
    # where no scale is given
    tol = 4 * torch.finfo(dt).eps
    assert out._t.dtype == dt and a.grad._t.dtype == dt
    assert torch.allclose(out._t.double(), w.double()[idx] * scale,
                          rtol=tol, atol=tol)
    assert torch.allclose(a.grad._t.double(), g * scale, rtol=tol,
                          atol=4 * tol)


def test_embedding_block_scale():
    net = gluon.nn.Embedding(7, 4, scale=3.0)
    net.initialize(mx.init.Normal(1.0))
    x = nd.array(np.array([1, 5]), dtype="int64")
    w = net.weight.data()._t.detach()
    assert torch.allclose(net(x)._t.detach(), w[[1, 5]] * 3.0)


@pytest.mark.parametrize("max_norm", [0.5, 100.0])
def test_clip(max_norm):
    ts = [torch.randn(3, 4), torch.randn(5).bfloat16(),
          torch.randn(2, 2).double(), torch.zeros(0)]
    before = [t.clone() for t in ts]
    total = float(sum((b.double() ** 2).sum() for b in before).sqrt())
    out = [nd.from_torch(torch.empty_like(t)) for t in ts]
    n1 = nd.multi_clip_global_norm([nd.from_torch(t) for t in ts], max_norm,
                                   out=out)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    n2 = nd.multi_clip_global_norm([nd.from_torch(t) for t in ts], max_norm)
    f = min(1.0, max_norm / (total + 1e-8))
    for t, o, b in zip(ts, out, before):
        assert torch.equal(t, o._t)
        assert torch.allclose(t.double(), b.double() * f,
                              rtol=torch.finfo(b.dtype).eps)
    assert abs(float(n1._t) - total) < 1e-6 * total
    assert torch.equal(n1._t, n2._t)


def test_clip_refuses():
    f, x = nd.multi_clip_global_norm, torch.ones(10)
    w = nd.from_torch
    for arrays, kw in [
            ([], {}), ([w(x), w(x)], {}), ([w(x[:6]), w(x[5:])], {}),
            ([w(x)], dict(out=[])), ([w(x.int())], {}),
            ([w(torch.ones(1).expand(10))], {}),
            ([w(x)], dict(out=[w(torch.ones(9))])),
            ([w(x)], dict(out=[w(torch.ones(10).double())])),
            ([w(x[:5]), w(x[5:])], dict(out=[w(x[5:]), w(x[:5])]))]:
        with pytest.raises(MXNetError):
            f(arrays, 1.0, **kw)
    with pytest.raises(MXNetError):
        f([w(x)], -1.0)
    with pytest.raises(MXNetError):
        f([w(x)], float("nan"))
    assert x.eq(1).all()


def second_order(idx, w, scale):
    """Gradient of the squared norm of the table's gradient."""
    from anand_mxnet_amd.ops.registry import RAW
    w = w.detach().requires_grad_()
    out = RAW["Embedding"](idx, w, scale=scale)
    g, = torch.autograd.grad((out ** 3).sum(), w, create_graph=True)
    second, = torch.autograd.grad((g ** 2).sum(), w)
    return g.detach(), second


def check_second_order(dt, scale, dev):
    """(x -> scale x[idx]) cubed: with c the count of a row's tokens the
    gradient is 3 c s^3 w^2, and that of its squared norm 36 c^2 s^6 w^3."""
    w = torch.randint(-2, 3, (5, 8)).to(dt)   # small whole numbers: exact
    idx = torch.tensor([[3, 3, 0], [4, 3, 1]])
    c = torch.tensor([1, 1, 0, 3, 1], dtype=torch.float64)[:, None]
    g, second = second_order(idx.to(dev), w.to(dev), scale)
    x = w.double()
    assert torch.equal(g.double().cpu(), 3 * c * scale ** 3 * x ** 2)
    assert torch.equal(second.double().cpu(),
                       36 * c ** 2 * scale ** 6 * x ** 3)


@pytest.mark.parametrize("dt", [torch.float32, torch.float64, torch.bfloat16,
                                torch.float16])
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_embedding_twice(dt, scale):
    check_second_order(dt, scale, "cpu")
