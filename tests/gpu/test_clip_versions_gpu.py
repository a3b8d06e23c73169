"""Clipping by a common norm and a backward that saved the arrays (GPU)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ratio,written", [(2.0, False), (0.5, True)])
@pytest.mark.parametrize("strided", [False, True])
def test_gluon_clip_marks_what_it_writes(ratio, written, strided):
    """An array below the limit is not written, and a backward that saved it
    goes on; one that was scaled makes it raise."""
    import anand_mxnet_amd as mx
    from anand_mxnet_amd import gluon
    x = torch.randn(64, 8, device="cuda", requires_grad=True)
    y = x.exp()  # its backward saves y
    t = y.detach()
    a = mx.nd.from_torch(t[:, ::2] if strided else t)
    norm = float(a._t.double().norm())
    before = t.clone()
    got = gluon.utils.clip_global_norm([a], ratio * norm)
    assert abs(got - norm) <= 1e-5 * norm
    assert torch.equal(t, before) == (not written)
    if written:
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()
    else:
        y.sum().backward()
        assert torch.equal(x.grad, before)


def test_clip_at_the_limit_counts_as_written():
    import anand_mxnet_amd as mx
    from anand_mxnet_amd import gluon
    t = torch.full((4,), 1.5, device="cuda")  # a norm of 3
    v = t._version
    gluon.utils.clip_global_norm([mx.nd.from_torch(t)], 3.0)
    assert t._version > v
    with torch.inference_mode():
        u = torch.ones(4, device="cuda")
        gluon.utils.clip_global_norm([mx.nd.from_torch(u)], 1.0)
        assert abs(float(u.norm()) - 1.0) < 1e-5
