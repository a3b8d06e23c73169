"""Which arguments automatic mixed precision casts."""
import sys

import pytest
import torch

from anand_mxnet_amd import nd
from anand_mxnet_amd.contrib import amp
from anand_mxnet_amd.contrib.amp import amp as amp_impl, lists
from anand_mxnet_amd.ops import nn as ops_nn, registry


@pytest.fixture
def amp_on():
    """amp.init() for one test: what it patches is put back."""
    mod = sys.modules["anand_mxnet_amd.ndarray"]
    names = lists.LP16_FUNCS + lists.FP32_FUNCS
    raw, ops = dict(registry.RAW), dict(registry.OPS)
    attrs = {n: getattr(mod, n) for n in names if hasattr(mod, n)}
    was = amp_impl._initialized
    amp_impl._initialized = False
    amp.init()
    yield
    registry.RAW.clear(), registry.RAW.update(raw)
    registry.OPS.clear(), registry.OPS.update(ops)
    for n in names:
        if n in attrs:
            setattr(mod, n, attrs[n])
        elif hasattr(mod, n):
            delattr(mod, n)
    amp_impl._initialized = was


@pytest.mark.parametrize("by_name", [True, False])
def test_distance_slopes_keep_their_bits(amp_on, monkeypatch, by_name):
    H = 12
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)])
    seen = {}

    def spy(q, k, v, *args):
        seen.update(q=q, slopes=args[4])
        return q

    monkeypatch.setattr(ops_nn, "_shaped_mha", spy)
    x = nd.from_torch(torch.randn(1, 3, H * 8))
    s = nd.from_torch(slopes.clone())
    if by_name:
        nd.multi_head_attention(x, x, x, H, distance_slopes=s)
    else:
        nd.multi_head_attention(x, x, x, H, None, 0.0, False, None, None,
                                None, s)
    assert seen["q"].dtype == torch.bfloat16
    assert torch.equal(seen["slopes"], slopes)


def test_float_indices_keep_their_rows(amp_on):
    w = torch.arange(1000.0)[:, None].expand(1000, 4).contiguous()
    idx = torch.tensor([255.0, 257.0, 511.0, 999.0])
    out = nd.Embedding(nd.from_torch(idx), nd.from_torch(w), input_dim=1000,
                       output_dim=4)._t
    assert out.dtype == torch.bfloat16
    assert torch.equal(out, w[idx.long()].bfloat16())
