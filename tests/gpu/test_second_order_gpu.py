"""Derivatives of the second order on the GPU: right, or an error."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(__file__)))
from test_embedding_clip import check_second_order  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16,
                                torch.float16])
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_embedding_twice(dt, scale):
    check_second_order(dt, scale, "cuda")


def test_embedding_forward_mode_raises():
    from anand_mxnet_amd.ops.registry import RAW
    w = torch.randn(5, 8, device="cuda")
    idx = torch.tensor([1, 3], device="cuda")
    with torch.enable_grad(), pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: RAW["Embedding"](idx, t), (w,),
                       (torch.ones_like(w),))
