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


def test_attention_twice_raises():
    """The first derivative is the same under create_graph; the second one
    raises, also where the queries had to be copied for the kernels."""
    from anand_mxnet_amd.ops.registry import RAW
    for odd in (0, 1):
        t = [torch.randn(2, 5, 2 * 16 + odd, device="cuda").bfloat16()
             .requires_grad_() for _ in range(3)]

        def f():
            return RAW["multi_head_attention"](
                *[x[..., :32] for x in t], 2, num_kv_heads=2, logit_cap=5.0)

        plain = torch.autograd.grad(f().sum(), t)
        g = torch.autograd.grad(f().sum(), t, create_graph=True)
        for x, y in zip(plain, g):
            assert torch.equal(x, y.detach())
        for y in g:
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad((y.float() ** 2).sum(), t,
                                    retain_graph=True, allow_unused=True)


def test_transforms_raise():
    """What the kernels cannot go through is refused, not dropped."""
    from anand_mxnet_amd.ops.registry import RAW
    w = torch.randn(3, 5, 8, device="cuda")
    idx = torch.tensor([1, 3], device="cuda")
    q = torch.randn(1, 5, 16, device="cuda").bfloat16()

    def attn(t):
        return RAW["multi_head_attention"](t, q, q, 2, num_kv_heads=2,
                                           logit_cap=5.0)

    def emb(t):
        return RAW["Embedding"](idx, t)

    with torch.enable_grad():
        for f in (lambda: torch.func.vmap(emb)(w),
                  lambda: torch.func.vmap(attn)(q[None]),
                  lambda: torch.func.jvp(attn, (q,), (q,)),
                  lambda: torch.func.grad(lambda t: emb(t).sum())(w[0])):
            with pytest.raises(RuntimeError):
                f()
