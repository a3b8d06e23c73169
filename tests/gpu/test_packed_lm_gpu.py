"""Embedding, attention on packed documents and norm clipping together on
the GPU."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(__file__)))

pytestmark = pytest.mark.gpu


def test_steps():
    import anand_mxnet_amd as mx
    from packed_lm import check_steps
    check_steps(mx.gpu(0), "bfloat16")


def test_documents_are_apart():
    import anand_mxnet_amd as mx
    from packed_lm import check_documents
    # logits of order one through two layers of bfloat16: attention adds the
    # same keys in other tiles, a step of 2**-7 here and there per layer
    check_documents(mx.gpu(0), "bfloat16", 0.125)


def test_cpu_and_gpu_agree():
    """The same weights and batch: gradients in bfloat16 against float32."""
    import anand_mxnet_amd as mx
    from anand_mxnet_amd import autograd
    from packed_lm import batch, build
    torch.manual_seed(5)
    cpu = build(mx.cpu(), "float32")
    gpu = build(mx.gpu(0), "bfloat16")
    ps = list(zip(cpu.collect_params().values(),
                  gpu.collect_params().values()))
    for a, b in ps:
        w = a.data(mx.cpu())._t.detach().bfloat16()
        a.data(mx.cpu())._t.data.copy_(w.float())
        b.data(mx.gpu(0))._t.data.copy_(w)
    grads = []
    for net, ctx in ((cpu, mx.cpu()), (gpu, mx.gpu(0))):
        tok, seg, _, _ = batch(ctx)
        with autograd.record():
            out = net(tok, seg)
            loss = (out * out).sum()
        loss.backward()
        grads.append([p.grad(ctx)._t.float().cpu()
                      for p in net.collect_params().values()])
    for (a, _), x, y in zip(ps, *grads):
        # a key bias adds the same q.b to all scores of a row, which a softmax
        # does not see: its gradient sum_ij dS_ij q_i is zero but for the
        # cap's bend, and what is left of cancelled terms has no relative
        # bound
        if not x.any() or a.name.endswith("key_bias"):
            continue
        # some 20 roundings of 2**-8 lie between weights and gradients
        rel = float((x - y).norm() / x.norm())
        assert rel < 20 * 2.0 ** -8, (a.name, rel)
