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


def test_hybridized_cell():
    """A cell replayed from a graph, its masks given by place and by name."""
    import numpy as np
    import anand_mxnet_amd as mx
    from anand_mxnet_amd import nd
    from anand_mxnet_amd.gluon.model_zoo.bert import MultiHeadAttentionCell
    cell = MultiHeadAttentionCell(128, 2, dropout=0.0, causal=True,
                                  num_kv_heads=1, logit_cap=10.0,
                                  distance_bias=True)
    cell.cast("bfloat16")
    cell.initialize(mx.init.Normal(0.1), ctx=mx.gpu(0))
    rng = np.random.default_rng(0)
    xs = [nd.array(rng.standard_normal((2, 50, 128)), ctx=mx.gpu(0),
                   dtype="bfloat16") for _ in range(3)]
    seg = nd.array(np.arange(100).reshape(2, 50) // 13, ctx=mx.gpu(0),
                   dtype="int32")
    plain = [cell(x)._t.clone() for x in xs]
    apart = [cell(x, segment_ids=seg)._t.clone() for x in xs]
    assert not torch.equal(plain[0], apart[0])
    cell.hybridize(static_alloc=True)
    for child in cell._children.values():  # one graph for the whole cell
        child.hybridize(False)
    for _ in range(2):
        for x, p, a in zip(xs, plain, apart):
            assert torch.equal(cell(x)._t, p)
            assert torch.equal(cell(x, segment_ids=seg)._t, a)
            assert torch.equal(cell(x, None, None, seg)._t, a)


def test_training_step_replays():
    """Forward, backward and clipping captured once and replayed on new
    inputs, eager steps of other leaves in between."""
    from anand_mxnet_amd.ops.registry import RAW
    mha, emb, clip = (RAW["multi_head_attention"], RAW["Embedding"],
                      RAW["multi_clip_global_norm"])
    torch.manual_seed(1)
    seg = (torch.arange(128, device="cuda") // 50).repeat(2, 1).int()

    def leaves():
        g = torch.Generator(device="cuda").manual_seed(7)
        return [torch.randn(s, generator=g, device="cuda").bfloat16()
                .requires_grad_(True) for s in ((40, 128), (128, 128))]

    def step(w, tok):
        x = emb(tok, w[0], scale=2.0)
        o = mha(x @ w[1], x, x, 2, causal=True, logit_cap=10.0,
                segment_ids=seg)
        return torch.autograd.grad(o, w, o.detach() * 0.1)

    toks = [torch.randint(0, 40, (2, 128), device="cuda") for _ in range(4)]
    eager = []
    for t in toks:
        g = [x.clone() for x in step(leaves(), t)]
        eager.append((clip(g, 0.5).clone(), g))
    w, tok = leaves(), toks[0].clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(2):
            step(w, tok)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(w, tok)
        norm = clip(list(got), 0.5)
    for i in (2, 0, 3, 1):
        tok.copy_(toks[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, eager[i][0])
        for a, b in zip(got, eager[i][1]):
            assert torch.equal(a, b)
        step(leaves(), toks[i])
