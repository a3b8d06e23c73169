"""A small causal language model on packed documents."""
import math

import numpy as np
import torch

import anand_mxnet_amd as mx
from anand_mxnet_amd import autograd, gluon, nd
from anand_mxnet_amd.gluon import nn
from anand_mxnet_amd.gluon.model_zoo.bert import TransformerEncoderCell

VOCAB, UNITS, HEADS = 320, 128, 2


class PackedLM(gluon.HybridBlock):
    def __init__(self, **kwargs):
        super().__init__(**kwargs)
        with self.name_scope():
            self.embed = nn.Embedding(VOCAB, UNITS, scale=math.sqrt(UNITS))
            self.cells = [TransformerEncoderCell(
                UNITS, 256, HEADS, dropout=0.0, causal=True, num_kv_heads=1,
                logit_cap=20.0, distance_bias=True, prefix=f"cell{i}_")
                for i in range(2)]
            for i, c in enumerate(self.cells):
                self.register_child(c, f"cell{i}")
            self.proj = nn.Dense(VOCAB, flatten=False, in_units=UNITS)

    def forward(self, tokens, segment_ids):
        x = self.embed(tokens)
        for c in self.cells:
            x = c(x, segment_ids=segment_ids)
        return self.proj(x)

    hybrid_forward = None


def build(ctx, dtype):
    net = PackedLM()
    net.cast(dtype)
    net.initialize(mx.init.Normal(0.05), ctx=ctx)
    return net


def batch(ctx, T=96):
    rng = np.random.default_rng(3)
    seg = np.full((2, T), -1, np.int32)
    seg[0, :40], seg[0, 40:80] = 0, 1
    seg[1, :T] = 0
    tok = rng.integers(0, VOCAB, (2, T))
    return (nd.array(tok, ctx=ctx, dtype="int64"),
            nd.array(seg, ctx=ctx, dtype="int32"), tok, seg)


def check_steps(ctx, dtype):
    """Three steps: the norm that clipping returns is that of the gradients,
    the gradients obey it, the parameters move and stay finite."""
    net = build(ctx, dtype)
    params = [p for p in net.collect_params().values()
              if p.grad_req != "null"]
    trainer = gluon.Trainer(net.collect_params(), "sgd",
                            {"learning_rate": 0.5, "momentum": 0.9,
                             "multi_precision": dtype != "float32"})
    loss_fn = gluon.loss.SoftmaxCrossEntropyLoss()
    tok, seg, _, _ = batch(ctx)
    for step in range(3):
        with autograd.record():
            out = net(tok, seg)
            loss = loss_fn(out.reshape(-1, VOCAB), tok.reshape(-1)).mean()
        loss.backward()
        grads = [p.list_grad()[0] for p in params]
        want = math.sqrt(sum(float((g._t.double() ** 2).sum())
                             for g in grads))
        limit = want / 3
        if step == 0:
            norm = float(nd.multi_clip_global_norm(grads, limit)._t)
        else:
            norm = gluon.utils.clip_global_norm(grads, limit)
        assert abs(norm - want) <= 1e-6 * want
        after = math.sqrt(sum(float((g._t.double() ** 2).sum())
                              for g in grads))
        # every element is rounded to its type once: the norm of what that
        # takes is at most half a step of the norm
        assert abs(after - limit) <= torch.finfo(
            grads[0]._t.dtype).eps * limit
        before = [p.data(ctx)._t.detach().clone() for p in params]
        trainer.step(1)
        assert any(not torch.equal(b, p.data(ctx)._t.detach())
                   for b, p in zip(before, params))
        assert all(torch.isfinite(p.data(ctx)._t).all() for p in params)
    rows = net.embed.weight.grad(ctx)._t
    hit = torch.zeros(VOCAB, dtype=torch.bool)
    hit[tok._t.cpu().flatten()] = True
    assert not rows[~hit.to(rows.device)].any()


def check_documents(ctx, dtype, tol):
    """A packed document gives what it gives alone, and its logits do not
    see the other documents or the padding."""
    net = build(ctx, dtype)
    tok, seg, tok_np, seg_np = batch(ctx)
    out = net(tok, seg)._t.detach().float()
    alone = net(nd.array(tok_np[:1, 40:80], ctx=ctx, dtype="int64"),
                nd.array(seg_np[:1, 40:80], ctx=ctx, dtype="int32"))
    assert (out[:1, 40:80] - alone._t.detach().float()).abs().max() <= tol
    other = tok_np.copy()
    other[0, :40] = (other[0, :40] + 7) % VOCAB
    other[0, 80:] = 1
    again = net(nd.array(other, ctx=ctx, dtype="int64"),
                seg)._t.detach().float()
    assert torch.equal(out[0, 40:80], again[0, 40:80])
