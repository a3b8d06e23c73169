"""Attention with shaped scores at the borders of its arguments (GPU)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(__file__)))

pytestmark = pytest.mark.gpu

FAR = [2 ** 31 - 1, 2 ** 31 - 200, 2 ** 30 - 1, 2 ** 30]


def _args(Tq, Tk):
    g = torch.Generator().manual_seed(5)
    return [torch.randn((2, T, 2 * 64), generator=g).bfloat16().cuda()
            for T in (Tq, Tk, Tk)]


def _run(ts, train, **kw):
    import anand_mxnet_amd as mx
    a = [mx.nd.from_torch(t.clone()) for t in ts]
    kw = {k: mx.nd.from_torch(v.cuda()) if isinstance(v, torch.Tensor) else v
          for k, v in kw.items()}
    if not train:
        return [mx.nd.multi_head_attention(*a, 2, num_kv_heads=2, **kw)._t]
    for x in a:
        x.attach_grad()
    with mx.autograd.record():
        out = mx.nd.multi_head_attention(*a, 2, num_kv_heads=2, **kw)
    out.backward(mx.nd.from_torch(torch.ones_like(ts[0])))
    return [out._t.detach()] + [x.grad._t for x in a]


@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("Tq,train", [(1, False), (130, False), (130, True)])
def test_offsets_near_the_end_of_32_bits(far, Tq, train):
    """A query behind every key sees them all, one before every key none,
    whatever the offset: no position overflows."""
    ts = _args(Tq, 150)
    ids = torch.zeros(2, Tq, dtype=torch.int32), \
        torch.zeros(2, 150, dtype=torch.int32)
    for seg in (False, True):  # with ids, single queries take blocks too
        kw = dict(segment_ids=ids[0], kv_segment_ids=ids[1]) if seg else {}
        want = _run(ts, train, kv_length=torch.tensor([150, 150]), **kw)
        for sign in (1, -1):
            off = torch.tensor([sign * far] * 2, dtype=torch.int32)
            got = _run(ts, train, causal=True, query_offset=off, **kw)
            for x, y in zip(got, want):
                assert torch.equal(x, y if sign > 0 else torch.zeros_like(y))


def _wide(B, H, Tq, Tk):
    """B equal sequences of H heads of 8, one sequence's memory."""
    g = torch.Generator().manual_seed(6)
    return [torch.randn((1, T, H * 8), generator=g).bfloat16().cuda()
            .expand(B, T, H * 8) for T in (Tq, Tk, Tk)]


@pytest.mark.parametrize("B,Tq,Tk,ids", [
    (1 << 21, 1, 1, False),            # 2**24 blocks of single queries
    (1 << 21, 1, 1, True),             # the same in blocks of 128
    (1 << 19, 1 << 10, 1, False),      # 2**25 blocks of 128 queries
])
def test_launches_past_2_to_the_32_threads_are_refused(B, Tq, Tk, ids):
    import anand_mxnet_amd as mx
    a = [mx.nd.from_torch(t) for t in _wide(B, 8, Tq, Tk)]
    kw = dict(num_kv_heads=8, logit_cap=30.0)
    if ids:
        kw.update(segment_ids=mx.nd.from_torch(torch.zeros(
            (B, Tq), dtype=torch.int32, device="cuda")))
    with pytest.raises(RuntimeError, match="too large"):
        mx.nd.multi_head_attention(*a, 8, **kw)


def test_backward_past_2_to_the_32_threads_is_refused_forward():
    """Heads above 64 columns: the keys' gradients take blocks of 512."""
    import anand_mxnet_amd as mx
    t = torch.zeros(1, 1, 8 * 72, dtype=torch.bfloat16, device="cuda")
    a = [mx.nd.from_torch(t.expand(1 << 20, 1, 8 * 72)) for _ in range(3)]
    a[1].attach_grad()
    with mx.autograd.record():
        with pytest.raises(RuntimeError, match="too large"):
            mx.nd.multi_head_attention(*a, 8, num_kv_heads=8, logit_cap=30.0)


@pytest.mark.parametrize("ids", [False, True])
def test_largest_launch(ids):
    import anand_mxnet_amd as mx
    B = (1 << 21) - 1
    ts = _wide(B, 8, 1, 1)
    kw = dict(num_kv_heads=8, logit_cap=30.0)
    if ids:
        kw.update(segment_ids=mx.nd.from_torch(torch.zeros(
            (B, 1), dtype=torch.int32, device="cuda")))
    out = mx.nd.multi_head_attention(*[mx.nd.from_torch(t) for t in ts], 8,
                                     **kw)._t
    assert torch.equal(out, ts[2])  # one key: its value


@pytest.mark.parametrize("i", range(4))
def test_nan_in_blind_queries(i):
    import anand_mxnet_amd as mx
    from test_shaped_attention import blind_cases, check_blind

    def same(x, y):
        assert torch.equal(x, y)
    check_blind(blind_cases()[i], torch.bfloat16,
                lambda t: mx.nd.from_torch(t.cuda()), same)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [None, 8.0])
def test_nan_in_blind_queries_of_long_sequences(D, cap):
    """Several tiles, shared heads, rows at both ends of them."""
    import anand_mxnet_amd as mx
    g = torch.Generator().manual_seed(8)
    T, H = 700, 4
    q, g0 = [torch.randn((2, T, H * D), generator=g).bfloat16()
             for _ in range(2)]
    k, v = [torch.randn((2, T, 2 * D), generator=g).bfloat16()
            for _ in range(2)]
    seg = torch.randint(0, 3, (2, T), generator=g, dtype=torch.int32)
    keys = seg.clone()
    seg[:, [0, 63, 64, 200, 255, 256, T - 1]] = 8  # no key has that id
    off = torch.tensor([-70, 0], dtype=torch.int32)
    pos = torch.arange(T)[None] + off[:, None]
    blind = (seg == 8) | (pos < 0)
    for b in range(2):  # causal: an id that begins behind the query
        for s in range(3):
            first = int((keys[b] == s).nonzero()[0])
            blind[b] |= (seg[b] == s) & (pos[b] < first)
    got = []
    for bad in (False, True):
        q2, g2 = q.clone(), g0.clone()
        if bad:
            q2[blind], g2[blind] = float("nan"), float("inf")
        a = [mx.nd.from_torch(t.cuda()) for t in (q2, k, v)]
        for x in a:
            x.attach_grad()
        with mx.autograd.record():
            out = mx.nd.multi_head_attention(
                *a, H, num_kv_heads=2, causal=True, logit_cap=cap,
                segment_ids=mx.nd.from_torch(seg.cuda()),
                kv_segment_ids=mx.nd.from_torch(keys.cuda()),
                query_offset=mx.nd.from_torch(off.cuda()))
        out.backward(mx.nd.from_torch(g2.cuda()))
        got.append([out._t.detach()] + [x.grad._t for x in a])
    assert blind.sum() > 80
    assert not got[0][0][blind].any() and not got[0][1][blind].any()
    for x, y in zip(*got):
        assert torch.isfinite(y).all() and torch.equal(x, y)


@pytest.mark.parametrize("off", [10 ** 6, 2 ** 26 + 3, -10 ** 6])
@pytest.mark.parametrize("Tq,causal,D", [(1, True, 64), (130, True, 128),
                                         (130, False, 64), (2, False, 128)])
def test_bias_far_from_the_keys(off, Tq, causal, D):
    """Queries far behind all keys, or before them: the weights are those of
    the distances' differences."""
    from shaped_attention_ref import check, reference, visible
    g = torch.Generator().manual_seed(12)
    B, Tk, H = 2, 150, 2
    q, dout = [torch.randn((B, Tq, H * D), generator=g).bfloat16()
               for _ in range(2)]
    k, v = [torch.randn((B, Tk, H * D), generator=g).bfloat16()
            for _ in range(2)]
    slopes = torch.tensor([0.5, 0.03])
    kv_len = torch.tensor([150, 77])
    ok, pos = visible(B, Tq, Tk, causal, kv_len=kv_len, off=off)
    # less the nearest key's distance: the same softmax, exact in 64 bits
    ref = reference(q, k, v, dout, H, H, ok, pos, slopes=slopes)
    kw = dict(causal=causal, query_offset=off, kv_length=kv_len,
              distance_slopes=slopes)
    for train in (False, True):
        if train:
            import anand_mxnet_amd as mx
            a = [mx.nd.from_torch(t.cuda()) for t in (q, k, v)]
            for x in a:
                x.attach_grad()
            kd = {n: mx.nd.from_torch(x.cuda())
                  if isinstance(x, torch.Tensor) else x
                  for n, x in kw.items()}
            with mx.autograd.record():
                out = mx.nd.multi_head_attention(*a, H, num_kv_heads=H, **kd)
            out.backward(mx.nd.from_torch(dout.cuda()))
            got = dict(out=out._t, dq=a[0].grad._t, dk=a[1].grad._t,
                       dv=a[2].grad._t)
        else:
            got = dict(out=_run([q.cuda(), k.cuda(), v.cuda()], False,
                                **kw)[0])
        for name, x in got.items():
            check(name, x, ref[name])
