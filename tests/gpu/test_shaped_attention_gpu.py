"""Attention with shaped scores on the GPU (attn_mod_*.hip) against the
definition in 64 bits, within bounds derived in shaped_attention_ref."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(__file__)))
from shaped_attention_ref import check, reference, visible  # noqa: E402

pytestmark = pytest.mark.gpu


def _docs(rng, B, T, n, pad):
    seg = np.full((B, T), -1, np.int32)
    for b in range(B):
        end = T - int(rng.integers(0, pad + 1))
        cuts = np.sort(rng.integers(0, end + 1, n - 1))
        edges = [0, *cuts, end]
        for i in range(n):
            seg[b, edges[i]:edges[i + 1]] = i * 3
    return seg


def _case(seed, B, Tq, Tk, H, Hkv, D, causal=False, cap=None, slopes=False,
          docs=0, pad=0, prefix=None, kv_len=None, off=None, std=1.5,
          scale=None):
    rng = np.random.default_rng(seed)

    def arr(*s, std=1.0):
        return torch.from_numpy(rng.standard_normal(s) * std) \
            .to(torch.bfloat16)

    c = dict(H=H, Hkv=Hkv, causal=causal, cap=cap, scale=scale,
             q=arr(B, Tq, H * D, std=std), k=arr(B, Tk, Hkv * D, std=std),
             v=arr(B, Tk, Hkv * D), dout=arr(B, Tq, H * D),
             slopes=None, seg=None, prefix=None, kv_len=None, off=None)
    if slopes:
        c["slopes"] = torch.tensor(
            [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)])
    if docs:
        c["seg"] = _docs(rng, B, Tk, docs, pad)
    for key, val in (("prefix", prefix), ("kv_len", kv_len), ("off", off)):
        if val is not None:
            c[key] = np.asarray(val, np.int32)
    return c


def _nd(x, grad=False):
    import anand_mxnet_amd as mx
    t = x if isinstance(x, torch.Tensor) else torch.from_numpy(x)
    a = mx.nd.from_torch(t.cuda())
    if grad:
        a.attach_grad()
    return a


def _kwargs(c):
    kw = dict(causal=c["causal"], softmax_scale=c["scale"],
              num_kv_heads=c["Hkv"], logit_cap=c["cap"])
    for key, name in (("slopes", "distance_slopes"), ("seg", "segment_ids"),
                      ("prefix", "prefix_length"), ("kv_len", "kv_length"),
                      ("off", "query_offset")):
        if c[key] is not None:
            kw[name] = _nd(c[key])
    return kw


def _ref(c, grads=True):
    B, Tq, _ = c["q"].shape
    off = 0 if c["off"] is None else c["off"]
    ok, pos = visible(B, Tq, c["k"].shape[1], c["causal"], c["seg"],
                      c["seg"], c["prefix"], c["kv_len"], off)
    return reference(c["q"], c["k"], c["v"], c["dout"] if grads else None,
                     c["H"], c["Hkv"], ok, pos, c["scale"], c["cap"],
                     c["slopes"])


def _train(c):
    import anand_mxnet_amd as mx
    q, k, v = _nd(c["q"], True), _nd(c["k"], True), _nd(c["v"], True)
    with mx.autograd.record():
        out = mx.nd.multi_head_attention(q, k, v, c["H"], **_kwargs(c))
    out.backward(_nd(c["dout"]))
    return {"out": out._t, "dq": q.grad._t, "dk": k.grad._t,
            "dv": v.grad._t}


def _infer(c):
    import anand_mxnet_amd as mx
    return mx.nd.multi_head_attention(_nd(c["q"]), _nd(c["k"]), _nd(c["v"]),
                                      c["H"], **_kwargs(c))._t


TRAIN = [
    # one token, one tile, tile edges, several blocks
    dict(B=1, Tq=1, Tk=1, H=1, Hkv=1, D=64, causal=True, cap=30.0),
    dict(B=2, Tq=63, Tk=63, H=2, Hkv=2, D=64, causal=True, cap=5.0),
    dict(B=1, Tq=64, Tk=64, H=2, Hkv=1, D=128, cap=20.0),
    dict(B=2, Tq=65, Tk=65, H=4, Hkv=2, D=128, causal=True, slopes=True),
    dict(B=1, Tq=129, Tk=129, H=2, Hkv=2, D=128, causal=True, cap=3.0,
         slopes=True),
    dict(B=2, Tq=300, Tk=300, H=4, Hkv=1, D=64, causal=True, slopes=True,
         docs=4, pad=40),
    dict(B=2, Tq=257, Tk=257, H=2, Hkv=2, D=64, docs=9, pad=100, cap=8.0),
    dict(B=1, Tq=200, Tk=200, H=3, Hkv=3, D=128, docs=2, pad=0,
         causal=True),
    # prefixes: none, inside a tile, past the end
    dict(B=3, Tq=150, Tk=150, H=2, Hkv=1, D=64, causal=True,
         prefix=[0, 70, 400], slopes=True),
    dict(B=2, Tq=140, Tk=140, H=2, Hkv=2, D=128, causal=True,
         prefix=[5, 100], docs=3, pad=20, cap=10.0),
    dict(B=2, Tq=100, Tk=100, H=2, Hkv=2, D=64, prefix=[5, 80], cap=10.0),
    # other head sizes
    dict(B=1, Tq=70, Tk=70, H=2, Hkv=2, D=8, causal=True, cap=4.0),
    dict(B=1, Tq=70, Tk=70, H=2, Hkv=1, D=32, causal=True, docs=2, pad=9),
    dict(B=2, Tq=97, Tk=97, H=2, Hkv=2, D=80, slopes=True, cap=6.0),
    dict(B=1, Tq=131, Tk=131, H=6, Hkv=2, D=96, causal=True, docs=3,
         pad=5),
    # other lengths of keys, lengths of zero and one, positions before 0
    dict(B=4, Tq=40, Tk=170, H=2, Hkv=1, D=64, causal=True,
         kv_len=[0, 1, 90, 170], off=[0, 0, 50, 130], cap=12.0),
    dict(B=2, Tq=150, Tk=33, H=2, Hkv=2, D=128, kv_len=[33, 7],
         slopes=True),
    dict(B=2, Tq=20, Tk=20, H=2, Hkv=2, D=64, causal=True, off=[-6, 3],
         slopes=True),
    # grouped heads only; a negative scale; large scores that saturate
    dict(B=1, Tq=90, Tk=90, H=8, Hkv=1, D=64),
    dict(B=1, Tq=60, Tk=60, H=2, Hkv=2, D=64, scale=-0.2, cap=9.0,
         causal=True),
    dict(B=1, Tq=80, Tk=80, H=2, Hkv=2, D=128, cap=50.0, std=6.0,
         causal=True),
    # queries divided among blocks in the backward, more than 64 tiles
    dict(B=1, Tq=1100, Tk=1100, H=2, Hkv=1, D=64, causal=True, docs=3,
         pad=50, slopes=True),
    dict(B=1, Tq=1030, Tk=1030, H=4, Hkv=1, D=128, causal=True, cap=10.0,
         prefix=[300]),
    dict(B=1, Tq=4200, Tk=70, H=1, Hkv=1, D=64, cap=10.0),
    dict(B=1, Tq=70, Tk=4200, H=1, Hkv=1, D=128, docs=0, slopes=True,
         kv_len=[4161]),
    # more than 2048 keys of heads of 64: whole tiles in the forward
    dict(B=1, Tq=130, Tk=2200, H=2, Hkv=2, D=64, causal=True, cap=10.0,
         off=[2050]),
    dict(B=1, Tq=70, Tk=2100, H=2, Hkv=1, D=64, slopes=True,
         kv_len=[2077]),
    dict(B=1, Tq=2100, Tk=2100, H=1, Hkv=1, D=64, causal=True, docs=5,
         pad=30),
    dict(B=1, Tq=40, Tk=2050, H=2, Hkv=2, D=48, causal=True, cap=7.0,
         slopes=True, off=[2000], prefix=[99]),
]


@pytest.mark.parametrize("i", range(len(TRAIN)))
def test_train(i):
    c = _case(100 + i, **TRAIN[i])
    ref = _ref(c)
    got = _train(c)
    for name in ("out", "dq", "dk", "dv"):
        check(name, got[name], ref[name])


@pytest.mark.parametrize("i", range(len(TRAIN)))
def test_infer(i):
    c = _case(100 + i, **TRAIN[i])
    check("out", _infer(c), _ref(c, grads=False)["out"])


@pytest.mark.parametrize(
    "i", [i for i in range(len(TRAIN)) if not TRAIN[i].get("docs")])
def test_both_forms(i):
    """Few queries and many take different kernels; each takes any number."""
    from anand_mxnet_amd import _C
    c = _case(100 + i, **TRAIN[i])
    want = _ref(c, grads=False)["out"]
    q, k, v = c["q"].cuda(), c["k"].cuda(), c["v"].cuda()
    D = q.shape[2] // c["H"]
    conf = (c["H"], c["Hkv"], c["scale"] or D ** -0.5, c["cap"] or 0.0,
            c["causal"])
    opt = [None if c[n] is None else torch.as_tensor(c[n]).cuda()
           for n in ("slopes", "prefix", "kv_len", "off")]
    check("split", _C.attn_decode(q, k, v, *conf, *opt, 0), want)
    check("blocks", _C.attn_mod_fwd(q, k, v, *conf, opt[0], None, None,
                                    *opt[1:], 0, False)[0], want)


def _drawn(seed):
    r = np.random.default_rng(seed)
    B, Hkv = int(r.integers(1, 4)), int(r.integers(1, 4))
    big = int(r.choice([40, 140, 300, 600]))
    Tk = int(r.integers(1, big))
    docs = int(r.choice([0, 0, 1, 2, 6]))
    kw = dict(B=B, Tq=Tk if docs else int(r.integers(1, big)), Tk=Tk,
              H=Hkv * int(r.integers(1, 4)), Hkv=Hkv,
              D=8 * int(r.integers(1, 17)), causal=bool(r.random() < 0.7),
              cap=float(r.choice([1.0, 5.0, 30.0, 100.0])),
              std=float(r.choice([0.3, 1.0, 2.5])))
    if docs:
        kw.update(docs=docs, pad=int(r.integers(0, Tk)))
    if r.random() < 0.5:
        kw["slopes"] = True
        if r.random() < 0.5:
            del kw["cap"]
    if r.random() < 0.3:
        kw["prefix"] = r.integers(-3, Tk + 10, B)
    if r.random() < 0.4:
        kw["kv_len"] = r.integers(0, Tk + 5, B)
    if r.random() < 0.4:
        kw["off"] = r.integers(-20, Tk + 20, B)
    if r.random() < 0.2:
        kw["scale"] = float(r.choice([-0.1, 0.3, 0.0]))
    return kw


@pytest.mark.parametrize("seed", range(40))
def test_drawn(seed):
    c = _case(1000 + seed, **_drawn(seed))
    ref = _ref(c)
    got = _train(c)
    for name in ref:
        check(name, got[name], ref[name])
    check("infer", _infer(c), ref["out"])


DECODE = [
    dict(B=1, Tq=1, Tk=1, H=1, Hkv=1, D=64, cap=20.0),
    dict(B=3, Tq=1, Tk=500, H=4, Hkv=4, D=64, kv_len=[500, 0, 33],
         off=[499, -1, 32], cap=20.0),
    dict(B=2, Tq=1, Tk=1500, H=8, Hkv=2, D=128, kv_len=[1500, 257],
         off=[1499, 256], slopes=True),
    dict(B=2, Tq=5, Tk=900, H=8, Hkv=1, D=64, kv_len=[900, 3],
         off=[895, -2], cap=9.0, slopes=True),
    dict(B=1, Tq=3, Tk=700, H=6, Hkv=2, D=96, kv_len=[640], off=[637]),
    dict(B=1, Tq=16, Tk=300, H=8, Hkv=2, D=128, kv_len=[299], off=[283],
         slopes=True, cap=30.0),
    dict(B=70, Tq=1, Tk=64, H=16, Hkv=16, D=64,
         kv_len=list(range(70)), off=[x - 1 for x in range(70)], cap=9.0),
]


@pytest.mark.parametrize("i", range(len(DECODE)))
def test_decode(i):
    c = _case(300 + i, causal=True, **DECODE[i])
    check("out", _infer(c), _ref(c, grads=False)["out"])


def test_unseen_places_may_hold_anything():
    """NaN and infinities behind kv_length and at negative ids."""
    nan, inf = float("nan"), float("inf")
    c = _case(7, 2, 130, 130, 2, 2, 64, causal=True, cap=10.0, docs=3,
              pad=0)
    c["seg"][:, 40:50] = -1
    c["seg"][:, 110:] = -5
    ref = _ref(c)
    for key in ("q", "k", "v", "dout"):
        c[key][:, 40:50] = nan
        c[key][:, 110:] = inf
    got = _train(c)
    for name in ref:
        check(name, got[name], ref[name])
    c = _case(8, 2, 20, 200, 4, 1, 128, causal=True, slopes=True,
              kv_len=[150, 0], off=[130, 0])
    ref = _ref(c)
    for key in ("k", "v"):
        c[key][0, 150:] = nan
        c[key][1] = -inf
    got = _train(c)
    for name in ref:
        check(name, got[name], ref[name])
    check("decode", _infer(c), ref["out"])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,off", [(3, 50), (70, 41), (150, 3)])
def test_keys_behind_the_last_query(D, Tq, off):
    """A cache without kv_length whose rest was never written."""
    from anand_mxnet_amd import _C
    last = off + Tq
    for prefix in (None, [last + 7, 0]):
        c = _case(9, 2, Tq, 230, 4, 2, D, causal=True, cap=10.0,
                  prefix=prefix, off=[off, off - 2])
        ref = _ref(c)
        for key in ("k", "v"):
            c[key][0, last + (7 if prefix else 0):] = float("nan")
            c[key][1, last - 2:] = float("inf")
        got = _train(c)
        for name in ref:
            check(name, got[name], ref[name])
        check("infer", _infer(c), ref["out"])
        pre = None if prefix is None else _nd(c["prefix"])._t
        args = (_nd(c["q"])._t, _nd(c["k"])._t, _nd(c["v"])._t, 4, 2,
                D ** -0.5, 10.0, True, None)
        opts = (pre, None, _nd(c["off"])._t, 0)
        check("split", _C.attn_decode(*args, *opts), ref["out"])
        check("blocks", _C.attn_mod_fwd(*args, None, None, *opts, False)[0],
              ref["out"])


def test_strided_operands():
    """Slices of one fused projection, a transposed batch, odd offsets."""
    import anand_mxnet_amd as mx
    c = _case(9, 2, 100, 100, 2, 2, 64, causal=True, cap=10.0)
    ref = _ref(c)
    fused = torch.cat([c["q"], c["k"], c["v"]], -1).cuda()
    q, k, v = fused.split(128, -1)
    kw = _kwargs(c)
    nd = mx.nd.from_torch
    for f in (lambda t: t,
              lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
              lambda t: torch.cat([t.new_zeros(3), t.flatten()])[3:]
              .reshape(t.shape),
              lambda t: torch.cat([t, t], -1)[..., ::2] * 0 + t):
        a = [nd(f(t)) for t in (q, k, v)]
        for x in a:
            x.attach_grad()
        with mx.autograd.record():
            out = mx.nd.multi_head_attention(*a, 2, **kw)
        g = c["dout"].cuda()
        out.backward(nd(f(g)))
        for name, t in zip(("out", "dq", "dk", "dv"),
                           (out._t, *[x.grad._t for x in a])):
            check(name, t, ref[name])
        check("infer", mx.nd.multi_head_attention(*a, 2, **kw)._t,
              ref["out"])


def test_same_bits_every_time():
    c = _case(10, 2, 333, 333, 8, 2, 64, causal=True, cap=10.0, docs=3,
              pad=30)
    a, b = _train(c), _train(c)
    for name in a:
        assert torch.equal(a[name], b[name]), name


def test_offsets_past_32_bits():
    """A cache whose rows lie 2**23 elements apart, 600 of them: their
    offsets pass 2**32 elements."""
    import anand_mxnet_amd as mx
    c = _case(11, 1, 2, 600, 2, 1, 64, causal=True, cap=10.0,
              kv_len=[600], off=[598])
    ref = _ref(c)
    base = torch.empty(600 * (1 << 23), dtype=torch.bfloat16, device="cuda")

    def far(t, at):
        w = torch.as_strided(base, (1, 600, 64), (0, 1 << 23, 1), at)
        w.copy_(t.cuda())
        return w

    k, v = far(c["k"], 0), far(c["v"], 4096)
    kw = _kwargs(c)
    nd = mx.nd.from_torch
    q = _nd(c["q"])
    check("decode", mx.nd.multi_head_attention(q, nd(k), nd(v), 2, **kw)._t,
          ref["out"])
    a = [nd(t) for t in (c["q"].cuda(), k, v)]
    for x in a:
        x.attach_grad()
    with mx.autograd.record():
        out = mx.nd.multi_head_attention(*a, 2, **kw)
    out.backward(_nd(c["dout"]))
    for name, t in zip(("out", "dq", "dk", "dv"),
                       (out._t, *[x.grad._t for x in a])):
        check(name, t, ref[name])


def test_side_stream_and_graph():
    """Called on a stream of its own, then captured and replayed with new
    inputs, eager calls in between."""
    import anand_mxnet_amd as mx
    nd = mx.nd.from_torch
    cs = [_case(20 + i, 2, 1, 700, 8, 2, 64, causal=True, cap=10.0,
                kv_len=[700, 90 + i], off=[699, 89 + i]) for i in range(4)]
    refs = [_ref(c, grads=False)["out"] for c in cs]
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        out = _infer(cs[0])
    st.synchronize()
    check("stream", out, refs[0])
    bufs = {key: cs[0][key].cuda() for key in ("q", "k", "v")}
    kv = torch.from_numpy(cs[0]["kv_len"]).cuda()
    off = torch.from_numpy(cs[0]["off"]).cuda()

    def call():
        return mx.nd.multi_head_attention(
            nd(bufs["q"]), nd(bufs["k"]), nd(bufs["v"]), 8, causal=True,
            num_kv_heads=2, logit_cap=10.0, kv_length=nd(kv),
            query_offset=nd(off))._t

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = call()
    for i in (1, 2, 3, 0):
        for key in bufs:
            bufs[key].copy_(cs[i][key])
        kv.copy_(torch.from_numpy(cs[i]["kv_len"]))
        off.copy_(torch.from_numpy(cs[i]["off"]))
        g.replay()
        check("replay", res, refs[i])
        assert torch.equal(call(), res)


def test_empty():
    import anand_mxnet_amd as mx
    for Tq, Tk in ((0, 5), (4, 0)):
        c = _case(12, 2, Tq, Tk, 2, 2, 64, cap=5.0)
        got = _train(c)
        assert got["out"].shape == (2, Tq, 128)
        for t in got.values():
            assert not t.any()
        assert not _infer(c).any()
    c = _case(12, 2, 4, 0, 2, 2, 64, cap=5.0)
    c["q"][:, 1] = float("nan")   # sees nothing all the same
    assert not _infer(c).any()
    for t in _train(c).values():
        assert not t.any()


def test_refuses_on_gpu():
    import anand_mxnet_amd as mx
    nd = mx.nd
    f = nd.multi_head_attention
    x = _nd(torch.zeros(1, 4, 2 * 132, dtype=torch.bfloat16))
    with pytest.raises(mx.base.MXNetError):
        f(x, x, x, 1, logit_cap=5.0)          # more than 128 columns
    y = _nd(torch.zeros(1, 4, 20, dtype=torch.bfloat16))
    with pytest.raises(mx.base.MXNetError):
        f(y, y, y, 1, logit_cap=5.0)          # not a multiple of 8
    z = _nd(torch.zeros(1, 4, 64))
    with pytest.raises(mx.base.MXNetError):
        f(z, z, z, 1, logit_cap=5.0)          # float32
    w = _nd(torch.zeros(1, 4, 64, dtype=torch.bfloat16))
    with pytest.raises(mx.base.MXNetError):   # ids on another device
        f(w, w, w, 1, segment_ids=nd.zeros((1, 4), dtype="int32"))
