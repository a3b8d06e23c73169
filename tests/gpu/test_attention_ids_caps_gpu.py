"""Attention with shaped scores (GPU): document ids in any order and of other
tokens than the keys', and caps at both ends of their range, against the
definition in 64 bits."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(__file__)))
from shaped_attention_ref import H8, check, reference, visible  # noqa: E402

pytestmark = pytest.mark.gpu


def _inputs(seed, B, Tq, Tk, H, Hkv, D, std=1.5):
    g = torch.Generator().manual_seed(seed)

    def arr(T, n, std=1.0):
        return (torch.randn((B, T, n * D), generator=g) * std).bfloat16()

    return arr(Tq, H, std), arr(Tk, Hkv, std), arr(Tk, Hkv), arr(Tq, H)


def _run(q, k, v, dout, H, train, **kw):
    import anand_mxnet_amd as mx

    def wrap(x):
        if isinstance(x, np.ndarray):
            x = torch.from_numpy(x)
        return mx.nd.from_torch(x.cuda()) if isinstance(x, torch.Tensor) \
            else x

    a = [wrap(t) for t in (q, k, v)]
    kw = {key: wrap(x) for key, x in kw.items()}
    if not train:
        return {"out": mx.nd.multi_head_attention(*a, H, **kw)._t}
    for x in a:
        x.attach_grad()
    with mx.autograd.record():
        out = mx.nd.multi_head_attention(*a, H, **kw)
    out.backward(wrap(dout))
    return {"out": out._t, "dq": a[0].grad._t, "dk": a[1].grad._t,
            "dv": a[2].grad._t}


def _ids(kind, rng, B, T):
    i = np.arange(T)[None] + np.zeros((B, 1), int)
    if kind == "random":        # in no order, some of them padding
        x = rng.integers(-2, 6, (B, T))
    elif kind == "round":       # neighbours always differ
        x = i % 3
    elif kind == "falling":     # documents in falling order, gaps between
        x = 700 - 100 * (i * 8 // T)
        x[:, ::17] = -1
    elif kind == "back":        # an id that comes back after another
        x = np.where((i // 50) % 2 == 0, 4, 9)
    elif kind == "large":       # both ends of 32 bits
        x = rng.choice([-2 ** 31, 0, 2 ** 31 - 1], (B, T))
    else:                       # none of them is a key's
        x = np.full((B, T), 77)
    return x.astype(np.int32)


IDS = [  # ids of queries and of keys, sizes
    ("random", "random", dict(B=2, Tq=130, Tk=130, H=2, Hkv=1, D=64)),
    ("round", "round", dict(B=1, Tq=200, Tk=75, H=2, Hkv=2, D=64)),
    ("falling", "falling", dict(B=2, Tq=140, Tk=333, H=4, Hkv=2, D=128)),
    ("back", "back", dict(B=1, Tq=260, Tk=260, H=2, Hkv=2, D=128)),
    ("large", "large", dict(B=2, Tq=70, Tk=129, H=2, Hkv=1, D=64)),
    ("random", "round", dict(B=2, Tq=1, Tk=500, H=4, Hkv=1, D=64)),
    ("round", "back", dict(B=1, Tq=3, Tk=2200, H=2, Hkv=1, D=64)),
    ("back", "random", dict(B=1, Tq=40, Tk=2200, H=2, Hkv=2, D=128)),
    ("random", "none", dict(B=2, Tq=100, Tk=65, H=2, Hkv=2, D=64)),
    ("none", "random", dict(B=1, Tq=65, Tk=190, H=2, Hkv=2, D=96)),
    ("falling", "round", dict(B=1, Tq=1100, Tk=90, H=4, Hkv=1, D=64)),
]


@pytest.mark.parametrize("i", range(len(IDS)))
@pytest.mark.parametrize("extra", [
    dict(), dict(causal=True, slopes=True), dict(causal=True, cap=9.0,
                                                 off=True, kv_len=True)])
def test_ids(i, extra):
    kq, kk, size = IDS[i]
    rng = np.random.default_rng(i)
    q, k, v, dout = _inputs(200 + i, **size)
    B, Tq, Tk, H = size["B"], size["Tq"], size["Tk"], size["H"]
    sq, sk = _ids(kq, rng, B, Tq), _ids(kk, rng, B, Tk)
    kw = dict(num_kv_heads=size["Hkv"], causal=extra.get("causal", False))
    slopes = cap = kv_len = None
    off = 0
    if extra.get("slopes"):
        slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / H)
                               for h in range(H)])
        kw["distance_slopes"] = slopes
    if extra.get("cap"):
        kw["logit_cap"] = cap = extra["cap"]
    if extra.get("off"):
        off = np.full(B, max(Tk - Tq, 0), np.int32)
        kw["query_offset"] = off
    if extra.get("kv_len"):
        kv_len = np.array([Tk - 5 * (b + 1) for b in range(B)], np.int32)
        kw["kv_length"] = kv_len
    ok, pos = visible(B, Tq, Tk, kw["causal"], sq, sk, None, kv_len, off)
    ref = reference(q, k, v, dout, H, size["Hkv"], ok, pos, None, cap, slopes)
    for train in (True, False):
        got = _run(q, k, v, dout, H, train, segment_ids=sq,
                   kv_segment_ids=sk, **kw)
        for name, x in got.items():
            check(name, x, ref[name])


def _cap_bounds(ref, q, k, v, dout, H, Hkv, ok, cap):
    """The bounds of `reference` with what a cap adds.

    z = -1 / (1 + t), t = exp(2 y), is held in 32 bits: exp2 and the
    reciprocal err by a unit in the last place (2**-23), the sum by half of
    one: |dz| <= z**2 t 2**-23 + |z| (2**-23 + 2**-24) <= 1.75 * 2**-23.  A
    score in units of log2 is mu z, mu = 2 cap log2(e), and the log-sum that
    the backward subtracts is rounded at that size: of a probability
    e_p = ln 2 (mu 1.75 * 2**-23 + mu 2**-24), beside H8.  All bounds grow
    with the error of a probability at most in proportion: 1 + 2 e_p / H8
    (its own, and the sum's).

    u = 1 - tanh(y)**2 = -4 (z**2 + z) errs by 4 |1 + 2 z| |dz| + 2**-24, and
    by 2 |tanh| u dy where the 32-bit product q.k of D terms moves y by dy =
    D 2**-24 |q|.|k| scale / cap, at most u exp(2 dy) within it."""
    e_z = 1.75 * 2.0 ** -23
    mu = 2 * cap / math.log(2)
    e_p = math.log(2) * (mu * e_z + mu * 2.0 ** -24)
    grow = 1 + 2 * e_p / H8
    B, Tq, HD = q.shape
    D, Tk, G = HD // H, k.shape[1], H // Hkv

    def split(x, n):
        return x.double().reshape(B, x.shape[1], n, D).transpose(1, 2)

    qh, gh = split(q, H), split(dout, H)
    kh = split(k, Hkv).repeat_interleave(G, 1)
    vh = split(v, Hkv).repeat_interleave(G, 1)
    scale = D ** -0.5
    t = torch.tanh(qh @ kh.transpose(-1, -2) * scale / cap)
    u = 1 - t * t
    m = ok[:, None].expand_as(t)
    p = torch.softmax((cap * t).masked_fill(~m, -math.inf), -1)
    dp = gh @ vh.transpose(-1, -2)
    ds0 = (p * (dp - (p * dp).sum(-1, keepdim=True))).abs()
    dy = D * 2.0 ** -24 * (qh.abs() @ kh.abs().transpose(-1, -2)) \
        * scale / cap
    e_u = 4 * e_z + 2.0 ** -24 + 2 * t.abs() * u * torch.exp(2 * dy) * dy
    e = ds0 * e_u * scale
    add = {"dq": (e @ kh.abs()).transpose(1, 2).reshape(B, Tq, HD),
           "dk": (e.transpose(-1, -2) @ qh.abs()).reshape(B, Hkv, G, Tk, D)
           .sum(2).transpose(1, 2).reshape(B, Tk, Hkv * D)}
    return {n: (x, b * grow + 1.1 * add.get(n, 0.0))
            for n, (x, b) in ref.items()}


@pytest.mark.parametrize("cap", [1e-3, 0.03, 300.0, 1e3])
@pytest.mark.parametrize("size", [
    dict(B=2, Tq=97, Tk=97, H=2, Hkv=2, D=64),
    dict(B=1, Tq=130, Tk=130, H=2, Hkv=1, D=128),
    dict(B=1, Tq=2, Tk=300, H=2, Hkv=1, D=64),
])
@pytest.mark.parametrize("std", [1.5, 8.0])
def test_caps(cap, size, std):
    q, k, v, dout = _inputs(300, **size, std=std)
    B, Tq, Tk, H = size["B"], size["Tq"], size["Tk"], size["H"]
    off = Tk - Tq
    ok, pos = visible(B, Tq, Tk, True, off=off)
    ref = reference(q, k, v, dout, H, size["Hkv"], ok, pos, None, cap)
    ref = _cap_bounds(ref, q, k, v, dout, H, size["Hkv"], ok, cap)
    for train in (True, False):
        got = _run(q, k, v, dout, H, train, num_kv_heads=size["Hkv"],
                   causal=True, logit_cap=cap, query_offset=off)
        for name, x in got.items():
            check(name, x, ref[name])
