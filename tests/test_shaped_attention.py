"""Attention with shaped scores on the CPU: values and gradients against the
definition in 64 bits, gradients against differences, refusals."""
import os
import sys

import numpy as np
import pytest
import torch

import anand_mxnet_amd as mx
from anand_mxnet_amd import nd
from anand_mxnet_amd.base import MXNetError

sys.path.insert(0, os.path.dirname(__file__))
from shaped_attention_ref import reference, visible  # noqa: E402

SEG = np.array([[0, 0, 0, 1, 1, -1, 2, 2, 2], [4, 4, 4, 4, 4, 4, 4, -3, -3]],
               np.int32)
CASES = [
    dict(logit_cap=3.0, causal=True),
    dict(slopes=True),
    dict(logit_cap=2.0, slopes=True, segment_ids=SEG, causal=True),
    dict(prefix_length=np.array([4, 0]), causal=True, slopes=True),
    dict(kv_length=np.array([0, 5]), query_offset=np.array([-1, 3]),
         causal=True),
    dict(query_offset=2, causal=True),
    dict(prefix_length=np.array([3, 8])),
]


def _setup(i):
    kw = dict(CASES[i])
    rng = np.random.default_rng(i)
    H, Hkv, D, T = 4, 2, 8, 9
    q = torch.from_numpy(rng.standard_normal((2, T, H * D)))
    k = torch.from_numpy(rng.standard_normal((2, T, Hkv * D)))
    v = torch.from_numpy(rng.standard_normal((2, T, Hkv * D)))
    g = torch.from_numpy(rng.standard_normal((2, T, H * D)))
    sl = torch.tensor([0.5, 0.25, 0.125, 0.0625]) if kw.pop("slopes", False) \
        else None
    seg = kw.get("segment_ids")
    ok, pos = visible(2, T, T, kw.get("causal", False), seg, seg,
                      kw.get("prefix_length"), kw.get("kv_length"),
                      kw.get("query_offset", 0))
    ref = reference(q, k, v, g, H, Hkv, ok, pos, None, kw.get("logit_cap"),
                    sl)
    for key in ("segment_ids", "prefix_length", "kv_length", "query_offset"):
        if isinstance(kw.get(key), np.ndarray):
            kw[key] = nd.from_torch(torch.from_numpy(kw[key]))
    if sl is not None:
        kw["distance_slopes"] = nd.from_torch(sl)
    return q, k, v, g, kw, ref


def _run(q, k, v, g, kw):
    a = [nd.from_torch(t.clone()) for t in (q, k, v)]
    for x in a:
        x.attach_grad()
    with mx.autograd.record():
        out = nd.multi_head_attention(*a, 4, num_kv_heads=2, **kw)
    out.backward(nd.from_torch(g.to(out._t.dtype)))
    return [out._t.detach()] + [x.grad._t for x in a]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_matches_definition(i):
    q, k, v, g, kw, ref = _setup(i)
    got = _run(q, k, v, g, kw)
    for t, name in zip(got, ("out", "dq", "dk", "dv")):
        # 64-bit sums of fewer than a thousand terms of order one
        assert torch.allclose(t, ref[name][0], rtol=1e-10, atol=1e-11), name


@pytest.mark.parametrize("i", range(len(CASES)))
def test_gradient_against_differences(i):
    q, k, v, g, kw, _ = _setup(i)
    _, dq, dk, dv = _run(q, k, v, g, kw)
    rng = np.random.default_rng(50 + i)
    eps = 1e-5
    for which, grad in ((0, dq), (1, dk), (2, dv)):
        step = torch.from_numpy(rng.standard_normal(grad.shape))
        vals = []
        for sgn in (1, -1):
            a = [q, k, v]
            a[which] = a[which] + sgn * eps * step
            out = nd.multi_head_attention(*[nd.from_torch(t) for t in a], 4,
                                          num_kv_heads=2, **kw)._t
            vals.append((out * g).sum())
        diff = float(vals[0] - vals[1]) / (2 * eps)
        # central difference: eps**2 times third derivatives (at most about
        # 1e3 here) and 1e-16 * 1e2 / eps of cancellation
        assert abs(diff - float((grad * step).sum())) < 1e-6


def test_bf16_cpu_and_empty_rows():
    q = nd.from_torch(torch.randn(1, 3, 16).bfloat16())
    out = nd.multi_head_attention(
        q, q, q, 2, segment_ids=nd.from_torch(torch.tensor([[0, -1, 0]])))
    assert out._t.dtype == torch.bfloat16
    assert not out._t[0, 1].any() and out._t[0, 0].any()


def test_nan_in_unseen_places():
    q = torch.randn(1, 4, 16)
    k = q.clone()
    k[:, 3] = float("nan")
    out = nd.multi_head_attention(
        nd.from_torch(q), nd.from_torch(k), nd.from_torch(k), 2,
        kv_length=nd.from_torch(torch.tensor([3])))
    assert torch.isfinite(out._t).all()
    out = nd.multi_head_attention(      # two queries before the last key
        nd.from_torch(q[:, :2]), nd.from_torch(k), nd.from_torch(k), 2,
        causal=True, query_offset=1)
    assert torch.isfinite(out._t).all()


def _x(*s):
    return nd.from_torch(torch.zeros(*s))


def _i(*s):
    return nd.from_torch(torch.zeros(*s, dtype=torch.int32))


@pytest.mark.parametrize("kw", [
    dict(logit_cap=0.0), dict(logit_cap=-1.0), dict(logit_cap=float("inf")),
    dict(logit_cap=float("nan")),
    dict(num_kv_heads=3), dict(num_kv_heads=1),
    dict(distance_slopes="bad"), dict(distance_slopes=_i(2)),
    dict(distance_slopes=_x(3)),
    dict(segment_ids=_x(2, 5)), dict(segment_ids=_i(2, 4)),
    dict(kv_segment_ids=_i(2, 5)),
    dict(prefix_length=_i(3), causal=True), dict(prefix_length=_x(2)),
    dict(kv_length=_i(1)), dict(kv_length=7.0),
    dict(query_offset=_i(2, 1)), dict(query_offset=1 << 40),
    dict(logit_cap=5.0, mask=_x(2, 2, 5, 5)),
])
def test_refuses(kw):
    q = _x(2, 5, 16)
    with pytest.raises(MXNetError):
        nd.multi_head_attention(q, q, q, 2, **kw)


def test_refuses_more():
    q, k = _x(2, 5, 16), _x(2, 6, 16)
    f = nd.multi_head_attention
    with pytest.raises(MXNetError):
        f(q, k, k, 2, segment_ids=_i(2, 5))          # keys' ids missing
    with pytest.raises(MXNetError):
        f(q, k, q, 2, logit_cap=1.0)                 # v unlike k
    with pytest.raises(MXNetError):
        f(q, _x(3, 5, 16), _x(3, 5, 16), 2, logit_cap=1.0)
    with pytest.raises(MXNetError):
        f(_x(2, 5, 15), q, q, 2, logit_cap=1.0)
    with pytest.raises(MXNetError):                  # heads of no columns
        f(_x(2, 5, 0), _x(2, 5, 0), _x(2, 5, 0), 2, logit_cap=1.0)
    s = nd.from_torch(torch.zeros(2))
    s.attach_grad()
    with pytest.raises(MXNetError):
        f(q, q, q, 2, distance_slopes=s)
    with mx.autograd.record():
        with pytest.raises(MXNetError):
            f(q, q, q, 2, logit_cap=1.0, dropout_p=0.1)
    # outside training dropout does nothing
    f(q, q, q, 2, logit_cap=1.0, dropout_p=0.1)


@pytest.mark.parametrize("far", [2 ** 31, 2 ** 32, 2 ** 40 + 1, 2 ** 63 - 1])
def test_integers_past_32_bits(far):
    """Lengths and positions behind every key see all of them, whatever
    their size; those before the first see none."""
    q, k = torch.randn(2, 3, 16), torch.randn(2, 7, 16)
    v = torch.randn(2, 7, 16)
    a = [nd.from_torch(t) for t in (q, k, v)]
    f = nd.multi_head_attention

    def ints(*x):
        return nd.from_torch(torch.tensor(x, dtype=torch.int64))

    want = f(*a, 2, kv_length=ints(7, 0))._t
    assert want[0].any() and not want[1].any()
    got = f(*a, 2, kv_length=ints(far, -far))._t
    assert torch.equal(got, want)
    got = f(*a, 2, causal=True, query_offset=ints(far, -far))._t
    assert torch.equal(got, want)
    want = f(*a, 2, causal=True, prefix_length=ints(7, 0))._t
    got = f(*a, 2, causal=True, prefix_length=ints(far, -far))._t
    assert torch.equal(got, want)


def test_second_derivative():
    """The composition on the CPU has one."""
    from anand_mxnet_amd.ops.registry import RAW
    t = [torch.randn(1, 3, 8, dtype=torch.float64).requires_grad_()
         for _ in range(3)]
    assert torch.autograd.gradgradcheck(
        lambda *x: RAW["multi_head_attention"](*x, 2, num_kv_heads=2,
                                               logit_cap=5.0, causal=True), t)


def test_refuses_no_kv_heads():
    q = _x(2, 5, 16)
    with pytest.raises(MXNetError):
        nd.multi_head_attention(q, q, q, 2, num_kv_heads=0)


@pytest.mark.parametrize("off", [1.5, 2.0, "3", [1, 2], np.zeros(2, int)])
def test_refuses_offsets_that_are_no_integers(off):
    q = _x(2, 5, 16)
    with pytest.raises(MXNetError):
        nd.multi_head_attention(q, q, q, 2, query_offset=off)
    nd.multi_head_attention(q, q, q, 2, query_offset=np.int64(2))


def blind_cases():
    """Sizes, which queries see nothing, and the arguments that make it so."""
    seg = np.array([[0, 0, 5, 1, 1, 7, 2, 2, 2]], np.int32)
    keys = np.array([[0, 0, 0, 1, 1, 2, 2, 4, 4]], np.int32)
    return [
        (dict(causal=True, query_offset=np.array([-4], np.int32)),
         [0, 1, 2, 3]),
        (dict(segment_ids=seg, kv_segment_ids=keys), [2, 5]),
        (dict(segment_ids=seg, kv_segment_ids=keys, causal=True,
              logit_cap=4.0), [2, 5]),
        (dict(kv_length=np.array([0], np.int32)), list(range(9))),
    ]


def check_blind(case, dtype, wrap, check):
    """NaN in queries that see nothing and in the gradients of their rows
    changes nothing anywhere."""
    kw, rows = case
    rng = np.random.default_rng(9)
    q, k, v, g = [torch.from_numpy(rng.standard_normal((1, 9, 16))).to(dtype)
                  for _ in range(4)]
    kw = {n: wrap(torch.from_numpy(x)) if isinstance(x, np.ndarray) else x
          for n, x in kw.items()}
    got = []
    for bad in (False, True):
        q2, g2 = q.clone(), g.clone()
        if bad:
            q2[:, rows], g2[:, rows] = float("nan"), float("nan")
        a = [wrap(t) for t in (q2, k, v)]
        for x in a:
            x.attach_grad()
        with mx.autograd.record():
            out = nd.multi_head_attention(*a, 2, num_kv_heads=2, **kw)
        out.backward(wrap(g2))
        got.append([out._t.detach()] + [x.grad._t for x in a])
    assert not got[0][0][:, rows].any() and not got[0][1][:, rows].any()
    for x, y in zip(*got):
        check(x, y)


@pytest.mark.parametrize("i", range(4))
def test_nan_in_blind_queries(i):
    def same(x, y):
        assert torch.equal(x, y)
    check_blind(blind_cases()[i], torch.float64, nd.from_torch, same)


def test_unsigned_lengths():
    """Unsigned integers of 32 bits above 2**31 are lengths too."""
    q = torch.randn(1, 4, 16)
    a = [nd.from_torch(q)] * 3
    want = nd.multi_head_attention(*a, 2, logit_cap=5.0)._t
    for dt, n in ((torch.uint32, 2 ** 31 + 5), (torch.uint8, 200),
                  (torch.int16, 4)):
        n = nd.from_torch(torch.tensor([n], dtype=torch.int64).to(dt))
        got = nd.multi_head_attention(*a, 2, logit_cap=5.0, kv_length=n)._t
        assert torch.equal(got, want)


@pytest.mark.parametrize("off", [10 ** 6, 2 ** 26 + 3, -10 ** 6])
def test_bias_far_from_the_keys(off):
    """In 32 bits too the weights are those of the distances' differences."""
    q, k = torch.randn(1, 3, 16), torch.randn(1, 9, 16)
    s = nd.from_torch(torch.tensor([0.5, 0.03]))
    f = nd.multi_head_attention
    got = f(*[nd.from_torch(t) for t in (q, k, k)], 2, distance_slopes=s,
            query_offset=off)._t
    want = f(*[nd.from_torch(t.double()) for t in (q, k, k)], 2,
             distance_slopes=s, query_offset=9 if off > 0 else -3)._t
    assert torch.allclose(got.double(), want, rtol=1e-4, atol=1e-5)


def test_no_keys():
    q, k = _x(1, 3, 16), _x(1, 0, 16)
    out = nd.multi_head_attention(
        q, k, k, 2, distance_slopes=nd.from_torch(torch.ones(2)))._t
    assert out.shape == (1, 3, 16) and not out.any()
