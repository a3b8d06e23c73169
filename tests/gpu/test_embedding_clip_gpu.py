"""Scaled embedding with its table gradient, and clipping by a common norm,
on the GPU against 64-bit references."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11,
        torch.float32: 2.0 ** -24}
# smallest step of a type: what a rounding to a subnormal may be off by
TINY = {torch.bfloat16: 1e-40, torch.float16: 2.0 ** -25,
        torch.float32: 1e-45}


def _embed(idx, w, dy, scale):
    import anand_mxnet_amd as mx
    nd = mx.nd.from_torch
    a = nd(w)
    a.attach_grad()
    with mx.autograd.record():
        out = mx.nd.Embedding(nd(idx), a, input_dim=w.shape[0],
                              output_dim=w.shape[1], scale=scale)
    out.backward(nd(dy))
    return out._t.detach(), a.grad._t


def _check_embed(idx, w, dy, scale):
    out, dw = _embed(idx, w, dy, scale)
    V, D = w.shape
    dt = w.dtype
    i = idx.cpu().long().flatten()
    ok = (i >= 0) & (i < V)
    safe = torch.where(ok, i, torch.zeros_like(i))
    want = w.cpu().double()[safe] * ok[:, None] * scale
    got = out.cpu().double().reshape(-1, D)
    # the scale reaches the kernel as float32, the product is rounded to 32
    # bits and then to the type
    rel = HALF[dt] + 2.0 ** -23
    assert ((got - want).abs() <= rel * want.abs() + TINY[dt]).all()
    d = dy.cpu().double().reshape(-1, D)[ok]
    g = torch.zeros(V, D, dtype=torch.float64)
    ab = torch.zeros(V, D, dtype=torch.float64)
    g.index_add_(0, i[ok], d)
    ab.index_add_(0, i[ok], d.abs())
    # a row of n terms: at most n sums in 32 bits, 2**-24 each of at most
    # the absolute sum, then the scale and the rounding
    n = torch.bincount(i[ok], minlength=V).double()[:, None]
    bound = scale * (n + 2) * 2.0 ** -24 * ab \
        + HALF[dt] * (g * scale).abs() * 1.001 + TINY[dt]
    assert dw.dtype == dt
    assert ((dw.cpu().double() - g * scale).abs() <= bound).all()
    assert not dw.cpu()[n[:, 0] == 0].any()


CASES = [
    # vocab, D, tokens, dtype, index type, scale, kind
    (1, 8, 1, "bfloat16", "int64", 1.0, "uniform"),
    (2, 768, 3000, "bfloat16", "int64", 1.0, "uniform"),
    (2, 64, 5000, "bfloat16", "int32", 2.0, "one"),
    (1000, 64, 148, "float16", "int64", 32.0, "uniform"),
    (1000, 1, 77, "float32", "int64", 3.0, "uniform"),
    (257, 33, 999, "bfloat16", "int32", 22.627416997969522, "zipf"),
    (5000, 100, 2000, "float32", "int32", 0.125, "zipf"),
    (5000, 512, 4001, "bfloat16", "int64", 32.0, "zipf"),
    (70000, 40, 33, "bfloat16", "int64", 1.0, "uniform"),
    (300000, 16, 3000, "float16", "int64", 1.0, "outside"),
    (50, 24, 1025, "float32", "int32", 1.0, "outside"),
    (3, 2056, 70, "bfloat16", "int64", 1.0, "uniform"),
    (40, 16, 64, "bfloat16", "int64", 1.0, "sorted"),
    # one list of a wave's tokens and several, few rows and many
    (900, 16, 8192, "bfloat16", "int32", 1.0, "zipf"),
    (900, 16, 16384, "bfloat16", "int32", 1.0, "outside"),
    (31, 8, 16385, "float32", "int64", 2.0, "uniform"),
    (40000, 8, 40001, "bfloat16", "int32", 1.0, "zipf"),
    (140000, 8, 20000, "bfloat16", "int64", 1.0, "uniform"),
]


def _make(seed, V, D, N, dt, it, kind):
    g = torch.Generator().manual_seed(seed)
    dt, it = getattr(torch, dt), getattr(torch, it)
    if kind == "one":
        idx = torch.full((N,), V - 1)
    elif kind == "zipf":
        p = torch.arange(1, V + 1).double().pow(-1.1)
        idx = torch.multinomial(p, N, replacement=True, generator=g)
    elif kind == "outside":
        idx = torch.randint(-V, 2 * V, (N,), generator=g)
    elif kind == "sorted":
        idx = torch.arange(N) % V
    else:
        idx = torch.randint(0, V, (N,), generator=g)
    w = torch.randn(V, D, generator=g).to(dt).cuda()
    dy = torch.randn(N, D, generator=g).to(dt).cuda()
    return idx.to(it).cuda(), w, dy


@pytest.mark.parametrize("i", range(len(CASES)))
def test_embedding(i):
    V, D, N, dt, it, scale, kind = CASES[i]
    idx, w, dy = _make(i, V, D, N, dt, it, kind)
    _check_embed(idx, w, dy, scale)


def test_embedding_shapes_and_strides():
    idx, w, dy = _make(50, 90, 48, 6 * 7, "bfloat16", "int64", "uniform")
    _check_embed(idx.reshape(6, 7), w, dy.reshape(6, 7, 48), 1.0)
    # indices, table and gradients that are views, or start off 16 bytes
    wide = torch.cat([idx, idx]).reshape(2, -1).t()[:, 0]
    _check_embed(wide, w, dy, 4.0)
    off = torch.cat([w.new_zeros(1), w.flatten()])[1:].reshape(w.shape)
    offd = torch.cat([dy.new_zeros(3), dy.flatten()])[3:].reshape(dy.shape)
    _check_embed(idx, off, offd, 4.0)
    _check_embed(idx, w, dy[:1].expand(42, 48), 1.0)
    # indices of other types, none at all
    _check_embed(idx.to(torch.uint8), w, dy, 1.0)
    _check_embed(idx.float(), w, dy, 1.0)
    _check_embed(idx[:0], w, dy[:0], 1.0)


def test_embedding_same_bits_and_far_index():
    idx, w, dy = _make(51, 300, 256, 20000, "bfloat16", "int64", "zipf")
    a = _embed(idx, w, dy, 1.0)
    b = _embed(idx, w, dy, 1.0)
    assert torch.equal(a[1], b[1])
    # 64-bit indices that fit the table when cut to 32 bits
    idx[::3] += 1 << 32
    _check_embed(idx, w, dy, 1.0)


def test_embedding_nan_stays_in_its_row():
    idx, w, dy = _make(52, 20, 64, 500, "float32", "int64", "uniform")
    idx[idx == 7] = 6
    idx[100] = 7
    dy[100] = float("nan")
    _, dw = _embed(idx, w, dy, 1.0)
    bad = torch.isnan(dw).any(1).cpu()
    assert bad[7] and int(bad.sum()) == 1


def test_embedding_graph_replays():
    import anand_mxnet_amd as mx
    from anand_mxnet_amd import _C
    sets = [_make(60 + i, 800, 96, 2500, "bfloat16", "int64", "zipf")
            for i in range(4)]
    idx, w, dy = (t.clone() for t in sets[0])
    _C.embedding_bwd(idx, dy, 800, 2.0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _C.embedding_fwd(idx, w, 2.0)
        dw = _C.embedding_bwd(idx, dy, 800, 2.0)
    for s in (sets[1], sets[2], sets[3], sets[0]):
        for t, x in zip((idx, w, dy), s):
            t.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _C.embedding_fwd(s[0], s[1], 2.0))
        assert torch.equal(dw, _C.embedding_bwd(s[0], s[2], 800, 2.0))


def test_embedding_refuses_too_many_tokens():
    """Places in the order of the tokens are 32 bits wide."""
    from anand_mxnet_amd import _C
    idx = torch.empty(0x7ffff000, dtype=torch.int32, device="cuda")
    dy = torch.empty(0x7ffff000, 0, device="cuda")
    with pytest.raises(RuntimeError, match="too large"):
        _C.embedding_bwd(idx, dy, 10, 1.0)


# ------------------------------------------------------------------ clip

def _shapes(n, rng):
    return [tuple(int(x) for x in rng.integers(1, 40, rng.integers(0, 4)))
            for _ in range(n)]


def _arrays(seed, n, dts, std=1.0):
    rng = np.random.default_rng(seed)
    out = []
    for i, s in enumerate(_shapes(n, rng)):
        x = torch.from_numpy(np.asarray(rng.standard_normal(s) * std))
        out.append(x.to(dts[i % len(dts)]).cuda())
    return out


def _check_clip(arrays, max_norm, got, norm, before):
    total = sum((b.double() ** 2).sum() for b in before)
    want = float(total.sqrt())
    # squares and sums in 64 bits; the result is rounded to 32
    assert abs(float(norm) - want) <= want * 2.0 ** -23
    f = min(1.0, max_norm / (want + 1e-8))
    for g, b in zip(got, before):
        if f == 1.0:
            assert torch.equal(g, b)
            continue
        w = b.double() * f
        # the factor and the product are rounded to 32 bits, then the type
        rel = HALF[b.dtype] + 2.0 ** -22
        assert ((g.double() - w).abs() <= rel * w.abs()
                + TINY[b.dtype]).all()


DTS = [[torch.bfloat16], [torch.float16], [torch.float32],
       [torch.float32, torch.bfloat16, torch.float16]]


@pytest.mark.parametrize("n", [1, 5, 140, 141, 300])
@pytest.mark.parametrize("d", range(len(DTS)))
@pytest.mark.parametrize("ratio", [0.1, 5.0])
def test_clip(n, d, ratio):
    import anand_mxnet_amd as mx
    arrays = _arrays(n * 10 + d, n, DTS[d])
    before = [a.clone() for a in arrays]
    total = float(sum((b.double() ** 2).sum() for b in before).sqrt())
    nds = [mx.nd.from_torch(a) for a in arrays]
    out = [torch.full_like(a, 7.0) for a in arrays]
    norm = mx.nd.multi_clip_global_norm(
        nds, total * ratio, out=[mx.nd.from_torch(o) for o in out])
    _check_clip(arrays, total * ratio, out, norm._t, before)
    assert all(torch.equal(a, b) for a, b in zip(arrays, before))
    norm = mx.nd.multi_clip_global_norm(nds, total * ratio)
    _check_clip(arrays, total * ratio, arrays, norm._t, before)


def test_clip_large_odd_and_views():
    import anand_mxnet_amd as mx
    g = torch.Generator(device="cuda").manual_seed(3)
    flat = torch.randn(3000001, device="cuda", generator=g)
    half = torch.randn(700003, device="cuda", generator=g).bfloat16()
    arrays = [flat[1:1000000], flat[1000003:1000004], half[5:700001],
              flat[1000010:2999810].reshape(-1, 11).t(), half[:3]]
    before = [a.clone() for a in arrays]
    keep = flat[0].clone(), half[700002].clone()
    norm = mx.nd.multi_clip_global_norm(
        [mx.nd.from_torch(a) for a in arrays], 3.0)
    _check_clip(arrays, 3.0, arrays, norm._t, before)
    assert torch.equal(flat[0], keep[0]) and torch.equal(half[700002],
                                                         keep[1])


def test_clip_extremes():
    import anand_mxnet_amd as mx
    f = mx.nd.multi_clip_global_norm
    nd = mx.nd.from_torch
    big = [torch.full((1000,), 1e30, device="cuda")]
    n = f([nd(b) for b in big], 1.0)
    assert abs(float(n._t) / (1e30 * 1000 ** 0.5) - 1) < 1e-6
    assert abs(float(big[0].double().norm()) - 1.0) < 1e-6
    small = [torch.full((1000,), 1e-30, device="cuda")]
    n = f([nd(b) for b in small], 1.0)
    assert abs(float(n._t) / (1e-30 * 1000 ** 0.5) - 1) < 1e-6
    bad = torch.ones(10, device="cuda")
    bad[3] = float("nan")
    keep = torch.ones(5, device="cuda")
    n = f([nd(bad), nd(keep)], 0.1)
    assert torch.isnan(n._t) and keep.eq(1).all() and bad[0] == 1
    z = torch.zeros(10, device="cuda")
    assert float(f([nd(z)], 0.0)._t) == 0.0
    o = torch.ones(10, device="cuda")
    f([nd(o)], 0.0)
    assert not o.any()
    e = [nd(torch.zeros(0, device="cuda")), nd(torch.ones(4, device="cuda"))]
    assert float(f(e, 10.0)._t) == 2.0


def test_clip_more_elements_than_32_bits():
    import anand_mxnet_amd as mx
    n = (1 << 32) + 1003
    x = torch.full((n,), 0.25, dtype=torch.bfloat16, device="cuda")
    norm = mx.nd.multi_clip_global_norm([mx.nd.from_torch(x)], 1e6)
    assert abs(float(norm._t) / (0.25 * n ** 0.5) - 1) < 2.0 ** -23
    assert float(x[0]) == float(x[-1]) == 0.25
    max_norm = float(norm._t) / 2        # the factor is 1/2 within 2**-23
    mx.nd.multi_clip_global_norm([mx.nd.from_torch(x)], max_norm)
    lo, hi = torch.aminmax(x)
    assert float(lo) == float(hi) == 0.125


def test_clip_graph_replays():
    import anand_mxnet_amd as mx
    nd = mx.nd.from_torch
    arrays = _arrays(5, 150, DTS[3])
    out = [torch.empty_like(a) for a in arrays]
    A, O = [nd(a) for a in arrays], [nd(o) for o in out]
    mx.nd.multi_clip_global_norm(A, 1.0, out=O)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = mx.nd.multi_clip_global_norm(A, 1.0, out=O)
    for seed in (6, 7, 8):
        for a in arrays:
            a.mul_(1.5)
        g.replay()
        torch.cuda.synchronize()
        want = [torch.empty_like(a) for a in arrays]
        n = mx.nd.multi_clip_global_norm(A, 1.0, out=[nd(w) for w in want])
        assert torch.equal(n._t, norm._t)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_clip_refuses():
    import anand_mxnet_amd as mx
    f, nd = mx.nd.multi_clip_global_norm, mx.nd.from_torch
    x = torch.ones(100, device="cuda")
    bad = [
        ([nd(x), nd(x)], {}),                          # twice the same
        ([nd(x[:60]), nd(x[50:])], {}),
        ([nd(x[:50]), nd(x[50:])], dict(out=[nd(x[50:]), nd(x[:50])])),
        ([nd(x)], dict(out=[nd(torch.ones(99, device="cuda"))])),
        ([nd(x)], dict(out=[nd(torch.ones(100, device="cuda").half())])),
        ([nd(x)], dict(out=[nd(torch.ones(100))])),
        ([nd(x), nd(torch.ones(3))], {}),
        ([nd(x.double())], {}),
        ([nd(x.int())], {}),
        ([nd(torch.ones(4, 4, device="cuda").t()[:2]),
          nd(x.double())], {}),
    ]
    for arrays, kw in bad:
        with pytest.raises(mx.base.MXNetError):
            f(arrays, 1.0, **kw)
    with pytest.raises(mx.base.MXNetError):
        f([nd(x)], -1.0)
    assert x.eq(1).all()
    # reading one array twice is no conflict
    a, b = torch.empty_like(x), torch.empty_like(x)
    n = f([nd(x), nd(x)], 1.0, out=[nd(a), nd(b)])
    assert abs(float(n._t) - 200 ** 0.5) < 1e-5 and torch.equal(a, b)


def test_gluon_clip_global_norm():
    import anand_mxnet_amd as mx
    from anand_mxnet_amd import gluon
    arrays = _arrays(9, 20, DTS[2])
    before = [a.clone() for a in arrays]
    n = gluon.utils.clip_global_norm([mx.nd.from_torch(a) for a in arrays],
                                     2.0)
    assert isinstance(n, float)
    _check_clip(arrays, 2.0, arrays, n, before)
    # what the kernels refuse still goes one by one
    d = torch.ones(9, device="cuda", dtype=torch.float64)
    assert gluon.utils.clip_global_norm([mx.nd.from_torch(d)], 1.5) == 3.0
    assert torch.allclose(d, torch.full_like(d, 0.5))
