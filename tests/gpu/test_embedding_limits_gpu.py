"""The gradient of an embedding's table at its largest sizes (GPU)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [1000])
def test_tokens_past_the_largest_launch(vocab):
    """More chunks of tokens than blocks that one launch may have: what
    follows is summed too.  Rows of one column that count their tokens."""
    from anand_mxnet_amd.ops.hip import _C
    n = (1 << 29) + 12345
    g = torch.Generator(device="cuda").manual_seed(1)
    idx = torch.randint(0, vocab, (n,), generator=g, device="cuda",
                        dtype=torch.int32)
    idx[-40:] = vocab - 1
    # whole numbers below 2**24: exact in 32 bits
    want = torch.bincount(idx, minlength=vocab)
    got = _C.embedding_bwd(idx, torch.ones(n, 1, device="cuda"), vocab)
    assert torch.equal(got[:, 0].long(), want)


@pytest.mark.parametrize("vocab", [2 ** 31 - 2, 2 ** 31 - 5000])
def test_rows_near_2_to_the_31(vocab):
    """The last rows of a table, and the rows that no token hits."""
    from anand_mxnet_amd.ops.hip import _C
    idx = torch.tensor([vocab - 1, 0, vocab - 8200, vocab - 1, vocab],
                       dtype=torch.int32, device="cuda")
    dy = torch.tensor([1., 2., 4., 8., 16.], device="cuda")[:, None].bfloat16()
    full = torch.full((vocab, 1), float("nan"), dtype=torch.bfloat16,
                      device="cuda")
    del full  # the gradient is likely to get this memory
    got = _C.embedding_bwd(idx, dy, vocab)
    for r, v in ((0, 2.), (vocab - 8200, 4.), (vocab - 1, 9.)):
        assert float(got[r, 0]) == v
        got[r, 0] = 0
    assert not got.any()


def _sum64(idx, dy, vocab, scale):
    """The gradient in 64 bits, and the bound of a sum in 32 bits that is
    rounded once: n terms err by n 2**-24 of their absolute sum, the scale
    and the type's rounding by a step each."""
    ok = (idx >= 0) & (idx < vocab)
    i, g = idx[ok].long(), dy[ok].double() * scale
    want = torch.zeros(vocab, dy.shape[1], dtype=torch.float64,
                       device=idx.device)
    mag, n = torch.zeros_like(want), torch.zeros(
        vocab, 1, dtype=torch.float64, device=idx.device)
    want.index_add_(0, i, g)
    mag.index_add_(0, i, g.abs())
    n.index_add_(0, i, torch.ones(len(i), 1, dtype=torch.float64,
                                  device=idx.device))
    tiny = torch.finfo(dy.dtype).smallest_normal
    return want, (n + 2) * 2.0 ** -24 * mag + \
        torch.finfo(dy.dtype).eps / 2 * want.abs() + tiny


CASES = [  # rows, columns, tokens: both orders, each number of passes
    (1, 8, 40000), (2, 24, 70000), (15, 7, 70001), (16, 8, 65537),
    (1000, 64, 28672), (1000, 64, 28673), (2047, 8, 50000),
    (2048, 8, 50000), (32768, 64, 45056), (32768, 64, 45057),
    (32769, 3, 131071), (250000, 16, 70000), (1 << 20, 16, 5),
    ((1 << 22) - 1, 4, 30000), (1 << 22, 4, 30000),
    (10000000, 8, 1), (10000000, 16, 300000), (500, 1, 2200000),
]


@pytest.mark.parametrize("vocab,D,n", CASES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_orders(vocab, D, n, dt):
    """Tokens spread, heaped on few rows, and outside the table, in both
    index types; the same bits in every run."""
    from anand_mxnet_amd.ops.hip import _C
    g = torch.Generator(device="cuda").manual_seed(vocab + n)
    dy = torch.randn(n, D, generator=g, device="cuda").to(dt)
    even = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    heap = (vocab ** torch.rand(n, generator=g, device="cuda",
                                dtype=torch.float64)).long() - 1
    out = torch.rand(n, generator=g, device="cuda") < 0.1
    heap[out] = torch.randint(-3, 3, (int(out.sum()),), generator=g,
                              device="cuda") + vocab
    wide = heap.clone()
    wide[::97] += 2 ** 40
    for idx in (even, heap.to(torch.int32), wide):
        want, bound = _sum64(idx, dy, vocab, 0.5)
        got = _C.embedding_bwd(idx, dy, vocab, 0.5)
        assert ((got.double() - want).abs() <= bound).all()
        again = _C.embedding_bwd(idx, dy, vocab, 0.5)
        assert torch.equal(got, again)
        del want, bound


def test_orders_replayed():
    """A captured gradient of each order gives the eager one's bits, with
    other tokens at each replay."""
    from anand_mxnet_amd.ops.hip import _C
    for vocab, n in ((1000, 4096), (1000, 65536), (1 << 20, 65536)):
        idx = torch.zeros(n, dtype=torch.int64, device="cuda")
        dy = torch.randn(n, 16, device="cuda")
        for _ in range(2):
            _C.embedding_bwd(idx, dy, vocab)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _C.embedding_bwd(idx, dy, vocab)
        for i in range(4):
            idx.copy_(torch.randint(0, vocab >> (3 * i), (n,),
                                    device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, _C.embedding_bwd(idx, dy, vocab))
