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
