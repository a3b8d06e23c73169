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
