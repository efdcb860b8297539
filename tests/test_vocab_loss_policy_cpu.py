"""The host's choices for a vocabulary loss, as the public function tells them, are those of the call."""
import pytest
import torch

from b200gemm import vocab_loss


@pytest.mark.parametrize("rows,vocab,hidden,top", [(1, 300, 64, 0), (999, 32003, 1000, 37), (8192, 128256, 4096, 0), (17, 300, 72, 5)])
def test_weights_of_rows_in_half_precision(rows, vocab, hidden, top):
    """A copy of hidden on 128-byte lines, and two launches, where the weights of rows leave G."""
    def of(dtype, reduction):
        return vocab_loss.policy(rows, vocab, hidden, top=top, dtype=dtype, reduction=reduction)
    plain = of(torch.bfloat16, "mean")
    for dtype, reduction in ((torch.bfloat16, "none"), (torch.bfloat16, "sum"), (torch.float16, "mean"), (torch.float16, "sum")):
        assert of(dtype, reduction) == plain
    weighed = of(torch.float16, "none")
    copy = -(-2 * rows * (-(-hidden // 64) * 64) // 256) * 256
    assert weighed.pop("workspace_backward") == plain.pop("workspace_backward") + copy
    assert weighed.pop("launches_backward") == plain.pop("launches_backward") + 2
    assert weighed == plain


def test_refusals():
    with pytest.raises(ValueError, match="reduction"):
        vocab_loss.policy(1, 1, 8, reduction="batchmean")
