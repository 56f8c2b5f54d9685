"""Log probabilities of tokens: what is refused, without a GPU, and how the rows are cut."""
import pytest
import torch

from hos_b200 import ops
from hos_b200.errors import KernelError
from hos_b200.sampling import TokenScores, log_probs


def test_logits_that_are_not_on_the_gpu_are_refused():
    with pytest.raises(KernelError, match="on the GPU"):
        log_probs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32), 1)


@pytest.mark.parametrize("top", [-1, 33])
def test_so_many_alternatives_are_refused(top):
    with pytest.raises(KernelError, match="alternatives"):
        log_probs(torch.zeros(2, 64), torch.zeros(2, dtype=torch.int32), top)


@pytest.mark.parametrize("held", [0, 2])
def test_scores_to_write_into_need_places_for_the_alternatives(held):
    with pytest.raises(KernelError, match="places for 3"):
        log_probs(torch.zeros(2, 64), torch.zeros(2, dtype=torch.int32), 3, TokenScores.empty(2, held, "cpu"))


def test_scores_to_write_into_have_the_sizes_asked_for():
    s = TokenScores.empty(3, 4, "cpu")
    assert s.logprob.shape == s.entropy.shape == (3,) and s.top_ids.shape == s.top_logprobs.shape == (3, 4)
    assert s.top_ids.dtype == torch.int32 and s.top_logprobs.dtype == torch.float32
    assert TokenScores.empty(3, 0, "cpu").top_ids is None


@pytest.mark.parametrize("rows", [1, 2, 18, 19, 64, 148, 600, 5000])
@pytest.mark.parametrize("vocab", [1, 7, 8192, 8193, 50000, 256000])
def test_blocks_of_a_row_are_what_the_kernel_takes(rows, vocab):
    threads, blocks = ops.log_probs_blocks(rows, vocab)
    assert threads in (128, 256, 1024) and blocks in (1, 2, 4, 8)
    assert blocks == 1 or (rows * blocks <= 148 and vocab > 32768 * blocks // 2)
