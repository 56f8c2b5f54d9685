"""What the 4-bit operators refuse on the host, before any kernel has an address (no GPU)."""
import pytest
import torch

from hos_b200 import ops
from hos_b200.cache import CacheManager
from hos_b200.engine.batch import build_step
from hos_b200.errors import KernelError, SpecError
from hos_b200.parts import attention4
from hos_b200.parts.base import KVNeed
from hos_b200.parts.weights4 import Weight4


def test_weights_that_are_not_on_the_gpu_are_refused():
    """Codes of a checkpoint lie on the host at first; a kernel would read the host's addresses."""
    codes, scales = torch.zeros(32, 128, dtype=torch.uint8), torch.ones(32, 2)
    with pytest.raises(SpecError, match="GPU"):
        Weight4.from_codes(codes, scales, None, 64)
    with pytest.raises(SpecError, match="GPU"):
        Weight4.from_codes(codes, scales, torch.zeros(32, 2, dtype=torch.uint8), 64)
    with pytest.raises(SpecError, match="GPU"):
        Weight4.from_matrix(torch.ones(32, 128))
    with pytest.raises(SpecError, match="GPU"):
        Weight4(torch.zeros(2, 2, 512, dtype=torch.uint8), torch.zeros(2, 2, 8, 1, 2, dtype=torch.bfloat16), 32, 128, 64, 1, False)


@pytest.mark.parametrize("group", [0, -64, 48, 33])
def test_groups_that_no_kernel_takes_are_refused(group):
    with pytest.raises(SpecError, match="groups"):
        Weight4.from_matrix(torch.ones(32, 128), group)
    with pytest.raises(SpecError, match="groups"):
        Weight4.from_codes(torch.zeros(32, 128, dtype=torch.uint8), torch.ones(32, 2), None, group)


def test_pages_and_steps_that_are_not_on_the_gpu_are_refused():
    cpu = torch.device("cpu")
    cache = CacheManager([KVNeed(2, 64, None, bits=4)], [None], [[]], 256, 256, torch.float32, cpu)
    with pytest.raises(KernelError, match="GPU"):
        ops.paged4(cache.stores[0].kv)
    with pytest.raises(KernelError, match="GPU"):
        attention4._check_step(1, build_step([[0]], [1], [0], cpu, 1), "attend")


@pytest.mark.parametrize("n,heads,kv,dim,longest,window,fill", [
    (2048, 32, 16, 128, 131072, None, 1.0), (2048, 32, 16, 128, 32768, None, 0.6), (512, 64, 8, 256, 131072, None, 0.1), (1, 8, 4, 256, 131072, None, 1.0),
    (300, 16, 1, 64, 10 ** 6, None, 0.5), (4096, 128, 8, 256, 200000, 4096, 0.9), (48, 32, 16, 128, 8000, 4096, 0.5), (20000, 8, 4, 256, 65536, None, 1.0)])
def test_the_workspace_of_attention_is_bounded(monkeypatch, n, heads, kv, dim, longest, window, fill):
    """The sums of shares take what the rows' outputs take a few times, or a fixed amount, however long the sequences are."""
    monkeypatch.setattr(attention4.ops, "sm_count", lambda: 148)
    items = kv * -(-(heads // kv) // 8)
    share, splits, cluster = attention4.bounded_shares(n, n, items, heads, dim, longest, window, fill)
    pages = attention4._pages(longest, window)
    assert share * splits >= pages and (splits - 1) * share < pages and splits <= attention4.MAX_SHARES
    assert splits == 1 or cluster or n * heads * splits * (dim + 2) * 4 <= attention4.MOST_PARTS
    fastest = attention4.shares(n, items, longest, window, fill)
    if n * heads * fastest[1] * (dim + 2) * 4 <= attention4.MOST_PARTS:               # room for all of them
        assert (share, splits, cluster) == fastest
