"""Prompt steps of fewer rows than their session has: what lies in memory that nothing wrote does not reach the sequences' rows."""
import random

import pytest
import torch
from helpers import TINY, make_folder, random_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture
def poison():
    """Memory that is taken is filled with NaN first."""
    was, fill = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory

    def on():
        torch.use_deterministic_algorithms(True, warn_only=True)
        torch.utils.deterministic.fill_uninitialized_memory = True
    yield on
    torch.use_deterministic_algorithms(was)
    torch.utils.deterministic.fill_uninitialized_memory = fill


@pytest.mark.parametrize("name", ["B", "C", "D", "E", "F", "G"])
@pytest.mark.parametrize("lengths", [[1], [5], [3, 20, 2, 1], [33], [40, 1], [70, 9, 1]])
def test_memory_that_nothing_wrote(tmp_path, name, lengths, poison):
    from hos_b200.engine import Runner
    folder = make_folder(tmp_path, name)
    rng = random.Random(len(lengths))
    rounds = [[random_tokens(rng, n, TINY[name][0]["vocab_size"]) for n in ns] for ns in (lengths, [3] * len(lengths), [1] * len(lengths))]
    got = []
    for filled in (False, True):
        r = Runner.from_folder(folder, dtype="bfloat16", max_tokens=4096)
        if filled:
            poison()
        slots = r.admit(len(lengths))
        got.append([r.step(slots, tokens) for tokens in rounds])
    for clean, filled in zip(*got):
        assert clean.isfinite().all() and torch.equal(clean, filled)


@pytest.mark.parametrize("rows", [3, 8, 20, 40])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (8, 1, 128), (4, 4, 48)])
def test_padding_rows_of_a_projection_formed_from_parts_are_zeros(rows, heads, kv, dim):
    from hos_b200 import ops
    from shared_cases import Tree
    t = Tree(kv, dim, slots=8)
    a = t.new(rows)
    step = t.step([a], [rows])
    step.token_seq[rows // 2:] = -1
    width = (heads + 2 * kv) * dim
    parts = torch.randn(2, rows, width, device="cuda")
    out = torch.full((rows, width), float("nan"), dtype=torch.bfloat16, device="cuda")
    freq = 1.0 / 10000 ** (torch.arange(0, dim, 2, device="cuda").float() / dim)
    ops.rope_kv_write(out, heads, step.token_pos, step.token_seq, step.seq_slot, step.seq_len_after, freq, dim, 0, t.view, kv, dim, partials=parts)
    assert out[:rows // 2].isfinite().all() and (out[rows // 2:] == 0).all()
