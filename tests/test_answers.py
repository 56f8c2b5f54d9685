"""Options and checks of scored answers that need no GPU."""
import pytest

from hos_b200 import sampling
from hos_b200.engine import cli


def test_options():
    a = cli.parse_args([])
    assert a.logprobs is None and a.answers == [] and not a.share_prefix
    a = cli.parse_args(["-p", "1,2", "--logprobs", "3", "--score", "4, 5", "--score", "6", "--share-prefix"])
    assert (a.logprobs, a.answers, a.share_prefix) == (3, [[4, 5], [6]], True)
    with pytest.raises(SystemExit):
        cli.parse_args(["--score", "x"])


def test_a_scored_token_is_its_id(capsys):
    import torch
    scores = sampling.TokenScores(torch.tensor([-1.0, -2.0]), torch.tensor([0.5, 0.25]), torch.tensor([[3, 7], [9, 4]]), torch.tensor([[-1.0, -1.5], [-0.5, -2.0]]))
    a, b = sampling.scored_tokens([3, 4], scores)
    assert a == 3 and [a, b] == [3, 4] and {a: 1}[3] == 1 and (a.logprob, a.entropy, a.top) == (-1.0, 0.5, [(3, -1.0), (7, -1.5)])
    plain, = sampling.scored_tokens([5], sampling.TokenScores(torch.tensor([-3.0]), torch.tensor([1.0]), None, None))
    assert plain == 5 and plain.top == []
    cli.report([a, plain, 8])
    lines = capsys.readouterr().err.splitlines()
    assert lines == ["[hos] 3 logprob -1.0000 entropy 0.5000 | 3:-1.0000 7:-1.5000", "[hos] 5 logprob -3.0000 entropy 1.0000"]
