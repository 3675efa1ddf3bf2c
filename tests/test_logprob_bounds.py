"""The bounds of logprob_bounds.py are narrow enough to see a lost part of a
row: mistakes planted in the definition, on the CPU."""
import pytest
import torch

from logprob_bounds import bounded64, head_chain, walk_chain
from score_util import check_logprobs


def values(logits, tokens, k):
    r = bounded64(logits, tokens, k, 0)
    f = lambda n, t: torch.tensor(r[n], dtype=t)  # noqa: E731
    return {"logprobs": f("logprobs", torch.float64), "entropy": f("entropy", torch.float64),
            "ids": f("ids", torch.int32), "top": f("top", torch.float64)}


def fails(got, ref):
    try:
        check_logprobs(got, ref)
    except AssertionError:
        return True
    return False


@pytest.mark.parametrize("V,chain", [(131072, walk_chain(131072, 4)), (131072, walk_chain(131072, 2)),
                                     (50021, walk_chain(50021, 2)), (600001, head_chain(130, 600001)),
                                     (290001, head_chain(300, 290001))])
def test_a_lost_tile_is_seen(V, chain):
    g = torch.Generator().manual_seed(V)
    tok = torch.tensor([[5]], dtype=torch.int32)
    for row in (torch.zeros(1, V), torch.randn(1, V, generator=g)):
        ref = bounded64(row, tok, 3, chain)
        right = values(row, tok, 3)
        assert not fails(right, ref)
        wrong = values(row.index_fill(1, torch.arange(V - 256, V), -float("inf")), tok, 3)
        for name in ("logprobs", "top"):  # each by itself
            assert fails({**right, name: wrong[name]}, ref), name
        # the sums of a row held to 12 bits
        low = {n: v.clone() for n, v in right.items()}
        low["logprobs"] += 2.0 ** -13
        assert fails(low, ref)


@pytest.mark.parametrize("V", [4096, 131072])
def test_a_lost_value_is_seen(V):
    """Two equal values that carry the row, as the seams of tiles have them."""
    row = torch.full((1, V), -25.0)
    row[0, [1023, 1024]] = 0.0
    tok = torch.tensor([[1023, 1024]], dtype=torch.int32)
    ref = bounded64(row, tok, 2, walk_chain(V, 4))
    right = values(row, tok, 2)
    assert not fails(right, ref)
    lost = row.clone()
    lost[0, 1024] = -25.0
    wrong = values(lost, tok, 2)
    for name in ("logprobs", "entropy", "ids", "top"):
        assert fails({**right, name: wrong[name]}, ref), name
