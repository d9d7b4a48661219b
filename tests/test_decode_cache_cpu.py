"""Refusals of decoders over the paged cache that need no GPU: a call's positions are checked before anything is planned."""

import pytest

torch = pytest.importorskip("torch")


class Untouched:
    """Stands in for the cache: a refused call must not reach it."""

    def forward(self, sequences, firsts):
        raise AssertionError("the call reached the cache")


@pytest.fixture
def model():
    from bitmask_speculation_b200.decode import build_decoder
    model = build_decoder(64, layers=1, dim=32, heads=2, dtype=torch.float32, device="cpu", seed=1)
    model._cache = Untouched()
    return model


@pytest.mark.parametrize("sequences,firsts,rows", [
    ([[1, 2, 3], [4, 5, 6]], [2, 0], [2, 1]),   # the first one's rows would run into the second's
    ([[1, 2, 3], [4, 5, 6]], [0, 2], [1, 2]),   # behind the last token of the batch
    ([[1, 2, 3]], [0], [4]),
    ([[1, 2, 3]], [-1], [1]),
    ([[1, 2, 3]], [0], [-1]),
    ([[1, 2, 3], [4, 5, 6]], [0, 0], [1]),      # a count for one of two
    ([[1, 2, 3]], [0], [1, 1]),
    ([[1, 2, 3], [4, 5, 6]], [0], [1, 1]),
])
def test_positions_outside_their_sequence(model, sequences, firsts, rows):
    with pytest.raises(ValueError):
        model.logits_batch(sequences, firsts, rows)


def test_single_sequences_are_checked_too(model):
    with pytest.raises(ValueError):
        model.logits([1, 2, 3], 2, 2)
