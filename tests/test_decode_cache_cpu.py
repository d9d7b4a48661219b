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


def test_weights_are_told_apart():
    from bitmask_speculation_b200 import decode
    build = lambda: decode.build_decoder(64, layers=2, dim=32, heads=2, dtype=torch.float32, device="cpu", seed=1)  # noqa: E731
    model = build()
    changes = (lambda m: m.load_state_dict(build().state_dict()), lambda m: m.embed.weight.detach().neg_(), lambda m: m.to(torch.float64),
               lambda m: setattr(m.blocks[1], "q", torch.nn.Linear(32, 32, bias=False)), lambda m: m.blocks.append(torch.nn.Linear(2, 2)),
               lambda m: setattr(m.norm, "weight", torch.nn.Parameter(torch.ones(32))))
    for change in changes:
        weights = decode._weights_of(model)
        assert decode._same_weights(model, weights)
        with torch.no_grad():
            change(model)
        assert not decode._same_weights(model, weights)
    with torch.inference_mode():  # parameters without a count of changes
        model = build()
        assert decode._same_weights(model, decode._weights_of(model))
