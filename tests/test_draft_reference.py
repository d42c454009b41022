"""The verification's definition (draft_reference.py) is lossless: over all random numbers, the first token is
distributed as the model's, whatever the draft proposed."""
import numpy as np
import pytest

import draft_reference as ref


def softmax(x):
    e = np.exp(x - x.max())
    return e / e.sum()


@pytest.mark.parametrize("mode,children", [("given", 0), ("given", 1), ("given", 3), ("drawn", 1), ("drawn", 3),
                                           ("distinct", 2), ("distinct", 4)])
def test_the_first_token_is_the_models(mode, children):
    rng = np.random.default_rng(children + len(mode))
    vocab, runs = 5, 20000
    logits = rng.standard_normal(vocab) * 1.5
    p, q = softmax(logits / 0.7), softmax(rng.standard_normal(vocab))
    q32 = q.astype(np.float32)
    seen = np.zeros(vocab)
    for _ in range(runs):
        if mode == "given":
            tokens = [0] + list(range(children))
        elif mode == "drawn":
            tokens = [0] + list(rng.choice(vocab, children, p=q))
        else:
            tokens = [0] + list(rng.choice(vocab, children, replace=False, p=q))
        rows = np.tile(logits, (children + 1, 1))
        out, _, _ = ref.verify(rows, tokens, [-1] + [0] * children, 0.7, rng.random(children + 1), rng.random(),
                               None if mode == "given" else np.tile(q32, (children + 1, 1)), mode == "distinct")
        seen[out[0]] += 1
    # a count's standard deviation is sqrt(runs p (1 - p)); five of them hold in all but one of 10^6 runs
    assert (np.abs(seen - runs * p) <= 5 * np.sqrt(runs * p * (1 - p))).all(), (seen / runs, p)


def test_masks_and_positions():
    parents = [-1, 0, 0, 1, 3, 2, -1]
    seen = ref.ancestors(parents)
    assert [list(np.nonzero(r)[0]) for r in seen] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4], [0, 2, 5], [6]]
    wide = ref.ancestors([-1] + list(range(129)))
    w = ref.words_of(wide, 3).view(np.uint64)
    assert w[0].tolist() == [1, 0, 0] and w[64].tolist() == [2 ** 64 - 1, 1, 0] and w[129].tolist() == [2 ** 64 - 1] * 2 + [3]
    assert ref.visible(ref.ancestors([-1, 0]), 2, 4).astype(int).tolist() == [[1, 1, 1, 0], [1, 1, 1, 1]]
    assert ref.visible(ref.ancestors([-1, 0]), -1, 1).astype(int).tolist() == [[0], [1]]
