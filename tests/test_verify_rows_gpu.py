"""verify_drafts: probabilities of a greedy sequence that are none."""
import math

import pytest

import test_verify_gpu as verify

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.mark.parametrize("what", [-math.inf, math.inf, math.nan, -0.25])
def test_greedy_sequences_flag_probabilities_that_are_none(torch, what):
    """A negative (-infinity among them), infinite or NaN probability ends the
    sequence with the row's largest number and bit 6, whatever the temperature."""
    for temp in (0.0, 1.0):
        s = verify.Step(torch, [1, 1, 1], 300, probs=True, temps=[temp], seed=6, banned=False)
        best = int(s.target[1].argmax())
        s.target[1, (best + 7) % 300] = what
        s.run()
        assert int(s.err) == 64
        assert int(s.out[1]) == ((best + 7) % 300 if what == math.inf else best)
        fine = verify.Step(torch, [1, 1, 1], 300, probs=True, temps=[temp], seed=6, banned=False)
        fine.run()
        assert int(fine.err) == 0 and s.out[::2].tolist() == fine.out[::2].tolist()
