"""verify_drafts: rows behind the last sequence, probabilities of a greedy
sequence that are none, and ties in full."""
import math

import pytest

import infernt_b200 as ib
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


def test_ties_in_full(torch):
    s = verify.Step(torch, [3, 2], 5000, temps=[0.0], seed=5, banned=False)
    s.target[:, [17, 4000, 900]] = 50.0
    s.tokens[1], s.tokens[2], s.tokens[4] = 17, 900, 4000
    s.run()
    assert s.out.tolist() == [17, 17, -1, 17, -1] and s.accepted.tolist() == [1, 0]
    assert s.kept.tolist() == [99, 100]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("probs", [False, True])
def test_rows_behind_the_last_sequence(torch, dtype, probs):
    """A captured step's batch has rows for the most tokens that it may get:
    those behind the last sequence stay as they are, whatever the target, the
    tokens and u hold there."""
    counts, spare = [4, 0, 1, 3], 9
    s = verify.Step(torch, counts, 1003, dtype=dtype, probs=probs, temps=[1.0, 0.0], seed=21)
    s.run()
    want, kept, acc = s.out.tolist(), s.kept.tolist(), s.accepted.tolist()
    rows = s.rows + spare

    def padded(x, fill):
        y = x.new_empty(rows, *x.shape[1:])
        y[:s.rows], y[s.rows:] = x[:s.rows], fill
        return y

    out = padded(s.out, 77)
    s.accepted.fill_(77)
    s.kept.fill_(77)
    workspace = torch.zeros(ib.verify_drafts_workspace_bytes(rows, len(counts)), dtype=torch.uint8, device="cuda")
    ib.verify_drafts(out, s.accepted, padded(s.target, math.nan), padded(s.tokens, 2 ** 30), s.q_start,
                     padded(s.u, math.nan), workspace, draft_probs=padded(s.draft, math.nan), temperature=s.temperature,
                     probabilities=probs, kv_len=s.kv_len, kept=s.kept, err=s.err)
    torch.cuda.synchronize()
    assert out.tolist() == want + [77] * spare and int(s.err) == 0
    assert s.kept.tolist() == kept and s.accepted.tolist() == acc
