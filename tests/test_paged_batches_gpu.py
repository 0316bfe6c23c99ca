"""Ragged batches whose device arrays hold something out of range: the error
bit is set whichever sequence it is, its rows stay, the others are served."""
import pytest

import infernt_b200 as ib
from paged_reference import Case, check_attention, new_workspace
from test_paged_rope_gpu import Rope

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def ws(torch):
    return new_workspace(torch)


@pytest.mark.parametrize("R", [64, 62])
@pytest.mark.parametrize("what", ["a length without new tokens", "a start above its end", "a negative length"])
def test_rope_reports_a_sequence_that_no_row_leads_to(torch, what, R):
    seqs = [(2, 50), (0, 60), (3, 40), (9, 30)] + [(1, 9)] * 40
    r = Rope(torch, seqs, 4, 2, 64, 16, rotary_dim=R)
    c = r.c
    if what == "a length without new tokens":
        c.kv_len[1] = 16 * c.table.shape[1] + 1
    elif what == "a negative length":
        c.kv_len[1] = -5
    else:
        # sequence 1 is [2, 1): rows 0 and 1 are sequence 0's, and row 1 sequence 2's too
        c.q_start[2] = 1
    r.run()
    assert int(c.err) == 1 << 4
    if what != "a start above its end":
        r.check()


# what is out of range -> (the sequence that it is in, those that are skipped)
BAD = {"length": (1, [1]), "negative": (1, [1]), "end": (2, [2]), "many": (1, [1]), "order": (0, [0, 1])}


@pytest.mark.parametrize("seqs", [[(2, 50), (3, 60), (2, 40)], [(80, 150), (90, 200), (70, 300)],
                                  [(2, 50), (90, 200), (2, 90)], [(90, 200), (91, 200), (1, 400)]])
@pytest.mark.parametrize("what", sorted(BAD))
def test_rows_of_a_bad_sequence_stay(torch, ws, what, seqs):
    """Attention and the rotary append: rows and pages of the sequence stay as
    they are, those of the others are right."""
    r = Rope(torch, list(seqs), 8, 2, 64, 16, spare_rows=3)
    c = r.c
    far, skipped = BAD[what]
    keep = c.q_start.clone()
    if what == "length":
        c.kv_len[far] = 16 * c.table.shape[1] + 1
    elif what == "negative":
        c.kv_len[far] = -1
    elif what == "end":
        c.q_start[3] = c.rows + 1
    elif what == "order":
        c.q_start[1] = c.rows + 5  # sequence 0 ends behind all rows, 1 starts there and ends before
    batch = c.batch()
    if what == "many":
        batch.max_q_len = max(n for i, (n, _) in enumerate(seqs) if i != far)
        if seqs[far][0] <= batch.max_q_len:
            pytest.skip("sequence %d is not the longest" % far)
    stay = torch.zeros(c.rows, dtype=torch.bool, device="cuda")
    stay[c.starts[-1]:] = True
    for s in skipped:
        stay[c.starts[s]:c.starts[s + 1]] = True
    ib.paged_rope_append(r.q_out, r.q, r.kn, r.vn, c.cache(), batch, ib.RopeParams(**r.params), err=c.err)
    torch.cuda.synchronize()
    assert int(c.err) == 1 << 4
    assert bool((r.q_out[stay] == 7).all())
    c.err.zero_()
    ib.paged_attention(c.out, c.q, c.cache(), batch, ws, lse=c.lse, err=c.err)
    torch.cuda.synchronize()
    assert int(c.err) == 1 << 4
    assert bool((c.out[stay] == 7).all()) and bool((c.lse[stay] == 7).all())
    # the others, by the tests' own checks: the skipped ones have no new tokens and no positions there
    c.q_start.copy_(keep)
    for s in skipped:
        c.seqs[s] = (0, 0)
    r.check()
    check_attention(c, rows=[0, 1, 2, 63, 64, 69, 79, 89, 90])
