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
