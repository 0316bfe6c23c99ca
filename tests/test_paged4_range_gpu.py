"""paged4_attention over values and queries at the ends of their types' ranges,
and the sizes of a call at theirs."""
import pytest

import infernt_b200 as ib
import paged4_reference as ref4
import paged_reference as ref
from test_paged4_attention_gpu import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def workspace(torch):
    return ref.new_workspace(torch)


@pytest.mark.parametrize("four", [True, False])
def test_a_call_for_no_new_tokens(torch, workspace, four):
    """max_q_len 0: sequences without new tokens leave all rows; one that has
    some all the same sets bit 4."""
    case = ref4.Case4(torch, [(0, 40), (0, 7)], 8, 2, 64, 16, "fp16", spare_rows=6)
    case.max_q = 0
    pools = [torch.zeros(*case.kc.shape[:3], 64, device="cuda", dtype=case.dtype) for _ in range(2)]
    call, cache = (ib.paged4_attention, case.cache()) if four else (ib.paged_attention, ib.PagedCache(*pools))
    call(case.out, case.q, cache, case.batch(), workspace, lse=case.lse, err=case.err)
    torch.cuda.synchronize()
    assert int(case.err) == 0 and bool((case.out == 7).all()) and bool((case.lse == 7).all())
    case.q_start[1:] = 2
    call(case.out, case.q, cache, case.batch(), workspace, lse=case.lse, err=case.err)
    torch.cuda.synchronize()
    assert int(case.err) == 16 and bool((case.out == 7).all())
