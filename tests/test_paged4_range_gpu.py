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


@pytest.mark.parametrize("n", [1, 5, 70])
@pytest.mark.parametrize("power", [-95, -80, -64, -50, 60, 115])
def test_v_vectors_all_tiny_or_all_large(torch, workspace, n, power):
    """Every V vector 2^power times an ordinary one: the bound is relative to
    the largest of them."""
    case = ref4.Case4(torch, [(n, 300), (n, 5000), (n, n)], 8, 2, 64, 16, "bf16", seed=n,
                      stretch=lambda k, v: (k, v * 2.0 ** power))
    run(torch, case, workspace)
    ref.check_attention(case, rows=range(0, n, 23))


@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("length", [33, 129, 161, 289, 20001])
@pytest.mark.parametrize("power", [40, 90])
def test_zeros_beside_large_values(torch, workspace, n, length, power):
    """One warp, and one CTA, has keys with V vectors of zeros alone, the others
    large ones: each one's weights still count in the sum."""
    def stretch(k, v):
        for s, (_, l) in enumerate(seqs):
            at = torch.arange(l, device="cuda")
            pages = torch.tensor(case.pages[s], device="cuda")[at // 16]
            zero = (at >= l // 32 * 32) | (at < l // 3)  # the first third, and the last part of 32
            v[pages[zero], :, at[zero] % 16] = 0.0
        return k, v

    seqs = [(n, length), (n, 64)]
    case = ref4.Case4(torch, seqs, 4, 2, 128, 16, "bf16", seed=n)  # whose pages the next one has too
    case = ref4.Case4(torch, seqs, 4, 2, 128, 16, "bf16", seed=n,
                      stretch=lambda k, v: stretch(k * 0.1, v * 2.0 ** power))
    run(torch, case, workspace)
    ref.check_attention(case)


@pytest.mark.parametrize("n", [1, 9, 70])
@pytest.mark.parametrize("power", [-120, -60, 60, 110, 124])
def test_queries_of_every_size(torch, workspace, n, power):
    """Queries 2^power times ordinary ones, keys as much smaller as the format
    goes: scores in FP32 as ever."""
    back = 2.0 ** -min(power, 94)
    case = ref4.Case4(torch, [(n, 200), (n, n + 3)], 8, 2, 64, 16, "bf16", seed=n,
                      stretch=lambda k, v: (k * back, v))
    case.q = (case.q.double() / 8 * 2.0 ** power).to(case.dtype)
    assert bool(case.q.isfinite().all())
    scale = 2.0 ** -max(0, power - 94) / 8
    run(torch, case, workspace, scale=scale)
    ref.check_attention(case, scale=scale, rows=range(0, n, 9))
    assert bool(case.out[:case.starts[-1]].isfinite().all())


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


@pytest.mark.parametrize("rest", [0, 3])
def test_a_long_chunk_over_a_wide_table(torch, workspace, rest):
    """8192 tokens of 64/8 heads, alone and beside sequences of a few, in a
    table of 2^20 positions: the same rows as in one that just holds them."""
    case = ref4.Case4(torch, [(8192, 8500), (rest, 300), (rest, 700)], 64, 8, 64, 1024, "bf16", seed=1)
    run(torch, case, workspace)
    out, lse = case.out.clone(), case.lse.clone()
    ref.check_attention(case, rows=[0, 1, 2, 5000, 8191])
    wide = torch.full((3, 1024), -1, dtype=torch.int32, device="cuda")
    wide[:, :case.table.shape[1]] = case.table
    case.table = wide
    case.out.fill_(7)
    run(torch, case, workspace)
    assert bool((out == case.out).all()) and bool((lse == case.lse).all())
