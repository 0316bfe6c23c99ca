"""What the operators over paged caches refuse, or serve, with memory of the
wrong kind among right ones: nothing is launched, nothing moves."""
import ctypes

import pytest

import infernt_b200 as ib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.mark.parametrize("n", [2, 5, 64, 300])
@pytest.mark.parametrize("kind", ["pageable", "pinned"])
def test_a_host_pool_among_device_pools(torch, n, kind):
    """At any place, behind pools of one allocation and of others."""
    page, pages = 64, 6
    x = torch.randint(0, 100, (n, pages, page), device="cuda", dtype=torch.uint8)
    apart = torch.randint(0, 100, (pages, page), device="cuda", dtype=torch.uint8)
    host = torch.zeros(pages, page, dtype=torch.uint8)
    host = host.pin_memory() if kind == "pinned" else host
    assert host.data_ptr() % 16 == 0
    before = x.clone()
    for at in sorted({1, n // 2, n - 1}):
        ptrs = [p.data_ptr() for p in x]
        ptrs[at - 1] = apart.data_ptr()
        ptrs[at] = host.data_ptr()
        status = ib.lib().infernt_pages_copy((ctypes.c_void_p * n)(*ptrs), n, page, pages, (ctypes.c_int * 1)(0),
                                             (ctypes.c_int * 1)(1), 1, None)
        assert status == 1 and b"not memory of the current device" in ib.lib().infernt_last_error()
    torch.cuda.synchronize()
    assert bool((x == before).all()) and not bool(host.any())
    ib.copy_pages(list(x) + [apart], [0], [1])
    torch.cuda.synchronize()
    assert bool((x[:, 1] == x[:, 0]).all()) and bool((apart[1] == apart[0]).all())


@pytest.mark.parametrize("page", [65536, 65500])
def test_overlapping_sequences_of_too_much_work(torch, page):
    """Every second sequence has all 16384 rows (q_start goes up and down): the
    units of the whole are more than 2^30, where a batch of so many rows has
    less than 2^27.  The call sets the error bit and computes nothing."""
    n, rows = 65535, 16384
    k = torch.zeros(1, 1, page, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(rows, 1, 64, device="cuda", dtype=torch.bfloat16)
    out, lse = torch.full_like(q, 7), torch.full((rows, 1), 7.0, device="cuda")
    q_start = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    q_start[1::2] = rows
    kv_len = torch.full((n,), page, dtype=torch.int32, device="cuda")
    batch = ib.RaggedBatch(q_start, kv_len, torch.zeros(n, 1, dtype=torch.int32, device="cuda"), rows, rows)
    ws = torch.zeros(ib.paged_attention_workspace_bytes(), dtype=torch.uint8, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    # what the schedule counts: a unit a tile of 64 keys and 3 an item of 256 rows (64 on pages that make no boxes)
    items = rows // (256 if page % 64 == 0 else 64)
    assert (n + 1) // 2 * items * ((page - rows) // 64 + 3) > 1 << 30
    ib.paged_attention(out, q, ib.PagedCache(k, k), batch, ws, lse=lse, err=err)
    torch.cuda.synchronize()
    assert int(err) == 1 << 4
    assert bool((out == 7).all()) and bool((lse == 7).all()) and not bool(ws[:2048].any())
    # the workspace and the kernels are as good as before
    q_start.fill_(rows)
    q_start[0] = 0
    kv_len.zero_()
    kv_len[0] = rows
    k.normal_()
    ib.paged_attention(out, q, ib.PagedCache(k, k), batch, ws, lse=lse, err=err)
    torch.cuda.synchronize()
    for r in (0, 63, 64, 16383):  # q is 0: the mean of the values so far, weights exact
        want = k[0, 0, :r + 1].double().mean(0)
        assert bool(((out[r, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + (r / 16 + 64) * 2.0 ** -22 * k[0, 0].abs().amax().double()).all())
