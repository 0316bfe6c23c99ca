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
