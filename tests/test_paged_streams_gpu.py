"""The operators over paged caches without `stream`, on torch's current
stream: in its order, and captured with what surrounds them."""
import pytest

import infernt_b200 as ib
from paged_reference import Case, check_attention, new_workspace

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


class Step:
    """q, k and v made from qkv, appended and attended; then a page copied."""

    def __init__(self, torch):
        c = Case(torch, [(1, 300), (90, 200)], 4, 2, 64, 16)
        self.torch, self.c, self.ws = torch, c, new_workspace(torch)
        self.qkv = torch.randn(c.rows, 8, 64, device="cuda")
        self.src = torch.zeros_like(self.qkv)
        self.rope = ib.RopeParams(rotary_dim=64)
        self.copies = torch.zeros(2, *c.k.shape, device="cuda", dtype=c.dtype)
        self.last = c.pages[1][199 // 16]

    def run(self):
        c = self.c
        self.src.copy_(self.qkv)
        ib.paged_rope_append(c.q, self.src[:, :4], self.src[:, 4:6], self.src[:, 6:], c.cache(), c.batch(), self.rope,
                             err=c.err)
        ib.paged_attention(c.out, c.q, c.cache(), c.batch(), self.ws, lse=c.lse, err=c.err)
        self.copies[0].copy_(c.k)
        self.copies[1].copy_(c.v)
        ib.copy_pages(self.copies, [self.last], [(self.last + 1) % c.k.shape[0]])
        ib.copy_pages([self.copies[0], self.copies[1]], [self.last], [(self.last + 2) % c.k.shape[0]])

    def check(self):
        self.torch.cuda.synchronize()
        c, last, n = self.c, self.last, self.c.k.shape[0]
        assert int(c.err) == 0
        # v is appended as it is: position 299 of sequence 0 is its new row
        assert bool((c.v[c.pages[0][299 // 16], :, 299 % 16] == self.qkv[0, 6:].to(c.dtype)).all())
        check_attention(c, rows=[0, 1, 45, 89])
        for at in (1, 2):
            assert bool((self.copies[0][(last + at) % n] == c.k[last]).all())
            assert bool((self.copies[1][(last + at) % n] == c.v[last]).all())


def busy(torch):
    """Milliseconds of work on the current stream, so that what does not wait for it comes first."""
    x = torch.randn(4096, 4096, device="cuda")
    for _ in range(20):
        x = x @ x
        x /= x.abs().amax()


def test_a_side_stream(torch):
    step = Step(torch)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        busy(torch)
        step.run()
    step.check()


def test_a_capture(torch):
    step = Step(torch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step.run()
    step.qkv.normal_()
    step.c.out.zero_()
    step.copies.zero_()
    g.replay()
    step.check()
