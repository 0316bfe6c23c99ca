"""Drafting steps whose batch has room for more tokens than come: one captured
step, replayed with other numbers of tokens a sequence (none among them), holds
the same rows as calls for exactly those, and leaves the rows behind them."""
import random

import pytest

import infernt_b200 as ib
import paged_reference as ref
from test_drafting_step_gpu import D, NKV, NQ, PAGE, V

pytestmark = pytest.mark.gpu

N, MOST, ROWS = 6, 5, 40


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


class Steps:
    """Buffers for `rows` tokens, and one step over them."""

    def __init__(self, torch, rows):
        self.torch, self.rows = torch, rows
        i32 = dict(dtype=torch.int32, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(4)
        self.embed = torch.randn(V, (NQ + 2 * NKV) * D, generator=g, device="cuda")
        self.out_w = torch.randn(NQ * D, V, generator=g, device="cuda") * 0.2
        self.tables = ib.PageTables.empty(N, 60, PAGE, 10)
        self.pools = [torch.zeros(60, NKV, PAGE, D // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.scales = torch.full((60, NKV, PAGE), -1, **i32)
        self.cache = ib.PagedCache4(*self.pools, self.scales, torch.bfloat16)
        self.rope = ib.RopeParams(theta=10000.0, rotary_dim=D)
        self.lens, self.new = torch.zeros(N, **i32), torch.zeros(N, **i32)
        self.q_start, self.kv_len = torch.zeros(N + 1, **i32), torch.zeros(N, **i32)
        self.accepted, self.err = torch.zeros(N, **i32), torch.zeros(1, **i32)
        self.temperature = torch.tensor([0.0, 1.0, 0.7, 0.0, 1.3, 2.0], device="cuda")
        self.ws = ref.new_workspace(torch)
        self.tokens, self.u = torch.zeros(rows, **i32), torch.zeros(rows, device="cuda")
        self.size(rows)

    def size(self, rows):
        torch, i32 = self.torch, dict(dtype=self.torch.int32, device="cuda")
        self.at = rows
        self.positions, self.slots, self.out = (torch.full((rows,), 77, **i32) for _ in range(3))
        self.q = torch.full((rows, NQ, D), 7.0, device="cuda", dtype=torch.bfloat16)
        self.attn = torch.full_like(self.q, 7.0)
        self.vws = torch.zeros(ib.verify_drafts_workspace_bytes(rows, N), dtype=torch.uint8, device="cuda")
        self.batch = ib.RaggedBatch(self.q_start, self.kv_len, self.tables.tensors[0], rows, MOST)

    def step(self):
        torch, n = self.torch, self.at
        ib.plan_batch(self.tables, self.lens, self.new, self.q_start, self.kv_len, self.positions, self.slots, err=self.err)
        qkv = self.embed[self.tokens[:n].long()].view(n, NQ + 2 * NKV, D)
        ib.paged4_rope_append(self.q, qkv[:, :NQ], qkv[:, NQ:NQ + NKV], qkv[:, NQ + NKV:], self.cache, self.batch, self.rope,
                              err=self.err)
        ib.paged4_attention(self.attn, self.q, self.cache, self.batch, self.ws, err=self.err)
        # (a sum of products in an order that does not depend on the number of rows)
        logits = (self.attn.float().view(n, NQ * D, 1) * self.out_w).sum(1)
        ib.verify_drafts(self.out, self.accepted, logits, self.tokens[:n], self.q_start, self.u[:n], self.vws,
                         temperature=self.temperature, kv_len=self.kv_len, kept=self.lens, err=self.err)


def test_replayed_steps_with_spare_rows(torch):
    r = random.Random(5)
    wide, exact = Steps(torch, ROWS), Steps(torch, ROWS)
    wide.step()  # no tokens at all; what libraries load at a first call, too
    torch.cuda.synchronize()
    assert int(wide.err) == 0 and wide.lens.tolist() == [0] * N and bool((wide.out == 77).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        wide.step()
    for _ in range(25):
        new = [r.choice([0, 1, 1, 2, MOST]) for _ in range(N)]
        total = sum(new)
        g = torch.Generator(device="cuda").manual_seed(r.randint(0, 1 << 30))
        tokens = torch.randint(0, V, (ROWS,), generator=g, dtype=torch.int32, device="cuda")
        u = torch.rand(ROWS, generator=g, device="cuda")
        for m in (wide, exact):
            m.new.copy_(torch.tensor(new, dtype=torch.int32))
            m.tokens.copy_(tokens)
            m.u.copy_(u)
        exact.size(max(1, total))
        for x in (wide.out, wide.positions, wide.slots):
            x.fill_(77)
        wide.q.fill_(7.0)
        wide.attn.fill_(7.0)
        graph.replay()
        exact.step()
        torch.cuda.synchronize()
        assert int(wide.err) == 0 and int(exact.err) == 0
        for x, y in zip((wide.lens, wide.kv_len, wide.q_start, wide.accepted, *wide.tables.tensors, *wide.pools, wide.scales),
                        (exact.lens, exact.kv_len, exact.q_start, exact.accepted, *exact.tables.tensors, *exact.pools,
                         exact.scales)):
            assert bool((x == y).all())
        for x, y in zip((wide.out, wide.positions, wide.slots, wide.q, wide.attn),
                        (exact.out, exact.positions, exact.slots, exact.q, exact.attn)):
            assert bool((x[:total] == y[:total]).all()) and bool((x[total:] == (7.0 if x.dim() == 3 else 77)).all())
    assert int(wide.lens.min()) > PAGE
