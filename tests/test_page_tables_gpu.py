"""plan_batch against a model of it with lists."""
import random

import pytest

import infernt_b200 as ib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


class Model:
    """Tables, the pages each sequence holds, the free pages in their order."""

    def __init__(self, n, pages, page, width):
        self.n, self.pages, self.page, self.width = n, pages, page, width
        self.tables = [[] for _ in range(n)]
        self.free = list(range(pages))

    def plan(self, lens, new, max_rows):
        """(q_start, kv_len, positions, slots, bits)"""
        bits, moves, wanted_pages, wanted_rows = 0, [], 0, 0
        for s in range(self.n):
            fine = lens[s] >= 0 and new[s] >= 0 and lens[s] + new[s] <= min(self.width * self.page, 1 << 30)
            bits |= 0 if fine else 16
            held = len(self.tables[s])
            need = -(-(lens[s] + new[s]) // self.page) if fine else held
            more, rows = max(0, need - held), new[s] if fine else 0
            wanted_pages += more
            wanted_rows += rows
            waits = (more > 0 and wanted_pages > len(self.free)) or (rows > 0 and wanted_rows > max_rows)
            bits |= 32 if waits else 0
            moves.append((need, new[s]) if fine and not waits else (held, 0))
        back, starts, kv, positions, slots = [], [0], [], [], []
        for s, (need, n) in enumerate(moves):
            t = self.tables[s]
            while len(t) < need:
                t.append(self.free.pop(0))
            back += t[need:]
            del t[need:]
            starts.append(starts[-1] + n)
            kv.append(lens[s] + n)
            for p in range(lens[s], lens[s] + n):
                positions.append(p)
                slots.append(t[p // self.page] * self.page + p % self.page)
        self.free += back
        return starts, kv, positions, slots, bits


class Pair:
    def __init__(self, torch, n, pages, page, width):
        self.torch, self.model = torch, Model(n, pages, page, width)
        self.tables = ib.PageTables.empty(n, pages, page, width)
        self.n = n

    def step(self, lens, new, max_rows, **kw):
        torch, n = self.torch, self.n
        i32 = dict(dtype=torch.int32, device="cuda")
        self.q_start, self.kv_len = torch.full((n + 1,), 9, **i32), torch.full((n,), 9, **i32)
        positions, slots = torch.full((max_rows,), -7, **i32), torch.full((max_rows,), -7, **i32)
        err = torch.zeros(1, **i32)
        ib.plan_batch(self.tables, torch.tensor(lens, **i32).view(n), torch.tensor(new, **i32).view(n), self.q_start,
                      self.kv_len, positions, slots, err=err, **kw)
        starts, kv, pos, sl, bits = self.model.plan(lens, new, max_rows)
        assert self.q_start.tolist() == starts and self.kv_len.tolist() == kv
        assert positions.tolist() == pos + [-7] * (max_rows - len(pos))
        assert slots.tolist() == sl + [-7] * (max_rows - len(sl))
        assert int(err) == bits
        self.check()
        return kv, bits

    def check(self):
        table, held, free, state = (t.tolist() for t in self.tables.tensors)
        m = self.model
        assert held == [len(t) for t in m.tables]
        assert table == [t + [-1] * (m.width - len(t)) for t in m.tables]
        head, count = state[:2]
        assert count == len(m.free) and state[2:] == [0, 0]
        assert [free[(head + i) % m.pages] for i in range(count)] == m.free


@pytest.mark.parametrize("n", [1, 2, 31, 33, 1000, 1024, 1025, 3000])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_lives_of_sequences(torch, n, page):
    """Prompts, drafts taken and rejected, sequences that end, a pool that runs
    short, row places that run short."""
    r = random.Random(n * page)
    pair = Pair(torch, n, max(4, n * 60 // page // 2), page, 120 // page + 2)
    lens = [0] * n
    seen = 0
    for step in range(12):
        new = []
        for s in range(n):
            if r.random() < 0.1:
                lens[s] = 0
            room = pair.model.width * page - lens[s]
            new.append(min(room, r.choice([0, 1, 1, 5, r.randint(0, 60)])))
        rows = max(1, sum(new) if r.random() < 0.7 else sum(new) // 2)
        kv, bits = pair.step(lens, new, rows)
        seen |= bits
        # some of the new tokens stay
        lens = [max(0, b - r.randint(0, max(0, b - a))) if b > a else a for a, b in zip(lens, kv)]
    assert seen == 32 or n <= 2


@pytest.mark.parametrize("rows", [4096, 4097, 60000])
def test_long_prompts(torch, rows):
    pair = Pair(torch, 9, 4000, 16, 2000)
    lens, new = [0] * 9, [1, 0, rows // 2, 33, 0, 0, rows // 4, 3, 64]
    kv, _ = pair.step(lens, new, rows)
    kv, _ = pair.step(kv, [1] * 9, rows)
    pair.step([x // 2 for x in kv], [0, 0, 7, 900, 0, 1, 0, 1, 2], rows)
    pair.step([0] * 9, [0] * 9, rows)
    assert pair.model.free != list(range(4000)) and len(pair.model.free) == 4000


def test_many_empty_sequences_between(torch):
    n = 65535
    pair = Pair(torch, n, 600, 16, 300)
    new = [0] * n
    new[0], new[n // 2], new[n - 1] = 33, 4100, 5
    pair.step([0] * n, new, 5000)


def test_what_needs_no_page_never_waits(torch):
    pair = Pair(torch, 4, 3, 16, 4)
    pair.step([0] * 4, [10, 10, 17, 3], 100)  # the third needs two pages: it waits, and so does the fourth
    assert pair.kv_len.tolist() == [10, 10, 0, 0]
    pair.step([10, 10, 0, 0], [6, 7, 0, 16], 100)  # the second needs another page, the last one left
    assert pair.kv_len.tolist() == [16, 17, 0, 0]
    pair.step([0, 17, 0, 0], [0, 2, 0, 3], 100)  # what the first gives back is for the next call
    assert pair.kv_len.tolist() == [0, 19, 0, 0]
    pair.step([0, 19, 0, 0], [0, 0, 0, 3], 100)
    assert pair.kv_len.tolist() == [0, 19, 0, 3]


def test_numbers_out_of_range(torch):
    pair = Pair(torch, 6, 20, 8, 4)
    pair.step([0] * 6, [8] * 6, 100)
    kv, bits = pair.step([8, -1, 8, 8, 33, 2 ** 31 - 1], [1, 1, -2, 25, 0, 2 ** 31 - 1], 100)
    assert bits == 16


@pytest.mark.parametrize("state", [[-1, 5], [20, 5], [0, 21], [0, -1], [2 ** 31 - 1, 2 ** 31 - 1]])
def test_a_ring_out_of_range_is_not_touched(torch, state):
    t = ib.PageTables.empty(3, 20, 8, 4)
    i32 = dict(dtype=torch.int32, device="cuda")
    t.tensors[3][:2] = torch.tensor(state, **i32)
    before = [x.clone() for x in t.tensors]
    q_start, kv, err = torch.full((4,), 9, **i32), torch.zeros(3, **i32), torch.zeros(1, **i32)
    lens = torch.tensor([0, 3, 5], **i32)
    ib.plan_batch(t, lens, torch.ones_like(lens), q_start, kv, err=err)
    assert int(err) == 16 and q_start.tolist() == [0] * 4 and kv.tolist() == [0, 3, 5]
    assert all(bool((a == b).all()) for a, b in zip(before, t.tensors))


@pytest.mark.parametrize("held", [[5, 0, 0], [-1, 0, 0], [2 ** 31 - 1, 4, 4], [4, 4, 4]])
def test_held_pages_that_were_never_given(torch, held):
    """Wrong counts do not lead out of the arrays."""
    i32 = dict(dtype=torch.int32, device="cuda")
    t = ib.PageTables.empty(3, 2, 8, 4)
    t.tensors[1].copy_(torch.tensor(held, **i32))
    q_start, err = torch.zeros(4, **i32), torch.zeros(1, **i32)
    lens = torch.zeros(3, **i32)
    for _ in range(3):
        ib.plan_batch(t, lens, lens.clone(), q_start, lens.clone(), err=err)
    torch.cuda.synchronize()
    assert bool((t.tensors[1] <= 2 ** 31 - 1).all())


def test_lengths_in_place_and_no_maps(torch):
    i32 = dict(dtype=torch.int32, device="cuda")
    t = ib.PageTables.empty(2000, 9000, 16, 8)
    lens, new = torch.randint(0, 30, (2000,), **i32), torch.randint(0, 9, (2000,), **i32)
    want = lens + new
    q_start = torch.zeros(2001, **i32)
    ib.plan_batch(t, lens, new, q_start, lens)
    assert bool((lens == want).all()) and q_start[1:].tolist() == new.cumsum(0).tolist()
    one = torch.zeros(5000 * 4, **i32)
    ib.plan_batch(t, lens, new, q_start, want, slots=one)  # slots alone, by the second kernel
    first = int(new.nonzero()[0])  # of the sequences that have rows
    at = int(lens[first])
    assert int(one[0]) == int(t.tensors[0][first, at // 16]) * 16 + at % 16


def test_captured(torch):
    """A graph of two calls, replayed: each sequence gains and loses pages."""
    i32 = dict(dtype=torch.int32, device="cuda")
    t = ib.PageTables.empty(3, 50, 4, 20)
    lens, new, zero = torch.zeros(3, **i32), torch.tensor([9, 2, 1], **i32), torch.zeros(3, **i32)
    q_start, kv, slots = torch.zeros(4, **i32), torch.zeros(3, **i32), torch.zeros(12, **i32)
    ib.plan_batch(t, lens, new, q_start, kv, slots=slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ib.plan_batch(t, lens, zero, q_start, kv)
        ib.plan_batch(t, lens, new, q_start, kv, slots=slots)
    model = Model(3, 50, 4, 20)
    model.plan([0] * 3, [9, 2, 1], 12)
    for at in ([0, 0, 0], [5, 1, 30], [0, 2, 0]):
        lens.copy_(torch.tensor(at, dtype=torch.int32))
        graph.replay()
        model.plan(at, [0] * 3, 1 << 29)
        starts, kvs, _, sl, _ = model.plan(at, [9, 2, 1], 12)
        assert kv.tolist() == kvs and q_start.tolist() == starts and slots.tolist()[:12] == sl
