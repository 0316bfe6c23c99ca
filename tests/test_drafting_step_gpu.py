"""A drafting step over 4-bit pages as one would be built: page tables, append,
attention, logits, verification, and the kept lengths into the next step's
tables, with no number through the host.  Steps launched one by one, held to
64-bit restatements of every stage, and the same steps as one replayed graph."""
import pytest

import infernt_b200 as ib
import paged4_reference as ref4
import paged_reference as ref

pytestmark = pytest.mark.gpu

N, DRAFTS, V, NQ, NKV, D, PAGE, WIDTH, PAGES = 5, 3, 400, 8, 2, 64, 16, 12, 50


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


class Model:
    """One attention layer between an embedding and logits."""

    def __init__(self, torch, seed):
        self.torch = torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        i32 = dict(dtype=torch.int32, device="cuda")
        rows = N * (DRAFTS + 1)
        self.embed = torch.randn(V, (NQ + 2 * NKV) * D, generator=g, device="cuda")
        self.out_w = torch.randn(NQ * D, V, generator=g, device="cuda") * 0.2
        self.tables = ib.PageTables.empty(N, PAGES, PAGE, WIDTH)
        shape = (PAGES, NKV, PAGE, D // 2)
        self.kc, self.vc = (torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.scales = torch.full(shape[:3], -1, **i32)  # vectors of NaN until they are written
        self.cache = ib.PagedCache4(self.kc, self.vc, self.scales, torch.bfloat16)
        self.rope = ib.RopeParams(theta=10000.0, rotary_dim=D)
        self.lens, self.new = torch.zeros(N, **i32), torch.full((N,), DRAFTS + 1, **i32)
        self.q_start, self.kv_len = torch.zeros(N + 1, **i32), torch.zeros(N, **i32)
        self.positions, self.slots = torch.zeros(rows, **i32), torch.zeros(rows, **i32)
        self.tokens = torch.randint(0, V, (rows,), generator=g, **i32)
        self.q = torch.zeros(rows, NQ, D, device="cuda", dtype=torch.bfloat16)
        self.attn, self.logits = torch.zeros_like(self.q), torch.zeros(rows, V, device="cuda")
        self.u = torch.rand(rows, generator=g, device="cuda")
        self.temperature = torch.tensor([0.0, 1.0, 0.7, 0.0, 1.3], device="cuda")
        self.out, self.accepted = torch.zeros(rows, **i32), torch.zeros(N, **i32)
        self.ws = ref.new_workspace(torch)
        self.vws = torch.zeros(ib.verify_drafts_workspace_bytes(rows, N), dtype=torch.uint8, device="cuda")
        self.err = torch.zeros(1, **i32)
        self.batch = ib.RaggedBatch(self.q_start, self.kv_len, self.tables.tensors[0], rows, DRAFTS + 1)

    def step(self):
        torch = self.torch
        ib.plan_batch(self.tables, self.lens, self.new, self.q_start, self.kv_len, self.positions, self.slots, err=self.err)
        qkv = self.embed[self.tokens.long()].view(-1, NQ + 2 * NKV, D)
        ib.paged4_rope_append(self.q, qkv[:, :NQ], qkv[:, NQ:NQ + NKV], qkv[:, NQ + NKV:], self.cache, self.batch, self.rope,
                              err=self.err)
        ib.paged4_attention(self.attn, self.q, self.cache, self.batch, self.ws, err=self.err)
        torch.matmul(self.attn.float().view(-1, NQ * D), self.out_w, out=self.logits)
        ib.verify_drafts(self.out, self.accepted, self.logits, self.tokens, self.q_start, self.u, self.vws,
                         temperature=self.temperature, kv_len=self.kv_len, kept=self.lens, err=self.err)
        # the next step: the token that was drawn, then guesses (the greedy ones of this step's rows)
        last = self.out.gather(0, (self.q_start[:-1] + self.accepted).long())
        guess = self.logits.argmax(-1).to(torch.int32).view(N, DRAFTS + 1)
        guess[:, 0] = last
        self.tokens.copy_(guess.view(-1))
        self.u.mul_(7.77).frac_()

    def state(self):
        return [x.clone() for x in (self.out, self.accepted, self.lens, self.kv_len, self.slots, self.positions, self.attn,
                                    self.kc, self.vc, self.scales, *self.tables.tensors)]


def test_steps(torch):
    m = Model(torch, 1)
    lens = [0] * N
    for _ in range(20):
        tokens, fed = m.tokens.clone(), m.u.clone()
        m.step()
        torch.cuda.synchronize()
        assert int(m.err) == 0
        starts, kv = m.q_start.tolist(), m.kv_len.tolist()
        assert starts == [i * (DRAFTS + 1) for i in range(N + 1)] and kv == [x + DRAFTS + 1 for x in lens]
        table, held = m.tables.tensors[0].tolist(), m.tables.tensors[1].tolist()
        assert held == [-(-x // PAGE) for x in kv]
        flat = [p for t, h in zip(table, held) for p in t[:h]]
        assert len(set(flat)) == len(flat) and all(0 <= p < PAGES for p in flat)
        for s in range(N):
            for i in range(DRAFTS + 1):
                p = lens[s] + i
                assert int(m.positions[starts[s] + i]) == p
                assert int(m.slots[starts[s] + i]) == table[s][p // PAGE] * PAGE + p % PAGE
        # the rows as they lie in the slots: within half a step of what was appended
        case = ref4.Case4(torch, [(DRAFTS + 1, x) for x in kv], NQ, NKV, D, PAGE)
        kw, vw = ref4.split_words(m.scales)
        case.kc, case.vc, case.pages, case.q, case.out = m.kc, m.vc, table, m.q, m.attn
        case.set_words(kw, vw)
        page, at = m.slots.long() // PAGE, m.slots.long() % PAGE
        new_v = m.embed[tokens.long()].view(-1, NQ + 2 * NKV, D)[:, NQ + NKV:].double()
        step = torch.ldexp((8 + ((vw >> 4) & 7)).double(), ((vw >> 7) & 255) - 130)[page, :, at]
        assert bool(((case.v[page, :, at] - new_v).abs() <= 0.5001 * step[..., None]).all())
        ref.check_attention(case, lse=False)
        # drafts: the greedy ones stand as far as they are the largest logits; what is kept
        best = m.logits.argmax(-1).tolist()
        for s in (0, 3):
            a = starts[s]
            n = 0
            while n < DRAFTS and int(tokens[a + n + 1]) == best[a + n]:
                n += 1
            assert int(m.accepted[s]) == n
            assert m.out[a:a + DRAFTS + 1].tolist() == best[a:a + n + 1] + [-1] * (DRAFTS - n)
        acc = m.accepted.tolist()
        assert m.lens.tolist() == [x - DRAFTS + n for x, n in zip(kv, acc)]
        lens = m.lens.tolist()
        assert not bool((fed == m.u).all())


def test_steps_as_a_graph(torch):
    one, two = Model(torch, 2), Model(torch, 2)
    start = two.state(), two.tokens.clone(), two.u.clone()
    two.step()  # what libraries load at a first call, outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two.step()
    for x, y in zip((two.out, two.accepted, two.lens, two.kv_len, two.slots, two.positions, two.attn, two.kc, two.vc,
                     two.scales, *two.tables.tensors), start[0]):
        x.copy_(y)
    two.tokens.copy_(start[1])
    two.u.copy_(start[2])
    for _ in range(40):
        one.step()
        graph.replay()
        torch.cuda.synchronize()
        assert int(one.err) == 0 and int(two.err) == 0
        assert all(bool((a == b).all()) for a, b in zip(one.state(), two.state()))
    assert int(one.lens.min()) > 2 * PAGE


def test_forked_pages(torch):
    """A page copied in its codes and scale words is the same page to a sequence
    that holds the copy."""
    case = ref4.Case4(torch, [(3, 75), (2, 40)], 8, 2, 128, 16, seed=6, hide=True)
    ws = ref.new_workspace(torch)
    ib.paged4_attention(case.out, case.q, case.cache(), case.batch(), ws, lse=case.lse, err=case.err)
    out, lse = case.out.clone(), case.lse.clone()
    n = case.kc.shape[0]
    codes = torch.zeros(2, 2 * n, *case.kc.shape[1:], dtype=torch.uint8, device="cuda")
    codes[0, :n], codes[1, :n] = case.kc, case.vc
    words = torch.zeros(1, 2 * n, *case.scales.shape[1:], dtype=torch.int32, device="cuda")
    words[0, :n] = case.scales
    order = list(range(n, 2 * n))[::-1]
    ib.copy_pages(codes, list(range(n)), order)
    ib.copy_pages(words, list(range(n)), order)
    codes[:, :n], words[:, :n] = 0, -1
    table = torch.tensor(order, dtype=torch.int32, device="cuda")[case.table.long().clamp(0, n - 1)].contiguous()
    batch = ib.RaggedBatch(case.q_start, case.kv_len, table, case.rows, case.max_q)
    case.out.fill_(7)
    ib.paged4_attention(case.out, case.q, ib.PagedCache4(codes[0], codes[1], words[0], case.dtype), batch, ws, lse=case.lse,
                        err=case.err)
    torch.cuda.synchronize()
    assert int(case.err) == 0 and bool((out == case.out).all()) and bool((lse == case.lse).all())


def test_models_on_streams_of_their_own(torch):
    """Two models' steps at once, each on its stream with its workspaces, are
    what they are one after the other."""
    alone = []
    for seed in (2, 3):
        m = Model(torch, seed)
        for _ in range(6):
            m.step()
        torch.cuda.synchronize()
        assert int(m.err) in (0, 1 << 5)
        alone.append(m.state())
    both, streams = [Model(torch, seed) for seed in (2, 3)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(6):
        for m, stream in zip(both, streams):
            with torch.cuda.stream(stream):
                m.step()
    torch.cuda.synchronize()
    for m, want in zip(both, alone):
        for x, y in zip(m.state(), want):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
