"""verify_drafts against a 64-bit restatement, row by row."""
import math
import random

import pytest

import infernt_b200 as ib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


class Step:
    """Drafts of `counts` tokens a sequence and the target's rows."""

    def __init__(self, torch, counts, V, dtype="float32", probs=False, draft=True, temps=None, seed=0, spread=2.0,
                 ld=None, banned=True):
        self.torch, self.V, self.probs, self.counts = torch, V, probs, counts
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = len(counts)
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        rows = self.rows = starts[-1]
        self.starts = starts
        ld = ld or V
        wide = torch.zeros(max(rows, 1), ld, device="cuda")
        wide.normal_(generator=g).mul_(spread)
        if banned and V > 8:
            wide[:, 3:V:5] = -math.inf
        self.temps = temps if temps is None else [temps[i % len(temps)] for i in range(n)]
        self.temperature = None if temps is None else torch.tensor(self.temps, device="cuda")
        warm = torch.ones(max(rows, 1), 1, device="cuda")
        for i in range(n):
            t = 1.0 if temps is None else self.temps[i]
            warm[starts[i]:starts[i + 1]] = t if t > 0 else 1.0
        q = torch.softmax((wide[:, :V] + torch.empty_like(wide[:, :V]).normal_(generator=g) * 0.5) / warm, -1)
        picked = torch.multinomial(q, 1, generator=g).squeeze(1)
        if probs:
            wide[:, :V] = torch.softmax(wide[:, :V] / warm, -1)
        wide = wide.to(getattr(torch, dtype))
        best = wide[:, :V].double().argmax(-1)
        greedy = torch.rand(picked.shape, generator=g, device="cuda") < 0.6
        tokens = torch.where(greedy, best, picked) if self.temps and min(self.temps) <= 0 else picked
        self.tokens = torch.cat((tokens[:1] * 0, tokens[:-1])).to(torch.int32)
        self.target = wide[:rows, :V] if rows else wide[:0, :V]
        self.draft = q[:rows].contiguous() if draft else None
        self.u = torch.rand(max(rows, 1), generator=g, device="cuda")
        self.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.out = torch.full((max(rows, 1),), 77, dtype=torch.int32, device="cuda")
        self.accepted = torch.full((n,), 77, dtype=torch.int32, device="cuda")
        self.kv_len = torch.arange(100, 100 + n, dtype=torch.int32, device="cuda")
        self.kept = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.workspace = torch.full((ib.verify_drafts_workspace_bytes(rows, n),), 255, dtype=torch.uint8, device="cuda")

    def run(self, **kw):
        ib.verify_drafts(self.out, self.accepted, self.target, self.tokens, self.q_start, self.u, self.workspace,
                         draft_probs=self.draft, temperature=self.temperature, probabilities=self.probs,
                         kv_len=self.kv_len, kept=self.kept, err=self.err, **kw)
        self.torch.cuda.synchronize()

    def row(self, r, t):
        """(p in 64 bits, the row's largest element's lowest index, whether the row is a distribution)"""
        torch, x = self.torch, self.target[r].double()
        number = x[~torch.isnan(x)]
        best = int((x == number.amax()).nonzero()[0]) if number.numel() and number.amax() > -math.inf else 0
        if self.probs:
            fine = bool(((x >= 0) & (x < math.inf)).all()) and bool((x > 0).any())
            return x, best, fine
        fine = bool((x < math.inf).all()) and bool((x > -math.inf).any())
        if t <= 0 or not fine:
            return x, best, fine
        y = (x - x.amax()) / float(torch.tensor(t, dtype=torch.float32))
        e = torch.where(x == -math.inf, 0.0, y.exp())
        return e / e.sum(), best, fine

    def want(self):
        """(out, accepted, bits, near) of every sequence; near: a comparison is so close that 32 bits may turn it"""
        torch, got = self.torch, []
        u = self.u.double().nan_to_num(0.0).clamp(0.0, 1 - 2.0 ** -24)
        for s, n in enumerate(self.counts):
            a, t, bits, near = self.starts[s], 1.0 if self.temps is None else self.temps[s], 0, False
            out, acc = [], 0
            for i in range(n):
                r, last = a + i, i == n - 1
                d = None if last else int(self.tokens[r + 1])
                known = d is not None and 0 <= d < self.V
                p, best, fine = self.row(r, t)
                if d is not None and not known:
                    bits |= 4
                if t <= 0:
                    if fine and known and d == best:
                        out.append(d)
                        continue
                    bits |= 0 if fine else 64
                    out.append(best)
                    break
                bad_at = known and self.probs and not (0 <= float(p[d]) < math.inf)
                if known and not bad_at and (fine or self.probs):
                    q = 1.0 if self.draft is None else float(self.draft[r, d])
                    x, y = float(u[r]) * q, float(p[d])
                    near |= abs(x - y) <= 1e-5 * max(x, y)
                    if x < y:
                        out.append(d)
                        continue
                if not fine:
                    bits |= 64
                    out.append(best)
                    break
                w = p
                if known:
                    if self.draft is None:
                        w = p.clone()
                        w[d] = 0
                    else:
                        q = self.draft[r].double()
                        w = (p - torch.where(q.isfinite(), q, math.inf)).clamp(min=0)
                    if not bool((w > 0).any()):
                        w = p
                c = w.cumsum(0)
                goal = float(u[a + n - 1]) * float(c[-1])
                past = ((c > goal) & (w > 0)).nonzero()
                token = int(past[0]) if past.numel() else int((w > 0).nonzero()[-1])
                near |= bool(((c - goal).abs() <= 1e-11 * c[-1])[max(0, token - 1):token + 1].any()) and goal > 0
                out.append(token)
                break
            acc = max(0, len(out) - 1)
            got.append((out + [-1] * (n - len(out)), acc, bits, near))
        return got

    def check(self, most_near=1):
        bits = nears = 0
        for s, (out, acc, b, near) in enumerate(self.want()):
            bits |= b
            nears += near
            if near:
                continue
            n, a = self.counts[s], self.starts[s]
            assert self.out[a:a + n].tolist() == out, (s, self.out[a:a + n].tolist(), out)
            assert int(self.accepted[s]) == acc
            assert int(self.kept[s]) == int(self.kv_len[s]) - max(0, n - 1 - acc)
        assert nears <= most_near and int(self.err) == bits
        return bits


COUNTS = [5, 1, 2, 9, 3, 0, 4, 8, 1, 6]


@pytest.mark.parametrize("V", [1, 2, 7, 127, 128, 129, 1000, 4099, 8192, 16385, 32000, 50257])
@pytest.mark.parametrize("draft", [True, False])
def test_logits(torch, V, draft):
    s = Step(torch, COUNTS, V, draft=draft, seed=V)
    s.run()
    assert s.check() == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("V", [130, 5003])
@pytest.mark.parametrize("temps", [[0.0], [1.0, 0.0, 0.3, 2.5], [0.02, 50.0]])
def test_temperatures_and_types(torch, dtype, V, temps):
    s = Step(torch, COUNTS, V, dtype=dtype, temps=temps, seed=int(10 * sum(temps)))
    s.run()
    assert s.check(2) == 0


@pytest.mark.parametrize("V", [1, 33, 4100, 40000])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("temps", [None, [1.0, 0.0]])
def test_probabilities(torch, V, draft, temps):
    s = Step(torch, COUNTS, V, probs=True, draft=draft, temps=temps, seed=V)
    s.run()
    assert s.check() == 0


@pytest.mark.parametrize("V", [152064, 300007])
def test_large_vocabularies(torch, V):
    s = Step(torch, [3, 1, 4], V, seed=1)
    s.run()
    assert s.check() == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("ld", [1003, 1005, 1008])
def test_rows_that_start_anywhere(torch, dtype, ld):
    s = Step(torch, COUNTS, 1001, dtype=dtype, ld=ld, seed=ld)
    if ld == 1005:  # not even the first row on 16 bytes
        s.target = s.target.new_zeros(s.rows * ld + 8)[1:1 + s.rows * ld].view(s.rows, ld)[:, :1001].copy_(s.target)
    s.run()
    assert s.check() == 0


@pytest.mark.parametrize("n", [1, 300, 2000])
def test_many_sequences(torch, n):
    r = random.Random(n)
    s = Step(torch, [r.randint(0, 6) for _ in range(n)], 97, seed=n, temps=[1.0, 0.7, 0.0])
    s.run()
    assert s.check(3) == 0


def test_many_drafts(torch):
    s = Step(torch, [200, 33], 64, spread=0.1, temps=[30.0, 1.0], seed=2)
    s.run()
    assert s.check(3) == 0


def test_every_draft_is_taken_or_none(torch):
    s = Step(torch, [4, 4, 4, 4], 500, seed=3)
    s.u[:8] = 0.0  # u q = 0 is below every probability above 0
    s.u[8:] = 1.0  # the largest below 1
    s.draft[12:] = 1.0  # of a draft that claimed certainty
    s.run()
    assert s.check() == 0
    assert s.accepted[:2].tolist() == [3, 3]


def test_the_draft_is_the_target(torch):
    """p = q: everything is taken (but for the last bit); where a draft is not,
    and nothing is left of p - q, the token is of p."""
    s = Step(torch, [3] * 50, 300, probs=True, seed=4, banned=False)
    s.draft = s.target.clone()
    s.u.mul_(0.999)
    s.run()
    assert s.check() == 0 and bool((s.accepted == 2).all())
    s.draft[:, 150:] *= 1.5  # above p there, p itself elsewhere
    s.draft[:, :150] = s.target[:, :150]
    s.u[:] = 0.9
    s.run()
    s.check()


def test_draws_are_distributed_as_the_target(torch):
    """Speculative sampling leaves the target's distribution: 40 000 first tokens, chi-square over 12 of them
    (the limit is the 1 - 10^-7 quantile of 11 degrees of freedom, 53.4)."""
    n, V = 40000, 12
    g = torch.Generator(device="cuda").manual_seed(8)
    logits = torch.randn(1, V, generator=g, device="cuda").repeat(2 * n, 1)
    q = torch.softmax(torch.randn(1, V, generator=g, device="cuda"), -1).repeat(2 * n, 1)
    tokens = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
    tokens[1::2] = torch.multinomial(q[:n], 1, generator=g).squeeze(1).to(torch.int32)
    out, acc = torch.zeros_like(tokens), torch.zeros(n, dtype=torch.int32, device="cuda")
    ws = torch.zeros(ib.verify_drafts_workspace_bytes(2 * n, n), dtype=torch.uint8, device="cuda")
    ib.verify_drafts(out, acc, logits, tokens, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda"),
                     torch.rand(2 * n, generator=g, device="cuda"), ws, draft_probs=q)
    seen = torch.bincount(out[::2].long(), minlength=V).double()
    want = torch.softmax(logits[0].double(), -1) * n
    assert float(((seen - want) ** 2 / want).sum()) < 53.4


def test_ties_go_to_the_lowest(torch):
    s = Step(torch, [3, 2], 5000, temps=[0.0], seed=5, banned=False)
    s.target[:, [17, 4000, 900]] = 50.0
    s.tokens[1] = 17
    s.tokens[2] = 900
    s.run()
    assert s.out.tolist() == [17, 17, -1, 17, -1] or s.out.tolist()[:2] == [17, 17]
    assert s.check() == 0


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temp", [1.0, 0.0])
def test_rows_that_are_no_distribution(torch, probs, temp):
    s = Step(torch, [2] * 8, 300, probs=probs, temps=[temp], seed=6, banned=False)
    s.target[0, 9] = math.nan
    s.target[2, 7] = math.inf
    s.target[4] = -math.inf if not probs else 0.0
    s.target[6] = math.nan
    s.target[9, 3] = math.nan  # of the last row: reached when the draft is taken
    if probs:
        s.target[10, 5] = -0.5
    s.u[8::2] = 0.0
    s.run()
    got = s.want()
    assert int(s.err) & 64 and (not probs or temp > 0 or int(s.err) == 64)
    for i, (out, acc, _, near) in enumerate(got):
        assert near or s.out[2 * i:2 * i + 2].tolist() == out, (i, s.out[2 * i:2 * i + 2].tolist(), out)


def test_tokens_outside_the_vocabulary(torch):
    s = Step(torch, [3, 3, 3], 100, temps=[1.0, 0.0], seed=7)
    s.tokens[1], s.tokens[4], s.tokens[8] = 100, -1, 2 ** 31 - 1
    s.u[6] = 0.0
    s.run()
    assert s.check() & 4


def test_numbers_outside_their_range(torch):
    """u below 0 and NaN are 0, from 1 on the largest below 1; a draft's
    distribution that is not finite leaves no weight there."""
    s = Step(torch, [2] * 6, 200, seed=9)
    s.u[:4] = torch.tensor([-1.0, math.nan, 2.0, 1.0], device="cuda")
    s.draft[4, 50:] = math.nan
    s.draft[6, :20] = math.inf
    s.u[4] = s.u[6] = 1.0
    s.run()
    assert s.check(2) == 0


def test_bad_rows_are_left(torch):
    s = Step(torch, [2, 3, 2], 50, seed=10)
    s.q_start[2] = 100
    s.run()
    assert int(s.err) == 16 and int(s.accepted[1]) == 77 and bool((s.out[2:5] == 77).all())
    assert s.out[:2].tolist() == s.want()[0][0]


def test_no_rows(torch):
    s = Step(torch, [0, 0], 50)
    s.run()
    assert s.accepted.tolist() == [0, 0] and s.kept.tolist() == s.kv_len.tolist()


def test_captured_on_another_stream(torch):
    s = Step(torch, COUNTS, 3000, seed=11)
    other = Step(torch, COUNTS, 3000, seed=12)
    s.run()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        ib.verify_drafts(s.out, s.accepted, s.target, s.tokens, s.q_start, s.u, s.workspace, draft_probs=s.draft,
                         kv_len=s.kv_len, kept=s.kept, err=s.err)
    for x in ("tokens", "u", "target", "draft"):
        getattr(s, x).copy_(getattr(other, x))
    s.out.fill_(5)
    graph.replay()
    torch.cuda.synchronize()
    assert s.check() == 0


def test_kept_in_place(torch):
    s = Step(torch, COUNTS, 300, seed=13)
    s.run()
    want = s.kept.tolist()
    lens = s.kv_len.clone()
    ib.verify_drafts(s.out, s.accepted, s.target, s.tokens, s.q_start, s.u, s.workspace, draft_probs=s.draft, kv_len=lens,
                     kept=lens)
    assert lens.tolist() == want
