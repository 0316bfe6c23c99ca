"""infernt_paged_attention over caches whose values are not finite: a value
reaches the rows that see it, in its column, as in the formula, and no other;
what it costs does not grow with the cache."""
import math
import random

import pytest

import infernt_b200 as ib
from paged_reference import HALF_STEP, Case, attention_row, check_attention, new_workspace

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def ws(torch):
    return new_workspace(torch)


def run(c, ws, window=0, sinks=0):
    ib.paged_attention(c.out, c.q, c.cache(), c.batch(), ws, window=window, sinks=sinks, lse=c.lse, err=c.err)
    c.torch.cuda.synchronize()
    assert int(c.err) == 0
    return c


def put(c, s, at, head, column, value):
    c.v[c.pages[s][at // c.page], head, at % c.page, column] = value


def check_classes(c, window, sinks, rows):
    """Finite results as paged_reference.check_attention holds them (the
    largest finite value for the largest one); infinities with their sign and
    NaN where the formula has them.  The smallest weight of these tests is far
    above 2^-29 of the largest, so that no visible value meets a 0."""
    torch, u, sc = c.torch, HALF_STEP[c.kind], 1.0 / math.sqrt(c.D)
    for s, (n, length) in enumerate(c.seqs):
        k, v = c.dense(c.k, s), c.dense(c.v, s)
        vmax = float(v[torch.isfinite(v)].abs().amax())
        for i in (x for x in rows if x < n):
            r, pos = c.starts[s] + i, length - n + i
            want, lse, big, _ = attention_row(c, c.q[r], k, v, pos, window, sinks, sc)
            got = c.out[r].double()
            ok = torch.isfinite(want)
            assert bool((torch.isfinite(got) == ok).all()), (s, i)
            assert bool((torch.isnan(got) == torch.isnan(want)).all()), (s, i)
            assert bool((got[~ok & ~torch.isnan(want)] == want[~ok & ~torch.isnan(want)]).all()), (s, i)
            es = (c.D + 2) * 2.0 ** -23 * sc * big
            tol = vmax * (2 * u + 4 * es + (pos + 65) * 2.0 ** -22)
            assert float((got - want)[ok].abs().amax()) <= tol, (s, i)
            far = (c.lse[r].double() - lse).abs()
            assert bool((far <= es + (pos + 9) * 2.0 ** -22 + 2.0 ** -21 * lse.abs()).all()), (s, i)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,nq,nkv,page", [(64, 4, 2, 16), (128, 8, 2, 32), (64, 2, 2, 24), (128, 3, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3), (64, 0), (7, 70)])
def test_scattered_values(torch, ws, window, sinks, D, nq, nkv, page, dtype):
    """Around every border: among the new tokens, at the windows' first keys,
    among the sinks, behind them, in whole tiles."""
    rng = random.Random(D + window)
    c = Case(torch, [(1, 500), (7, 300), (20, 90), (64, 64), (100, 400), (300, 900), (5, 1200)], nq, nkv, D, page, dtype)
    for s, (n, length) in enumerate(c.seqs):
        first = length - n
        for at in [first, length - 1, rng.randrange(first, length), rng.randrange(first, length), sinks, sinks - 1,
                   first - window, first - window + 1, length - window, rng.randrange(length)]:
            if 0 <= at < length:
                put(c, s, at, rng.randrange(nkv), rng.randrange(D), rng.choice([INF, -INF, NAN, INF, -INF]))
    run(c, ws, window, sinks)
    check_classes(c, window, sinks, rows=list(range(0, 24)) + [63, 64, 65, 98, 99, 127, 128, 200, 255, 256, 298, 299])


@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs", [[(1, 70001)], [(300, 20000), (1, 9000)], [(40, 30000)], [(1, 3000)] * 70])
def test_a_value_that_all_rows_see(torch, ws, seqs, D, value):
    """Position 3 of sequence 0: every row of the KV head sees it, in its
    column.  All other columns, heads and sequences have the same bits as
    without it."""
    c = Case(torch, seqs, 4, 2, D, 64)
    run(c, ws)
    before, lse = c.out.clone(), c.lse.clone()
    put(c, 0, 3, 1, 9, value)
    run(c, ws)
    n = seqs[0][0]
    assert not bool(torch.isfinite(c.out[:n, 2:, 9].float()).any())
    c.out[:n, 2:, 9] = before[:n, 2:, 9]
    assert bool((c.out == before).all()) and bool((c.lse == lse).all())


@pytest.mark.parametrize("new", [2, 33, 257])
def test_the_last_token_of_a_long_cache(torch, ws, new):
    """Hidden from all rows but the last, over 60000 positions: the others
    keep the bits that they have without it."""
    n = 60000
    c = Case(torch, [(new, n), (1, 700)], 4, 1, 128, 64)
    run(c, ws)
    before, lse = c.out.clone(), c.lse.clone()
    for column, value in ((3, INF), (4, -INF), (5, NAN)):
        put(c, 0, n - 1, 0, column, value)
    run(c, ws)
    last = c.out[new - 1].float()
    assert bool((last[:, 3] == INF).all()) and bool((last[:, 4] == -INF).all()) and bool(torch.isnan(last[:, 5]).all())
    c.out[new - 1, :, 3:6] = before[new - 1, :, 3:6]
    assert bool((c.out == before).all()) and bool((c.lse == lse).all())


def test_a_window_moves_past_the_value(torch, ws):
    n, window = 9000, 500
    c = Case(torch, [(1200, n)], 4, 1, 64, 64)
    at = n - 900
    put(c, 0, at, 0, 0, INF)
    run(c, ws, window)
    shown = torch.tensor([at <= n - 1200 + i < at + window for i in range(1200)], device="cuda")
    assert bool((c.out[shown][..., 0] == INF).all())
    assert bool(torch.isfinite(c.out[~shown].float()).all()) and bool(torch.isfinite(c.out[..., 1:].float()).all())
    check_attention(c, window, rows=[0, 299, 800, 801, 850, 1199])  # (its tolerance is infinite for rows that see it)


def test_the_time_does_not_depend_on_the_values(torch, ws):
    """4096 tokens at 12288 positions with an infinite value at position 3,
    then with one among the new tokens: within twice the finite call's time."""
    c = Case(torch, [(4096, 12288)], 8, 2, 128, 32)

    def time():
        best = INF
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ib.paged_attention(c.out, c.q, c.cache(), c.batch(), ws, err=c.err)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    finite = time()
    put(c, 0, 3, 0, 0, INF)
    assert time() <= 2 * finite
    put(c, 0, 12288 - 2000, 1, 0, NAN)
    assert time() <= 2 * finite
    assert int(c.err) == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs", [[(1, 300), (5, 200)], [(90, 300)], [(90, 300), (1, 400)]])
def test_the_largest_values_of_bf16(torch, ws, seqs, D):
    """Values near 2^120, scores that rise along the cache by up to 7 in base 2
    within a tile: no sum passes FP32's range on the way to a finite result."""
    c = Case(torch, seqs, 2, 1, D, 16)
    c.v.copy_(torch.randn(c.v.shape, device="cuda").sign() * (1.0 + torch.rand(c.v.shape, device="cuda")) * 2.0 ** 120)
    c.q.zero_()
    c.q[:, :, 0] = 1.0
    for pages, (_, n) in zip(c.pages, c.seqs):
        for p in range(n):
            c.k[pages[p // 16], :, p % 16, 0] = math.sqrt(D) * math.log(2.0) * (7.0 if p >= 64 else 0.0)
    run(c, ws)
    check_attention(c)
