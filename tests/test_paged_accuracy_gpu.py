"""infernt_paged_attention against 64 bits with bounds that shrink with the
row's own sums (paged_bounds), where the cache is long, items are split, tiles
end at a window's border, and what was taken out of V could be missed."""
import math

import pytest

import infernt_b200 as ib
from paged_bounds import check_rows
from paged_reference import Case, new_workspace

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def ws(torch):
    return new_workspace(torch)


def run(c, ws, window=0, sinks=0, scale=0.0):
    ib.paged_attention(c.out, c.q, c.cache(), c.batch(), ws, window=window, sinks=sinks, scale=scale, lse=c.lse, err=c.err)
    c.torch.cuda.synchronize()
    assert int(c.err) == 0
    return c


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,nq,nkv,page", [(128, 8, 1, 64), (64, 8, 2, 16)])
def test_long_caches(torch, ws, D, nq, nkv, page, dtype):
    c = run(Case(torch, [(1, 70001), (20, 66000), (300, 30000)], nq, nkv, D, page, dtype), ws)
    check_rows(c, rows=[0, 1, 19, 63, 64, 255, 256, 299])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs", [[(1, 9000)], [(2, 9000)], [(90, 9000)], [(1, 1 + 97 * i) for i in range(70)],
                                  [(700, 3000)], [(65, 4000), (300, 700), (1, 5000), (9, 2000)]])
def test_split_items(torch, ws, seqs, D):
    c = run(Case(torch, seqs, 4, 1, D, 64, fill=math.nan), ws)
    check_rows(c, rows=[0, 1, 8, 31, 63, 64, 88, 89, 255, 256, 299, 699])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(300, 5), (1000, 0), (64, 300), (2000, 1)])
def test_windows(torch, ws, window, sinks, D, dtype):
    c = run(Case(torch, [(700, 6000), (1, 5001), (513, 513), (1, 9), (30, 3000)], 8, 2, D, 32, dtype, fill=math.inf),
            ws, window, sinks)
    check_rows(c, window, sinks, rows=[0, 1, 29, 31, 63, 64, 255, 256, 300, 511, 512, 600, 699])


@pytest.mark.parametrize("page", [1, 8, 24, 48, 64, 100, 256])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(torch, ws, page, D):
    c = run(Case(torch, [(1, 3333), (400, 2700), (1, 5), (7, 800)], 8, 2, D, page, fill=math.nan), ws)
    check_rows(c, rows=[0, 1, 6, 63, 64, 127, 128, 255, 256, 399])


@pytest.mark.parametrize("nq,nkv", [(1, 1), (3, 1), (12, 1), (32, 4), (128, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_head_layouts(torch, ws, nq, nkv, dtype):
    c = run(Case(torch, [(1, 2000), (70, 1500), (3, 40), (1, 1)], nq, nkv, 128, 16, dtype, fill=math.nan), ws)
    check_rows(c, rows=[0, 1, 2, 31, 32, 64, 69])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("q_scale,scale", [(4.0, 0.0), (8.0, 0.0), (1.0, 0.5), (1.0, 0.004), (30.0, 0.0)])
def test_peaked_and_flat_scores(torch, ws, q_scale, scale, dtype):
    for D in (64, 128):
        c = run(Case(torch, [(1, 4000), (300, 2000), (5, 700)], 8, 2, D, 32, dtype, q_scale=q_scale), ws, scale=scale)
        check_rows(c, scale=scale, rows=[0, 1, 4, 63, 64, 150, 255, 256, 299])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rise", [0.5, 3.0, 20.0])
def test_scores_that_rise_along_the_cache(torch, ws, rise, dtype):
    """Every tile's largest score passes the last one's by `rise` in base 2, so
    that references move (or do not), and tiles are computed twice."""
    for D in (64, 128):
        c = Case(torch, [(1, 1500), (200, 1500), (70, 3000)], 4, 2, D, 64, dtype)
        c.q[..., 0] = 1.0
        for pages, (_, n) in zip(c.pages, c.seqs):
            for t in range(-(-n // 64)):
                c.k[pages[t], :, :, 0] = t * rise * math.sqrt(D) * math.log(2.0)
        run(c, ws)
        check_rows(c, rows=[0, 1, 63, 64, 69, 127, 128, 199])


def test_every_sequence_a_chunk_of_its_own_length(torch, ws):
    c = run(Case(torch, [(64 + 3 * i, 200 + 91 * i) for i in range(30)], 4, 1, 64, 16, fill=math.nan), ws)
    check_rows(c, rows=[0, 31, 63, 64, 100, 140])
