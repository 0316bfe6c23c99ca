"""paged4_attention against 64 bits over what the 4-bit pages stand for
(paged_reference.check_attention has the bounds: the codes' values are exact
in the kernels, so they are those of 16-bit pages)."""
import math

import pytest

import infernt_b200 as ib
import paged4_reference as ref4
import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def workspace(torch):
    return ref.new_workspace(torch)


def run(torch, case, workspace, window=0, sinks=0, scale=0.0, lse=True):
    ib.paged4_attention(case.out, case.q, case.cache(), case.batch(), workspace, window=window, sinks=sinks, scale=scale,
                        lse=case.lse if lse else None, err=case.err)
    torch.cuda.synchronize()
    assert int(case.err) == 0
    assert not bool(workspace[:2048].any())  # tickets


# sequences (new tokens, length); the items' rows are new x nq / nkv: one to four blocks of 8, several items, chunks
SHAPES = [
    ([(1, 1)], 4, 1, 64, 16),
    ([(1, 37)], 32, 4, 64, 16),
    ([(1, 300), (1, 1), (1, 129), (1, 128)], 8, 8, 128, 32),
    ([(2, 2), (2, 77), (2, 640)], 8, 2, 128, 24),
    ([(3, 900), (1, 513), (4, 4)], 10, 2, 64, 100),
    ([(5, 700), (5, 5), (5, 1025)], 32, 8, 128, 16),
    ([(7, 333), (1, 40)], 24, 3, 64, 1),
    ([(16, 200), (13, 900)], 16, 4, 128, 8),
    ([(1, 260)], 128, 1, 64, 64),
    ([(1, 450), (2, 260)], 32, 1, 128, 3),
    ([(17, 300), (1, 700), (3, 64)], 16, 4, 64, 32),
    ([(40, 40), (64, 333), (1, 90)], 8, 4, 128, 24),
    ([(130, 400), (33, 1000)], 12, 3, 128, 1),
    ([(300, 301)], 20, 4, 64, 7),
    ([(0, 50), (1, 20), (0, 0), (2, 9)], 8, 2, 64, 16),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_shapes(torch, workspace, shape, dtype):
    seqs, nq, nkv, D, page = SHAPES[shape]
    case = ref4.Case4(torch, seqs, nq, nkv, D, page, dtype, seed=shape, spare_rows=2, hide=True, q_scale=1.5)
    run(torch, case, workspace)
    ref.check_attention(case)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [8, 9, 16, 17, 24, 25, 32, 33, 40, 48, 49, 64, 65])
def test_rows_at_the_items_borders(torch, workspace, rows, D):
    """Query rows that fill one to four blocks of eight, of one item or two, and
    one more; alone and beside shorter and longer sequences."""
    for seqs in ([(rows, 500), (rows, rows)], [(rows, 700), (1, 300), (0, 9), (3, 3), (100, 400)]):
        case = ref4.Case4(torch, seqs, 2, 2, D, 16, "bf16" if rows % 2 else "fp16", seed=rows, spare_rows=1, hide=True)
        run(torch, case, workspace)
        ref.check_attention(case)


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 2), (64, 0), (100, 4), (127, 130), (1000, 1), (5000, 3)])
@pytest.mark.parametrize("seqs", [[(1, 700), (1, 130)], [(5, 640), (2, 90)], [(20, 1500)], [(100, 900), (1, 400)]])
def test_windows(torch, workspace, seqs, window, sinks):
    case = ref4.Case4(torch, seqs, 8, 2, 64 if window % 2 else 128, 24, "bf16" if sinks % 2 else "fp16", seed=window,
                      hide=True)
    run(torch, case, workspace, window, sinks)
    ref.check_attention(case, window, sinks, rows=range(0, 100, 7))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("seqs,nq,nkv,D", [([(1, 20000)], 4, 1, 128), ([(6, 9000), (1, 12000)], 8, 2, 64),
                                           ([(2, 30011)], 8, 1, 128), ([(90, 6000)], 8, 2, 128)])
def test_long_sequences_are_split(torch, workspace, seqs, nq, nkv, D, dtype):
    case = ref4.Case4(torch, seqs, nq, nkv, D, 32, dtype, seed=3)
    run(torch, case, workspace, scale=0.05)
    ref.check_attention(case, scale=0.05, rows=range(0, 90, 11))


def test_rows_before_the_first_position_see_nothing(torch, workspace):
    for n in (5, 30):
        case = ref4.Case4(torch, [(n, 3), (n, n + 1)], 8, 4, 64, 16, seed=n)
        run(torch, case, workspace)
        ref.check_attention(case)


@pytest.mark.parametrize("n", [1, 4, 9, 70])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scales_of_every_size(torch, workspace, n, dtype):
    """Vectors of zeros, of the least and of the largest values side by side:
    the weights' reference follows the values, the sum of weights does not
    leave FP32.  The bound is relative to the largest value that is seen."""
    top = 13 if dtype == "fp16" else 100

    def stretch(k, v):
        at = torch.arange(v.shape[0] * v.shape[2], device="cuda").view(v.shape[0], 1, v.shape[2], 1)
        power = torch.tensor([-30.0, 0.0, float(top), -5.0, 3.0], device="cuda").double()[at % 5]
        return k, torch.where(at % 7 == 0, 0.0, v * 2.0 ** power)

    case = ref4.Case4(torch, [(n, 260), (n, n)], 8, 2, 64, 16, dtype, stretch=stretch, seed=n)
    run(torch, case, workspace)
    ref.check_attention(case)
    small = ref4.Case4(torch, [(n, 500)], 8, 2, 128, 16, dtype, stretch=lambda k, v: (k, v * 0), seed=n)
    run(torch, small, workspace)
    ref.check_attention(small)
    assert not bool(small.out[:n].any())


@pytest.mark.parametrize("n", [1, 3, 12, 40])
def test_vectors_of_nan(torch, workspace, n):
    """A K vector of NaN: the rows that see it are NaN, out and lse; a V vector:
    out alone.  Rows that do not see it are as if it were not there."""
    D, G, L = 128, 4, 300
    for which in (0, 1):
        case = ref4.Case4(torch, [(n, L), (n, L - 60)], 2 * G, 2, D, 16, seed=n + which, hide=True)
        bad = [5, L - n + n // 2]  # seen by all rows of the first sequence; by some
        for p in bad[1:] if n > 1 else bad[:1]:
            w = [x.clone() for x in case.words]
            w[which][case.pages[0][p // 16], 1, p % 16] = ref4.NONE
            plain = ref4.Case4(torch, [(n, L), (n, L - 60)], 2 * G, 2, D, 16, seed=n + which, hide=True)
            case.set_words(*w)
            run(torch, case, workspace)
            run(torch, plain, workspace)
            ref.check_attention(plain)
            for i in range(n):
                sees = p <= L - n + i
                got, lse = case.out[i].view(2, G, D), case.lse[i].view(2, G)
                assert bool(torch.isnan(got[1]).all()) == sees and not bool(torch.isnan(got[0]).any())
                assert bool(torch.isnan(lse[1]).all()) == (sees and which == 0)
                if not sees:
                    assert bool((case.out[i] == plain.out[i]).all())
            assert bool((case.out[n:] == plain.out[n:]).all())


@pytest.mark.parametrize("n,length", [(1, 300), (1, 30000), (3, 700), (5, 20000), (40, 700), (40, 9000)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_query_rows_that_are_not_finite(torch, workspace, n, length, what):
    """A NaN or an infinity in a head's row (an infinity in all of it, so that
    every score is one or NaN): that row's out and lse are NaN, whether its item
    is split or not, and all others as without it."""
    case, plain = (ref4.Case4(torch, [(n, length), (n, n + 64)], 8, 2, 128, 16, "fp16", seed=n, hide=True) for _ in range(2))
    r = n // 2
    case.q[r, 1, 5] = what
    case.q[r, 6] = what
    run(torch, plain, workspace)
    run(torch, case, workspace)
    bad = torch.zeros(case.rows, 8, dtype=torch.bool, device="cuda")
    bad[r, 1] = bad[r, 6] = True
    assert bool(torch.isnan(case.out[bad]).all()) and bool(torch.isnan(case.lse[bad]).all())
    case.q.copy_(plain.q)
    case.out[bad], case.lse[bad] = plain.out[bad], plain.lse[bad]
    ref.check_attention(case, rows=range(0, n, 7))


@pytest.mark.parametrize("n", [1, 6, 50])
@pytest.mark.parametrize("page", [16, 5])
def test_as_over_unpacked_pages(torch, workspace, n, page):
    """The values are numbers of the type: both kinds of pages give the same
    rows but for each kernel's half steps of the probabilities (of vmax at most
    in all) and of the result, and what scores in FP32 and weights below the
    normal numbers leave (1e-3; of lse, scores of 128 products off by 2^-24 of
    their sizes' sum, some 10, each: 1e-4)."""
    case = ref4.Case4(torch, [(n, 1000), (n, n + 70)], 8, 2, 128, page, "fp16", seed=n)
    run(torch, case, workspace)
    pools = [torch.zeros(*case.kc.shape[:3], 128, device="cuda", dtype=case.dtype) for _ in range(2)]
    wide = ib.PagedCache(*pools)
    every = torch.arange(case.kc.shape[0], dtype=torch.int32, device="cuda")
    ib.paged4_unpack(case.cache(), wide, every, every)
    assert bool((pools[0].double() == case.k).all()) and bool((pools[1].double() == case.v).all())
    out, lse = torch.zeros_like(case.out), torch.zeros_like(case.lse)
    ib.paged_attention(out, case.q, wide, case.batch(), workspace, lse=lse)
    vmax = float(case.v.abs().amax())
    assert float((out.double() - case.out.double()).abs().amax()) <= vmax * 4 * ref.HALF_STEP["fp16"] + 1e-3
    assert float((lse - case.lse).abs().amax()) <= 1e-4


def test_strides_and_no_lse(torch, workspace):
    case = ref4.Case4(torch, [(3, 200), (1, 64)], 8, 2, 64, 16, seed=1)
    wide = torch.zeros(case.rows, 20, 64, device="cuda", dtype=case.dtype)
    wide[:, 4:12] = case.q
    case.q = wide[:, 4:12]
    out = torch.full((case.rows, 16, 64), 7.0, device="cuda", dtype=case.dtype)
    case.out = out[:, 8:]
    run(torch, case, workspace, lse=False)
    ref.check_attention(case, lse=False)
    assert bool((out[:, :8] == 7).all())


@pytest.mark.parametrize("n", [1, 40])
def test_bad_pages_are_zeros(torch, workspace, n):
    case = ref4.Case4(torch, [(n, 100), (n, 64)], 4, 2, 64, 16, seed=2)
    case.table[0, 2] = case.kc.shape[0]
    case.table[1, 1] = -5
    ib.paged4_attention(case.out, case.q, case.cache(), case.batch(), workspace, lse=case.lse, err=case.err)
    torch.cuda.synchronize()
    assert int(case.err) == 8
    zero = (set(range(case.kc.shape[0])) - {p for r in case.pages for p in r}).pop()  # a spare page, as zeros
    case.k[zero], case.v[zero] = 0, 0
    case.pages[0][2] = case.pages[1][1] = zero
    ref.check_attention(case)


def test_bad_sequences_are_left(torch, workspace):
    case = ref4.Case4(torch, [(2, 30), (2, 40), (2, 20)], 4, 2, 64, 16, seed=2)
    case.kv_len[1] = 16 * case.table.shape[1] + 1
    ib.paged4_attention(case.out, case.q, case.cache(), case.batch(), workspace, lse=case.lse, err=case.err)
    torch.cuda.synchronize()
    assert int(case.err) == 16
    assert bool((case.out[2:4] == 7).all())
    case.seqs = [(2, 30), (0, 40), (2, 20)]
    ref.check_attention(case)


@pytest.mark.parametrize("n", [1, 40])
def test_a_captured_call_follows_its_lengths(torch, workspace, n):
    case = ref4.Case4(torch, [(n, 400), (n, 200)], 8, 2, 128, 32, seed=5)
    batch, cache = case.batch(), case.cache()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ib.paged4_attention(case.out, case.q, cache, batch, workspace, lse=case.lse, err=case.err)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ib.paged4_attention(case.out, case.q, cache, batch, workspace, lse=case.lse, err=case.err)
    for lens in ([400, 200], [333, 64], [64, 399]):
        case.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        case.pages[1] = case.pages[0]
        case.table[1] = case.table[0]
        case.out.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        case.seqs = [(n, lens[0]), (n, lens[1])]
        case.pages = [case.table[i].tolist() for i in range(2)]
        ref.check_attention(case)


def test_the_same_call_twice_is_the_same(torch, workspace):
    case = ref4.Case4(torch, [(1, 9000), (5, 3000), (70, 2000), (1, 64)], 8, 2, 128, 16, seed=9)
    run(torch, case, workspace)
    out, lse = case.out.clone(), case.lse.clone()
    for _ in range(5):
        run(torch, case, workspace)
        assert bool((out == case.out).all()) and bool((lse == case.lse).all())


def test_offsets_past_32_bits(torch, workspace):
    """Codes and values of a pool's last pages lie past 2^32 bytes."""
    page, nkv, D = 4096, 4, 128
    pages = (1 << 32) // (page * nkv * D // 2) + 2
    k = torch.zeros(pages, nkv, page, D // 2, dtype=torch.uint8, device="cuda")
    v = torch.zeros_like(k)
    scales = torch.zeros(pages, nkv, page, dtype=torch.int32, device="cuda")
    small = ref4.Case4(torch, [(3, 200)], 8, nkv, D, page, seed=4)
    at = pages - 1
    k[at], v[at], scales[at] = small.kc[small.pages[0][0]], small.vc[small.pages[0][0]], small.scales[small.pages[0][0]]
    run(torch, small, workspace)
    out, lse = small.out.clone(), small.lse.clone()
    table = torch.full_like(small.table, at)
    batch = ib.RaggedBatch(small.q_start, small.kv_len, table, small.rows, small.max_q)
    small.out.fill_(0)
    ib.paged4_attention(small.out, small.q, ib.PagedCache4(k, v, scales, small.dtype), batch, workspace, lse=small.lse)
    torch.cuda.synchronize()
    assert bool((out == small.out).all()) and bool((lse == small.lse).all())
    assert math.isfinite(float(out.float().sum()))
