"""infernt_paged_attention against 64 bits row by row (tolerances derived in
paged_reference.check_attention): single tokens, short and long chunks, mixed
batches, head layouts, page sizes, windows with sinks, what hidden rows hold,
rows that see nothing, strides, bad device data, streams and graphs."""
import math

import pytest

import infernt_b200 as ib
from paged_reference import HALF_STEP, Case, attention_row, check_attention, new_workspace

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def ws(torch):
    return new_workspace(torch)


def run(case, ws, window=0, sinks=0, scale=0.0, stream=None, lse=True):
    ib.paged_attention(case.out, case.q, case.cache(), case.batch(), ws, window=window, sinks=sinks, scale=scale,
                       lse=case.lse if lse else None, err=case.err, stream=stream)
    case.torch.cuda.synchronize()
    return case


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 300, 1000]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("nq,nkv,D,page", [(32, 4, 64, 16), (32, 8, 128, 32)])
def test_single_tokens(torch, ws, nq, nkv, D, page, dtype):
    c = run(Case(torch, [(1, n) for n in LENGTHS], nq, nkv, D, page, dtype, fill=math.nan, spare_rows=3), ws)
    check_attention(c)
    assert int(c.err) == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("chunk,length", [(2, 2), (3, 70), (15, 15), (16, 80), (17, 200), (33, 33), (64, 130),
                                          (65, 65), (130, 300), (300, 301), (257, 1025)])
def test_chunks(torch, ws, chunk, length, dtype):
    c = run(Case(torch, [(chunk, length)], 8, 2, 128, 32, dtype, fill=math.inf, spare_rows=2), ws)
    check_attention(c)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (3, 1), (5, 1), (4, 4), (6, 2), (10, 2), (12, 1), (16, 1), (24, 1),
                                    (128, 1), (21, 3)])
def test_head_layouts(torch, ws, nq, nkv, D):
    c = run(Case(torch, [(1, 77), (9, 140), (1, 1), (40, 200)], nq, nkv, D, 16, fill=math.nan), ws)
    check_attention(c)


@pytest.mark.parametrize("page", [1, 3, 7, 8, 16, 24, 40, 64, 100, 128, 192, 256, 1000])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(torch, ws, page, D):
    c = run(Case(torch, [(1, 333), (150, 270), (1, 5)], 8, 2, D, page, fill=math.nan), ws)
    check_attention(c)
    assert int(c.err) == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (63, 0), (64, 64), (65, 1), (100, 70), (128, 200),
                                          (250, 4), (999, 5), (5000, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_windows(torch, ws, window, sinks, dtype):
    c = run(Case(torch, [(1, 1000), (1, 260), (1, 3), (200, 600), (70, 70), (5, 900)], 8, 2, 64, 16, dtype,
                 fill=math.nan), ws, window, sinks)
    check_attention(c, window, sinks)


@pytest.mark.parametrize("window,sinks", [(300, 5), (1000, 0), (40, 300)])
def test_long_windowed_chunk(torch, ws, window, sinks):
    """D = 128, a chunk over several tiles of rows; a sample of its rows."""
    c = run(Case(torch, [(700, 2000), (1, 1500), (513, 513)], 16, 4, 128, 64, fill=math.nan), ws, window, sinks)
    check_attention(c, window, sinks, rows=[0, 1, 31, 63, 64, 255, 256, 300, 511, 512, 600, 699])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [4, 8])
def test_windows_that_begin_with_a_tile(torch, ws, G, D):
    """The first key of the last rows of a block of query rows is the first of
    a tile of keys, while the first rows' windows begin in the tile before."""
    for window in (448, 449, 447, 64, 128):
        c = run(Case(torch, [(256, 2048)], 2 * G, 2, D, 64), ws, window)
        check_attention(c, window, rows=[0, 1, 31, 32, 62, 63, 64, 127, 128, 191, 255])


@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 2)])
def test_rows_that_see_nothing(torch, ws, window, sinks):
    """More new tokens than positions: the first rows have negative positions
    (a batch padded in front); no positions at all; no new tokens."""
    seqs = [(5, 3), (1, 0), (70, 1), (0, 40), (130, 64), (0, 0), (4, 4)]
    c = run(Case(torch, seqs, 8, 2, 64, 16, fill=math.nan, spare_rows=4), ws, window, sinks)
    check_attention(c, window, sinks)
    assert bool((c.out[:2] == 0).all()) and bool((c.out[5] == 0).all())
    assert int(c.err) == 0


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("chunk,length", [(6, 40), (100, 200), (300, 500)])
def test_hidden_rows_that_are_not_finite(torch, ws, chunk, length, bad):
    """Keys and values of one new token are not finite: the tokens before it
    do not see it, and it reaches those after it as in the formula."""
    c = Case(torch, [(chunk, length)], 4, 2, 128, 16)
    at = length - chunk // 2
    page, row = c.pages[0][at // 16], at % 16
    c.v[page, 0, row, 5] = bad
    c.k[page, 1, row, 7] = bad
    run(c, ws)
    first = at - (length - chunk)
    check_attention(c, rows=range(first))
    G = 2
    seen = c.out[first:chunk].float()
    assert not bool(torch.isfinite(seen[:, :G, 5]).any())        # V of KV head 0, column 5
    assert bool(torch.isfinite(seen[:, :G, :5]).all())           # its other columns
    v = c.dense(c.v, 0)
    k = c.dense(c.k, 0)
    s = torch.einsum("d,pd->p", c.q[first, G].double(), k[:at + 1, 1]) / math.sqrt(128)
    want = torch.softmax(s, 0) @ v[:at + 1, 1]
    assert bool((torch.isfinite(want) == torch.isfinite(seen[0, G])).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_scores_that_are_not_finite(torch, ws, bad):
    """One key of a KV head is not finite: every row that sees it has no
    finite result there, wherever in a tile it lies; the other head is whole."""
    for at in list(range(64, 130)) + [5, 190]:
        c = Case(torch, [(100, 300)], 4, 2, 64, 16)
        c.k[c.pages[0][at // 16], 1, at % 16] = bad
        run(c, ws)
        assert not bool(torch.isfinite(c.out[:, 2:].float()).any()), at
        assert bool(torch.isfinite(c.out[:, :2].float()).all()), at


@pytest.mark.parametrize("new", [2, 100])
def test_a_first_score_of_minus_infinity(torch, ws, new):
    """Position 0 has no weight where its score is -infinity, also in rows
    whose tile holds a hidden value that is not finite."""
    n = 150
    c = Case(torch, [(new, n)], 4, 2, 64, 16)
    c.q.abs_().add_(0.1)
    c.k[c.pages[0][0], :, 0] = -math.inf
    c.v[c.pages[0][(n - 1) // 16], :, (n - 1) % 16] = math.nan
    run(c, ws)
    k, v = c.dense(c.k, 0)[1:], c.dense(c.v, 0)[1:]
    for i in range(new - 1):
        pos = n - new + i
        out, lse, big, vmax = attention_row(c, c.q[i], k, v, pos - 1, 0, 0, 0.125)
        es = (64 + 2) * 2.0 ** -23 * 0.125 * big  # as in check_attention
        assert float((c.out[i].double() - out).abs().amax()) <= vmax * (2 * HALF_STEP["bf16"] + 4 * es +
                                                                       (pos + 65) * 2.0 ** -22), i
        far = (c.lse[i].double() - lse).abs()
        assert bool((far <= es + (pos + 9) * 2.0 ** -22 + 2.0 ** -21 * lse.abs()).all()), i
    assert bool(torch.isnan(c.out[new - 1]).all())


def test_hidden_by_a_window(torch, ws):
    """A value behind the window of the later rows of a tile, in the window of
    the earlier ones."""
    c = Case(torch, [(200, 400)], 4, 1, 64, 16)
    at = 250
    c.v[c.pages[0][at // 16], 0, at % 16] = math.nan
    run(c, ws, 64, 2)
    hidden = [i for i in range(200) if not (200 + i - 64 < at <= 200 + i)]
    check_attention(c, 64, 2, rows=hidden)
    shown = [i for i in range(200) if i not in set(hidden)]
    assert bool(torch.isnan(c.out[shown]).all())


@pytest.mark.parametrize("q_scale,scale", [(8.0, 0.0), (1.0, 0.5), (1.0, 0.004), (30.0, 0.0)])
def test_peaked_scores(torch, ws, q_scale, scale):
    c = run(Case(torch, [(1, 900), (100, 700)], 8, 2, 128, 32, q_scale=q_scale), ws, scale=scale)
    check_attention(c, scale=scale)


def test_strided_rows_and_no_lse(torch, ws):
    """q a slice of stacked rows, out with rows further apart."""
    c = Case(torch, [(1, 90), (60, 100), (1, 64)], 8, 2, 64, 16)
    stacked = torch.randn(c.rows, 12, 64, device="cuda").to(c.dtype)
    wide = torch.full((c.rows, 11, 64), 3.0, device="cuda").to(c.dtype)
    stacked[:, :8] = c.q
    c.q, c.out = stacked[:, :8], wide[:, :8]
    run(c, ws, lse=False)
    check_attention(c, lse=False)
    assert bool((wide[:, 8:] == 3).all()) and bool((c.lse == 7).all())


def test_mixed_step(torch, ws):
    """Decodes, short drafts and two prompts' chunks in one call."""
    seqs = [(1, 900), (1, 33), (5, 120), (300, 300), (1, 1), (40, 640), (128, 1030), (1, 4000)]
    c = run(Case(torch, seqs, 32, 8, 128, 32, fill=math.nan, spare_rows=5), ws)
    check_attention(c, rows=[0, 1, 4, 39, 40, 63, 64, 127, 128, 200, 299])


@pytest.mark.parametrize("n", [130, 700])
def test_many_sequences(torch, ws, n):
    seqs = [(1 + (i % 7 == 3) * (i % 5), 1 + (i * 37) % 211) for i in range(n)]
    seqs = [(min(a, b), b) for a, b in seqs]
    c = run(Case(torch, seqs, 4, 2, 64, 16, fill=math.nan), ws)
    check_attention(c)


def test_many_sequences_with_chunks(torch, ws):
    """More sequences than a block has threads, some of them long enough for
    the tensor cores' kernel, some with many blocks of rows."""
    seqs = [(60 if i % 90 == 7 else 300 if i == 500 else 1, 1 + (i * 53) % 90) for i in range(900)]
    seqs = [(a, max(a, b)) for a, b in seqs]
    c = run(Case(torch, seqs, 4, 2, 64, 16, fill=math.nan), ws)
    check_attention(c)


@pytest.mark.parametrize("new", [1, 30, 200])
@pytest.mark.parametrize("window,sinks", [(100, 5), (300, 0), (64, 70)])
def test_pages_behind_a_window_are_not_read(torch, ws, new, window, sinks):
    """Pages that only hold positions between the sinks and the window may
    have been given back: their table entries mean nothing."""
    c = Case(torch, [(new, 1500), (1, 40)], 8, 2, 64, 16)
    first = max(0, 1500 - new - window + 1)
    for i in range(first // 16):
        if i * 16 >= sinks:
            c.table[0, i] = -7
    run(c, ws, window, sinks)
    assert int(c.err) == 0
    check_attention(c, window, sinks)


def test_every_sequence_a_chunk(torch, ws):
    """All sequences as long as the longest, so that one kernel has them all;
    then the same rows with a shorter sequence among them."""
    c = run(Case(torch, [(100, 130), (100, 1000), (100, 100)], 8, 2, 128, 32, fill=math.nan), ws)
    check_attention(c, rows=[0, 1, 31, 32, 63, 64, 99])
    c = run(Case(torch, [(100, 130), (7, 1000), (100, 100)], 8, 2, 128, 32, fill=math.nan), ws)
    check_attention(c, rows=[0, 1, 6, 31, 32, 63, 64, 99])


def test_the_workspace_is_left_for_the_next_call(torch):
    """Counters are zero after calls that split items in either kernel."""
    ws = new_workspace(torch)
    for seqs in ([(1, 9000), (1, 4000)], [(300, 3000)], [(200, 2000), (1, 5000)]):
        c = run(Case(torch, seqs, 8, 2, 128, 32), ws)
        check_attention(c, rows=[0, 100, 199, 299])
        assert not bool(ws[:2048].any()) and not bool(ws[24 << 20:(24 << 20) + 2048].any())


def test_pages_shared_by_sequences(torch, ws):
    c = Case(torch, [(1, 100), (1, 100), (3, 90)], 8, 2, 64, 16)
    c.pages[1], c.pages[2] = c.pages[0], c.pages[0][:6] + [-1]
    c.table.copy_(torch.tensor(c.pages, dtype=torch.int32))
    check_attention(run(c, ws))


@pytest.mark.parametrize("page", [-1, 99, 2 ** 31 - 1, -2 ** 31])
def test_a_page_outside_the_pool(torch, ws, page):
    """Its rows are read as zeros, the error bit is set, the others are right."""
    for seqs in ([(1, 100), (1, 90)], [(80, 100), (1, 90)]):
        c = Case(torch, seqs, 8, 2, 128, 16)
        c.table[0, 2] = page
        run(c, ws)
        assert int(c.err) == 1 << 3
        c.pages[0][2] = c.k.shape[0]
        zero = c.k.new_zeros(1, *c.k.shape[1:])
        c.k, c.v = torch.cat((c.k, zero)), torch.cat((c.v, zero))
        check_attention(c)


@pytest.mark.parametrize("what", ["long", "negative", "order", "rows", "many"])
def test_sequences_out_of_range_are_skipped(torch, ws, what):
    c = Case(torch, [(2, 50), (3, 60), (2, 40)], 8, 2, 64, 16)
    if what == "long":
        c.kv_len[1] = 16 * c.table.shape[1] + 1
    elif what == "negative":
        c.kv_len[1] = -1
    elif what == "order":
        c.q_start[1] = 100
    elif what == "rows":
        c.q_start[3] = 1000
    batch = c.batch()
    if what == "many":
        batch.max_q_len = 2
    ib.paged_attention(c.out, c.q, c.cache(), batch, ws, lse=c.lse, err=c.err)
    torch.cuda.synchronize()
    assert int(c.err) == 1 << 4
    if what in ("long", "negative", "many"):
        assert bool((c.out[2:5] == 7).all()) and bool((c.lse[2:5] == 7).all())
        c.seqs[1] = (0, 0)
        check_attention(c)
    elif what == "rows":
        assert bool((c.out[5:] == 7).all())


def test_host_memory_is_refused(torch, ws):
    c = Case(torch, [(1, 10), (2, 20)], 4, 2, 64, 16)
    cache, batch = c.cache(), c.batch()
    cpu = {k: getattr(c, k).cpu() for k in ("q", "out", "lse", "k", "v", "q_start", "kv_len", "table", "err")}
    with_cpu = ib.RaggedBatch
    for call in (lambda: ib.paged_attention(c.out, cpu["q"], cache, batch, ws),
                 lambda: ib.paged_attention(cpu["out"], c.q, cache, batch, ws),
                 lambda: ib.paged_attention(c.out, c.q, cache, batch, ws, lse=cpu["lse"]),
                 lambda: ib.paged_attention(c.out, c.q, cache, batch, ws, err=cpu["err"]),
                 lambda: ib.paged_attention(c.out, c.q, cache, batch, ws.cpu()),
                 lambda: ib.paged_attention(c.out, c.q, ib.PagedCache(cpu["k"], cpu["v"]), batch, ws),
                 lambda: ib.paged_attention(c.out, c.q, cache, with_cpu(cpu["q_start"], c.kv_len, c.table, 3, 2), ws),
                 lambda: ib.paged_attention(c.out, c.q, cache, with_cpu(c.q_start, cpu["kv_len"], c.table, 3, 2), ws),
                 lambda: ib.paged_attention(c.out, c.q, cache, with_cpu(c.q_start, c.kv_len, cpu["table"], 3, 2), ws)):
        with pytest.raises(ib.InferntError):
            call()
    run(c, ws)
    check_attention(c)


def test_two_streams_with_their_own_workspaces(torch, ws):
    a = Case(torch, [(1, 3000), (200, 900)], 32, 8, 128, 32, seed=1)
    b = Case(torch, [(1, 2500), (1, 77), (90, 400)], 32, 4, 64, 16, seed=2)
    mine = [ws, new_workspace(torch)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, w, st in zip((a, b), mine, streams):
            ib.paged_attention(c.out, c.q, c.cache(), c.batch(), w, lse=c.lse, err=c.err, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for c in (a, b):
        check_attention(c, rows=[0, 1, 63, 64, 89, 150, 199])


def test_captured_call_follows_the_device_arrays(torch, ws):
    """A captured call replayed with other lengths, starts and pages."""
    c = Case(torch, [(1, 500), (1, 70), (40, 200)], 8, 2, 64, 16, spare_pages=100)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run(c, ws, stream=st.cuda_stream)
    check_attention(c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ib.paged_attention(c.out, c.q, c.cache(), c.batch(), ws, lse=c.lse, err=c.err, stream=st.cuda_stream)
    width = c.table.shape[1]
    for seqs in ([(2, 40), (39, 300), (1, 512)], [(1, 0), (0, 5), (40, 40)], [(1, 500), (1, 70), (40, 200)]):
        free = list(range(c.k.shape[0]))
        c.pages = [[free.pop() for _ in range(-(-n // 16))] for _, n in seqs]
        c.pages = [r + [-1] * (width - len(r)) for r in c.pages]
        starts = [0]
        for n, _ in seqs:
            starts.append(starts[-1] + n)
        c.seqs, c.starts = seqs, starts
        c.table.copy_(torch.tensor(c.pages, dtype=torch.int32))
        c.kv_len.copy_(torch.tensor([n for _, n in seqs], dtype=torch.int32))
        c.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        c.out.fill_(7)
        c.lse.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert int(c.err) == 0
        check_attention(c)


def test_the_same_call_twice_gives_the_same_bits(torch, ws):
    c = Case(torch, [(1, 4000), (1, 2100), (300, 1500), (1, 65)], 32, 8, 128, 32)
    first = run(c, ws).out.clone(), c.lse.clone()
    for _ in range(3):
        run(c, ws)
        assert bool((c.out == first[0]).all()) and bool((c.lse == first[1]).all())


def test_offsets_past_32_bits(torch, ws):
    """Pools of 2^31 + values: the sequences' pages at both ends."""
    page, nkv, D = 64, 8, 128
    pages = (1 << 31) // (nkv * page * D) + 40
    c = Case(torch, [(1, 700), (70, 400)], 16, nkv, D, page)
    small_k, small_v = c.k, c.v
    k = torch.empty(pages, nkv, page, D, device="cuda", dtype=c.dtype)
    v = torch.empty_like(k)
    rows, last = [], pages
    for r, (_, n) in zip(c.pages, c.seqs):
        new = []
        for i, p in enumerate(r):
            if p < 0:
                new.append(-1)
                continue
            last -= 1
            k[last].copy_(small_k[p])
            v[last].copy_(small_v[p])
            new.append(last)
        rows.append(new)
    c.k, c.v, c.pages = k, v, rows
    c.table.copy_(torch.tensor(rows, dtype=torch.int32))
    check_attention(run(c, ws), rows=[0, 1, 35, 69])


def test_long_context(torch, ws):
    """One token and a short chunk over 70000 positions (FP32 sums of many terms)."""
    c = run(Case(torch, [(1, 70001), (20, 66000)], 8, 1, 128, 64), ws)
    check_attention(c, rows=[0, 1, 19])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [2, 90])
def test_split_rows_with_a_hidden_value_that_is_not_finite(torch, ws, new, D):
    """Items shared by many blocks, whose last token's value is not finite:
    the joined rows before it are computed again, the last one shows it."""
    n = 9000
    c = Case(torch, [(new, n)], 4, 1, D, 64)
    c.v[c.pages[0][(n - 1) // 64], 0, (n - 1) % 64, 3] = math.inf
    for _ in range(2):
        run(c, ws)
        check_attention(c, rows=[0, new // 2 - 1, new - 2])
        assert bool(torch.isinf(c.out[new - 1, :, 3]).all()) and bool(torch.isfinite(c.out[new - 1, :, 4:].float()).all())
        assert int(c.err) == 0
