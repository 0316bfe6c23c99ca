"""Copies of pages (bit for bit, nothing else moves), and the operators over
paged caches together as a server uses them: append, attend, fork, copy on
write, compact; then the same through the paged batched engine."""
import math

import pytest

import infernt_b200 as ib
from paged_reference import Case, check_attention, new_workspace
from test_paged_rope_gpu import Rope

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.mark.parametrize("pools,pages,shape,moves", [
    (1, 2, (8,), 1), (2, 10, (2, 1, 4), 5), (64, 40, (4, 16, 64), 3), (65, 40, (4, 16, 64), 20), (3, 101, (5, 24, 8), 33),
    (44, 90, (2, 7, 64), 45), (300, 70, (16,), 35), (2, 9000, (8,), 4400), (5, 6, (2, 1024, 128), 3)])
def test_copies(torch, pools, pages, shape, moves):
    g = torch.Generator(device="cuda").manual_seed(pages)
    x = torch.randint(-2 ** 15, 2 ** 15, (pools, pages) + shape, device="cuda", generator=g, dtype=torch.int16)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(moves)).tolist()
    src, dst = order[:moves], order[moves:2 * moves]
    want = x.clone()
    want[:, dst] = x[:, src]
    ib.copy_pages(x, src, dst)
    assert bool((x == want).all())
    apart = [p.clone() for p in want]  # pools that lie apart, back again
    ib.copy_pages(apart, dst, src)
    torch.cuda.synchronize()
    for a, w in zip(apart, want):
        w = w.clone()
        w[src] = w[dst]
        assert bool((a == w).all())


def test_one_page_into_several(torch):
    x = torch.arange(3 * 8 * 32, device="cuda", dtype=torch.int32).view(3, 8, 32)
    want = x.clone()
    want[:, [1, 5, 7]] = x[:, [2, 2, 4]]
    ib.copy_pages(x, [2, 2, 4], [1, 5, 7])
    assert bool((x == want).all())


def test_offsets_past_32_bits(torch):
    x = torch.zeros(1, 9, 1 << 29, device="cuda", dtype=torch.uint8)
    x[0, 8] = torch.randint(0, 255, (1 << 29,), device="cuda", dtype=torch.uint8)
    ib.copy_pages(x, [8], [7])
    assert bool((x[0, 7] == x[0, 8]).all()) and not bool(x[0, :7].any())


def test_captured_copy_keeps_its_list(torch):
    x = torch.randint(0, 100, (4, 10, 64), device="cuda", dtype=torch.int32)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ib.copy_pages(x, [1, 2], [7, 8], stream=st.cuda_stream)
    assert not bool((x[:, 7] == x[:, 1]).all())
    x[:, 1] += 1000
    g.replay()
    torch.cuda.synchronize()
    assert bool((x[:, [7, 8]] == x[:, [1, 2]]).all())


def test_host_memory_is_refused(torch):
    with pytest.raises(ib.InferntError):
        ib.copy_pages(torch.zeros(2, 4, 16), [0], [1])
    with pytest.raises(ValueError):
        ib.copy_pages([torch.zeros(4, 16, device="cuda"), torch.zeros(4, 16)], [0], [1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_attend_fork_and_compact(torch, dtype):
    """Two prompts, one forked three ways, all decoded some steps on shared
    pages, then compacted: every row of every step against 64 bits over rows
    that a plain copy of the sequences keeps."""
    page, nkv, nq, D, num = 16, 2, 8, 64, 40
    pool = ib.PagePool(num, page, 6)
    k = torch.full((num, nkv, page, D), math.nan, device="cuda", dtype=torch.float32)
    ref = Rope(torch, [(1, 1)], nq, nkv, D, page, "fp32", dtype, theta=500000.0)
    t = ref.c.dtype
    k = k.to(t)
    v = k.clone()
    ws, g = new_workspace(torch), torch.Generator(device="cuda").manual_seed(9)
    told = {}  # sequence -> (K rows, V rows) as 64-bit values of what was appended

    def step(new):
        """new: {sequence: tokens}; their rows appended and attended."""
        seqs, copies = sorted(new), ([], [])
        for s in seqs:
            n = told[s][0].shape[0] if s in told else 0
            pool.resize(s, n + new[s])
            a, b = pool.write(s, n, n + new[s])
            copies[0].extend(a), copies[1].extend(b)
        ib.copy_pages([k, v], *copies)
        c = Case.__new__(Case)
        c.torch, c.nq, c.nkv, c.D, c.page, c.kind, c.dtype = torch, nq, nkv, D, page, dtype, t
        c.seqs = [(new[s], (told[s][0].shape[0] if s in told else 0) + new[s]) for s in seqs]
        rows = [pool.pages(s) for s in seqs]
        width = max(len(r) for r in rows)
        c.pages = [r + [-1] * (width - len(r)) for r in rows]
        c.table = torch.tensor(c.pages, dtype=torch.int32, device="cuda")
        c.starts = [0]
        for n, _ in c.seqs:
            c.starts.append(c.starts[-1] + n)
        c.rows, c.max_q = c.starts[-1] + 1, max(n for n, _ in c.seqs)
        c.q_start = torch.tensor(c.starts, dtype=torch.int32, device="cuda")
        c.kv_len = torch.tensor([n for _, n in c.seqs], dtype=torch.int32, device="cuda")
        c.k, c.v = k, v
        qkv = torch.randn(c.rows, nq + 2 * nkv, D, device="cuda", generator=g)
        q, kn, vn = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
        c.q = torch.full((c.rows, nq, D), 7.0, device="cuda").to(t)
        c.out = c.q.clone()
        c.lse = torch.full((c.rows, nq), 7.0, device="cuda")
        ib.paged_rope_append(c.q, q, kn, vn, c.cache(), c.batch(), ib.RopeParams(**ref.params))
        ib.paged_attention(c.out, c.q, c.cache(), c.batch(), ws, lse=c.lse)
        torch.cuda.synchronize()
        for i, s in enumerate(seqs):
            a, n, length = c.starts[i], *c.seqs[i]
            kk, _ = ref.turn(kn[a:a + n], torch.arange(length - n, length, device="cuda"))
            old = told.get(s, (kk[:0], kk[:0]))
            told[s] = (torch.cat((old[0], kk)), torch.cat((old[1], vn[a:a + n].to(t).double())))
            # the cache holds what this sequence appended, whoever shared its pages
            u = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}[dtype]
            assert bool(((c.dense(k, i) - told[s][0]).abs() <= 1.01 * u * told[s][0].abs() + 2.0 ** -17).all())
            assert bool((c.dense(v, i) == told[s][1]).all())
        check_attention(c)

    step({0: 37, 1: 20})
    for s in (2, 3, 4):
        pool.fork(0, s, 37 - s)
        told[s] = tuple(x[:37 - s] for x in told[0])
    assert pool.stats()[1] > 0
    for _ in range(3):
        step({0: 1, 1: 1, 2: 1, 3: 1, 4: 5})
    pool.resize(0, 0)
    del told[0]
    ib.copy_pages([k, v], *pool.compact())
    free, _, highest = pool.stats()
    assert highest == num - free - 1
    step({1: 1, 2: 1, 3: 9, 4: 1})
    step({0: 50, 4: 2})


def test_fork_in_the_engine():
    """A sequence forked in the paged batched engine (shared pages, its last
    page copied) decodes as one that was prefilled itself, bit for bit, and
    leaves the one it came from as it was."""
    cfg = ib.ModelConfig(vocab_size=1024, hidden_size=512, num_layers=2, num_attention_heads=8, num_key_value_heads=2,
                         intermediate_size=1024, max_seq_len=256, weight_dtype=ib.DTYPE_BF16)
    page, prompt = 32, ib.prompt(71, 3, 3, 1024)
    ea = ib.BatchEngine(cfg, 3, seed=4, pages=(page, 30))
    eb = ib.BatchEngine(cfg, 3, seed=4, pages=(page, 30))
    for s in range(3):
        eb.set_pages(s, range(8 * s, 8 * s + 8))
        first = eb.prefill(s, prompt)[0]
    pool = ib.PagePool(30, page, 3)
    pool.resize(0, 71)
    ea.set_pages(0, pool.pages(0))
    assert ea.prefill(0, prompt)[0] == first
    for s in (1, 2):
        pool.fork(0, s, 71)
    tokens, pos = [first, 5, 900], 71
    for _ in range(40):  # over the end of a page
        for s in range(3):
            pool.resize(s, pos + 1)
            ea.copy_pages(*pool.write(s, pos, pos + 1))
            ea.set_pages(s, pool.pages(s))
        got = ea.step(tokens, [pos] * 3)
        assert got == eb.step(tokens, [pos] * 3)
        assert (ea.logits() == eb.logits()).all()
        tokens, pos = got, pos + 1
    assert pool.stats()[1] == 2  # the two full pages of the prompt are still shared
    src, dst = pool.compact()
    ea.copy_pages(src, dst)
    for s in range(3):
        ea.set_pages(s, pool.pages(s))
    assert ea.step(tokens, [pos - 1] * 3) == eb.step(tokens, [pos - 1] * 3)
    ec = ib.BatchEngine(cfg, 1, seed=4)
    with pytest.raises(ib.InferntError):
        ec.copy_pages([0], [1])
    for bad in (([0], [30]), ([0], [0]), ([0, 1], [2, 2])):
        with pytest.raises(ib.InferntError):
            ea.copy_pages(*bad)
    for e in (ea, eb, ec):
        e.close()
