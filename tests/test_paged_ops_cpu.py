"""The operators over paged caches on a host without a GPU: refusals of bad
arguments (no kernel is launched, no address is read), the page pool against
a plain model of it, and the Python wrappers' own checks."""
import ctypes
import random

import pytest

import infernt_b200 as ib

A = 4096  # an aligned address that nothing reads


def cache(**kw):
    c = ib.PagedCache.__new__(ib.PagedCache)
    ctypes.Structure.__init__(c, A, A, 8, 2, 16, 64, ib.DTYPE_BF16)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def batch(**kw):
    b = ib.RaggedBatch.__new__(ib.RaggedBatch)
    ctypes.Structure.__init__(b, A, A, A, 2, 10, 10, 4)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def attention(c=None, b=None, out=2 * A, ldo=256, q=A, ldq=256, nq=4, window=0, sinks=0, scale=0.0, ws=A):
    return ib.lib().infernt_paged_attention(out, ldo, q, ldq, nq, ctypes.byref(c or cache()),
                                            ctypes.byref(b or batch()), window, sinks, scale, None, ws, None, None)


BAD_CACHES = [dict(k=None), dict(v=None), dict(k=A + 8), dict(num_pages=0), dict(num_kv_heads=0), dict(page_size=0),
              dict(head_dim=96), dict(head_dim=0), dict(dtype=ib.DTYPE_F32), dict(dtype=3),
              dict(num_pages=1 << 20, page_size=1 << 11)]
BAD_BATCHES = [dict(num_seqs=-1), dict(num_seqs=65536), dict(num_rows=-1), dict(num_rows=1 << 30),
               dict(max_q_len=-1), dict(table_stride=-1), dict(q_start=None), dict(kv_len=None),
               dict(block_table=None)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches_are_refused(kw):
    assert attention(c=cache(**kw)) == 1
    assert rope(c=cache(**kw)) == 1


@pytest.mark.parametrize("kw", BAD_BATCHES)
def test_bad_batches_are_refused(kw):
    assert attention(b=batch(**kw)) == 1
    assert rope(b=batch(**kw)) == 1


@pytest.mark.parametrize("kw", [
    dict(out=None), dict(q=None), dict(out=A), dict(ws=None), dict(q=A + 2), dict(out=A + 8), dict(ws=A + 4), dict(nq=0),
    dict(nq=3), dict(nq=2 * 129), dict(ldq=255), dict(ldq=260), dict(ldo=248), dict(window=-1),
    dict(sinks=-1, window=4), dict(sinks=4), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(scale=-0.1), dict(b=batch(num_rows=1 << 29), nq=4),
    dict(b=batch(num_rows=1 << 27, max_q_len=1 << 27, table_stride=1 << 20))])
def test_bad_attention_arguments_are_refused(kw):
    assert attention(**kw) == 1
    assert ib.lib().infernt_last_error() != b""


@pytest.mark.parametrize("field", ["q_start", "kv_len", "block_table"])
def test_misaligned_batch_arrays_are_refused(field):
    assert attention(b=batch(**{field: A + 2})) == 1
    assert rope(b=batch(**{field: A + 2})) == 1


def test_misaligned_lse_and_err_are_refused():
    f, c, b = ib.lib().infernt_paged_attention, ctypes.byref(cache()), ctypes.byref(batch())
    for lse, err in ((A + 2, None), (None, A + 1), (None, A + 2)):
        assert f(2 * A, 256, A, 256, 4, c, b, 0, 0, 0.0, lse, A, err, None) == 1
    p = ib.RopeParams(rotary_dim=64)
    assert ib.lib().infernt_paged_rope_append(A, 256, A, 256, 4, A, 128, A, 128, ib.DTYPE_BF16, c, b, ctypes.byref(p),
                                              A + 2, None) == 1


def test_empty_batches_are_no_work():
    assert attention(b=batch(num_seqs=0)) == 0
    assert attention(b=batch(num_rows=0)) == 0
    assert rope(b=batch(num_seqs=0)) == 0
    assert ib.lib().infernt_pages_copy(None, 0, 16, 4, None, None, 0, None) == 0


def rope(c=None, b=None, p=None, q_out=A, ldo=256, q=A, ldq=256, nq=4, k=A, ldk=128, v=A, ldv=128, src=ib.DTYPE_BF16):
    return ib.lib().infernt_paged_rope_append(
        q_out, ldo, q, ldq, nq, k, ldk, v, ldv, src, ctypes.byref(c or cache()), ctypes.byref(b or batch()),
        ctypes.byref(p) if p is not None else ctypes.byref(ib.RopeParams(rotary_dim=64)), None, None)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(q_out=None), dict(k=None), dict(v=None), dict(q=None, q_out=None, k=None, v=None),
    dict(src=5), dict(nq=0), dict(ldq=255), dict(ldo=10), dict(ldk=127), dict(ldv=1), dict(q=A + 1), dict(q_out=A + 1),
    dict(q=A + 2, src=ib.DTYPE_F32), dict(src=ib.DTYPE_F16), dict(q=A, q_out=A, ldo=512)])
def test_bad_rope_arguments_are_refused(kw):
    # q_out == q in the last two: another type, another stride
    assert rope(**kw) == 1


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=66), dict(rotary_dim=64, theta=0.0),
    dict(rotary_dim=64, theta=float("nan")), dict(rotary_dim=64, scaling="linear", factor=0.0),
    dict(rotary_dim=64, scaling="llama3", factor=8.0, original_max_len=0),
    dict(rotary_dim=64, scaling="llama3", factor=8.0, original_max_len=8192, low=4.0, high=4.0),
    dict(rotary_dim=64, scaling="yarn", factor=8.0, original_max_len=8192, theta=1.0)])
def test_bad_rope_parameters_are_refused(kw):
    assert rope(p=ib.RopeParams(**kw)) == 1


def test_unknown_scaling_name():
    with pytest.raises(ValueError):
        ib.RopeParams(scaling="dynamic")


def copy(pools, page_bytes, num_pages, src, dst):
    n = len(src)
    return ib.lib().infernt_pages_copy((ctypes.c_void_p * max(1, len(pools)))(*pools), len(pools), page_bytes, num_pages,
                                       (ctypes.c_int * max(1, n))(*src), (ctypes.c_int * max(1, n))(*dst), n, None)


MANY = list(range(40))


@pytest.mark.parametrize("args", [
    ([A], 24, 4, [0], [1]), ([A], 0, 4, [0], [1]), ([A + 8], 16, 4, [0], [1]), ([None], 16, 4, [0], [1]),
    ([A], 16, 0, [0], [1]), ([A], 16, 4, [-1], [1]), ([A], 16, 4, [4], [1]), ([A], 16, 4, [0], [4]),
    ([A], 16, 4, [0], [-1]), ([A], 16, 4, [0, 1], [2, 2]), ([A], 16, 4, [0, 1], [1, 2]), ([A], 16, 4, [1], [1]),
    ([A], 16, 100, MANY, MANY[1:] + [50]), ([A], 16, 100, MANY, [60] * 40)])
def test_bad_page_copies_are_refused(args):
    assert copy(*args) == 1


def test_the_engine_call_needs_an_engine():
    assert ib.lib().infernt_batch_engine_copy_pages(None, None, None, 0) == 1


# ------------------------------------------------------------- page pool


def test_pool_refusals():
    with pytest.raises(ib.InferntError):
        ib.PagePool(0, 16, 1)
    with pytest.raises(ib.InferntError):
        ib.PagePool(4, 0, 1)
    p = ib.PagePool(4, 16, 3)
    for call in (lambda: p.resize(3, 1), lambda: p.resize(-1, 1), lambda: p.resize(0, -1), lambda: p.fork(0, 0, 0),
                 lambda: p.fork(0, 1, 1), lambda: p.write(0, 0, 1), lambda: p.write(0, 2, 1), lambda: p.pages(7)):
        with pytest.raises(ib.InferntError):
            call()
    p.resize(0, 17)
    p.resize(1, 1)
    with pytest.raises(ib.InferntError):
        p.fork(0, 1, 16)  # sequence 1 holds pages
    with pytest.raises(ib.InferntError) as e:
        p.resize(2, 33)  # three pages, one is free
    assert e.value.status == 4
    assert p.pages(2) == [] and p.stats() == (1, 0, 2)


def test_a_failed_write_changes_nothing():
    p = ib.PagePool(3, 4, 2)
    p.resize(0, 8)
    p.fork(0, 1, 8)
    with pytest.raises(ib.InferntError) as e:
        p.write(1, 0, 8)  # two copies, one free page
    assert e.value.status == 4
    assert p.pages(1) == p.pages(0) == [0, 1] and p.stats() == (1, 2, 1)
    assert p.write(1, 4, 8) == ([1], [2])
    assert p.pages(1) == [0, 2] and p.stats() == (0, 1, 2)
    assert p.write(0, 4, 8) == ([], [])  # sequence 0 is its page's only holder now


@pytest.mark.parametrize("seed", range(6))
def test_pool_against_a_model_with_contents(seed):
    """Random forks, growth, writes, frees and compactions; the pages hold
    what their sequences wrote, so a lost share, a missing copy or a wrong
    move shows."""
    rng = random.Random(seed)
    num, size, seqs = rng.choice([5, 12, 40]), rng.choice([1, 4]), 6
    p = ib.PagePool(num, size, seqs)
    content = [None] * (num * size)                 # per page row
    told = {s: [] for s in range(seqs)}             # what each sequence should read back

    def run(copies):
        src, dst = copies
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for a, b in zip(src, dst):
            content[b * size:(b + 1) * size] = content[a * size:(a + 1) * size]

    for step in range(400):
        s = rng.randrange(seqs)
        do = rng.choice(["grow", "grow", "grow", "rewrite", "fork", "free", "cut", "compact"])
        try:
            if do == "grow":
                n = len(told[s]) + rng.randint(1, 2 * size)
                p.resize(s, n)
                try:
                    run(p.write(s, len(told[s]), n))
                except ib.InferntError:
                    p.resize(s, len(told[s]))
                    raise
                pages = p.pages(s)
                for i in range(len(told[s]), n):
                    told[s].append((s, step, i))
                    content[pages[i // size] * size + i % size] = told[s][i]
            elif do == "rewrite" and told[s]:
                a = rng.randrange(len(told[s]))
                b = rng.randint(a, len(told[s]))
                run(p.write(s, a, b))
                pages = p.pages(s)
                for i in range(a, b):
                    told[s][i] = (s, step, i)
                    content[pages[i // size] * size + i % size] = told[s][i]
            elif do == "fork":
                d = rng.randrange(seqs)
                if d != s and not told[d]:
                    n = rng.randint(0, len(told[s]))
                    p.fork(s, d, n)
                    told[d] = told[s][:n]
            elif do == "free":
                p.resize(s, 0)
                told[s] = []
            elif do == "cut":
                told[s] = told[s][:rng.randint(0, len(told[s]))]
                p.resize(s, len(told[s]))
            elif do == "compact":
                run(p.compact())
                free, _, highest = p.stats()
                assert highest == num - free - 1
        except ib.InferntError as e:
            assert e.status == 4
        held = {}
        for t in range(seqs):
            pages = p.pages(t)
            assert len(pages) == -(-len(told[t]) // size) and len(set(pages)) == len(pages)
            for i, x in enumerate(told[t]):
                assert content[pages[i // size] * size + i % size] == x, (seed, step, t, i)
            for q in pages:
                held[q] = held.get(q, 0) + 1
        assert p.stats() == (num - len(held), sum(c > 1 for c in held.values()), max(held, default=-1))


def test_wrapper_checks():
    torch = pytest.importorskip("torch")
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ib.PagedCache(k, k[:, :, :, :32])
    with pytest.raises(ValueError):
        ib.PagedCache(k, k.half())
    with pytest.raises(ValueError):
        ib.PagedCache(k.transpose(1, 2), k.transpose(1, 2))
    with pytest.raises(ValueError):
        ib.PagedCache(k.double(), k.double())
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        ib.RaggedBatch(i32, i32, torch.zeros(3, 4, dtype=torch.int32), 4, 4)
    with pytest.raises(ValueError):
        ib.RaggedBatch(i32, i32[:2], torch.zeros(2, 4, dtype=torch.int64), 4, 4)
    c = ib.PagedCache(k, k)
    b = ib.RaggedBatch(i32, i32[:2], torch.zeros(2, 4, dtype=torch.int32), 4, 4)
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16)
    ws = torch.zeros(ib.paged_attention_workspace_bytes(), dtype=torch.uint8)
    for bad in (lambda: ib.paged_attention(q, q.half(), c, b, ws), lambda: ib.paged_attention(q[:2], q, c, b, ws),
                lambda: ib.paged_attention(q.clone(), q.transpose(0, 1), c, b, ws),
                lambda: ib.paged_attention(q.clone(), q, c, b, ws[:100]),
                lambda: ib.paged_attention(q.clone(), q, c, b, ws, lse=torch.zeros(4, 3)),
                lambda: ib.paged_rope_append(q, q, k[0, 0], k[0, 0], c, b, ib.RopeParams()),
                lambda: ib.paged_rope_append(q.half(), q, None, None, c, b, ib.RopeParams()),
                lambda: ib.copy_pages([k, k[:2]], [0], [1]), lambda: ib.copy_pages([k], [0], [1, 2]),
                lambda: ib.copy_pages([], [0], [1])):
        with pytest.raises(ValueError):
            bad()
