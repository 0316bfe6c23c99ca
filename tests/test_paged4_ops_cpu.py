"""The operators over 4-bit pages, page tables and drafts on a host without a
GPU: refusals of bad arguments (no kernel is launched, no address is read) and
the Python wrappers' own checks."""
import ctypes

import pytest

import infernt_b200 as ib
import test_paged_ops_cpu as wide

A = 4096  # an aligned address that nothing reads


def cache(**kw):
    c = ib.PagedCache4.__new__(ib.PagedCache4)
    ctypes.Structure.__init__(c, A, A, A, 8, 2, 16, 64, ib.DTYPE_BF16)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attention(c=None, b=None, out=2 * A, ldo=256, q=A, ldq=256, nq=4, window=0, sinks=0, scale=0.0, ws=A, lse=None,
              err=None):
    return ib.lib().infernt_paged4_attention(out, ldo, q, ldq, nq, ctypes.byref(c or cache()),
                                             ctypes.byref(b or wide.batch()), window, sinks, scale, lse, ws, err, None)


def rope(c=None, b=None, p=None, q_out=A, ldo=256, q=A, ldq=256, nq=4, k=A, ldk=128, v=A, ldv=128, src=ib.DTYPE_BF16,
         err=None):
    return ib.lib().infernt_paged4_rope_append(
        q_out, ldo, q, ldq, nq, k, ldk, v, ldv, src, ctypes.byref(c or cache()), ctypes.byref(b or wide.batch()),
        ctypes.byref(p if p is not None else ib.RopeParams(rotary_dim=64)), err, None)


def unpack(c=None, to=None, src=A, dst=A, n=3, err=None):
    return ib.lib().infernt_paged4_unpack(ctypes.byref(c or cache()), ctypes.byref(to or wide.cache()), src, dst, n, err,
                                          None)


@pytest.mark.parametrize("kw", wide.BAD_CACHES + [dict(scales=None), dict(scales=A + 2)])
def test_bad_caches_are_refused(kw):
    assert attention(c=cache(**kw)) == 1
    assert rope(c=cache(**kw)) == 1
    assert unpack(c=cache(**kw)) == 1
    assert ib.lib().infernt_paged4_attention(2 * A, 256, A, 256, 4, None, ctypes.byref(wide.batch()), 0, 0, 0.0, None, A,
                                             None, None) == 1


@pytest.mark.parametrize("kw", wide.BAD_BATCHES)
def test_bad_batches_are_refused(kw):
    assert attention(b=wide.batch(**kw)) == 1
    assert rope(b=wide.batch(**kw)) == 1


@pytest.mark.parametrize("kw", [
    dict(out=None), dict(q=None), dict(out=A), dict(ws=None), dict(q=A + 2), dict(out=A + 8), dict(ws=A + 4), dict(nq=0),
    dict(nq=3), dict(nq=2 * 129), dict(ldq=255), dict(ldq=260), dict(ldo=248), dict(window=-1),
    dict(sinks=-1, window=4), dict(sinks=4), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-0.1),
    dict(lse=A + 2), dict(err=A + 1), dict(b=wide.batch(num_rows=1 << 29), nq=4),
    dict(b=wide.batch(num_rows=1 << 27, max_q_len=1 << 27, table_stride=1 << 20)), dict(b=wide.batch(q_start=A + 2))])
def test_bad_attention_arguments_are_refused(kw):
    assert attention(**kw) == 1
    assert ib.lib().infernt_last_error().startswith(b"paged4_attention: ")


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(q_out=None), dict(k=None), dict(v=None), dict(q=None, q_out=None, k=None, v=None),
    dict(src=5), dict(nq=0), dict(ldq=255), dict(ldo=10), dict(ldk=127), dict(ldv=1), dict(q=A + 1), dict(q_out=A + 1),
    dict(q=A + 2, src=ib.DTYPE_F32), dict(src=ib.DTYPE_F16), dict(q=A, q_out=A, ldo=512), dict(err=A + 1),
    dict(p=ib.RopeParams(rotary_dim=66)), dict(p=ib.RopeParams(rotary_dim=64, theta=0.0))])
def test_bad_rope_arguments_are_refused(kw):
    assert rope(**kw) == 1
    assert ib.lib().infernt_last_error().startswith(b"paged4_rope_append: ")


@pytest.mark.parametrize("kw", [
    dict(to=wide.cache(num_kv_heads=3)), dict(to=wide.cache(page_size=8)), dict(to=wide.cache(head_dim=128)),
    dict(to=wide.cache(dtype=ib.DTYPE_F16)), dict(to=wide.cache(k=None)), dict(src=None), dict(dst=None), dict(n=-1),
    dict(src=A + 2), dict(dst=A + 1), dict(err=A + 3)])
def test_bad_unpack_arguments_are_refused(kw):
    assert unpack(**kw) == 1
    assert ib.lib().infernt_last_error().startswith(b"paged4_unpack: ")


def test_nothing_is_no_work():
    assert attention(b=wide.batch(num_seqs=0)) == 0 and attention(b=wide.batch(num_rows=0)) == 0
    assert rope(b=wide.batch(num_seqs=0)) == 0
    assert unpack(n=0, src=None, dst=None) == 0
    assert verify(num_seqs=0) == 0


def tables(**kw):
    t = ib.PageTables.__new__(ib.PageTables)
    ctypes.Structure.__init__(t, A, A, A, A, 3, 20, 16, 4)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def plan(t=None, lens=A, new=2 * A, q_start=A, kv=A, positions=None, slots=None, rows=10, err=None):
    return ib.lib().infernt_paged_batch_plan(ctypes.byref(t) if t is not False else None, lens, new, q_start, kv, positions,
                                             slots, rows, err, None)


@pytest.mark.parametrize("kw", [
    dict(t=False), dict(t=tables(block_table=None)), dict(t=tables(held=None)), dict(t=tables(free_pages=None)),
    dict(t=tables(state=None)), dict(t=tables(num_seqs=-1)), dict(t=tables(num_seqs=65536)), dict(t=tables(num_pages=0)),
    dict(t=tables(page_size=0)), dict(t=tables(table_stride=-1)), dict(t=tables(num_pages=1 << 20, page_size=1 << 11)),
    dict(t=tables(num_pages=1, page_size=1 << 30)), dict(t=tables(held=A + 2)), dict(lens=None), dict(new=None),
    dict(q_start=None), dict(kv=None), dict(kv=2 * A), dict(rows=-1), dict(rows=1 << 30), dict(lens=A + 1),
    dict(positions=A + 2), dict(slots=A + 1), dict(err=A + 2)])
def test_bad_plans_are_refused(kw):
    kw.setdefault("t", tables())
    assert plan(**kw) == 1
    assert ib.lib().infernt_last_error().startswith(b"paged_batch_plan: ")


def verify(out=A, acc=A, target=A, ld=100, dtype=0, probs=0, draft=None, draft_ld=0, tokens=A, q_start=A, num_seqs=2,
           num_rows=5, vocab=100, temps=None, u=A, kv=None, kept=None, ws=A, err=None):
    return ib.lib().infernt_verify_drafts(out, acc, target, ld, dtype, probs, draft, draft_ld, tokens, q_start, num_seqs,
                                          num_rows, vocab, temps, u, kv, kept, ws, err, None)


@pytest.mark.parametrize("kw", [
    dict(out=None), dict(acc=None), dict(target=None), dict(tokens=None), dict(q_start=None), dict(u=None), dict(ws=None),
    dict(ld=99), dict(dtype=3), dict(dtype=-1), dict(draft=A, draft_ld=99), dict(num_seqs=-1), dict(num_seqs=65536),
    dict(num_rows=-1), dict(num_rows=1 << 30), dict(vocab=0), dict(vocab=1 << 30, ld=1 << 31), dict(kv=A), dict(kept=A),
    dict(ws=A + 8), dict(target=A + 2), dict(target=A + 1, dtype=1), dict(u=A + 2), dict(tokens=A + 1), dict(temps=A + 2),
    dict(err=A + 1)])
def test_bad_verifications_are_refused(kw):
    assert verify(**kw) == 1
    assert ib.lib().infernt_last_error().startswith(b"verify_drafts: ")


def test_arrays_that_overlap_are_refused():
    """What a call writes may lie in nothing else of it, kept in kv_len and
    kv_len in len apart."""
    def at(n, step=1 << 20):  # arrays far from each other
        return A + n * step

    def message(status):
        assert status in (1, 6)  # 6: there is no device whose memory they could be
        return ib.lib().infernt_last_error()

    names = dict(out=at(0), acc=at(1), target=at(2), draft=at(3), draft_ld=100, tokens=at(4), q_start=at(5), temps=at(6),
                 u=at(7), kv=at(8), kept=at(9), ws=at(10), err=at(11))
    assert b"overlap" not in message(verify(**names))  # no memory of a device
    assert b"overlap" not in message(verify(**{**names, "kept": at(8)}))
    for bad in (dict(tokens=at(0)), dict(tokens=at(0) + 16), dict(q_start=at(1) - 8), dict(kv=at(9) + 4), dict(kept=at(5)),
                dict(acc=at(0) + 16), dict(u=at(0) - 4), dict(temps=at(1)), dict(out=at(2) + 4 * 499), dict(err=at(4) + 16),
                dict(kept=at(3) + 400), dict(ws=at(7)), dict(u=at(10) + 5 * 512 - 4)):
        assert b"overlap" in message(verify(**{**names, **bad})), bad
    assert b"overlap" not in message(verify(**{**names, "tokens": at(0) + 20}))
    t = tables(block_table=at(0), held=at(1), free_pages=at(2), state=at(3))
    args = dict(t=t, lens=at(4), new=at(5), q_start=at(6), kv=at(7), positions=at(8), slots=at(9), err=at(10))
    assert b"overlap" not in message(plan(**args))
    assert b"overlap" not in message(plan(**{**args, "kv": at(4)}))
    for bad in (dict(kv=at(5)), dict(kv=at(4) + 4), dict(q_start=at(4) - 12), dict(positions=at(9) + 36), dict(slots=at(0) + 44),
                dict(lens=at(1)), dict(new=at(2) + 76), dict(err=at(3) + 12)):
        assert b"overlap" in message(plan(**{**args, **bad})), bad


# ---------------------------------------------------------------- the Python wrappers


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def pools(torch, pages=4, heads=2, page=16, dim=64):
    return (torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8), torch.zeros(pages, heads, page, dim // 2,
            dtype=torch.uint8), torch.zeros(pages, heads, page, dtype=torch.int32))


def test_cache_wrapper(torch):
    k, v, s = pools(torch)
    c = ib.PagedCache4(k, v, s, torch.float16)
    assert (c.num_pages, c.num_kv_heads, c.page_size, c.head_dim, c.dtype) == (4, 2, 16, 64, ib.DTYPE_F16)
    for bad in ((k[0], v, s, torch.bfloat16), (k, v[:3], s, torch.bfloat16), (k, v, s[:, :1], torch.bfloat16),
                (k.int(), v.int(), s, torch.bfloat16), (k, v, s.float(), torch.bfloat16), (k, v, s, torch.float32),
                (k.transpose(1, 2), v.transpose(1, 2), s.transpose(1, 2), torch.bfloat16)):
        with pytest.raises(ValueError):
            ib.PagedCache4(*bad)


def test_table_wrapper(torch):
    t = ib.PageTables.empty(3, 20, 16, 4, device="cpu")
    assert (t.num_seqs, t.num_pages, t.page_size, t.table_stride) == (3, 20, 16, 4)
    table, held, free, state = t.tensors
    assert free.tolist() == list(range(20)) and state.tolist() == [0, 20, 0, 0]
    for bad in ((table[0], held, free, state, 16), (table, held[:2], free, state, 16), (table, held, free, state[:3], 16),
                (table.long(), held, free, state, 16), (table, held.float(), free, state, 16),
                (table.t(), held, free, state, 16), (table, held, free, state, 1 << 31)):
        with pytest.raises(ValueError):
            ib.PageTables(*bad)
    i32 = dict(dtype=torch.int32)
    good = [t, torch.zeros(3, **i32), torch.zeros(3, **i32), torch.zeros(4, **i32), torch.zeros(3, **i32)]
    for at, bad in ((1, torch.zeros(2, **i32)), (2, torch.zeros(3)), (3, torch.zeros(3, **i32)), (4, torch.zeros(2, **i32))):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError):
            ib.plan_batch(*args)
    with pytest.raises((ValueError, ib.InferntError)):  # host memory
        ib.plan_batch(*good)


def test_verify_wrapper(torch):
    i32 = dict(dtype=torch.int32)
    good = dict(out_tokens=torch.zeros(5, **i32), accepted=torch.zeros(2, **i32), target=torch.zeros(5, 30),
                tokens=torch.zeros(5, **i32), q_start=torch.zeros(3, **i32), u=torch.zeros(5),
                workspace=torch.zeros(ib.verify_drafts_workspace_bytes(5, 2), dtype=torch.uint8))
    for bad in (dict(out_tokens=torch.zeros(4, **i32)), dict(target=torch.zeros(30)), dict(target=torch.zeros(30, 5).t()),
                dict(target=torch.zeros(5, 30).double()), dict(tokens=torch.zeros(5)), dict(q_start=torch.zeros(2, **i32)),
                dict(u=torch.zeros(4)), dict(u=torch.zeros(5).half()), dict(workspace=torch.zeros(10)),
                dict(draft_probs=torch.zeros(4, 30)), dict(draft_probs=torch.zeros(5, 31)),
                dict(draft_probs=torch.zeros(5, 30).half()), dict(temperature=torch.zeros(1)),
                dict(kv_len=torch.zeros(2, **i32), kept=torch.zeros(1, **i32))):
        with pytest.raises(ValueError):
            ib.verify_drafts(**{**good, **bad})
    with pytest.raises((ValueError, ib.InferntError)):  # host memory
        ib.verify_drafts(**good)


def test_unpack_wrapper(torch):
    c = ib.PagedCache4(*pools(torch), torch.bfloat16)
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    to, one = ib.PagedCache(k, k.clone()), torch.zeros(1, dtype=torch.int32)
    for src, dst in ((one, one[:0]), (one.long(), one), (one, one.float())):
        with pytest.raises(ValueError):
            ib.paged4_unpack(c, to, src, dst)
