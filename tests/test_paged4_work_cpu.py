"""Which calls of attention over 4-bit pages have more work than its 32-bit
counts can hold: those of the kernels that would run, no others (no kernel is
launched here)."""
import pytest

import infernt_b200 as ib
import test_paged4_ops_cpu as four
import test_paged_ops_cpu as wide


def message(**kw):
    nq, nkv, dim, page = kw.pop("nq"), kw.pop("nkv"), kw.pop("dim", 128), kw.pop("page", 64)
    cache = four.cache(num_kv_heads=nkv, head_dim=dim, page_size=page, num_pages=1000)
    status = four.attention(c=cache, b=wide.batch(**kw), nq=nq, ldq=nq * dim, ldo=nq * dim)
    assert status in (1, 6)  # 6: there is no device whose memory the arrays could be
    return ib.lib().infernt_last_error()


@pytest.mark.parametrize("kw", [
    # a chunk over a table of 2^20 positions: the tcgen05 kernel alone
    dict(num_seqs=1, num_rows=8192, max_q_len=8192, table_stride=1 << 14, nq=64, nkv=8),
    # the same beside 63 sequences of a few tokens: both kernels
    dict(num_seqs=64, num_rows=8192 + 63 * 3, max_q_len=8192, table_stride=1 << 14, nq=64, nkv=8),
    # 2048 sequences of a token each over tables of 2^19 positions: the few-row kernel alone
    dict(num_seqs=2048, num_rows=2048, max_q_len=1, table_stride=1 << 13, nq=64, nkv=8)])
def test_calls_within_the_counts_are_taken(kw):
    assert b"split the call" not in message(**kw)


@pytest.mark.parametrize("kw", [
    dict(num_seqs=1, num_rows=1 << 21, max_q_len=1 << 21, table_stride=1 << 14, nq=64, nkv=8),
    dict(num_seqs=60000, num_rows=60000 + 8192, max_q_len=8192, table_stride=1 << 14, nq=64, nkv=8),
    dict(num_seqs=60000, num_rows=60000, max_q_len=1, table_stride=1 << 14, nq=64, nkv=8),
    dict(num_seqs=20000, num_rows=120000, max_q_len=6, table_stride=1 << 12, nq=64, nkv=8)])
def test_calls_past_the_counts_are_refused(kw):
    assert message(**kw).startswith(b"paged4_attention: ") and b"split the call" in message(**kw)
