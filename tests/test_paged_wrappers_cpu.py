"""What the wrappers of the operators over paged caches refuse before a call:
an error word or a workspace of the wrong kind, pools of no pages, numbers that
do not fit a C int."""
import pytest

import infernt_b200 as ib

torch = pytest.importorskip("torch")


@pytest.fixture
def args(monkeypatch):
    """A small batch, and a library whose calls fail the test."""
    class Unreached:
        def __getattr__(self, name):
            def call(*a):
                raise AssertionError("%s is reached" % name)
            return call

    monkeypatch.setattr(ib, "_workspace_bytes", 64)
    monkeypatch.setattr(ib, "_lib", Unreached())
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    i32 = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(2, 4, dtype=torch.int32)
    return dict(cache=ib.PagedCache(k, k), i32=i32, table=table, batch=ib.RaggedBatch(i32, i32[:2], table, 4, 4),
                q=torch.zeros(4, 4, 64, dtype=torch.bfloat16), kv=torch.zeros(4, 2, 64, dtype=torch.bfloat16),
                ws=torch.zeros(64, dtype=torch.uint8))


BAD_ERR = [torch.zeros(1, dtype=torch.uint8), torch.zeros(4, dtype=torch.bfloat16), torch.zeros(1),
           torch.zeros(1, dtype=torch.int64), torch.zeros(0, dtype=torch.int32)]


@pytest.mark.parametrize("err", BAD_ERR)
def test_an_error_word_of_another_type(args, err):
    with pytest.raises(ValueError):
        ib.paged_attention(args["q"].clone(), args["q"], args["cache"], args["batch"], args["ws"], err=err)
    with pytest.raises(ValueError):
        ib.paged_rope_append(args["q"], args["q"], args["kv"], args["kv"], args["cache"], args["batch"],
                             ib.RopeParams(rotary_dim=64), err=err)


@pytest.mark.parametrize("ws", [torch.zeros(1, dtype=torch.uint8).expand(64), torch.zeros(128, dtype=torch.uint8)[::2]])
def test_a_workspace_with_gaps(args, ws):
    with pytest.raises(ValueError):
        ib.paged_attention(args["q"].clone(), args["q"], args["cache"], args["batch"], ws)


@pytest.mark.parametrize("pools", [torch.zeros(3, 0, 16), [torch.zeros(0, 16)], [torch.zeros(0, 16)] * 2])
def test_pools_of_no_pages(args, pools):
    with pytest.raises(ValueError):
        ib.copy_pages(pools, [], [])


@pytest.mark.parametrize("kw", [dict(window=2 ** 31), dict(window=2 ** 32 + 5), dict(window=9, sinks=2 ** 32)])
def test_windows_past_an_int(args, kw):
    with pytest.raises(ValueError):
        ib.paged_attention(args["q"].clone(), args["q"], args["cache"], args["batch"], args["ws"], **kw)


def test_other_numbers_past_an_int(args):
    for rows, most in ((2 ** 32, 4), (4, 2 ** 32 + 4)):
        with pytest.raises(ValueError):
            ib.RaggedBatch(args["i32"], args["i32"][:2], args["table"], rows, most)
    with pytest.raises(ValueError):
        ib.RopeParams(rotary_dim=2 ** 32 + 64)
    with pytest.raises(ValueError):
        ib.RopeParams(rotary_dim=64, original_max_len=2 ** 32 + 1)
    for src, dst in (([2 ** 32], [1]), ([0], [2 ** 32 + 1]), ([-2 ** 32], [1])):
        with pytest.raises(ValueError):
            ib.copy_pages(torch.zeros(3, 4, 16), src, dst)
    one = torch.empty(256, dtype=torch.bfloat16).as_strided((1, 4, 64), (2 ** 32 + 256, 64, 1))
    rows = torch.empty(0, dtype=torch.bfloat16, device="meta").as_strided((4, 4, 64), (2 ** 32 + 256, 64, 1))
    with pytest.raises(ValueError):
        ib._rows(rows, 4, 4, 64, "q")
    assert ib._rows(one, 1, 4, 64, "q") == 256  # one row has no stride of its own
