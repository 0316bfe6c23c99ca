"""Which stream the operators' wrappers pass on: the one that they are given,
else torch's current one on the tensors' device (a stand-in library records it)."""
import pytest

import infernt_b200 as ib


class Recorder:
    def __init__(self):
        self.streams = []

    def __getattr__(self, name):
        if name.endswith("workspace_bytes"):
            return lambda: 64
        return lambda *args: self.streams.append(args[-1]) or 0


@pytest.mark.parametrize("given", [None, 0, 77])
def test_the_stream_that_is_passed_on(monkeypatch, given):
    torch = pytest.importorskip("torch")
    lib = Recorder()
    monkeypatch.setattr(ib, "_lib", lib)
    monkeypatch.setattr(ib, "_workspace_bytes", 64)
    monkeypatch.setattr(ib, "_current_stream", lambda t: 1000 + t.shape[0])
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    cache = ib.PagedCache(k, k)
    i32 = torch.zeros(3, dtype=torch.int32)
    batch = ib.RaggedBatch(i32, i32[:2], torch.zeros(2, 4, dtype=torch.int32), 4, 4)
    q, kv, ws = torch.zeros(5, 4, 64, dtype=k.dtype), torch.zeros(6, 2, 64, dtype=k.dtype), torch.zeros(64, dtype=torch.uint8)
    kw = {} if given is None else {"stream": given}
    ib.paged_attention(q.clone(), q, cache, batch, ws, **kw)
    ib.paged_rope_append(q, q, None, None, cache, batch, ib.RopeParams(rotary_dim=64), **kw)
    ib.paged_rope_append(q, q, kv, kv, cache, batch, ib.RopeParams(rotary_dim=64), **kw)
    ib.copy_pages(torch.zeros(3, 4, 16), [0], [1], **kw)
    ib.copy_pages([torch.zeros(7, 16), torch.zeros(7, 16)], [0], [1], **kw)
    assert lib.streams == ([1005, 1005, 1006, 1003, 1007] if given is None else [given] * 5)


def test_a_host_tensor_has_no_stream():
    torch = pytest.importorskip("torch")
    assert ib._current_stream(torch.zeros(1)) is None
