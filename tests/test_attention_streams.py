"""Which stream the attention operators hand to the library, without a GPU: a recorder in the library's place, and host
tensors that say they are CUDA tensors."""

import pytest
import torch

from voxwerk_b200 import attention


class Tensor:
    """A host tensor in a CUDA tensor's place."""

    is_cuda = True

    def __init__(self, *shape, dtype=torch.bfloat16):
        self._t = torch.zeros(shape, dtype=dtype)
        self.device = torch.device("cuda", 0)

    def __getattr__(self, name):
        return getattr(self._t, name)


class Library:
    """Records (call, stream), and fails where it is told to."""

    def __init__(self):
        self.calls, self.status = [], 0

    def __getattr__(self, name):
        def call(handle, *args):
            self.calls.append((name, args[-1]))
            return self.status if name == "vw_synchronize" else 0
        return call


class FakeDevice:
    handle, device = None, 0


@pytest.fixture
def calls(monkeypatch):
    """The three operators as calls of a stream, the recorder, and the current stream's handle (a list of one)."""
    library, current, capturing = Library(), [0], [False]
    monkeypatch.setattr(attention, "lib", library)

    class Stream:
        @property
        def cuda_stream(self):
            return current[0]
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    cache = attention.KvCache(Tensor(4, 16, 2, 64), Tensor(4, 16, 2, 64))
    batch = attention.KvBatch(Tensor(2, 2, dtype=torch.int32), Tensor(2, dtype=torch.int32))
    q, k, out = Tensor(2, 4, 64), Tensor(2, 2, 64), Tensor(2, 4, 64)
    operators = [
        ("vw_rope_append", lambda s: attention.rope_append(FakeDevice, q, k, k, cache, batch, None, out, stream=s)),
        ("vw_prompt_attention", lambda s: attention.prompt_attention(FakeDevice, q, cache, batch, out, stream=s)),
        ("vw_decode_attention", lambda s: attention.decode_attention(FakeDevice, q, cache, batch, out, stream=s)),
    ]
    return operators, library, current, capturing


@pytest.mark.parametrize("current,handle", [(0, 1), (0x5550, 0x5550)], ids=["default", "other"])
def test_without_a_stream_a_call_is_in_order_with_the_current_one(calls, current, handle):
    """It runs on torch's current stream (the default stream's handle is cudaStreamLegacy, 1: NULL would be another
    stream), and returns after it with what the kernels reported."""
    operators, library, now, _ = calls
    now[0] = current
    for name, call in operators:
        library.calls.clear()
        call(None)
        assert library.calls == [(name, handle), ("vw_synchronize", handle)]
        library.status = 2
        with pytest.raises(Exception):
            call(None)
        library.status = 0


def test_a_given_stream_only_enqueues(calls):
    operators, library, now, _ = calls
    now[0] = 0x5550
    for name, call in operators:
        for stream, handle in ((0x7770, 0x7770), (0, 1)):   # 0: torch's default stream
            library.calls.clear()
            call(stream)
            assert library.calls == [(name, handle)]


def test_a_call_that_waits_is_refused_inside_a_capture(calls):
    operators, library, now, capturing = calls
    now[0], capturing[0] = 0x5550, True
    for name, call in operators:
        library.calls.clear()
        with pytest.raises(ValueError, match="captur"):
            call(None)
        assert library.calls == []
        call(0x5550)
        assert library.calls == [(name, 0x5550)]


def test_a_batch_serves_calls_of_different_numbers_of_rows_at_a_time(calls):
    """Two threads may share a KvBatch: the struct that one call hands over is not changed by the next."""
    _, library, _, _ = calls
    cache = attention.KvCache(Tensor(4, 16, 2, 64), Tensor(4, 16, 2, 64))
    batch = attention.KvBatch(Tensor(2, 2, dtype=torch.int32), Tensor(2, dtype=torch.int32))
    given = []
    library.vw_prompt_attention = library.vw_decode_attention = library.vw_rope_append = \
        lambda handle, cache, batch, *rest: given.append(batch._obj) or 0
    for n in (2, 5, 3):
        q, k = Tensor(n, 4, 64), Tensor(n, 2, 64)
        attention.prompt_attention(FakeDevice, q, cache, batch, Tensor(n, 4, 64), stream=1)
        attention.decode_attention(FakeDevice, q, cache, batch, Tensor(n, 4, 64), stream=1)
        attention.rope_append(FakeDevice, q, k, k, cache, batch, None, Tensor(n, 4, 64), stream=1)
    assert [b.n_rows for b in given] == [2, 2, 2, 5, 5, 5, 3, 3, 3]
    assert all(b.n_seqs == 2 and b.page_table == batch.page_table.data_ptr() for b in given)
