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

    def get_device(self):
        return 0

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


def test_tensors_of_another_gpu_are_refused(calls):
    """The kernels would read them through addresses that the handle's device may not map."""
    _, library, _, _ = calls

    class Elsewhere(Tensor):
        def get_device(self):
            return 1

    def make(where, **other):
        t = lambda name, *a, **k: (Elsewhere if name == where else Tensor)(*a, **k)
        ints = dict(dtype=torch.int32)
        cache = attention.KvCache(t("cache", 4, 16, 2, 64), t("cache", 4, 16, 2, 64))
        batch = attention.KvBatch(t("batch", 2, 2, **ints), t("batch", 2, **ints))
        prefix = attention.KvPrefix(t("prefix", 1, 2, **ints), t("prefix", 1, **ints), t("prefix", 2, **ints))
        rope = attention.RopeTable(t("rope", 9, 32, dtype=torch.float32), t("rope", 9, 32, dtype=torch.float32))
        q, k, v, out = t("q", 2, 4, 64), t("k", 2, 2, 64), t("v", 2, 2, 64), t("out", 2, 4, 64)
        norm, lse = t("norm", 64, dtype=torch.float32), t("lse", 2, 4, dtype=torch.float32)
        positions = t("positions", 2, **ints)
        return (lambda: attention.rope_append(FakeDevice, q, k, v, cache, batch, rope, out, q_norm=norm, k_norm=norm,
                                              positions=positions, stream=1),
                lambda: attention.prompt_attention(FakeDevice, q, cache, batch, out, lse=lse, stream=1),
                lambda: attention.decode_attention(FakeDevice, q, cache, batch, out, prefix=prefix, lse=lse, stream=1))

    for call in make(None):
        call()
    assert len(library.calls) == 3
    library.calls.clear()
    for where, callers in (("cache", (0, 1, 2)), ("batch", (0, 1, 2)), ("q", (0, 1, 2)), ("out", (0, 1, 2)), ("k", (0,)),
                           ("v", (0,)), ("rope", (0,)), ("norm", (0,)), ("positions", (0,)), ("lse", (1, 2)),
                           ("prefix", (2,))):
        for i in callers:
            with pytest.raises(ValueError, match="cuda:1"):
                make(where)[i]()
    assert library.calls == []


def test_synchronize_waits_for_the_stream_that_was_given(monkeypatch):
    """0 is the default stream here as in the operators: what they enqueued there is waited for, and its errors are read."""
    from voxwerk_b200 import sampler
    library = Library()
    monkeypatch.setattr(sampler, "lib", library)
    device = sampler.Device.__new__(sampler.Device)
    device._h, device.device = None, 0
    monkeypatch.setattr(sampler.Device, "handle", None)
    for stream, handle in ((None, None), (0, 1), (0x7770, 0x7770)):
        library.calls.clear()
        device.synchronize(stream)
        assert library.calls == [("vw_synchronize", handle)]
