"""The Python cache against torch's streams, without a GPU: every call waits
for torch's current stream and is waited for by it, unless it is the library's."""
import pytest
import torch


class Library:
    """The library with its stream and its launching calls replaced."""

    def __init__(self, real, log, stream):
        self.real, self.log, self.stream = real, log, stream

    def kq_b200_get_stream(self):
        return self.stream

    def kq_b200_set_stream(self, stream, _):
        self.log.append(("set", stream))
        return 0

    def kq_b200_order_stream(self, stream, library_first, _):
        first, then = (self.stream, stream) if library_first else (stream, self.stream)
        self.log.append((then, "waits for", first))
        return 0

    def __getattr__(self, name):
        if name in ("kq_b200_kv8_plan", "kq_b200_kv8_append", "kq_b200_kv8_read", "kq_b200_kv8_attend"):
            return lambda *_: self.log.append(("call", name)) or 0
        return getattr(self.real, name)


class Stream:
    def __init__(self, handle):
        self.cuda_stream = handle


@pytest.mark.parametrize("torch_stream,library", [(0, 7), (5, 7), (7, 7), (0, 1)])
def test_calls_in_the_order_of_torch(kq, monkeypatch, torch_stream, library):
    log = []
    real = kq.lib()
    monkeypatch.setattr(kq, "lib", lambda: Library(real, log, library))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: {3: torch_stream}[device], raising=False)
    cache = kq.Kv8Cache(1, 64, 16, 4, device="cpu")
    cache.device = 3
    step = kq.Kv8Step(1, 3, torch.zeros(1, 2, dtype=torch.int32), 16)
    one, row = torch.zeros(1, dtype=torch.int32), torch.zeros(3, 1, 64)
    calls = {"plan": lambda: cache.plan(step, one, one, one, one, one), "append": lambda: cache.append(step, row, row),
             "read": lambda: cache.read_pages(one, torch.zeros(2048)),
             "attend": lambda: cache.attend(step, row, row.clone(), scale=1.0)}
    for name, call in calls.items():
        log.clear()
        call()
        only = [("call", "kq_b200_kv8_" + name)]
        here = torch_stream or 1   # CUDA's name of the default stream
        assert log == (only if here == library else [(library, "waits for", here), *only, (here, "waits for", library)])


def test_set_stream_names_the_default_stream(kq, monkeypatch):
    """Handle 0 would be the library's own stream."""
    log = []
    real = kq.lib()
    monkeypatch.setattr(kq, "lib", lambda: Library(real, log, 7))
    for stream in (None, Stream(0), Stream(5)):
        kq.set_stream(stream)
    assert log == [("set", None), ("set", 1), ("set", 5)]
