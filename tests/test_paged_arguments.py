"""CPU-only checks of what the paged cache's Python calls refuse and where they allocate, with
tensors that only claim to lie on a GPU; the library is replaced by a recorder, so nothing runs."""
import contextlib
import importlib
import types

import pytest

torch = pytest.importorskip("torch")
g2 = importlib.import_module("cuda-gpt2-inference_amd")


class OnGpu(torch.Tensor):
    """A host tensor that says it is on GPU `at`."""

    @staticmethod
    def of(shape, dtype=torch.float32, at=1):
        t = torch.zeros(shape, dtype=dtype).as_subclass(OnGpu)
        t.at = at
        return t

    at = 1  # of views
    is_cuda = property(lambda self: True)

    def get_device(self):
        return self.at


class Recorder:
    """Stands in for the library: takes every call for a good one."""

    def __init__(self, **results):
        self.calls, self.results = [], results

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return self.results.get(name, 0)
        return call


@pytest.fixture
def library(monkeypatch):
    r = Recorder(attention_decode_paged_workspace=g2.PAGED_COUNTER_BYTES + 1024)
    monkeypatch.setattr(g2, "lib", lambda: r)
    return r


@pytest.fixture
def cache(monkeypatch, library):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    return g2.PagedCache(OnGpu.of((8, 2, 16, 64)), OnGpu.of((8, 2, 16, 64)), OnGpu.of((2, 4), torch.int32))


def step(cache, **other):
    a = dict(out=OnGpu.of((2, 4 * 64)), cache=cache, inp=OnGpu.of((2, 8 * 64)), lengths=OnGpu.of((2,), torch.int32), B=2, NH=4)
    a.update(other)
    g2.attention_decode_paged(**a)


def test_a_workspace_on_another_gpu_is_refused(cache, library):
    step(cache)
    step(cache, workspace=OnGpu.of((g2.PAGED_COUNTER_BYTES,), torch.uint8))
    assert [name for name, _ in library.calls] == ["attention_decode_paged_status"] * 2
    with pytest.raises(TypeError, match="workspace.*cuda:1"):
        step(cache, workspace=OnGpu.of((g2.PAGED_COUNTER_BYTES,), torch.uint8, at=0))
    with pytest.raises(TypeError, match="workspace.*cuda:1"):
        step(cache, workspace=bytearray(g2.PAGED_COUNTER_BYTES))
    with pytest.raises(ValueError, match="contiguous"):
        step(cache, workspace=OnGpu.of((2 * g2.PAGED_COUNTER_BYTES,), torch.uint8)[::2])
    assert len(library.calls) == 2, "a refused call reached the library"


@pytest.mark.parametrize("launchers", [None, 0x5000])
def test_a_workspace_is_zeroed_on_the_stream_of_the_launchers(cache, library, monkeypatch, launchers):
    """Its counters have to be zero when the first call's kernel reads them, whatever torch's own
    current stream has to do before."""
    library.results["gpt2hip_get_stream"] = launchers
    order, current = [], ["torch's current stream"]

    @contextlib.contextmanager
    def stream(s):
        current.append(s.cuda_stream)
        yield
        current.pop()

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda raw, device=None: types.SimpleNamespace(cuda_stream=raw))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: types.SimpleNamespace(cuda_stream=0))
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, **k: (order.append(current[-1]), zeros(*a, **{**k, "device": "cpu"}))[1])
    space = g2.attention_decode_paged_workspace(cache, 2, 4)
    assert space.nbytes == g2.PAGED_COUNTER_BYTES + 1024 and not space.any()
    assert order == [launchers or 0]


class Rows:
    """A float32 array of any shape and strides on GPU 1, without its memory."""

    dtype = torch.float32

    def __init__(self, shape, strides):
        self.shape, self.strides = shape, strides

    def stride(self):
        return self.strides

    def get_device(self):
        return 1

    def data_ptr(self):
        return 1 << 20


WRAP = 1 << 32  # what a C int cannot tell from 0


def test_strides_and_counts_beyond_a_c_int_are_refused(cache, library):
    starts, lengths = OnGpu.of((3,), torch.int32), OnGpu.of((2,), torch.int32)
    step(cache, inp=Rows((2, 512), (2 ** 31 - 1, 1)))
    g2.kv_store_paged(cache, Rows((5, 512), (512, 1)), starts, lengths, 5, 2, 4)
    del library.calls[:]
    for strides in ((WRAP + 512, 1), (2 ** 31, 1)):
        with pytest.raises(ValueError, match="32 bits"):
            step(cache, inp=Rows((2, 512), strides))
        with pytest.raises(ValueError, match="32 bits"):
            g2.kv_store_paged(cache, Rows((5, 512), strides), starts, lengths, 5, 2, 4)
    for N in (WRAP + 5, 2 ** 31, -WRAP + 5):
        with pytest.raises(ValueError, match="32 bits"):
            g2.kv_store_paged(cache, Rows((WRAP + 9, 512), (512, 1)), starts, lengths, N, 2, 4)
    for NH in (WRAP + 4, -WRAP + 4):
        with pytest.raises(ValueError, match="32 bits"):
            g2.kv_store_paged(cache, Rows((5, 64 * WRAP + 512), (512, 1)), starts, lengths, 5, 2, NH)
    assert not library.calls


def test_evict_and_workspace_refuse_numbers_beyond_a_c_int(cache, library):
    other = g2.PagedCache(cache.keys, cache.values, OnGpu.of((2, 4), torch.int32))
    arrays = [OnGpu.of((2, 2, 16), torch.int32), OnGpu.of((2, 2, 64)), OnGpu.of((2,), torch.int32), OnGpu.of((2, 2, 64)),
              OnGpu.of((2,), torch.int32)]
    g2.kv_evict_paged(other, cache, *arrays, 2, 16, 4)
    del library.calls[:]
    for recent in (WRAP + 4, -WRAP + 4):
        with pytest.raises(g2.GPT2HipError, match="recent"):
            g2.kv_evict_paged(other, cache, *arrays, 2, 16, recent)
    with pytest.raises(g2.GPT2HipError, match="budget"):
        g2.kv_evict_paged(other, cache, Rows((2, 2, WRAP + 16), (2 * WRAP, WRAP, 1)), *arrays[1:], 2, WRAP + 16, 4)
    for B, NH in ((WRAP + 2, 4), (2, WRAP + 4), (-WRAP + 2, 4)):
        with pytest.raises(g2.GPT2HipError, match="arguments"):
            g2.attention_decode_paged_workspace(cache, B, NH)
    assert not library.calls


def test_a_cache_of_more_pages_than_a_c_int_counts_is_refused(cache):
    class Wide(OnGpu):
        shape = property(lambda self: torch.Size((WRAP + 8, 2, 16, 64)))

    keys = torch.zeros((8, 2, 16, 64)).as_subclass(Wide)
    with pytest.raises(ValueError, match="32 bits"):
        g2.PagedCache(keys, keys, OnGpu.of((2, 4), torch.int32))
