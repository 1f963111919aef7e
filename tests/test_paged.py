"""CPU-only checks of the paged key/value cache's launchers: every refusal, before any HIP call."""
import ctypes
import importlib

import pytest

g2 = importlib.import_module("cuda-gpt2-inference_amd")
FAKE = 1 << 20  # a non-null, well-aligned address that nothing dereferences


def cache(**other):
    c = dict(keys=FAKE, values=FAKE, table=FAKE, type=0, num_pages=8, page_size=16, max_pages=4, kv_heads=2,
             head_size=64)
    c.update(other)
    return g2.GPT2PagedCache(**c)


def store(c, inp=FAKE, stride=8 * 64, starts=FAKE, lengths=FAKE, N=3, B=2, NH=4):
    return g2.lib().kv_store_paged_status(ctypes.addressof(c) if c else None, inp, stride, starts, lengths, N, B, NH)


def attend(c, out=FAKE, inp=FAKE, stride=8 * 64, lengths=FAKE, win=None, wout=None, B=2, NH=4, append=1, ws=None,
           nbytes=0):
    return g2.lib().attention_decode_paged_status(out, ctypes.addressof(c) if c else None, inp, stride, lengths, win,
                                                  wout, B, NH, append, ws, nbytes)


def evict(d, s, kept=FAKE, wout=FAKE, lout=FAKE, win=2 * FAKE, lengths=2 * FAKE, B=2, budget=32, recent=4):
    return g2.lib().kv_evict_paged_status(ctypes.addressof(d) if d else None, ctypes.addressof(s) if s else None, kept,
                                          wout, lout, win, lengths, B, budget, recent)


def message():
    return g2.lib().gpt2hip_last_error()


BAD_CACHES = [
    (dict(type=3), b"type"), (dict(type=-1), b"type"),
    (dict(num_pages=0), b"shape"), (dict(page_size=0), b"shape"), (dict(page_size=-4), b"shape"),
    (dict(max_pages=0), b"shape"), (dict(kv_heads=0), b"shape"), (dict(head_size=0), b"shape"),
    (dict(head_size=257), b"256"),
    (dict(max_pages=1 << 26, page_size=16), b"2^30"),
    (dict(num_pages=1 << 27, page_size=16, kv_heads=2), b"2^32"),
    (dict(keys=None), b"null"), (dict(values=None), b"null"), (dict(table=None), b"null"),
    (dict(keys=FAKE + 2), b"aligned"), (dict(type=1, values=FAKE + 1), b"aligned"),
]


@pytest.mark.parametrize("other,word", BAD_CACHES, ids=[str(i) for i in range(len(BAD_CACHES))])
def test_every_launcher_refuses_a_bad_cache(other, word):
    bad, good = cache(**other), cache(keys=3 * FAKE)
    for rc in (store(bad), attend(bad), evict(bad, good), evict(good, bad)):
        assert rc == 1 and word in message(), message()
    assert g2.lib().attention_decode_paged_workspace(ctypes.addressof(bad), 2, 4, 0) == 0


def test_store_refusals():
    c = cache()
    assert store(None) == 1 and b"null cache" in message()
    assert store(c, N=-1) == 1 and store(c, B=-1) == 1 and store(c, NH=-1) == 1
    assert store(c, stride=8 * 64 - 1) == 1 and b"stride" in message()
    for k in ("inp", "starts", "lengths"):
        assert store(c, **{k: None}) == 1 and b"null" in message()
    assert store(c, N=0, inp=None) == 0 and store(c, B=0, lengths=None) == 0


def test_attend_refusals():
    c = cache()
    assert attend(None) == 1 and b"null cache" in message()
    assert attend(c, B=-1) == 1 and attend(c, NH=0) == 1 and attend(c, NH=3) == 1
    assert attend(c, stride=8 * 64 - 1) == 1 and b"stride" in message()
    assert attend(c, append=0, stride=4 * 64 - 1) == 1 and b"stride" in message()
    assert attend(c, win=FAKE) == 1 and attend(c, wout=FAKE) == 1 and b"together" in message()
    for k in ("out", "inp", "lengths"):
        assert attend(c, **{k: None}) == 1 and b"null" in message()
    assert attend(c, ws=FAKE + 64, nbytes=1 << 20) == 1 and b"256-byte" in message()
    # weights need room for the counters, the scores and the rows' maxima and sums
    least = g2.PAGED_COUNTER_BYTES + 2 * 4 * (64 + 2) * 4
    assert attend(c, win=FAKE, wout=FAKE) == 1 and str(least).encode() in message()
    assert attend(c, win=FAKE, wout=FAKE, ws=FAKE, nbytes=least - 1) == 1
    assert attend(c, B=0, out=None, inp=None) == 0


def test_workspace_size():
    f = g2.lib().attention_decode_paged_workspace
    c = cache(max_pages=64)
    p = ctypes.addressof(c)
    assert f(p, 0, 4, 0) == 0 and f(p, 2, 3, 0) == 0 and f(None, 2, 4, 0) == 0
    plain, scored = f(p, 2, 4, 0), f(p, 2, 4, 1)
    assert g2.PAGED_COUNTER_BYTES < plain and scored - plain == 2 * 4 * (1024 + 2) * 4
    # many sequences need no split, few long ones do
    assert f(p, 4000, 4, 0) == g2.PAGED_COUNTER_BYTES and f(p, 1, 4, 0) >= g2.PAGED_COUNTER_BYTES + 4 * 66 * 4 * 4


def test_evict_refusals():
    d, s = cache(table=5 * FAKE), cache()
    assert evict(None, s) == 1 and evict(d, None) == 1
    assert evict(cache(table=5 * FAKE, type=1), s) == 1 and b"differ" in message()
    assert evict(cache(table=5 * FAKE, kv_heads=1), s) == 1 and evict(cache(table=5 * FAKE, head_size=32), s) == 1
    assert evict(d, s, B=-1) == 1 and evict(d, s, budget=0) == 1 and evict(d, s, recent=-1) == 1
    assert evict(d, s, budget=8, recent=9) == 1
    assert evict(d, s, budget=65) == 1 and b"does not fit" in message()
    assert evict(s, s) == 1 and b"pages of its own" in message()
    for k in ("kept", "wout", "lout", "win", "lengths"):
        assert evict(d, s, **{k: None}) == 1 and b"null" in message()
    assert evict(d, s, wout=2 * FAKE) == 1 and evict(d, s, lout=2 * FAKE) == 1 and b"inputs" in message()
    assert evict(d, s, B=0, kept=None) == 0


def test_python_wrapper_refuses_host_memory_and_wrong_shapes():
    torch = pytest.importorskip("torch")
    k = torch.zeros(4, 2, 16, 64)
    with pytest.raises(TypeError):
        g2.PagedCache(k, k, torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(TypeError):
        g2.PagedCache(k, k.half(), torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(TypeError):
        g2.PagedCache(k.double(), k.double(), torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(ValueError):
        g2.PagedCache(k, k[:2], torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(ValueError):
        g2.PagedCache(k, k, torch.zeros(4, dtype=torch.int32))
