"""CPU-only: sizes at the ends of what the paged cache's launchers take.  A launch holds fewer than
2^32 threads in all; calls that would need more are refused before anything runs."""
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


def refused(rc):
    message = g2.lib().gpt2hip_last_error()
    assert rc == 1 and b"grid too large" in message, (rc, message)


@pytest.mark.parametrize("N", [(1 << 26) - 3, 1 << 27, (1 << 31) - 3, (1 << 31) - 1])
def test_store_refuses_more_rows_than_a_launch_holds(N):
    refused(g2.lib().kv_store_paged_status(ctypes.addressof(cache()), FAKE, 8 * 64, FAKE, FAKE, N, 2, 4))


@pytest.mark.parametrize("B,NH,head_size", [(1 << 23, 2, 64), (1 << 24, 2, 64), (1 << 24, 8, 64), (1 << 30, 2, 64),
                                            ((1 << 31) - 1, 2, 64), (1 << 23, 2, 7), (1 << 23, 8, 250)])
def test_attend_refuses_more_workgroups_than_a_launch_holds(B, NH, head_size):
    c = cache(head_size=head_size)
    stride = (NH + 4) * head_size
    refused(g2.lib().attention_decode_paged_status(FAKE, ctypes.addressof(c), FAKE, stride, FAKE, None, None, B, NH, 1, None, 0))


@pytest.mark.parametrize("max_pages,budget,B", [(4, 32, 1 << 24), (4, 64, (1 << 31) - 1), (512, 32, 1 << 21),
                                                (512, 4096, 1 << 20), (1 << 12, 1 << 15, 1 << 20)])
def test_evict_refuses_more_workgroups_than_a_launch_holds(max_pages, budget, B):
    c, d = cache(max_pages=max_pages), cache(table=3 * FAKE, max_pages=max_pages)
    refused(g2.lib().kv_evict_paged_status(ctypes.addressof(d), ctypes.addressof(c), FAKE, FAKE, FAKE, 2 * FAKE, 2 * FAKE, B,
                                           budget, 4))
