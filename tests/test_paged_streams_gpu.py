"""The paged cache on streams other than torch's current one."""
import importlib

import pytest
import torch

from test_paged_gpu import Case, say

g2 = importlib.import_module("cuda-gpt2-inference_amd")

pytestmark = pytest.mark.gpu


def test_a_workspace_made_while_torchs_stream_is_busy():
    """The launchers run on a stream of their own; torch's current stream is held up by a kernel of
    some tens of milliseconds.  Memory that has been written before comes back as the workspace:
    it is zero when the split call reads its counters."""
    c = Case(70, "f16", 1, 2, 2, 64, 16, [6000], 6001)
    cache, inp = c.gpu(), c.inp.cuda()
    out = torch.zeros((1, 128), device="cuda")
    space = g2.attention_decode_paged_workspace(cache, 1, 2)
    assert space.nbytes > g2.PAGED_COUNTER_BYTES, "not a split call"
    g2.attention_decode_paged(out, cache, inp, c.dl, 1, 2, workspace=space)
    want = out.clone()
    size = space.nbytes
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        used = torch.full((size,), 3, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    del used, space
    try:
        g2.set_stream(side)
        for _ in range(3):
            out.zero_()
            torch.cuda.synchronize()
            say("torch's stream is held up")
            torch.cuda._sleep(50_000_000)
            mine = g2.attention_decode_paged_workspace(cache, 1, 2)
            g2.attention_decode_paged(out, cache, inp, c.dl, 1, 2, workspace=mine)
            side.synchronize()
            assert torch.equal(out, want)
            assert not mine[: g2.PAGED_COUNTER_BYTES].any()
            with torch.cuda.stream(side):
                mine.fill_(3)
            torch.cuda.synchronize()
            del mine
    finally:
        g2.set_stream(None)
