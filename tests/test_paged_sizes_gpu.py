"""The paged cache where a call would need more threads than a launch holds (2^32: the rest would be
left out without an error)."""
import importlib

import pytest
import torch

from test_paged_gpu import Case, say

g2 = importlib.import_module("cuda-gpt2-inference_amd")

pytestmark = pytest.mark.gpu


def test_attend_weights_of_a_table_wider_than_a_launch():
    """2^30 - 1024 positions that a table can name, five kv heads: the weights' launch would need
    more than 2^32 threads.  The lengths are short; 21 GB of accumulated weights and as much of
    workspace, of which next to nothing is touched."""
    KVH, HS, page, pages, n = 5, 8, 1024, (1 << 20) - 1, 3000
    assert KVH * pages * page > 1 << 32
    c = Case(80, "f16", 1, KVH, KVH, HS, page, [n], n + 1, spare=0)
    small = c.gpu()
    out, want = torch.zeros((1, KVH * HS), device="cuda"), torch.zeros((1, KVH * HS), device="cuda")
    w = torch.zeros((1, KVH, c.cap), device="cuda")
    g2.attention_decode_paged(want, small, c.inp.cuda(), c.dl, 1, KVH, weights_in=w, weights_out=w,
                              workspace=g2.attention_decode_paged_workspace(small, 1, KVH, weights=True))
    table = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
    table[:, : c.table.shape[1]] = c.table.cuda()
    cache = g2.PagedCache(c.dk, c.dv, table)
    wide = torch.empty((1, KVH, pages * page), device="cuda")
    wide[:, :, : n + 1000] = 0
    ws = g2.attention_decode_paged_workspace(cache, 1, KVH, weights=True)
    say(f"workspace {ws.nbytes / 2**30:.1f} GiB")
    g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 1, KVH, weights_in=wide, weights_out=wide, workspace=ws)
    exp, tol, p, ptol = c.expect(0, True)
    assert ((out[0].cpu().double() - exp).abs() <= tol).all()
    assert ((wide[0, :, : n + 1].cpu().double() - p).abs() <= ptol).all()
    assert not wide[:, :, n + 1: n + 1000].any()
    del wide, ws, cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_store_with_starts_far_in_front_of_the_rows(kind):
    """A sequence whose first row lies 2^31 in front of row 0: its positions do not fit and nothing
    is stored; one that begins a little in front of row 0 has its later rows here."""
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[kind]
    g = torch.Generator().manual_seed(81)
    rows = torch.randn((5, 2 * 2 * 8), generator=g)
    for start, length in ((-(1 << 31), 0), (-(1 << 31), (1 << 31) - 1), (-(1 << 31) + 3, 5), (-2, 7), (-2, 0), (0, (1 << 31) - 1)):
        say(f"starts {start} lengths {length}")
        keys = torch.full((4, 2, 4, 8), 9.0, dtype=dtype, device="cuda")
        values = keys.clone()
        table = torch.tensor([[2, 0, 3], [1, 1, 1]], dtype=torch.int32).cuda()
        g2.kv_store_paged(g2.PagedCache(keys, values, table), rows.cuda(), torch.tensor([start, 3, 3], dtype=torch.int32).cuda(),
                          torch.tensor([length, 0], dtype=torch.int32).cuda(), 5, 2, 0)
        want_k, want_v = torch.full((4, 2, 4, 8), 9.0, dtype=dtype), torch.full((4, 2, 4, 8), 9.0, dtype=dtype)
        for r in range(3):
            pos = length + r - start
            if pos < 12:
                at, slot = int(table[0, pos // 4]), pos % 4
                want_k[at, :, slot] = rows[r, :16].view(2, 8).to(dtype)
                want_v[at, :, slot] = rows[r, 16:].view(2, 8).to(dtype)
        assert torch.equal(keys.cpu(), want_k) and torch.equal(values.cpu(), want_v)
