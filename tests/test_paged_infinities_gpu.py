"""Infinities and NaN in the values of the paged cache, on the GPU: an output is what
sum_i p_i v_i is by IEEE arithmetic, whichever kernel a call takes -- an infinity where values of
one sign are infinite, a NaN where both signs are or a value is a NaN -- and every channel that
holds finite values stays within the bound of a cache without any.

The softmax weights of these rows are far above 2^-126 (scores of a few units), so that in fp32
as in float64 none of them is 0.  fp16 caches make such values themselves: 1e5 is stored as inf."""
import importlib

import pytest
import torch

from test_paged_gpu import TYPES, Case, attention_bound, same_bits, say

g2 = importlib.import_module("cuda-gpt2-inference_amd")

pytestmark = pytest.mark.gpu

INF = float("inf")


def put(c, b, i, h, channel, x):
    """Makes x the value of position i of sequence b, kv head h, in the pages and in float64."""
    c.values[c.table[b, i // c.page], h, i % c.page, channel] = x
    c.v64[b][h, i, channel] = x


def check(c, append=True, workspace=True, weights=False):
    """Outputs against float64: the same infinities and NaN, and what is finite within the bound."""
    cache = c.gpu()
    B, NH, KVH, HS = c.B, c.NH, c.KVH, c.HS
    out = torch.full((B, NH * HS), 7.0, device="cuda")
    ws = g2.attention_decode_paged_workspace(cache, B, NH, weights=weights) if workspace else None
    w = wo = None
    if weights:
        w = torch.zeros((B, KVH, c.cap), device="cuda")
        wo = torch.full_like(w, -5.0)
    inp = c.inp.cuda() if append else c.inp[:, : NH * HS].contiguous().cuda()
    g2.attention_decode_paged(out, cache, inp, c.dl, B, NH, append=append, weights_in=w, weights_out=wo, workspace=ws)
    torch.cuda.synchronize()
    for b in range(B):
        k, v = c.rows(b, append)
        q = c.inp[b, : NH * HS].double().reshape(KVH, NH // KVH, HS)
        s = torch.matmul(q, k.transpose(1, 2)) / HS ** 0.5
        p = torch.softmax(s, -1)
        # one column at a time: a product over blocks may not multiply an infinity by a weight alone
        exp = torch.stack([(p * v[:, None, :, d]).sum(-1) for d in range(HS)], -1)
        finite_v = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
        tol, ptol = attention_bound(q, k, finite_v, p, s)
        got = out[b].cpu().double().view(KVH, NH // KVH, HS)
        special = ~torch.isfinite(exp)
        assert torch.equal(torch.isnan(got), torch.isnan(exp)), f"row {b}: NaN in the wrong places"
        assert torch.equal(got[special & ~torch.isnan(exp)], exp[special & ~torch.isnan(exp)]), f"row {b}: infinities"
        assert ((got - exp).abs() <= tol)[~special].all(), f"row {b}: {float((got - exp).abs()[~special].max()):.3e}"
        if weights:
            n = p.shape[-1]
            assert ((wo[b, :, :n].cpu().double() - p.sum(1)).abs() <= ptol + 2.0 ** -24 * p.sum(1)).all(), f"weights of row {b}"


FORMS = [  # NH, KVH, HS, page, lengths
    (1, 1, 64, 16, [40, 1000, 333]), (4, 2, 64, 16, [40, 1000, 333]),           # the kernel of one or two heads
    (6, 2, 64, 16, [40, 1000, 333]), (5, 1, 128, 24, [17, 900, 64]),            # matrix instructions, one tile to several
    (16, 1, 64, 16, [16, 700, 255]), (16, 2, 200, 7, [33, 500, 129]), (9, 1, 72, 16, [15, 600, 128]),
    (20, 1, 96, 16, [31, 400, 65]), (40, 2, 64, 32, [50, 300, 90]),             # more heads than a workgroup takes
    (8, 1, 128, 16, [6000, 3000, 5]), (3, 1, 64, 16, [9000, 1, 8999]),          # split over the length
    (4, 1, 20, 16, [40, 300, 5]),                                               # rows of no whole 16 bytes
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("NH,KVH,HS,page,lengths", FORMS)
def test_infinite_values(kind, NH, KVH, HS, page, lengths):
    say(f"infinite values {kind} NH={NH} KVH={KVH} HS={HS} lengths={lengths}")
    c = Case(NH + HS, kind, 3, NH, KVH, HS, page, lengths, max(lengths) + 1)
    for b, n in enumerate(lengths):
        h = b % KVH
        if b == 2:
            continue  # a sequence of finite values beside them
        put(c, b, 0, h, 1, INF)                                  # the first position
        put(c, b, n - 1, h, HS - 1, -INF)                        # the last one, in the last channel
        put(c, b, n // 3, h, 2, INF), put(c, b, n // 2, h, 2, -INF)  # both signs: NaN
        put(c, b, n // 2, h, 3, float("nan"))
        for i in range(0, n, 3):
            put(c, b, i, h, 4, -INF)                             # in every tile
        # where the first head of the group looks most: its weight is exactly 1 relative to the maximum
        q = c.inp[b, h * (NH // KVH) * HS:][:HS].double()
        put(c, b, int((c.k64[b][h] @ q).argmax()), h, 5, INF)
    for workspace in (True, False):
        check(c, workspace=workspace, weights=workspace)
    check(c, append=False)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("NH,KVH", [(2, 2), (8, 2), (16, 1)])
def test_a_new_row_whose_value_is_stored_as_an_infinity(kind, NH, KVH):
    """What a call appends is part of its own output, and of the next call's."""
    say(f"new row {kind} NH={NH} KVH={KVH}")
    n = 100
    c = Case(5, kind, 2, NH, KVH, 64, 16, [n, n], n + 2)
    values = c.inp[0, (NH + KVH) * 64:].view(KVH, 64)
    values[0, 6] = 1e5 if kind == "f16" else INF
    values[KVH - 1, 9] = -1e5 if kind == "f16" else -INF
    check(c)
    # the same row among the positions held
    for b in range(2):
        k, v = c.rows(b, True)
        c.k64[b], c.v64[b] = k, v
        c.keys[c.table[b, n // 16], :, n % 16] = k[:, n].to(c.kind)
        c.values[c.table[b, n // 16], :, n % 16] = v[:, n].to(c.kind)
    c.lengths = [n + 1, n + 1]
    check(c, append=False)
    check(c, append=False, workspace=False)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("NH", [3, 16])
def test_an_infinite_value_of_a_position_that_weighs_nothing(kind, NH):
    """Score -inf: the weight is 0 exactly, and 0 times an infinity is a NaN in that channel only."""
    say(f"weight 0 {kind} NH={NH}")
    n = 200
    c = Case(6, kind, 1, NH, 1, 64, 16, [n], n + 1)
    c.inp[0, : NH * 64: 64] = -1.0
    c.keys[c.table[0, 70 // 16], 0, 70 % 16, 0] = INF
    c.k64[0][0, 70, 0] = INF
    put(c, 0, 70, 0, 3, INF)
    put(c, 0, 71, 0, 4, INF)
    cache = c.gpu()
    out = torch.zeros((1, NH * 64), device="cuda")
    g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 1, NH)
    got = out.view(NH, 64).cpu()
    assert torch.isnan(got[:, 3]).all() and (got[:, 4] == INF).all()
    assert torch.isfinite(got[:, [d for d in range(64) if d not in (3, 4)]]).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_outputs_beside_infinities_keep_their_bits(kind):
    """Channels without an infinity are the same bits as in a cache that holds none."""
    n = 777
    c = Case(8, kind, 2, 12, 2, 128, 16, [n, 5000], 5001)
    cache = c.gpu()
    outs = []
    for value in (None, INF):
        if value is not None:
            for b, i in ((0, 3), (0, 700), (1, 4000)):
                c.dv[c.table[b, i // 16].long(), 0, i % 16, 11] = value
        out = torch.zeros((2, 12 * 128), device="cuda")
        g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 2, 12, append=True,
                                  workspace=g2.attention_decode_paged_workspace(cache, 2, 12))
        outs.append(out.view(2, 2, 6, 128).cpu())
    assert (outs[1][:, 0, :, 11] == INF).all()
    outs[1][:, 0, :, 11] = outs[0][:, 0, :, 11]
    assert same_bits(outs[0], outs[1])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("NH", [1, 8])
def test_sums_of_values_that_pass_fp32_are_not_finite(kind, NH):
    """Values are summed before the division: finite ones whose sum passes 2^128 leave an infinity or a
    NaN in their channel, never another number, and no trace in the other channels."""
    say(f"overflow {kind} NH={NH}")
    n = 2000
    c = Case(9, kind, 1, NH, 1, 64, 16, [n], n + 1)
    c.inp[:, : NH * 64] = 0
    plain = c.v64[0][0].clone()
    for i in range(n):
        put(c, 0, i, 0, 5, 3e38 if i % 64 < 32 else -1.5e38)   # both signs in every wave
        put(c, 0, i, 0, 6, 3e38)
        put(c, 0, i, 0, 7, 3e38 if i < n // 2 else -1.5e38)
    cache = c.gpu()
    for ws in (None, g2.attention_decode_paged_workspace(cache, 1, NH)):
        out = torch.zeros((1, NH * 64), device="cuda")
        g2.attention_decode_paged(out, cache, c.inp[:, : NH * 64].contiguous().cuda(), c.dl, 1, NH, append=False, workspace=ws)
        got = out.cpu().double().view(NH, 64)
        assert not torch.isfinite(got[:, 6]).any()
        for d in (5, 7):
            # not finite, or right where a sum happens to stay below 2^128
            exact = float(c.v64[0][0, :, d].mean())
            assert (~torch.isfinite(got[:, d]) | ((got[:, d] - exact).abs() <= 2.0 ** -24 * 4 * n * 3e38)).all()
        others = [d for d in range(64) if d not in (5, 6, 7)]
        assert ((got[:, others] - plain[:, others].mean(0)).abs() <= 4 * n * 2.0 ** -24 * plain[:, others].abs().mean(0)).all()
