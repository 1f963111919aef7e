"""That attention_decode_paged counts every position of every sequence once, however a call is cut
into tiles, waves and ranges.

Counting.  With queries of 0 every score is 0 and every weight exactly 1 before the division.
Values are whole numbers of -8 .. 8 without 0, so that all partial sums are whole numbers (in an
fp16 cache with shared keys: multiples of 2^14) below 2^24 of their unit and exact; what is rounded
is one division by n, and the powers of two that parts meet with are exact or off by 2^-22 of the
sum.  So out * n is the sum of the values to |sum| 2^-20 <= 8 n 2^-20, below 1/4 for n <= 32768,
while a position that is lost, or seen twice, or taken for another one, moves some channel by 1 or
more; and every weight is G / n to (G + 8) 2^-23.

A bound for random scores that stays useful on long caches.  u = 2^-24, x = s log2(e) base-2
scores, X = max |x|, A = max sum_j |q_j k_j| log2(e) / sqrt(HS), T = steps of a wave, at most
n / (rows that a workgroup's waves take per step) + 1.
* A score is off by 2 (HS + 4) u A (twice the usual bound, for sums inside a matrix instruction).
* A term is exp2(x - m1) exp2(m1 - m2) ... with rising maxima m1 <= m2 <= ..: each difference is
  rounded relative to itself and they add up to m - x <= 2 X, so the exponents are off by 2 u X in
  all, and by 2 u (X + 16) where a maximum is kept 14 lower.
* Each exp2 is off by 2 u and its product by u: at most T + 48 of them (one per step; eight ranges
  share one when they are joined, at most 256 ranges; row groups, waves, slices one each).
E = ln2 (2 (HS + 4) u A + 2 u X + 2 u (X + 16)) + 3 (T + 48) u bounds a term's relative error.  A
term goes through at most D = (rows of a step) T + 320 additions (a step's rows one after the other,
lanes, waves, ranges), the denominator through as many: |out - exact| <= 2 (E + D u) sum_i p_i |v_i|."""
import importlib
import math

import pytest
import torch

from test_paged_gpu import TYPES, Case, say, spread

g2 = importlib.import_module("cuda-gpt2-inference_amd")

U = 2.0 ** -24


def counting(seed, kind, B, NH, KVH, HS, page, lengths, max_len):
    """A Case whose queries are 0 and whose values are whole numbers of -8 .. 8 without 0."""
    c = Case(seed, kind, B, NH, KVH, HS, page, lengths, max_len)

    def whole(shape):
        x = torch.randint(1, 9, shape, generator=c.g)
        return torch.where(torch.rand(shape, generator=c.g) < 0.5, -x, x).double()

    for b, n in enumerate(lengths):
        n = max(n, 0)
        c.v64[b] = whole((KVH, n, HS))
        m = min(n, c.cap)
        used = -(-m // page)
        rows = torch.full((KVH, used * page, HS), float("nan"), dtype=c.kind)
        rows[:, :m] = c.v64[b][:, :m].to(c.kind)
        c.values[c.table[b, :used].long()] = rows.view(KVH, used, page, HS).transpose(0, 1)
    c.inp[:, : NH * HS] = 0
    c.inp[:, (NH + KVH) * HS:] = whole((B, KVH * HS)).float()
    return c


def miscounted(out, v):
    """out (KVH, G, HS) of one row, v (KVH, n, HS): where out is not the mean of the n values."""
    return (out.double() * v.shape[1] - v.sum(1)[:, None]).abs() >= 0.25


def check_counts(c, append=True, weights=False, workspace="full"):
    cache = c.gpu()
    B, NH, KVH, HS = c.B, c.NH, c.KVH, c.HS
    G = NH // KVH
    inp = c.inp.cuda() if append else c.inp[:, : NH * HS].contiguous().cuda()
    out = torch.full((B, NH * HS), 99.0, device="cuda")
    ws = None
    if workspace == "full":
        ws = g2.attention_decode_paged_workspace(cache, B, NH, weights=weights)
    elif workspace:
        ws = torch.zeros(workspace, dtype=torch.uint8, device="cuda")
    if ws is not None:
        ws[g2.PAGED_COUNTER_BYTES:] = 0xFF
    w = wo = None
    if weights:
        w = torch.zeros((B, KVH, c.cap), device="cuda")
        wo = torch.full_like(w, -5.0)
    g2.attention_decode_paged(out, cache, inp, c.dl, B, NH, append=append, weights_in=w, weights_out=wo, workspace=ws)
    out = out.cpu().view(B, KVH, G, HS)
    for b, n in enumerate(c.lengths):
        total = n + (1 if append else 0)
        if n < 0 or total > c.cap or total == 0:
            continue
        assert total <= 32768
        _, v = c.rows(b, append)
        assert not miscounted(out[b], v).any(), f"row {b} n={n}"
        if weights:
            got = wo[b].cpu().double()
            assert ((got[:, :total] * total / G - 1).abs() <= (G + 8) * 2 * U).all(), f"weights of row {b} n={n}"
            assert (got[:, total:] == -5).all()


def test_the_count_shows_every_position_lost_repeated_or_mistaken():
    """On the CPU: at the shapes below, outputs as they would be with one mistake each."""
    for HS, n in ((8, 30000), (8, 1000), (20, 12000), (64, 6000), (16, 17)):
        c = counting(HS + n, "f32", 1, 1, 1, HS, 16, [n], n + 1)
        v = c.rows(0, True)[1]
        total, N = v.sum(1), v.shape[1]
        assert not miscounted((total / N).float()[:, None], v).any()
        lost = (total - v[0]) / (N - 1)         # position by position, with the sum of weights ..
        lost_above = (total - v[0]) / N          # .. and without
        twice = (total + v[0]) / (N + 1)
        for out in (lost, lost_above, twice):
            assert miscounted(out.float()[None], v).any(-1).all(), (HS, n)
        for step in (1, 4, 16, 64, 128):
            if step < N:
                other = (total - v[0, step:] + v[0, :-step]) / N
                # two positions may hold the same eight numbers; no test passes for many of them
                alike = (v[0, step:] == v[0, :-step]).all(-1)
                assert torch.equal(miscounted(other.float()[None], v).any(-1)[0], ~alike) and alike.sum() < 3


SPLIT = [  # NH, KVH, HS, page, cap
    (2, 2, 64, 16, 6000), (4, 2, 128, 24, 4000), (3, 1, 80, 1, 5000), (8, 1, 96, 7, 5000), (40, 2, 64, 16, 5000),
    (5, 1, 33, 16, 6000), (2, 1, 256, 32, 2000), (16, 2, 200, 50, 2500), (1, 1, 8, 16, 30000), (2, 1, 20, 1000, 12000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("NH,KVH,HS,page,cap", SPLIT)
def test_counts_of_split_sequences(kind, NH, KVH, HS, page, cap):
    say(f"count split {kind} NH={NH} KVH={KVH} HS={HS} page={page} cap={cap}")
    c = counting(NH + HS, kind, 5, NH, KVH, HS, page, [cap, cap - 1, 1, -1, cap // 2 + 3], cap + 1)
    one = 5 * NH * (HS + 4) * 4
    for workspace in ("full", None, g2.PAGED_COUNTER_BYTES + 2 * one, g2.PAGED_COUNTER_BYTES + 5 * one):
        check_counts(c, workspace=workspace)
    check_counts(c, append=False, weights=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("B,NH,KVH,HS,top", [
    (140, 4, 4, 64, 150), (140, 8, 4, 128, 150), (64, 4, 4, 64, 1100), (64, 4, 4, 128, 600), (64, 4, 4, 256, 300),
    (64, 4, 4, 32, 2100), (90, 12, 3, 64, 200), (90, 15, 3, 128, 100), (90, 12, 3, 256, 60), (170, 16, 4, 64, 60),
    (2, 20, 1, 96, 9000), (3, 1, 1, 64, 20000), (8, 32, 8, 128, 6000),
])
def test_counts_of_every_form_of_the_kernels(kind, B, NH, KVH, HS, top):
    say(f"count {kind} B={B} NH={NH} KVH={KVH} HS={HS} top={top}")
    c = counting(B + HS, kind, B, NH, KVH, HS, 16, spread(B, top), top + 1)
    check_counts(c)
    check_counts(c, append=False, weights=True)


@pytest.mark.gpu
@pytest.mark.parametrize("append", [True, False])
@pytest.mark.parametrize("B,NH,KVH,cap,lengths", [
    (3, 2, 2, 4000, [4000, 0, 700]), (5, 1, 1, 6000, [6000, 1, -1, 5999, 2500]), (4, 6, 2, 3000, [3001, 9000, 2999, 10]),
    (1, 1, 1, 32000, [31999]), (2, 3, 3, 32000, [31999, 1]), (8, 1, 1, 20000, [19999] + [3] * 7),
    (64, 1, 1, 4000, None), (65, 1, 1, 4000, None), (130, 2, 1, 2000, None), (200, 1, 1, 3200, None),
    (256, 1, 1, 2000, None), (257, 1, 1, 2000, None),
])
def test_counts_of_dealt_sequences(B, NH, KVH, cap, lengths, append):
    say(f"count dealt B={B} NH={NH} KVH={KVH} cap={cap} append={append}")
    for kind in ("f16", "f32"):
        check_counts(counting(B + NH, kind, B, NH, KVH, 64, 16, lengths or spread(B, cap), cap), append=append, weights=B % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("NH,KVH", [(2, 2), (2, 1), (8, 1)])
def test_counts_around_the_ends_of_tiles_and_ranges(kind, NH, KVH):
    lengths = [0, 1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 384, 385, 511, 512, 513, 640]
    say(f"count lengths {kind} NH={NH} KVH={KVH}")
    for HS in (64, 128):
        check_counts(counting(NH, kind, len(lengths), NH, KVH, HS, 24, lengths, 700))
        for n in (128, 4095, 4096, 4097):
            check_counts(counting(NH + n, kind, 1, NH, KVH, HS, 16, [n], 4200), weights=True)


# ---------------------------------------------------------------- random scores, long caches
def rows_per_step(kind, G, HS):
    """(rows a workgroup's waves take per step, rows a term is added to one after the other in a step),
    the least and the most that any form of the kernels has."""
    size = TYPES[kind].itemsize
    if HS * size % 16:
        return (32, 8) if G < 3 else (16, 4)
    if G < 3:
        lanes = 8
        while lanes * 16 < HS * size:
            lanes *= 2
        return (32 if G == 1 else 16) * 64 // lanes, 8
    blocks = (2 if size == 4 else 4) if HS <= 64 else (1 if size == 4 else 2) if HS <= 128 else 1
    return 4 * 16 * blocks, 16 * blocks


def useful_bound(kind, q, k, v, p, s):
    HS, G, n = q.shape[-1], q.shape[-2], k.shape[-2]
    log2e = 1 / math.log(2)
    A = torch.matmul(q.abs(), k.abs().transpose(-1, -2)).amax(-1, keepdim=True) * log2e / math.sqrt(HS)
    X = s.abs().amax(-1, keepdim=True) * log2e
    step, chain = rows_per_step(kind, G, HS)
    T = n // step + 1
    E = math.log(2) * (2 * (HS + 4) * U * A + 2 * U * X + 2 * U * (X + 16)) + 3 * (T + 48) * U
    D = chain * T + 320
    return 2 * (E + D * U) * torch.matmul(p, v.abs()) + 2.0 ** -126 * v.abs().sum(-2, keepdim=True)


def exact_row(c, b, append=True):
    k, v = c.rows(b, append)
    q = c.inp[b, : c.NH * c.HS].double().reshape(c.KVH, c.NH // c.KVH, c.HS)
    s = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(c.HS)
    p = torch.softmax(s, -1)
    return q, k, v, p, s


LONG = [(1, 1, 8, 30000), (2, 2, 64, 20000), (2, 1, 128, 9000), (3, 1, 64, 20000), (8, 1, 128, 9000), (16, 1, 64, 12000),
        (4, 2, 200, 5000), (3, 1, 33, 6000)]


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("NH,KVH,HS,n", LONG)
def test_the_bound_shows_a_shortest_range_left_out(kind, NH, KVH, HS, n):
    """On the CPU: an output of zeros, and one without the 256 first or last positions, is outside."""
    c = Case(NH + HS, kind, 1, NH, KVH, HS, 16, [n], n + 1, keys_std=0.5)
    q, k, v, p, s = exact_row(c, 0)
    exp, tol = torch.matmul(p, v), useful_bound(kind, q, k, v, p, s)
    assert (exp.abs() > tol).any(-1).all(), "a head of zeros would pass"
    for left in (slice(256, None), slice(None, -256)):
        out = torch.matmul(p[..., left] / p[..., left].sum(-1, keepdim=True), v[:, left])
        assert ((out - exp).abs() > tol).any(-1).all(), "a head would pass"


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("NH,KVH,HS,n", LONG)
def test_long_caches_within_the_bound(kind, NH, KVH, HS, n):
    say(f"long {kind} NH={NH} KVH={KVH} HS={HS} n={n}")
    lengths = [n, n // 3, 200]
    c = Case(NH + HS, kind, 3, NH, KVH, HS, 16, lengths, n + 1, keys_std=0.5)
    cache = c.gpu()
    for ws in (g2.attention_decode_paged_workspace(cache, 3, NH), None):
        out = torch.zeros((3, NH * HS), device="cuda")
        g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 3, NH, workspace=ws)
        for b in range(3):
            q, k, v, p, s = exact_row(c, b)
            err = (out[b].cpu().double().view(KVH, NH // KVH, HS) - torch.matmul(p, v)).abs()
            tol = useful_bound(kind, q, k, v, p, s)
            say(f"  row {b}: worst {float((err / tol).max()):.3f} of the bound")
            assert (err <= tol).all()
