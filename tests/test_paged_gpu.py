"""GPU parity of the paged key/value cache (kv_store_paged, attention_decode_paged,
kv_evict_paged) against plain float64 implementations of the same operators.

Tolerances of the attention.  With u = 2^-24 (half a step of fp32), x = s log2(e) the base-2
scores of one row and X = max |x|: the dot product of HS terms, the scaling of q and the constant
are off by at most (HS + 4) u A, A = max_i sum_j |q_j k_ij| log2(e) / sqrt(HS); the difference to
the running maximum by 2 u X; exp2 itself by 2 u relative.  A term that has been rescaled goes
through at most 24 more exp2 factors that matter less than it (the factors of a row group's
maxima multiply to one exp2, each rounded once, their arguments off by 2 u X each while the
maximum rises; a rise by less than one step changes nothing): R rescales at most, R <= tiles of
a wave + 8 joins.  A sum of n terms adds n u.  So each weight is off by
E = ln2 (2 (HS + 4) u A + 2 (R + 2) u X) + (R + 4) 2 u relative before the sums, and
|out - exact| <= (2 E + 2 (n + 8) u) sum_i p_i |v_i|; a weight (a sum over G heads, one division
each) <= (2 E + (n + G + 8) u) of its value plus u of what it is added to.
"""
import importlib
import math
import sys

import numpy as np
import pytest
import torch

g2 = importlib.import_module("cuda-gpt2-inference_amd")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def attention_bound(q, k, v, p, s):
    """(tolerance of out, tolerance of the weights summed over a group) as derived above; q (KVH, G, HS),
    k, v (KVH, n, HS), scores s and softmax p (KVH, G, n), all float64."""
    HS, G, n = q.shape[-1], q.shape[-2], k.shape[-2]
    log2e = 1 / math.log(2)
    A = float(torch.matmul(q.abs(), k.abs().transpose(-1, -2)).max()) * log2e / math.sqrt(HS)
    X = float(s.abs().max()) * log2e
    R = n / 4 + 8  # a tile holds at least one row, and a workgroup has four waves
    E = math.log(2) * (2 * (HS + 4) * U * A + 2 * (R + 2) * U * X) + (R + 4) * 2 * U
    low = 2.0 ** -126
    return ((2 * E + 2 * (n + 8) * U) * torch.matmul(p, v.abs()) + low * v.abs().sum(-2, keepdim=True),
            (2 * E + (n + G + 8) * U) * p.sum(-2) + G * low)


class Case:
    """Pools filled with NaN except for the positions held, and everything in float64 beside them."""

    def __init__(self, seed, kind, B, NH, KVH, HS, page, lengths, max_len, spare=3, keys_std=1.0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.kind = g, TYPES[kind]
        self.B, self.NH, self.KVH, self.HS, self.page = B, NH, KVH, HS, page
        self.lengths = list(lengths)
        P = -(-max_len // page)
        self.cap = P * page
        pool = B * P + spare
        order = torch.randperm(pool, generator=g)[: B * P].reshape(B, P)
        self.table = order.to(torch.int32)
        self.keys = torch.full((pool, KVH, page, HS), float("nan"), dtype=self.kind)
        self.values = self.keys.clone()
        self.k64, self.v64 = [], []
        for b, n in enumerate(self.lengths):
            n = max(n, 0)
            k = (torch.randn((KVH, n, HS), generator=g) * keys_std).to(self.kind)
            v = torch.randn((KVH, n, HS), generator=g).to(self.kind)
            m, used = min(n, self.cap), -(-min(n, self.cap) // page)
            for pages, rows in ((self.keys, k), (self.values, v)):
                whole = torch.full((KVH, used * page, HS), float("nan"), dtype=self.kind)
                whole[:, :m] = rows[:, :m]
                pages[order[b, :used]] = whole.view(KVH, used, page, HS).transpose(0, 1)
            self.k64.append(k.double())
            self.v64.append(v.double())
        self.inp = torch.randn((B, (NH + 2 * KVH) * HS), generator=g)

    def gpu(self):
        self.dk, self.dv, self.dt = self.keys.cuda(), self.values.cuda(), self.table.cuda()
        self.dl = torch.tensor(self.lengths, dtype=torch.int32).cuda()
        return g2.PagedCache(self.dk, self.dv, self.dt)

    def rows(self, b, append):
        """float64 keys and values that sequence b's query sees."""
        k, v = self.k64[b], self.v64[b]
        if append:
            kn = self.inp[b, self.NH * self.HS:(self.NH + self.KVH) * self.HS].reshape(self.KVH, 1, self.HS)
            vn = self.inp[b, (self.NH + self.KVH) * self.HS:].reshape(self.KVH, 1, self.HS)
            k = torch.cat([k, kn.to(self.kind).double()], 1)
            v = torch.cat([v, vn.to(self.kind).double()], 1)
        return k, v

    def expect(self, b, append):
        """(out, its tolerance, weights summed over a group, their tolerance) in float64."""
        k, v = self.rows(b, append)
        G = self.NH // self.KVH
        q = self.inp[b, : self.NH * self.HS].double().reshape(self.KVH, G, self.HS)
        s = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(self.HS)
        p = torch.softmax(s, -1)
        out = torch.matmul(p, v)
        tol, ptol = attention_bound(q, k, v, p, s)
        return out.reshape(-1), tol.reshape(-1), p.sum(1), ptol


def spread(count, top):
    """count lengths of 0 .. top, short and long ones in turn, a few of them unused places."""
    return [-1 if i % 23 == 22 else (i * 7919) % (top + 1) if i % 3 else (i * 31) % (top // 8 + 1) for i in range(count)]


def same_bits(a, b):
    it = {4: torch.int32, 2: torch.int16}[a.element_size()]
    return torch.equal(a.cpu().view(it), b.cpu().view(it))


def check_attend(c, append=True, weights=False, workspace="full", view=False, calls=1):
    cache = c.gpu()
    B, NH, KVH, HS = c.B, c.NH, c.KVH, c.HS
    pad = 257
    flat = torch.full((B * NH * HS + 2 * pad,), 7.0, device="cuda")
    out = flat[pad:-pad].view(B, NH * HS)
    inp = c.inp.cuda()
    if not append:
        inp = inp[:, : NH * HS].contiguous()
    if view:
        wide = torch.full((B, inp.shape[1] + 13), float("nan"), device="cuda")
        wide[:, 5:5 + inp.shape[1]] = inp
        inp = wide[:, 5:5 + inp.shape[1]]
    ws = None
    if workspace == "full":
        ws = g2.attention_decode_paged_workspace(cache, B, NH, weights=weights)
    elif workspace:
        ws = torch.zeros(workspace, dtype=torch.uint8, device="cuda")
    if ws is not None:
        ws[g2.PAGED_COUNTER_BYTES:] = 0xFF  # NaN everywhere behind the counters
    w = wo = None
    if weights:
        w = torch.rand((B, KVH, c.cap), generator=c.g).cuda() * 3
        wo = torch.full_like(w, -5.0)
    for _ in range(calls):
        g2.attention_decode_paged(out, cache, inp, c.dl, B, NH, append=append, weights_in=w, weights_out=wo, workspace=ws)
    torch.cuda.synchronize()
    assert ws is None or (ws[: g2.PAGED_COUNTER_BYTES] == 0).all(), "a counter was left behind"
    assert (flat[:pad] == 7).all() and (flat[-pad:] == 7).all(), "write outside the output"
    want_k, want_v = c.keys.clone(), c.values.clone()
    for b, n in enumerate(c.lengths):
        got = out[b].cpu().double()
        if n < 0:
            assert (got == 7).all(), f"unused row {b} was written"
            if weights:
                assert (wo[b] == -5).all()
            continue
        if n + (1 if append else 0) > c.cap:
            assert torch.isnan(got).all(), b
            if weights:
                assert (wo[b] == -5).all()
            continue
        total = n + (1 if append else 0)
        if total == 0:
            assert (got == 0).all()
            if weights:
                assert (wo[b] == -5).all()
            continue
        if append:
            k, v = c.rows(b, True)
            want_k[c.table[b, n // c.page], :, n % c.page] = k[:, n].to(c.kind)
            want_v[c.table[b, n // c.page], :, n % c.page] = v[:, n].to(c.kind)
        exp, tol, p, ptol = c.expect(b, append)
        err = (got - exp).abs()
        assert (err <= tol).all(), f"row {b} n={n}: worst {float((err - tol).max()):.3e} above tolerance, err {float(err.max()):.3e}"
        if weights:
            before = w[b].cpu().double()[:, :total].clone()
            if append:
                before[:, n] = 0
            gw = wo[b].cpu().double()
            werr = (gw[:, :total] - before - p).abs()
            assert (werr <= ptol + U * (before + p)).all(), f"weights of row {b} n={n}: {float(werr.max()):.3e}"
            assert (gw[:, total:] == -5).all(), "weights behind the last position were written"
    assert same_bits(c.dk, want_k) and same_bits(c.dv, want_v), "the pages differ"
    return out


SHAPES = [  # NH, KVH, HS
    (12, 12, 64), (25, 25, 64), (8, 2, 128), (32, 4, 96), (6, 3, 80), (7, 1, 64), (3, 3, 256), (9, 3, 32), (10, 5, 16),
    (2, 1, 8), (16, 1, 64), (12, 1, 64), (40, 2, 128), (24, 2, 256), (18, 6, 72), (4, 1, 136), (15, 5, 8),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("NH,KVH,HS", SHAPES)
def test_attend_over_heads_and_types(kind, NH, KVH, HS):
    say(f"attend {kind} NH={NH} KVH={KVH} HS={HS}")
    lengths = [0, 1, 15, 16, 63, 131, 300]
    check_attend(Case(NH * 1000 + HS, kind, len(lengths), NH, KVH, HS, 16, lengths, 301))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("B,NH,KVH,HS,top,weights", [
    (140, 4, 4, 64, 150, False),     # more than 512 (sequence, kv head) pairs: workgroups that follow each other
    (140, 8, 4, 128, 150, True),     # the same, two query heads per kv head
    (64, 4, 4, 64, 1100, True),      # one workgroup per compute unit with much to do
    (64, 4, 4, 128, 600, False), (64, 4, 4, 256, 300, False), (64, 4, 4, 32, 2100, False),
    (90, 12, 3, 64, 200, True),      # matrix kernel: 270 pairs
    (90, 15, 3, 128, 100, False), (90, 12, 3, 256, 60, False),
    (170, 16, 4, 64, 60, False),     # and more than 512
    (2, 20, 1, 96, 9000, True),      # few pairs, long, more heads than a workgroup takes
    (3, 1, 1, 64, 20000, True),
])
def test_attend_every_form_of_the_kernels(kind, B, NH, KVH, HS, top, weights):
    """Sizes on both sides of every line that the plan of a call draws."""
    say(f"attend {kind} B={B} NH={NH} KVH={KVH} HS={HS} top={top}")
    check_attend(Case(B + HS, kind, B, NH, KVH, HS, 16, spread(B, top), top + 1), weights=weights)


@pytest.mark.parametrize("append", [True, False])
@pytest.mark.parametrize("B,NH,KVH,cap,lengths", [
    (3, 2, 2, 4000, [4000, 0, 700]), (5, 1, 1, 6000, [6000, 1, -1, 5999, 2500]), (2, 8, 1, 5000, [-1, -1]),
    (6, 4, 4, 2000, [0, 0, 0, 0, 0, 0]), (4, 6, 2, 3000, [3001, 9000, 2999, 10]),
    (64, 1, 1, 4000, None), (65, 1, 1, 4000, None), (130, 2, 1, 2000, None), (130, 1, 1, 4000, None),
    (200, 1, 1, 3200, None),
])
def test_attend_deals_positions_to_workgroups(B, NH, KVH, cap, lengths, append):
    """Sequences of every length under one plan: a few to three hundred ranges, one to four sequences
    per lane that looks through the lengths, unused places, empty and oversized sequences among them."""
    say(f"deal B={B} NH={NH} KVH={KVH} cap={cap} append={append}")
    for kind in ("f16", "f32") if B < 60 else ("f16",):
        c = Case(B + NH, kind, B, NH, KVH, 64, 16, lengths or spread(B, cap), cap, keys_std=0.5)
        check_attend(c, append=append, weights=B % 2 == 0)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("NH,KVH,HS,page,cap", [
    (2, 2, 64, 16, 6000), (4, 2, 128, 24, 4000), (3, 1, 80, 1, 5000), (8, 1, 96, 7, 5000), (40, 2, 64, 16, 5000),
    (5, 1, 33, 16, 6000), (2, 1, 256, 32, 2000), (16, 2, 200, 50, 2500), (1, 1, 8, 16, 30000), (2, 1, 20, 1000, 12000),
])
def test_attend_split_forms(kind, NH, KVH, HS, page, cap):
    """Caches long enough for several ranges per sequence, in every form of the kernels."""
    say(f"split {kind} NH={NH} KVH={KVH} HS={HS} page={page} cap={cap}")
    c = Case(NH + HS, kind, 5, NH, KVH, HS, page, [cap, cap - 1, 1, -1, cap // 2 + 3], cap + 1, keys_std=0.5)
    whole = g2.PAGED_COUNTER_BYTES + 16
    assert g2.attention_decode_paged_workspace(c.gpu(), 5, NH).nbytes > whole
    check_attend(c)
    check_attend(c, append=False, weights=True)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 128, 1000])
@pytest.mark.parametrize("append", [True, False])
def test_attend_over_lengths_and_page_sizes(page, append):
    """Around the ends of tiles (8 .. 64 rows), of the shortest range (128) and of pages; unused
    places, empty sequences and sequences that do not fit among them."""
    lengths = [0, -1, 1, 2, 7, 8, 9, 31, 32, 33, 127, 128, 129, 255, 256, 257, 383, 385, 511, 513, 640, -7, 700]
    say(f"attend page={page} append={append}")
    for kind in ("f32", "bf16"):
        c = Case(page, kind, len(lengths), 4, 2, 64, page, lengths, 640)
        check_attend(c, append=append)


@pytest.mark.parametrize("kind,HS,NH,KVH", [("f16", 20, 4, 2), ("bf16", 7, 3, 3), ("f32", 50, 6, 2), ("f32", 1, 2, 1),
                                            ("bf16", 250, 8, 1), ("f16", 129, 9, 1)])
def test_attend_head_sizes_of_no_whole_number_of_16_bytes(kind, HS, NH, KVH):
    say(f"attend {kind} HS={HS} NH={NH} KVH={KVH}")
    lengths = [0, 5, 64, 200, 333]
    check_attend(Case(HS, kind, len(lengths), NH, KVH, HS, 9, lengths, 400), weights=True)


@pytest.mark.parametrize("kind", list(TYPES))
def test_attend_pages_that_are_not_16_byte_aligned(kind):
    say(f"attend misaligned {kind}")
    c = Case(5, kind, 3, 4, 2, 64, 16, [3, 100, 250], 300)
    want = check_attend(c)
    for name in ("dk", "dv"):
        t = getattr(c, name)
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        setattr(c, name, flat[1:].view(t.shape))
    cache = g2.PagedCache(c.dk, c.dv, c.dt)
    out = torch.empty((3, 4 * 64), device="cuda")
    g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 3, 4)
    for b in range(3):
        exp, tol, _, _ = c.expect(b, True)
        assert ((out[b].cpu().double() - exp).abs() <= tol).all()
        assert ((out[b] - want[b]).cpu().double().abs() <= 2 * tol).all()


@pytest.mark.parametrize("NH,KVH,HS,kind", [(4, 4, 64, "f32"), (8, 2, 128, "bf16"), (12, 1, 64, "f16"), (6, 6, 64, "bf16")])
@pytest.mark.parametrize("append", [True, False])
def test_attend_weights(NH, KVH, HS, kind, append):
    lengths = [0, -1, 1, 40, 129, 1023, 1024, 1500, 2047, 2048, 5000]
    say(f"weights {kind} NH={NH} KVH={KVH} HS={HS} append={append}")
    check_attend(Case(77, kind, len(lengths), NH, KVH, HS, 16, lengths, 2048), append=append, weights=True)


def test_attend_weights_in_place():
    c = Case(78, "f32", 4, 4, 2, 64, 16, [0, 100, -1, 700], 704)
    cache = c.gpu()
    w = torch.rand((4, 2, c.cap), device="cuda")
    apart = w.clone()
    out = torch.zeros((4, 256), device="cuda")
    ws = g2.attention_decode_paged_workspace(cache, 4, 4, weights=True)
    other = w.clone()
    g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 4, 4, weights_in=w, weights_out=apart, workspace=ws)
    g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 4, 4, weights_in=other, weights_out=other, workspace=ws)
    assert torch.equal(apart, other)


def test_attend_split_as_far_as_the_workspace_goes():
    """None, room for one range, for three, and the full size: the same row to rounding each time."""
    lengths = [4000, 1, 2500]
    one = 3 * 4 * (64 + 2) * 4
    for ws in (None, 256, g2.PAGED_COUNTER_BYTES, g2.PAGED_COUNTER_BYTES + one, g2.PAGED_COUNTER_BYTES + 3 * one + 100, "full"):
        say(f"workspace {ws}")
        check_attend(Case(9, "f32", 3, 4, 4, 64, 32, lengths, 4001), workspace=ws)


def test_attend_rows_at_a_stride():
    check_attend(Case(10, "bf16", 5, 6, 2, 64, 16, [0, 17, 200, -1, 500], 512), view=True)
    check_attend(Case(11, "f32", 5, 6, 2, 64, 16, [0, 17, 200, -1, 500], 512), view=True, append=False)


@pytest.mark.parametrize("kind,NH", [("f32", 2), ("f32", 8), ("f16", 8), ("bf16", 8)])
def test_attend_large_scores(kind, NH):
    """Scores of some hundreds: one position has all the weight, exp must neither overflow nor lose it."""
    check_attend(Case(12, kind, 2, NH, 2, 64, 16, [300, 700], 701, keys_std=60.0), weights=True)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("scale", [1e-12, 1e-3, 1e4])
def test_attend_queries_of_any_size(kind, scale):
    """Queries far below and above 1, keys that make up for it: pieces of queries lose nothing."""
    c = Case(19, kind, 2, 8, 2, 64, 16, [300, 700], 701, keys_std=min(1 / scale, 1e3) if kind != "f16" else 1.0)
    c.inp[:, : 8 * 64] *= scale
    c.inp[0, 64:128] *= torch.logspace(-6, 0, 64)
    check_attend(c)


@pytest.mark.parametrize("kind,NH", [("f32", 1), ("f16", 1), ("bf16", 2), ("f32", 5), ("f16", 5), ("bf16", 5), ("bf16", 16)])
def test_attend_infinite_keys_weigh_nothing(kind, NH):
    """Positions whose score is -inf (a key with an infinity against a negative query) weigh nothing,
    even when they are all that a row group, a wave or a range has seen."""
    say(f"infinite keys {kind} NH={NH}")
    n = 900
    c = Case(13, kind, 1, NH, 1, 64, 16, [n], n + 1)
    c.inp[0, : NH * 64: 64] = -1.0
    live = [5, 640]
    for i in range(n):
        if i not in live:
            c.keys[c.table[0, i // 16], 0, i % 16] = 0.0
            c.keys[c.table[0, i // 16], 0, i % 16, 0] = float("inf")
    cache = c.gpu()
    out = torch.zeros((1, NH * 64), device="cuda")
    for ws in (None, g2.attention_decode_paged_workspace(cache, 1, NH)):
        g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 1, NH, workspace=ws)
        k, v = c.rows(0, True)
        rows = live + [n]
        q, k, v = c.inp[0, : NH * 64].double().view(1, NH, 64), k[:, rows], v[:, rows]
        s = torch.matmul(q, k.transpose(1, 2)) / 8.0
        p = torch.softmax(s, -1)
        tol, _ = attention_bound(q, k, v, p, s)
        assert ((out[0].cpu().double() - torch.matmul(p, v).reshape(-1)).abs() <= tol.reshape(-1)).all()


def test_attend_nan_in_a_key_shows_and_stays_in_its_row():
    c = Case(14, "f32", 3, 2, 2, 64, 16, [200, 200, 200], 208)
    c.keys[c.table[1, 3], 0, 4, 7] = float("nan")
    cache = c.gpu()
    out = torch.zeros((3, 128), device="cuda")
    g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 3, 2, workspace=g2.attention_decode_paged_workspace(cache, 3, 2))
    bad = torch.isnan(out).cpu()
    assert bad[1, :64].all() and not bad[1, 64:].any() and not bad[0].any() and not bad[2].any()


def test_attend_pages_that_do_not_exist_give_nan_rows_only():
    lengths = [100, 100, 100, 40]
    c = Case(15, "f32", 4, 4, 2, 64, 16, lengths, 160)
    c.table[1, 2] = -1          # among the pages read
    c.table[2, 6] = c.keys.shape[0]  # the page of the new row
    c.table[3, 3] = 1 << 30     # behind the last position: never looked at
    cache = c.gpu()
    out = torch.zeros((4, 256), device="cuda")
    for ws in (None, g2.attention_decode_paged_workspace(cache, 4, 4)):
        g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 4, 4, workspace=ws)
        bad = torch.isnan(out).cpu()
        assert bad[1].all() and bad[2].all() and not bad[0].any() and not bad[3].any()
        for b in (0, 3):
            exp, tol, _, _ = c.expect(b, True)
            assert ((out[b].cpu().double() - exp).abs() <= tol).all()


@pytest.mark.parametrize("kind,NH", [("f16", 2), ("f32", 4), ("bf16", 10)])
def test_attend_split_nan_and_pages_that_do_not_exist(kind, NH):
    """One range of many sees it: its whole row shows it, in the weights too, and no other row does."""
    lengths = [4000, 4000, 3999, 4000]
    c = Case(16, kind, 4, NH, 2, 64, 16, lengths, 4016)
    c.table[1, 200] = c.keys.shape[0]
    c.keys[c.table[2, 30], 0, 4, 7] = float("nan")
    c.table[3, 250] = -1  # the page of the new row
    cache = c.gpu()
    ws = g2.attention_decode_paged_workspace(cache, 4, NH, weights=True)
    out = torch.zeros((4, NH * 64), device="cuda")
    w = torch.rand((4, 2, c.cap), device="cuda")
    wo = torch.full_like(w, 7.0)
    for _ in range(2):
        g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 4, NH, weights_in=w, weights_out=wo, workspace=ws)
        bad, badw = torch.isnan(out).cpu(), torch.isnan(wo).cpu()
        half = NH * 32  # what the heads of the first kv head write
        for b in range(4):
            n = lengths[b] + 1
            both = b in (1, 3)
            assert bad[b, :half].all() if both or b == 2 else not bad[b, :half].any(), b
            assert bad[b, half:].all() if both else not bad[b, half:].any(), b
            assert badw[b, 0, :n].all() if both or b == 2 else not badw[b, 0, :n].any(), b
            assert badw[b, 1, :n].all() if both else not badw[b, 1, :n].any(), b
        assert (wo[:, :, 4001:] == 7.0).all()
        exp, tol, _, _ = c.expect(0, True)
        assert ((out[0].cpu().double() - exp).abs() <= tol).all()
    assert not ws[: g2.PAGED_COUNTER_BYTES].any()


def test_attend_is_repeatable_and_replays_in_a_graph():
    """The same bits eagerly, on another stream and in replays of one captured call, with eager
    work and other lengths between the replays."""
    c = Case(16, "bf16", 3, 8, 2, 128, 16, [900, 30, 2000], 2100)
    cache = c.gpu()
    inp = c.inp.cuda()
    w = torch.rand((3, 2, c.cap), device="cuda")

    def call(out, wo, ws):
        g2.attention_decode_paged(out, cache, inp, c.dl, 3, 8, weights_in=w, weights_out=wo, workspace=ws)

    def eager():
        out, wo = torch.zeros((3, 1024), device="cuda"), torch.zeros_like(w)
        call(out, wo, g2.attention_decode_paged_workspace(cache, 3, 8, weights=True))
        torch.cuda.synchronize()
        return out, wo

    first, again = eager(), eager()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    out, wo = torch.zeros((3, 1024), device="cuda"), torch.zeros_like(w)
    ws = g2.attention_decode_paged_workspace(cache, 3, 8, weights=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            g2.set_stream(side)
            call(out, wo, ws)
    finally:
        g2.set_stream(None)
    for lengths in ([900, 30, 2000], [5, -1, 777], [900, 30, 2000], [0, 2099, 64]):
        c.dl.copy_(torch.tensor(lengths, dtype=torch.int32))
        c.dk.copy_(c.keys), c.dv.copy_(c.values)
        c.dk.nan_to_num_(0.5), c.dv.nan_to_num_(0.25)
        out.zero_(), wo.zero_()
        want = eager()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(wo, want[1]), lengths


def test_calls_of_different_sizes_share_a_workspace_one_after_the_other():
    cases = [Case(40 + i, kind, B, NH, KVH, 64, 16, lengths, max(lengths) + 1)
             for i, (kind, B, NH, KVH, lengths) in enumerate([
                 ("f32", 2, 3, 3, [2000, 900]), ("bf16", 1, 8, 1, [3000]), ("f16", 7, 4, 2, [10, 500, 3, 900, 64, 0, 77]),
                 ("f32", 1, 1, 1, [5000])])]
    caches = [c.gpu() for c in cases]
    need = max(g2.attention_decode_paged_workspace(k, c.B, c.NH, weights=True).numel() for k, c in zip(caches, cases))
    shared = torch.zeros(need, dtype=torch.uint8, device="cuda")

    def run(i, ws):
        c = cases[i]
        out = torch.zeros((c.B, c.NH * 64), device="cuda")
        w = torch.zeros((c.B, c.KVH, c.cap), device="cuda")
        own = ws if ws is not None else g2.attention_decode_paged_workspace(caches[i], c.B, c.NH, weights=True)
        g2.attention_decode_paged(out, caches[i], c.inp.cuda(), c.dl, c.B, c.NH, weights_in=w, weights_out=w, workspace=own)
        return out, w

    alone = [run(i, None) for i in range(4)]
    for i in (0, 1, 2, 3, 3, 1, 0, 2, 1, 2, 0, 3):
        # a larger workspace than a call asks for changes nothing
        got = run(i, shared)
        assert torch.equal(got[0], alone[i][0]) and torch.equal(got[1], alone[i][1]), i
    assert (shared[: g2.PAGED_COUNTER_BYTES] == 0).all()


def test_two_streams_with_a_workspace_each():
    """Calls that overlap on the GPU: the same bits as one after the other."""
    cases = [Case(50, "f32", 2, 3, 3, 64, 16, [3000, 900], 3001), Case(51, "bf16", 2, 16, 2, 128, 16, [2500, 3000], 3001)]
    caches = [c.gpu() for c in cases]
    inps = [c.inp.cuda() for c in cases]
    spaces = [g2.attention_decode_paged_workspace(k, 2, c.NH) for k, c in zip(caches, cases)]
    outs = [torch.zeros((8, 2, c.NH * c.HS), device="cuda") for c in cases]
    want = []
    for i in range(2):
        g2.attention_decode_paged(outs[i][0], caches[i], inps[i], cases[i].dl, 2, cases[i].NH, workspace=spaces[i])
        want.append(outs[i][0].clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        for k in range(8):
            for i in range(2):
                g2.set_stream(streams[i])
                g2.attention_decode_paged(outs[i][k], caches[i], inps[i], cases[i].dl, 2, cases[i].NH, workspace=spaces[i])
    finally:
        g2.set_stream(None)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(outs[i][k], want[i]) for k in range(8))


def test_store_and_evict_replay_in_a_graph():
    g = torch.Generator().manual_seed(60)
    B, KVH, HS, page, P = 3, 2, 64, 16, 6
    pages = torch.randperm(2 * B * P, generator=g).to(torch.int32).view(2, B, P).cuda()
    keys, values = (torch.randn((2 * B * P, KVH, page, HS), generator=g).cuda() for _ in range(2))
    src, dst = g2.PagedCache(keys, values, pages[0]), g2.PagedCache(keys, values, pages[1])
    rows = torch.randn((60, 2 * KVH * HS), generator=g).cuda()
    starts, held = torch.tensor([0, 20, 50, 60], dtype=torch.int32).cuda(), torch.zeros(3, dtype=torch.int32).cuda()
    lengths, weights = torch.zeros(3, dtype=torch.int32).cuda(), torch.rand((B, KVH, P * page), generator=g).cuda()
    kept = torch.zeros((B, KVH, 40), dtype=torch.int32).cuda()
    wo, lo = torch.zeros_like(weights), torch.zeros_like(lengths)

    def call():
        g2.kv_store_paged(src, rows, starts, held, 60, B, 0)
        g2.kv_evict_paged(dst, src, kept, wo, lo, weights, lengths, B, 40, 5)

    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            g2.set_stream(side)
            call()
    finally:
        g2.set_stream(None)
    for at, n in (([0, 0, 0], [20, 30, 10]), ([30, 5, 80], [50, 35, 90]), ([0, -1, 7], [20, -1, 17])):
        state = []
        for replay in (False, True):
            keys.copy_(torch.arange(keys.numel(), device="cuda").view_as(keys) % 997), values.copy_(-keys)
            rows.mul_(1.0), kept.fill_(-9), wo.fill_(-5), lo.fill_(-9)
            held.copy_(torch.tensor(at, dtype=torch.int32)), lengths.copy_(torch.tensor(n, dtype=torch.int32))
            torch.cuda.synchronize()
            graph.replay() if replay else call()
            torch.cuda.synchronize()
            state.append([t.clone() for t in (keys, values, kept, wo, lo)])
        assert all(torch.equal(x, y) for x, y in zip(*state)), n


def test_attend_pool_beyond_32_bit_offsets():
    """Pages whose first element lies behind 2^32 elements: 2^18 pages of (2, 64, 256) bf16 and more."""
    NH, KVH, HS, page = 4, 2, 256, 64
    pool = (1 << 17) + 50
    say(f"pool of {pool} pages, {pool * KVH * page * HS * 2 / 2**30:.1f} GiB each of keys and values")
    c = Case(17, "bf16", 2, NH, KVH, HS, page, [150, 700], 704, spare=0)
    low = c.table.clone()
    c.table = (pool - 1 - low).to(torch.int32)
    keys = torch.empty((pool, KVH, page, HS), dtype=torch.bfloat16, device="cuda")
    values = torch.empty_like(keys)
    for b in range(2):
        for i in range(low.shape[1]):
            keys[c.table[b, i].item()] = c.keys[low[b, i]].cuda()
            values[c.table[b, i].item()] = c.values[low[b, i]].cuda()
    cache = g2.PagedCache(keys, values, c.table.cuda())
    dl = torch.tensor(c.lengths, dtype=torch.int32).cuda()
    out = torch.zeros((2, NH * HS), device="cuda")
    g2.attention_decode_paged(out, cache, c.inp.cuda(), dl, 2, NH, workspace=g2.attention_decode_paged_workspace(cache, 2, NH))
    for b in range(2):
        exp, tol, _, _ = c.expect(b, True)
        assert ((out[b].cpu().double() - exp).abs() <= tol).all()
        n = c.lengths[b]
        k, v = c.rows(b, True)
        assert torch.equal(keys[c.table[b, n // page].item(), :, n % page].cpu().double(), k[:, n])
    # and the last page takes part in a store and an eviction
    starts, held = torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.tensor([9], dtype=torch.int32).cuda()
    one = g2.PagedCache(keys, values, torch.tensor([[pool - 1]], dtype=torch.int32).cuda())
    two = g2.PagedCache(keys, values, torch.tensor([[pool - 40]], dtype=torch.int32).cuda())
    row = torch.randn((1, 2 * KVH * HS), device="cuda")
    g2.kv_store_paged(one, row, starts, held, 1, 1, 0)
    want = row[0, : KVH * HS].view(KVH, HS).bfloat16()
    assert torch.equal(keys[pool - 1, :, 9], want)
    w = torch.zeros((1, KVH, page), device="cuda")
    w[:, :, 9] = 1.0
    kept = torch.zeros((1, KVH, 1), dtype=torch.int32, device="cuda")
    wo, lo = torch.zeros((1, KVH, page), device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    g2.kv_evict_paged(two, one, kept, wo, lo, w, torch.tensor([12], dtype=torch.int32).cuda(), 1, 1, 0)
    assert (kept == 9).all() and torch.equal(keys[pool - 40, :, 0], want)


# ------------------------------------------------------------------ store
def plain_store(keys, values, table, inp, starts, lengths, NH, cap):
    KVH, page, HS = keys.shape[1:]
    for b in range(len(lengths)):
        for r in range(starts[b], starts[b + 1]):
            pos = lengths[b] + r - starts[b]
            if lengths[b] < 0 or pos >= cap or r >= inp.shape[0]:
                continue
            at = int(table[b, pos // page])
            if not 0 <= at < keys.shape[0]:
                continue
            keys[at, :, pos % page] = inp[r, NH * HS:(NH + KVH) * HS].view(KVH, HS).to(keys.dtype)
            values[at, :, pos % page] = inp[r, (NH + KVH) * HS:(NH + 2 * KVH) * HS].view(KVH, HS).to(keys.dtype)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("NH,KVH,HS,page", [(12, 12, 64, 16), (8, 2, 128, 24), (0, 3, 20, 5), (5, 1, 7, 16), (2, 2, 256, 1)])
def test_store(kind, NH, KVH, HS, page):
    say(f"store {kind} NH={NH} KVH={KVH} HS={HS} page={page}")
    r = torch.Generator().manual_seed(page + HS)
    tokens, lengths = [3, 0, 40, 1, 17, 9], [0, 4, 33, 47, -1, 10]
    first = 2  # rows in front of the first sequence, and five behind the last
    starts = [first]
    for t in tokens:
        starts.append(starts[-1] + t)
    N, B, cap = starts[-1] + 5, len(tokens), -(-48 // page) * page
    P = cap // page
    pool = B * P + 2
    table = torch.randperm(pool, generator=r)[: B * P].reshape(B, P).to(torch.int32)
    table[5, 12 // page] = pool  # a page that does not exist
    inp = torch.randn((N, (NH + 2 * KVH) * HS), generator=r) * 3
    inp[4, -1], inp[5, -1], inp[6, -1] = float("nan"), float("inf"), 1e5
    inp[7, -1], inp[8, -1] = 1e-42, -0.0
    keys = torch.randn((pool, KVH, page, HS), generator=r).to(TYPES[kind])
    values = torch.randn((pool, KVH, page, HS), generator=r).to(TYPES[kind])
    dk, dv = keys.cuda(), values.cuda()
    cache = g2.PagedCache(dk, dv, table.cuda())
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    wide = torch.full((N, inp.shape[1] + 4), 9.0, device="cuda")
    wide[:, : inp.shape[1]] = inp.cuda()
    plain_store(keys, values, table, inp, starts, lengths, NH, cap)
    for rows in (inp.cuda(), wide[:, : inp.shape[1]]):
        g2.kv_store_paged(cache, rows, i32(starts), i32(lengths), N, B, NH)
        torch.cuda.synchronize()
        for got, want in ((dk, keys), (dv, values)):
            got, want = got.cpu(), want
            nan = torch.isnan(want)
            assert torch.equal(torch.isnan(got), nan)
            assert same_bits(torch.where(nan, torch.zeros_like(got), got), torch.where(nan, torch.zeros_like(want), want))


def test_store_many_sequences():
    """More sequences than lanes of a wave, many of them with no row at all."""
    r = np.random.default_rng(3)
    B, page, KVH, HS, P = 700, 4, 2, 16, 3
    tokens = r.integers(0, 3, B) * r.integers(0, 4, B)
    starts = np.concatenate([[0], np.cumsum(tokens)]).astype(np.int32)
    lengths = r.integers(0, 8, B).astype(np.int32)
    N = int(starts[-1])
    table = torch.from_numpy(r.permutation(B * P).reshape(B, P).astype(np.int32))
    inp = torch.randn((N, 2 * KVH * HS))
    keys, values = torch.zeros((B * P, KVH, page, HS)), torch.zeros((B * P, KVH, page, HS))
    dk, dv = keys.cuda(), values.cuda()
    g2.kv_store_paged(g2.PagedCache(dk, dv, table.cuda()), inp.cuda(), torch.from_numpy(starts).cuda(),
                      torch.from_numpy(lengths).cuda(), N, B, 0)
    plain_store(keys, values, table, inp, starts.tolist(), lengths.tolist(), 0, P * page)
    assert torch.equal(dk.cpu(), keys) and torch.equal(dv.cpu(), values)


# ------------------------------------------------------------------ evict
def plain_pick(w, n, budget, recent):
    """Positions that stay of n, by sorting (float64, ties to the lowest position, NaN the largest)."""
    if n <= budget:
        return list(range(n))
    older = n - recent
    key = [(-math.inf if math.isnan(x) else -x, 0 if math.isnan(x) else 1, i) for i, x in enumerate(w[:older].tolist())]
    return sorted(i for _, _, i in sorted(key)[: budget - recent]) + list(range(older, n))


def check_evict(seed, kind, lengths, budget, recent, KVH=2, HS=64, page=16, dst_page=None, max_len=None, weights=None,
                bad_src=None, bad_dst=None):
    g = torch.Generator().manual_seed(seed)
    B, dst_page = len(lengths), dst_page or page
    cap_len = max_len or max(max(lengths), 1)
    P, D = -(-cap_len // page), -(-budget // dst_page)
    src_k = torch.randn((B * P + 1, KVH, page, HS), generator=g).to(TYPES[kind])
    src_v = torch.randn((B * P + 1, KVH, page, HS), generator=g).to(TYPES[kind])
    dst_k = torch.randn((B * D + 1, KVH, dst_page, HS), generator=g).to(TYPES[kind])
    dst_v = torch.randn((B * D + 1, KVH, dst_page, HS), generator=g).to(TYPES[kind])
    st = torch.randperm(B * P + 1, generator=g)[: B * P].reshape(B, P).to(torch.int32)
    dt = torch.randperm(B * D + 1, generator=g)[: B * D].reshape(B, D).to(torch.int32)
    if bad_src:
        st[bad_src] = -3
    if bad_dst:
        dt[bad_dst] = 1 << 20
    w = torch.rand((B, KVH, P * page), generator=g) ** 6 if weights is None else weights(B, KVH, P * page, g)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    dsk, dsv, ddk, ddv = src_k.cuda(), src_v.cuda(), dst_k.cuda(), dst_v.cuda()
    kept = torch.full((B, KVH, budget), -9, dtype=torch.int32, device="cuda")
    wo = torch.full((B, KVH, D * dst_page), -5.0, device="cuda")
    lo = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    g2.kv_evict_paged(g2.PagedCache(ddk, ddv, dt.cuda()), g2.PagedCache(dsk, dsv, st.cuda()), kept, wo, lo, w.cuda(),
                      i32(lengths), B, budget, recent)
    torch.cuda.synchronize()
    kept, wo, lo = kept.cpu(), wo.cpu(), lo.cpu()
    assert same_bits(dsk, src_k) and same_bits(dsv, src_v), "the source was written"
    for b, n in enumerate(lengths):
        if n < 0:
            assert lo[b] == -9 and (kept[b] == -9).all() and (wo[b] == -5).all()
            continue
        if n > P * page:
            assert lo[b] == -1 and (kept[b] == -1).all() and (wo[b] == -5).all()
            continue
        m = min(n, budget)
        assert lo[b] == m
        for h in range(KVH):
            want = plain_pick(w[b, h].double().numpy(), n, budget, recent)
            assert kept[b, h, :m].tolist() == want, (b, h)
            assert (kept[b, h, m:] == -1).all() and (wo[b, h, m:] == -5).all()
            for j, i in enumerate(want):
                s, d = int(st[b, i // page]), int(dt[b, j // dst_page])
                if not 0 <= s < len(src_k) or not 0 <= d < len(dst_k):
                    assert math.isnan(wo[b, h, j])
                    continue
                assert same_bits(wo[b, h, j].reshape(1), w[b, h, i].reshape(1))
                dst_k[d, h, j % dst_page] = src_k[s, h, i % page]
                dst_v[d, h, j % dst_page] = src_v[s, h, i % page]
    assert same_bits(ddk, dst_k) and same_bits(ddv, dst_v), "the pages differ"


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (64, 0), (64, 64), (100, 17), (300, 3), (511, 64)])
def test_evict(kind, budget, recent):
    say(f"evict {kind} budget={budget} recent={recent}")
    check_evict(budget + recent, kind, [0, 1, 63, -1, 100, 101, 300, 512, 999], budget, recent, max_len=512)


@pytest.mark.parametrize("KVH,HS,page,dst_page", [(1, 128, 24, 24), (3, 20, 16, 7), (2, 7, 5, 16), (4, 96, 16, 32), (1, 256, 1, 3)])
def test_evict_head_and_page_sizes(KVH, HS, page, dst_page):
    for kind in TYPES:
        say(f"evict {kind} KVH={KVH} HS={HS} page={page}")
        check_evict(HS, kind, [200, 77, 130], 90, 11, KVH=KVH, HS=HS, page=page, dst_page=dst_page)


@pytest.mark.parametrize("n,budget", [(1000, 600), (1024 + 64, 200), (4000, 1000), (9001, 4000), (20000, 5000), (32768 + 10, 700),
                                      (40000, 12345)])
def test_evict_lengths_of_every_form(n, budget):
    """Lengths on both sides of what the choice keeps in registers, up to more than it can."""
    say(f"evict n={n} budget={budget}")
    check_evict(n, "bf16", [n, n - 1, budget + 1], budget, 32, KVH=1, HS=8, page=64)


def ties(B, KVH, cap, g):
    return torch.randint(0, 3, (B, KVH, cap), generator=g).float()


def special(B, KVH, cap, g):
    w = torch.randint(0, 9, (B, KVH, cap), generator=g)
    return torch.tensor([0.0, -0.0, 1.0, -1.0, float("inf"), float("-inf"), float("nan"), 1e-42, -1e-42])[w]


def zeros(B, KVH, cap, g):
    return torch.zeros((B, KVH, cap))


def behind(B, KVH, cap, g):
    """What lies behind the last position is larger than anything that takes part."""
    w = torch.rand((B, KVH, cap), generator=g)
    w[..., 300:] = float("inf")
    return w


@pytest.mark.parametrize("weights", [ties, special, zeros, behind], ids=lambda f: f.__name__)
@pytest.mark.parametrize("budget,recent", [(10, 0), (150, 20), (299, 5)])
def test_evict_ties_and_special_weights(weights, budget, recent):
    check_evict(budget, "f32", [300, 299, 256], budget, recent, max_len=320, weights=weights, HS=16)


def negative(B, KVH, cap, g):
    """Nothing but large negative weights: the smallest ranks there are."""
    return -torch.rand((B, KVH, cap), generator=g) * 3e38


@pytest.mark.parametrize("n,budget", [(300, 100), (9001, 8000), (20000, 19000), (20000, 40)])
def test_evict_negative_weights(n, budget):
    check_evict(8, "f32", [n, n - 7], budget, 10, KVH=1, HS=8, page=64, weights=negative)


def test_evict_many_that_stay_nearly_whole():
    """More than a thousand (sequence, kv head) pairs, most positions stay: choice and copy apart."""
    check_evict(10, "bf16", [48 - i % 9 for i in range(520)], 40, 3, KVH=2, HS=8, page=8)


def test_evict_one_value_apart():
    """Weights that differ in their last bits only."""
    def close(B, KVH, cap, g):
        return (torch.randint(0, 40, (B, KVH, cap), generator=g) + 0x3F800000).to(torch.int32).view(torch.float32)
    for n, budget in ((900, 400), (9001, 4000), (30000, 7000)):
        check_evict(9, "f16", [n, n - 3], budget, 0, KVH=1, HS=8, page=64, weights=close)


def test_evict_ties_beyond_the_registers():
    check_evict(4, "f16", [40000, 39999], 20000, 100, KVH=1, HS=8, page=64, weights=ties)


def lowest(B, KVH, cap, g):
    return torch.where(torch.rand((B, KVH, cap), generator=g) < 0.9, -math.inf, torch.rand((B, KVH, cap), generator=g))


@pytest.mark.parametrize("weights", [special, lowest, zeros], ids=lambda f: f.__name__)
@pytest.mark.parametrize("n,budget", [(1023, 900), (4095, 5), (20001, 15000), (40001, 30000)])
def test_evict_special_weights_of_every_form(n, budget, weights):
    """Ranks at both ends of their order, next to what is behind the last position."""
    say(f"evict special n={n} budget={budget}")
    check_evict(11, "f16", [n, budget + 6, n - 1], budget, 4, KVH=1, HS=8, page=64, weights=weights)


def test_evict_pages_that_do_not_exist():
    check_evict(5, "f32", [300, 300, 300], 100, 10, bad_src=(1, 4), bad_dst=(2, 2))


# ------------------------------------------------------------------ together
def test_prompts_steps_and_evictions_together():
    """Ragged prompts are stored, tokens are decoded with weights, the cache is brought down to a
    budget and decoding goes on, with a sequence that leaves in between: every step against a
    float64 simulation that keeps plain lists."""
    g = torch.Generator().manual_seed(21)
    B, NH, KVH, HS, page, P, budget, recent = 4, 6, 3, 64, 16, 12, 60, 10
    G, cap = NH // KVH, P * page
    tokens = [70, 1, 33, 120]
    starts = np.concatenate([[0], np.cumsum(tokens)]).astype(np.int32)
    N = int(starts[-1])
    row = (NH + 2 * KVH) * HS
    pool = 2 * B * P
    keys = torch.full((pool, KVH, page, HS), float("nan"), device="cuda", dtype=torch.float32)
    values = keys.clone()
    tables = torch.randperm(pool, generator=g).to(torch.int32).view(2, B, P).cuda()
    caches = [g2.PagedCache(keys, values, t) for t in tables]
    prompt = torch.randn((N, row), generator=g)
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    g2.kv_store_paged(caches[0], prompt.cuda(), torch.from_numpy(starts).cuda(), lengths, N, B, NH)
    lengths += torch.tensor(tokens, dtype=torch.int32, device="cuda")
    sim = []
    for b in range(B):
        x = prompt[starts[b]:starts[b + 1]].double()
        k = x[:, NH * HS:(NH + KVH) * HS].view(-1, KVH, HS).transpose(0, 1)
        v = x[:, (NH + KVH) * HS:].view(-1, KVH, HS).transpose(0, 1)
        sim.append([k, v, torch.zeros((KVH, k.shape[1]), dtype=torch.float64)])
    weights = torch.zeros((B, KVH, cap), device="cuda")
    ws = g2.attention_decode_paged_workspace(caches[0], B, NH, weights=True)
    out = torch.zeros((B, NH * HS), device="cuda")
    at = 0
    for step in range(24):
        inp = torch.randn((B, row), generator=g)
        g2.attention_decode_paged(out, caches[at], inp.cuda(), lengths, B, NH, weights_in=weights, weights_out=weights, workspace=ws)
        lengths = torch.where(lengths >= 0, lengths + 1, lengths)
        for b in range(B):
            if sim[b] is None:
                continue
            k, v, w = sim[b]
            x = inp[b].double()
            k = torch.cat([k, x[NH * HS:(NH + KVH) * HS].view(KVH, 1, HS)], 1)
            v = torch.cat([v, x[(NH + KVH) * HS:].view(KVH, 1, HS)], 1)
            q = x[: NH * HS].view(KVH, G, HS)
            s = torch.matmul(q, k.transpose(1, 2)) / 8.0
            p = torch.softmax(s, -1)
            w = torch.cat([w, torch.zeros((KVH, 1), dtype=torch.float64)], 1) + p.sum(1)
            sim[b] = [k, v, w]
            tol, _ = attention_bound(q, k, v, p, s)
            assert ((out[b].cpu().double() - torch.matmul(p, v).reshape(-1)).abs() <= tol.reshape(-1)).all(), (step, b)
        if step == 9:
            lengths[1] = -1  # it has ended
            sim[1] = None
        if step % 8 == 7:
            kept = torch.full((B, KVH, budget), -1, dtype=torch.int32, device="cuda")
            new_w, new_l = torch.zeros_like(weights), torch.full_like(lengths, -1)
            g2.kv_evict_paged(caches[1 - at], caches[at], kept, new_w, new_l, weights, lengths, B, budget, recent)
            at, weights, lengths = 1 - at, new_w, new_l
            for b in range(B):
                if sim[b] is None:
                    continue
                k, v, w = sim[b]
                m = min(k.shape[1], budget)
                assert int(lengths[b]) == m
                idx = kept[b, :, :m].cpu().long()
                for h in range(KVH):
                    # the simulation's own choice, where its weights are further apart than fp32 can confuse
                    want = plain_pick(w[h].numpy(), k.shape[1], budget, recent)
                    if idx[h].tolist() != want:
                        odd = set(idx[h].tolist()) ^ set(want)
                        assert max(w[h, list(odd)]) - min(w[h, list(odd)]) < 1e-4, (b, h)
                sim[b] = [k.gather(1, idx[..., None].expand(-1, -1, HS)), v.gather(1, idx[..., None].expand(-1, -1, HS)),
                          w.gather(1, idx)]


def test_decoding_equals_the_causal_attention_row_by_row():
    """attention_forward over a whole sequence, and the same sequence fed token by token: each side
    is within the launchers' 1e-5 + 1e-4 |x| of the exact row, so they are within twice that."""
    B, T, NH, HS, page = 2, 40, 12, 64, 16
    C = NH * HS
    g = torch.Generator().manual_seed(22)
    qkv = torch.randn((B, T, 3 * C), generator=g).cuda()
    whole = torch.empty((B, T, C), device="cuda")
    g2.attention_forward(whole, None, None, qkv, B, T, C, NH)
    keys = torch.empty((B * 3, NH, page, HS), device="cuda")
    cache = g2.PagedCache(keys, torch.empty_like(keys), torch.arange(B * 3, dtype=torch.int32).view(B, 3).cuda())
    out = torch.empty((B, C), device="cuda")
    for t in range(T):
        g2.attention_decode_paged(out, cache, qkv[:, t], torch.full((B,), t, dtype=torch.int32, device="cuda"), B, NH)
        assert torch.allclose(out, whole[:, t], rtol=2e-4, atol=2e-5), t


def test_a_cache_on_another_gpu_is_refused():
    c = Case(30, "f32", 1, 1, 1, 64, 16, [5], 16)
    cache = c.gpu()
    out = torch.zeros((1, 64), device="cuda")
    cache._device += 1  # as if its tensors lay there
    with pytest.raises(ValueError, match="current device"):
        g2.attention_decode_paged(out, cache, c.inp.cuda(), c.dl, 1, 1)
    with pytest.raises(ValueError, match="current device"):
        g2.kv_store_paged(cache, c.inp.cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"), c.dl, 1, 1, 1)


def test_python_refusals():
    c = Case(31, "f32", 2, 2, 1, 64, 16, [5, 6], 32)
    cache = c.gpu()
    inp, out = c.inp.cuda(), torch.zeros((2, 128), device="cuda")
    ok = dict(out=out, cache=cache, inp=inp, lengths=c.dl, B=2, NH=2)
    for other, error in ((dict(out=out.double()), TypeError), (dict(out=out.cpu()), TypeError), (dict(out=out[:, :64]), ValueError),
                         (dict(out=out.t().contiguous().t()), ValueError), (dict(lengths=c.dl.long()), TypeError),
                         (dict(lengths=c.dl[:1]), ValueError), (dict(inp=inp[:, :-1]), ValueError), (dict(inp=inp[:1]), ValueError),
                         (dict(inp=inp.t()), ValueError), (dict(inp=inp.cpu()), TypeError), (dict(B=3), ValueError),
                         (dict(weights_in=torch.zeros((2, 1, 32), device="cuda")), g2.GPT2HipError),
                         (dict(weights_in=torch.zeros((2, 1, 31), device="cuda")), ValueError)):
        with pytest.raises(error):
            g2.attention_decode_paged(**{**ok, **other})
    g2.attention_decode_paged(**ok)
    torch.cuda.synchronize()
