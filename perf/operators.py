"""What a decoding server asks of a paged key/value cache, as cases that can be timed and checked.

Three operators: the rows of new prompts are stored into pages (``kv_store_paged``), one new
token per sequence is appended and attends to its pages (``attention_decode_paged``), and a
cache that has grown beyond its budget keeps the positions that the attention weighed most
(``kv_evict_paged``).  ``run`` makes the framework's calls where ``own`` is true and computes
the same operators with elementary torch operations otherwise.

Keys and values are held in pages of shape (page, kv head, slot, channel); row b of a table
lists the pages of sequence b in order.  A packed row is q | k | v, head after head.
"""
import importlib
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MOST_BYTES = 0.98e9    # keys and values of a drawn case
MOST_ROW_FLOATS = 2e8  # floats of the packed rows of a drawn prompt batch


def listed():
    return [
        # one sequence early in a chat with the smallest configuration: latency counts
        dict(name="attend one short", op="attend", type="f32", B=1, NH=12, KVH=12, HS=64, page=16, lo=100, hi=100, weights=False),
        # a batch in mid-flight, every sequence at another length, one of them just begun
        dict(name="attend ragged f32", op="attend", type="f32", B=16, NH=12, KVH=12, HS=64, page=16, lo=1, hi=1023, weights=False),
        # a full server of the widest configuration (25 heads), cache in 16 bits
        dict(name="attend full bf16", op="attend", type="bf16", B=64, NH=25, KVH=25, HS=64, page=32, lo=200, hi=1023, weights=False),
        # long contexts with query heads that share their keys
        dict(name="attend long shared", op="attend", type="bf16", B=8, NH=32, KVH=8, HS=128, page=64, lo=28000, hi=32767, weights=False),
        # one very long sequence alone: the work has to be split over the cache's length
        dict(name="attend one long f16", op="attend", type="f16", B=1, NH=20, KVH=20, HS=64, page=128, lo=65001, hi=65001, weights=False),
        # decoding under a budget: the step also accumulates what each position weighed
        dict(name="attend weights f32", op="attend", type="f32", B=12, NH=16, KVH=16, HS=64, page=16, lo=300, hi=1000, weights=True),
        # the same with shared keys, a head size and a page size that are no powers of two
        dict(name="attend weights odd", op="attend", type="bf16", B=4, NH=32, KVH=4, HS=96, page=24, lo=5000, hi=9001, weights=True),
        # two prompts of a few tokens each join a running batch
        dict(name="store short", op="store", type="bf16", B=2, NH=12, KVH=12, HS=64, page=16, lo=5, hi=11, held=0),
        # a batch of ordinary prompts of ragged lengths
        dict(name="store prompts", op="store", type="f32", B=8, NH=12, KVH=12, HS=64, page=16, lo=129, hi=1023, held=0),
        # further pieces of long prompts behind what is held already, into 16 bits
        dict(name="store long", op="store", type="bf16", B=4, NH=32, KVH=8, HS=128, page=64, lo=4001, hi=8192, held=517),
        # a batch at its full context is brought down to half of it
        dict(name="evict half", op="evict", type="f32", B=8, NH=12, KVH=12, HS=64, page=16, lo=900, hi=1024, budget=512, recent=64),
        # long contexts with shared keys are brought down to a quarter
        dict(name="evict long", op="evict", type="bf16", B=4, NH=32, KVH=8, HS=128, page=64, lo=30000, hi=32768, budget=8192, recent=512),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "store", "evict"])
    kind = rng.choice(["f32", "f16", "bf16"])
    NH, KVH, HS = rng.choice([(12, 12, 64), (16, 16, 64), (20, 20, 64), (25, 25, 64), (32, 8, 128), (32, 4, 96), (16, 2, 64), (24, 8, 80), (12, 1, 64)])
    page = rng.choice([16, 16, 24, 32, 64, 128])
    size = TYPES[kind].itemsize
    B = _spread(rng, 1, 64)
    row = 2 * KVH * HS * size
    top = int(min(65536, MOST_BYTES / (row * B)))
    if op == "store":
        top = int(min(8192, top, MOST_ROW_FLOATS / ((NH + 2 * KVH) * HS * B)))
    if op == "evict":
        top = int(min(32768, top, MOST_BYTES / (row * B) / 1.6))
    hi = _spread(rng, 1, max(1, top)) if op == "store" else _spread(rng, min(16, top), top)
    lo = _spread(rng, 1, hi) if rng.random() < 0.7 else hi
    case = dict(op=op, type=kind, B=B, NH=NH, KVH=KVH, HS=HS, page=page, lo=lo, hi=hi)
    if op == "attend":
        case["weights"] = rng.random() < 0.35
    elif op == "store":
        case["held"] = rng.choice([0, 0, rng.randint(1, 600)])
    else:
        case["budget"] = max(1, int(hi * rng.uniform(0.1, 0.9)))
        case["recent"] = int(case["budget"] * rng.uniform(0.0, 0.5))
    return case


def _lengths(case):
    """The B lengths of a case: lo..hi, spread over the batch, the longest first."""
    lo, hi, B = case["lo"], case["hi"], case["B"]
    return [hi - int((hi - lo) * ((b * 0.6180339887) % 1.0)) for b in range(B)] if B > 1 else [hi]


def work(case):
    n, size = _lengths(case), TYPES[case["type"]].itemsize
    B, NH, KVH, HS, page = (case[k] for k in ("B", "NH", "KVH", "HS", "page"))
    row = 2 * KVH * HS
    if case["op"] == "attend":
        # the positions held, the packed rows, the row appended, the output, the pages' numbers
        moved = sum(n) * row * size + B * ((NH + 2 * KVH) * HS * 4 + row * size + NH * HS * 4)
        moved += sum(-(-(x + 1) // page) for x in n) * 4
        if case["weights"]:
            moved += KVH * 4 * (sum(n) + sum(x + 1 for x in n))
        return {"bytes": moved, "flops": 4 * NH * HS * sum(x + 1 for x in n)}
    if case["op"] == "store":
        return {"bytes": sum(n) * row * (4 + size), "flops": 0}
    kept = sum(min(x, case["budget"]) for x in n)
    # every weight is read; what is kept is read and written, with its weight and its number
    return {"bytes": KVH * 4 * sum(n) + kept * (2 * row * size + KVH * 8), "flops": 0}


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    n, kind = _lengths(case), TYPES[case["type"]]
    B, NH, KVH, HS, page = (case[k] for k in ("B", "NH", "KVH", "HS", "page"))
    order = torch.randperm(B, generator=gen, device=dev)
    lengths = torch.tensor(n, dtype=torch.int32, device=dev)[order]
    op, longest = case["op"], max(n)
    s = dict(case=case, B=B, NH=NH, KVH=KVH, HS=HS, page=page)

    held = {"attend": longest + 1, "store": longest + case.get("held", 0), "evict": longest}[op]
    width = -(-held // page)
    kept_width = -(-case["budget"] // page) if op == "evict" else 0
    # every sequence has its pages anywhere in the pool, which other sequences have used before
    pool = B * (width + kept_width) + 5
    pages = torch.randperm(pool, generator=gen, device=dev).to(torch.int32)
    table = pages[: B * width].reshape(B, width).contiguous()
    keys = torch.empty((pool, KVH, page, HS), dtype=kind, device=dev).normal_(generator=gen)
    values = torch.empty((pool, KVH, page, HS), dtype=kind, device=dev).normal_(generator=gen)
    s.update(keys=keys, values=values, table=table)

    if op == "store":
        starts = torch.zeros(B + 1, dtype=torch.int32, device=dev)
        starts[1:] = lengths.cumsum(0)
        N = sum(n)
        s.update(N=N, starts=starts, inp=torch.randn((N, (NH + 2 * KVH) * HS), generator=gen, device=dev))
        s["lengths"] = torch.full((B,), case["held"], dtype=torch.int32, device=dev)
    else:
        s["lengths"] = lengths
    if op == "attend":
        inp = torch.randn((B, (NH + 2 * KVH) * HS), generator=gen, device=dev)
        inp[:, : NH * HS] *= 2.0  # queries that prefer some keys to others
        s.update(inp=inp, out=torch.zeros((B, NH * HS), device=dev))
    if op == "evict" or case.get("weights"):
        # few positions weigh much, most weigh next to nothing, some exactly nothing
        w = torch.rand((B, KVH, width * page), generator=gen, device=dev)
        w = 20.0 * w ** 12
        w[w < 1e-9] = 0.0
        s["weights_in"] = w
    if op == "attend" and case["weights"]:
        s["weights_out"] = torch.zeros_like(s["weights_in"])
    if op == "evict":
        budget = case["budget"]
        s.update(budget=budget, recent=case["recent"],
                 kept_table=pages[B * width: B * (width + kept_width)].reshape(B, kept_width).contiguous(),
                 kept=torch.full((B, KVH, budget), -1, dtype=torch.int32, device=dev),
                 weights_out=torch.zeros((B, KVH, kept_width * page), device=dev),
                 lengths_out=torch.zeros(B, dtype=torch.int32, device=dev))
    if own:
        g2 = importlib.import_module("cuda-gpt2-inference_amd")
        s["g2"] = g2
        s["cache"] = g2.PagedCache(keys, values, table)
        if op == "attend":
            s["workspace"] = g2.attention_decode_paged_workspace(s["cache"], B, NH, weights=case["weights"])
        if op == "evict":
            s["kept_cache"] = g2.PagedCache(keys, values, s["kept_table"])
    return s


# ---- the operators in elementary operations ------------------------------------------------

def _plain_store(s):
    NH, KVH, HS, page = s["NH"], s["KVH"], s["HS"], s["page"]
    rows = torch.arange(s["N"], device=s["inp"].device)
    seq = torch.searchsorted(s["starts"].long(), rows, right=True) - 1
    pos = s["lengths"].long()[seq] + rows - s["starts"].long()[seq]
    at, slot = s["table"].long()[seq, pos // page], pos % page
    k = s["inp"][:, NH * HS:(NH + KVH) * HS].reshape(-1, KVH, HS)
    v = s["inp"][:, (NH + KVH) * HS:].reshape(-1, KVH, HS)
    s["keys"][at, :, slot] = k.to(s["keys"].dtype)
    s["values"][at, :, slot] = v.to(s["values"].dtype)
    return {"keys": s["keys"], "values": s["values"]}


def _gathered(pages, table):
    """(B, kv head, position, channel) in 32 bits."""
    x = pages[table.long()].permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4]).float()


def _plain_attend(s):
    B, NH, KVH, HS, page = s["B"], s["NH"], s["KVH"], s["HS"], s["page"]
    inp, n = s["inp"], s["lengths"].long()
    at, slot = s["table"].long().gather(1, (n // page)[:, None])[:, 0], n % page
    s["keys"][at, :, slot] = inp[:, NH * HS:(NH + KVH) * HS].reshape(B, KVH, HS).to(s["keys"].dtype)
    s["values"][at, :, slot] = inp[:, (NH + KVH) * HS:].reshape(B, KVH, HS).to(s["values"].dtype)
    q = inp[:, : NH * HS].reshape(B, KVH, NH // KVH, HS)
    k = _gathered(s["keys"], s["table"])
    held = torch.arange(k.shape[2], device=k.device)[None] <= n[:, None]
    scores = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(HS))
    del k
    scores = scores.masked_fill(~held[:, None, None], float("-inf"))
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    v = _gathered(s["values"], s["table"]).masked_fill_(~held[:, None, :, None], 0.0)
    out = {"out": torch.matmul(p, v).reshape(B, NH * HS), "keys": s["keys"], "values": s["values"]}
    if s["case"]["weights"]:
        before = torch.arange(held.shape[1], device=held.device)[None] < n[:, None]
        w = torch.where(before[:, None], s["weights_in"], torch.zeros_like(s["weights_in"])) + p.sum(2)
        out["weights"] = torch.where(held[:, None], w, s["weights_out"])
    return out


def _plain_evict(s):
    page, budget, dev = s["page"], s["budget"], s["keys"].device
    w, n = s["weights_in"], s["lengths"].long()
    pos = torch.arange(w.shape[2], device=dev)[None]
    rank = w.masked_fill((pos >= (n - s["recent"])[:, None])[:, None], float("inf"))
    rank = rank.masked_fill((pos >= n[:, None])[:, None], float("-inf"))
    take = min(budget, w.shape[2])
    first = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :take]
    left = n.clamp(max=budget)
    live = (torch.arange(take, device=dev)[None] < left[:, None])[:, None].expand_as(first)
    at = torch.sort(first.masked_fill(~live, w.shape[2]), dim=-1)[0]
    src = at.clamp(max=w.shape[2] - 1)
    kept = s["kept"].clone()
    kept[..., :take] = at.masked_fill(~live, -1).to(torch.int32)
    b = torch.arange(s["B"], device=dev)[:, None, None]
    h = torch.arange(s["KVH"], device=dev)[None, :, None]
    j = torch.arange(take, device=dev)[None, None]
    to, frm = s["kept_table"].long()[b, j // page], s["table"].long()[b, src // page]
    for pages in (s["keys"], s["values"]):
        pages[to, h, j % page] = torch.where(live[..., None], pages[frm, h, src % page], pages[to, h, j % page])
    weights = s["weights_out"].clone()
    weights[..., :take] = torch.where(live, w.gather(2, src), weights[..., :take])
    return {"kept": kept, "keys": s["keys"], "values": s["values"], "weights": weights, "lengths": left.to(torch.int32)}


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"store": _plain_store, "attend": _plain_attend, "evict": _plain_evict}[op](s)
    g2 = s["g2"]
    if op == "store":
        g2.kv_store_paged(s["cache"], s["inp"], s["starts"], s["lengths"], s["N"], s["B"], s["NH"])
        return {"keys": s["keys"], "values": s["values"]}
    if op == "attend":
        g2.attention_decode_paged(s["out"], s["cache"], s["inp"], s["lengths"], s["B"], s["NH"], weights_in=s.get("weights_in"),
                                  weights_out=s.get("weights_out"), workspace=s["workspace"])
        out = {"out": s["out"], "keys": s["keys"], "values": s["values"]}
        if s["case"]["weights"]:
            out["weights"] = s["weights_out"]
        return out
    g2.kv_evict_paged(s["kept_cache"], s["cache"], s["kept"], s["weights_out"], s["lengths_out"], s["weights_in"], s["lengths"],
                      s["B"], s["budget"], s["recent"])
    return {"kept": s["kept"], "keys": s["keys"], "values": s["values"], "weights": s["weights_out"], "lengths": s["lengths_out"]}


# ---- the same from the definitions, sequence by sequence, in 64 bits -----------------------

def exact(case, seed):
    s = prepare(case, seed)
    NH, KVH, HS, page = s["NH"], s["KVH"], s["HS"], s["page"]
    keys, values, table = s["keys"], s["values"], s["table"].cpu().tolist()
    n = s["lengths"].cpu().tolist()

    def put(b, first, rows):
        """Stores packed rows as the positions of sequence b from `first` on, rounded as the cache holds them."""
        k = rows[:, NH * HS:(NH + KVH) * HS].reshape(-1, KVH, HS).to(keys.dtype)
        v = rows[:, (NH + KVH) * HS:].reshape(-1, KVH, HS).to(values.dtype)
        i = 0
        while i < len(rows):
            page_at, slot = divmod(first + i, page)
            m = min(page - slot, len(rows) - i)
            keys[table[b][page_at], :, slot:slot + m] = k[i:i + m].transpose(0, 1)
            values[table[b][page_at], :, slot:slot + m] = v[i:i + m].transpose(0, 1)
            i += m

    def sequence(pages, b, count):
        """(kv head, position, channel) of the first `count` positions of sequence b, in 64 bits."""
        x = pages[s["table"][b].long()].transpose(0, 1).reshape(KVH, -1, HS)
        return x[:, :count].double()

    if case["op"] == "store":
        starts = s["starts"].cpu().tolist()
        for b in range(s["B"]):
            put(b, n[b], s["inp"][starts[b]:starts[b + 1]])
        return {"keys": keys.double(), "values": values.double()}

    if case["op"] == "attend":
        out, weights = [], s["weights_out"].double() if case["weights"] else None
        for b in range(s["B"]):
            put(b, n[b], s["inp"][b:b + 1])
            q = s["inp"][b, : NH * HS].double().reshape(KVH, NH // KVH, HS)
            k, v = sequence(keys, b, n[b] + 1), sequence(values, b, n[b] + 1)
            p = torch.softmax((q @ k.transpose(1, 2).contiguous()) / math.sqrt(HS), dim=-1)
            out.append((p @ v).reshape(-1))
            if weights is not None:
                weights[b, :, : n[b] + 1] = p.sum(1)
                weights[b, :, : n[b]] += s["weights_in"][b, :, : n[b]].double()
        got = {"out": torch.stack(out), "keys": keys.double(), "values": values.double()}
        if weights is not None:
            got["weights"] = weights
        return got

    budget, recent = s["budget"], s["recent"]
    kept_table, kept, weights = s["kept_table"].cpu().tolist(), s["kept"], s["weights_out"].double()
    for b in range(s["B"]):
        m = min(n[b], budget)
        free = n[b] - recent if n[b] > budget else 0  # positions that have to earn their place
        w = s["weights_in"][b, :, : n[b]].double()
        older = torch.argsort(w[:, :free], dim=1, descending=True, stable=True)[:, : m - (n[b] - free)]
        newer = torch.arange(free, n[b], device=w.device).expand(KVH, -1)
        rows = torch.cat([torch.sort(older, dim=1)[0], newer], dim=1)
        kept[b, :, :m] = rows.to(torch.int32)
        weights[b, :, :m] = w.gather(1, rows)
        for pages in (keys, values):
            x = pages[s["table"][b].long()].transpose(0, 1).reshape(KVH, -1, HS)
            x = x.gather(1, rows[:, :, None].expand(-1, -1, HS))
            for i in range(0, m, page):
                pages[kept_table[b][i // page], :, : min(page, m - i)] = x[:, i:i + page]
    return {"kept": kept, "keys": keys.double(), "values": values.double(), "weights": weights,
            "lengths": torch.tensor([min(x, budget) for x in n], dtype=torch.int32)}
