"""One serving step over the paged KV cache, operator by operator: what is timed, and what each operator computes.

  tables  page tables and slot maps of a batch from its sequences' lengths (pages from a free list)
  append  rotary positions on q and k, k and v written to their cache slots
  attend  attention of each sequence's new tokens over its pages (one token, a chunk, a long prompt; mixed)
  sample  temperature, top-k, top-p, min-p and a draw from given uniform numbers, row by row

`own` False runs the plain forms below (elementary torch operations); True makes the calls of tinybrain_b200.serving.
The cache layout is the framework's: pool [pages][layers][K, V][kv heads][16 tokens][head dim] fp32, page tables
[sequences][logical page] int32 with -1 for an evicted page, whose rows read as zeros.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 16
LAYERS = 2  # layers in the pool: the strides of a real cache, one layer used
LAYER = 1


# --------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of the benchmark's 64 sequences: one new token each
        {"name": "tables decode 64", "op": "tables", "batch": 64, "new_min": 1, "new_max": 1, "len_min": 512, "len_max": 4224, "single": 0.0, "mix": 4},
        # a large mixed step: most sequences decode, some bring a prompt chunk
        {"name": "tables mixed 4096", "op": "tables", "batch": 4096, "new_min": 0, "new_max": 517, "len_min": 1, "len_max": 8192, "single": 0.8, "mix": 11},
        # the same decode step's rows, TinyLlama heads
        {"name": "append decode 64", "op": "append", "rows": 64, "heads": 32, "kv": 4, "dim": 64, "positions": 4352, "mix": 5},
        # a long prefill, 7B heads
        {"name": "append prompt 8192", "op": "append", "rows": 8192, "heads": 32, "kv": 32, "dim": 128, "positions": 8192, "mix": 6},
        # the smallest call: one token of one sequence with a short context
        {"name": "attend one token", "op": "attend", "batch": 1, "new_min": 1, "new_max": 1, "len_min": 129, "len_max": 129, "single": 0.0, "heads": 32, "kv": 4, "dim": 64, "evicted": 0, "mix": 1},
        # the benchmark's decode step: 64 sequences, contexts 512 to 4224
        {"name": "attend decode 64", "op": "attend", "batch": 64, "new_min": 1, "new_max": 1, "len_min": 512, "len_max": 4224, "single": 0.0, "heads": 32, "kv": 4, "dim": 64, "evicted": 0, "mix": 4},
        # one 64-token chunk of a 1920-token prompt, the runner's chunk size
        {"name": "attend chunk 64", "op": "attend", "batch": 1, "new_min": 64, "new_max": 64, "len_min": 1920, "len_max": 1920, "single": 0.0, "heads": 32, "kv": 4, "dim": 64, "evicted": 0, "mix": 3},
        # a mixed ragged step, 7B heads: single tokens, odd chunks, an idle sequence, evicted pages
        {"name": "attend mixed", "op": "attend", "batch": 13, "new_min": 0, "new_max": 301, "len_min": 1, "len_max": 2047, "single": 0.5, "heads": 32, "kv": 32, "dim": 128, "evicted": 2, "mix": 7},
        # the last 2048 tokens of an 8192-token prompt
        {"name": "attend prompt 2048", "op": "attend", "batch": 1, "new_min": 2048, "new_max": 2048, "len_min": 8192, "len_max": 8192, "single": 0.0, "heads": 32, "kv": 4, "dim": 64, "evicted": 0, "mix": 2},
        # one sequence's next token, the benchmark's vocabulary
        {"name": "sample one row", "op": "sample", "rows": 1, "vocab": 32000, "pad": 0, "mix": 1},
        # the benchmark's 64 sequences, each with its own settings
        {"name": "sample 64 rows", "op": "sample", "rows": 64, "vocab": 32000, "pad": 0, "mix": 2},
        # a large batch and a large vocabulary
        {"name": "sample 256 large", "op": "sample", "rows": 256, "vocab": 131072, "pad": 0, "mix": 3},
    ]


def _log(rng, lo, hi):
    """A whole number of lo .. hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


HEADS = [(32, 4, 64), (32, 32, 128), (8, 2, 64), (16, 4, 32), (16, 2, 64), (8, 8, 16), (32, 8, 128)]


def draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend", "sample"])
    mix = rng.randrange(1 << 20)
    while op == "tables":
        most = _log(rng, 1, 517)
        case = {"op": op, "batch": _log(rng, 1, 4096), "new_min": rng.randint(0, 1), "new_max": most, "len_min": 1,
                "len_max": max(most + 1, _log(rng, 64, 8192)), "single": rng.choice([0.0, 0.8, 1.0]), "mix": mix}
        if sum(_lengths(case)[1]):
            return case
    if op == "append":
        h, kv, d = rng.choice(HEADS)
        return {"op": op, "rows": _log(rng, 1, 8192), "heads": h, "kv": kv, "dim": d, "positions": _log(rng, 64, 8192), "mix": mix}
    if op == "sample":
        return {"op": op, "rows": _log(rng, 1, 256), "vocab": _log(rng, 100, 131072), "pad": rng.choice([0, 0, 1, 3, 8]), "mix": mix}
    while True:
        h, kv, d = rng.choice(HEADS)
        batch, most, total = _log(rng, 1, 64), rng.choice([1, _log(rng, 2, 2048)]), _log(rng, 16, 8192)
        case = {"op": op, "batch": batch, "new_min": rng.randint(0, 1), "new_max": min(most, total), "len_min": 1, "len_max": total,
                "single": rng.choice([0.0, 0.5]), "heads": h, "kv": kv, "dim": d, "evicted": rng.choice([0, 0, 1, 3]), "mix": mix}
        total, new = _lengths(case)
        if sum(new) and batch * max(new) * max(total) * h <= 2048 * 8192 * 32 and batch * max(total) * kv * d <= 1 << 26:
            return case


def _lengths(case):
    """Every sequence's length with its new tokens, and how many of them are new."""
    r = random.Random(case["mix"])
    total, new = [], []
    for _ in range(case["batch"]):
        t = r.randint(case["len_min"], case["len_max"])
        n = 1 if r.random() < case["single"] else r.randint(case["new_min"], case["new_max"])
        total.append(t)
        new.append(min(n, t))
    return total, new


def _pages(n):
    return -(-n // PAGE)


# -------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(new):
    return _ints([0] + list(np.cumsum(new)))


def prepare(case, seed):
    return {"tables": _prepare_tables, "append": _prepare_append, "attend": _prepare_attend, "sample": _prepare_sample}[case["op"]](case, seed)


def _prepare_tables(case, seed):
    g = _gen(seed)
    total, new = _lengths(case)
    cached = [t - n for t, n in zip(total, new)]
    stride = _pages(case["len_max"]) + 1
    held = sum(_pages(c) for c in cached)
    need = sum(_pages(t) for t in total) - held
    order = torch.randperm(held + need + 7, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["batch"], stride), -1, dtype=torch.int32, device="cuda")
    owned = torch.arange(stride, device="cuda")[None] < _ints([_pages(c) for c in cached])[:, None]
    table[owned] = order[:held]
    rows = sum(new)
    room = rows + 5  # a step's buffers are larger than the step
    blank = lambda n, t=torch.int32: torch.full((n,), -7, dtype=t, device="cuda")  # noqa: E731
    return {"op": "tables", "rows": rows, "cached": _ints(cached), "new": _ints(new), "free": order[held:].clone(), "table": table,
            "row_offsets": blank(case["batch"] + 1), "total": blank(case["batch"]), "row_seq": blank(room), "row_pos": blank(room),
            "row_slot": blank(room, torch.int64), "info": blank(4)}


def _prepare_append(case, seed):
    g = _gen(seed)
    T, H, kv, d = case["rows"], case["heads"], case["kv"], case["dim"]
    r = random.Random(case["mix"])
    pages = _pages(T) + _pages(T) // 4 + 2
    slots = torch.randperm(pages * PAGE, generator=g, device="cuda")[:T].clone()
    if T > 1:  # prompts fill pages in order: all but the last rows are runs of 16
        runs = torch.randperm(pages, generator=g, device="cuda")[: _pages(T)]
        slots = (runs[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)[:T].clone()
        slots[r.randrange(T)] = -1  # an evicted page: nothing is written
    pos = torch.randint(0, case["positions"], (T,), generator=g, device="cuda", dtype=torch.int32)
    angle = torch.arange(case["positions"], dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    rope = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    qkv = torch.randn(T, (H + 2 * kv) * d, generator=g, device="cuda")  # the fused projection's output
    pool = torch.randn(pages, LAYERS, 2, kv, PAGE, d, generator=g, device="cuda")
    return {"op": "append", "H": H, "kv": kv, "d": d, "q": qkv[:, : H * d], "k": qkv[:, H * d : (H + kv) * d], "v": qkv[:, (H + kv) * d :],
            "row_pos": pos, "row_slot": slots, "rope": rope, "pool": pool, "q_out": torch.zeros(T, H * d, device="cuda")}


def _prepare_attend(case, seed):
    g = _gen(seed)
    H, kv, d = case["heads"], case["kv"], case["dim"]
    total, new = _lengths(case)
    stride = _pages(max(total)) + 1
    count = [_pages(t) for t in total]
    pages = sum(count) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(total), stride), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(stride, device="cuda")[None] < _ints(count)[:, None]] = order[: sum(count)]
    if case["evicted"]:  # the oldest pages of the longer sequences are gone
        for s, c in enumerate(count):
            if c > case["evicted"] + 2:
                table[s, : case["evicted"]] = -1
    rows = sum(new)
    seq = np.repeat(np.arange(len(new)), new)
    index = np.concatenate([np.arange(n) for n in new])
    return {"op": "attend", "H": H, "kv": kv, "d": d, "max_new": max(new), "max_len": max(total),
            "q": 2.0 * torch.randn(rows, H * d, generator=g, device="cuda"),
            "pool": torch.randn(pages, LAYERS, 2, kv, PAGE, d, generator=g, device="cuda"),
            "table": table, "row_offsets": _offsets(new), "total": _ints(total), "new": _ints(new),
            "row_seq": torch.from_numpy(seq).cuda(), "row_index": torch.from_numpy(index).cuda(),
            "out": torch.zeros(rows, H * d, device="cuda")}


def _prepare_sample(case, seed):
    g = _gen(seed)
    T, V = case["rows"], case["vocab"]
    r = random.Random(case["mix"])
    # a language model's row: a bulk, and a few dozen tokens well above it
    full = 2.0 * torch.randn(T, V + case["pad"], generator=g, device="cuda")
    peaks = torch.randint(0, V, (T, min(V, 40)), generator=g, device="cuda")
    full.scatter_add_(1, peaks, 12.0 * torch.rand(peaks.shape, generator=g, device="cuda"))
    full[torch.rand(full.shape, generator=g, device="cuda") < 0.01] = -math.inf  # tokens a grammar forbids
    full[:, V // 3] = torch.finfo(torch.float32).min  # and one masked with the type's lowest value
    if T > 8:
        full[r.randrange(T)] = -math.inf  # nothing is left
    pick = lambda v, t: torch.tensor([r.choice(v) for _ in range(T)], dtype=t, device="cuda")  # noqa: E731
    return {"op": "sample", "logits": full[:, :V], "uniform": torch.rand(T, generator=g, device="cuda"),
            "temperature": pick([0.7, 0.8, 1.0, 1.3] + [0.0] * (T > 1), torch.float32), "top_k": pick([0, 0, 1, 40, 1000], torch.int32),
            "top_p": pick([1.0, 0.95, 0.9, 0.5], torch.float32), "min_p": pick([0.0, 0.0, 0.05, 0.1], torch.float32),
            "token": torch.zeros(T, dtype=torch.int32, device="cuda"), "prob": torch.zeros(T, device="cuda"), "entropy": torch.zeros(T, device="cuda")}


# ---------------------------------------------------------------------- runs
def run(state):
    s = state
    if own:
        from tinybrain_b200 import serving

        if s["op"] == "tables":
            serving.build_page_tables(s["cached"], s["new"], s["free"], s["table"], s["row_offsets"], s["total"], s["row_seq"], s["row_pos"],
                                      s["row_slot"], s["info"])
        elif s["op"] == "append":
            serving.rope_append(s["q"], s["k"], s["v"], s["row_pos"], s["row_slot"], s["rope"], s["pool"], s["q_out"], layer=LAYER)
        elif s["op"] == "attend":
            serving.paged_attention_chunk(s["q"], s["row_offsets"], s["total"], s["pool"], s["table"], s["out"], layer=LAYER, max_new=s["max_new"],
                                          max_len=s["max_len"])
        else:
            serving.sample_rows(s["logits"], s["uniform"], s["token"], s["prob"], s["entropy"], temperature=s["temperature"], top_k=s["top_k"],
                                top_p=s["top_p"], min_p=s["min_p"])
    else:
        {"tables": _tables, "append": _append, "attend": _attend, "sample": _sample}[s["op"]](s)
    names = {"tables": ("table", "row_offsets", "total", "row_seq", "row_pos", "row_slot", "info"), "append": ("q_out", "pool"), "attend": ("out",),
             "sample": ("token", "prob", "entropy")}[s["op"]]
    return {n: s[n] for n in names}


def _tables(s):
    """Sequence q holds ceil(c / 16) pages and needs ceil((c + n) / 16): the missing ones come off the free list's front,
    sequence by sequence. Its n rows follow those of the sequences before it; a row's slot is page * 16 + position % 16."""
    cached, new, table = s["cached"].long(), s["new"].long(), s["table"]
    total = cached + new
    before, after = (cached + PAGE - 1) // PAGE, (total + PAGE - 1) // PAGE
    taken = (after - before).cumsum(0)
    first = taken - (after - before)
    logical = torch.arange(table.shape[1], device=table.device)[None]
    fresh = (logical >= before[:, None]) & (logical < after[:, None])
    at = (first[:, None] + logical - before[:, None]).clamp(0, max(0, s["free"].numel() - 1))
    table.copy_(torch.where(fresh, s["free"][at], table))
    offsets = torch.cat([new.new_zeros(1), new.cumsum(0)])
    s["row_offsets"].copy_(offsets)
    s["total"].copy_(total)
    rows = s["rows"]
    seq = torch.repeat_interleave(torch.arange(new.numel(), device=table.device), new, output_size=rows)
    pos = cached[seq] + torch.arange(rows, device=table.device) - offsets[seq]
    page = table[seq, pos // PAGE].long()
    s["row_seq"][:rows] = seq.to(torch.int32)
    s["row_pos"][:rows] = pos.to(torch.int32)
    s["row_slot"][:rows] = torch.where(page < 0, -1, page * PAGE + pos % PAGE)
    s["info"].copy_(torch.stack([offsets[-1], taken[-1], torch.zeros_like(taken[-1]), torch.full_like(taken[-1], -1)]))


def _append(s):
    """Pairs (x0, x1) of neighbouring dims become (x0 cos - x1 sin, x0 sin + x1 cos), the table's row at the token's position."""
    T, kv, d = s["q"].shape[0], s["kv"], s["d"]
    cs = s["rope"][s["row_pos"].long()][:, None]  # [T, 1, d / 2, (cos, sin)]

    def turned(x):
        x = x.reshape(T, -1, d // 2, 2)
        a, b = x[..., 0], x[..., 1]
        return torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1)

    s["q_out"].copy_(turned(s["q"]).reshape(T, -1))
    both = torch.stack([turned(s["k"]).reshape(T, kv, d), s["v"].reshape(T, kv, d)], 1)  # [T, 2, kv, d]
    slot = s["row_slot"]
    at = s["pool"].permute(0, 4, 1, 2, 3, 5)[:, :, LAYER]  # [page, token, 2, kv, d]
    page, token = slot.clamp(min=0) // PAGE, slot.clamp(min=0) % PAGE
    keep = (slot >= 0)[:, None, None, None]
    # a row without a slot repeats what another one writes: the first row that has one
    stand = (slot >= 0).to(torch.int8).argmax()
    none = slot < 0
    at[torch.where(none, page[stand], page), torch.where(none, token[stand], token)] = torch.where(keep, both, both[stand][None])


def _attend(s):
    """softmax(q k / sqrt(d)) v over the positions up to the row's own; evicted pages read as zeros."""
    H, kv, d, n, L = s["H"], s["kv"], s["d"], s["max_new"], s["max_len"]
    B, G = s["table"].shape[0], H // kv
    total, new = s["total"].long(), s["new"].long()
    pos = torch.arange(L, device=total.device)
    page = s["table"][:, pos // PAGE].long()
    held = (page >= 0) & (pos[None] < total[:, None])
    rows = s["pool"][:, LAYER].permute(0, 3, 1, 2, 4)[page.clamp(min=0), pos % PAGE]  # [B, L, 2, kv, d]
    rows = torch.where(held[..., None, None, None], rows, 0.0)
    i = torch.arange(n, device=total.device)
    q = s["q"][(s["row_offsets"][:-1].long()[:, None] + i).clamp(max=s["q"].shape[0] - 1)]
    q = q.reshape(B, n, kv, G, d).permute(0, 2, 1, 3, 4).reshape(B, kv, n * G, d)
    score = (q @ rows[:, :, 0].permute(0, 2, 3, 1)) / math.sqrt(d)
    seen = pos <= (total - new)[:, None, None] + i[None, :, None]  # [B, n, L]
    seen = (seen & (pos < total[:, None])[:, None]).repeat_interleave(G, 1)[:, None]
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    o = (p @ rows[:, :, 1].permute(0, 2, 1, 3)) / p.sum(-1, keepdim=True)
    o = o.reshape(B, kv, n, G, d).permute(0, 2, 1, 3, 4).reshape(B, n, H * d)
    s["out"].copy_(o[s["row_seq"], s["row_index"]])


def _sample(s):
    """Weights exp((x - max) / T). In descending order (equal values: lowest index first) top-k keeps the first k, top-p the
    shortest prefix of those with top_p of their mass, min-p those of at least min_p times the largest weight. The token is the
    first, in index order, whose running mass passes u times the kept mass. T = 0 takes the maximum. An empty row gives -1."""
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    T, V = x.shape
    temp = s["temperature"].double()[:, None]
    top = x.amax(1, keepdim=True)
    empty = top == -math.inf
    y = torch.where(x == top, 0.0, (x - top) / torch.where(temp > 0, temp, 1.0))
    y = torch.where(x == -math.inf, -math.inf, y)
    w = y.exp()
    order = x.sort(dim=1, descending=True, stable=True).indices
    k = s["top_k"].long()[:, None]
    k = torch.where((k <= 0) | (k > V), V, k)
    k = torch.where(temp > 0, k, 1)
    rank = torch.arange(V, device=x.device)[None]
    ws = torch.where(rank < k, w.gather(1, order), 0.0)
    run_ = ws.cumsum(1)
    p = s["top_p"].double()[:, None]
    keep = (rank < k) & ((p >= 1) | (rank == 0) | (run_ - ws < p * run_[:, -1:]))
    keep &= ws >= s["min_p"].double()[:, None]
    keep = torch.zeros_like(keep).scatter_(1, order, keep) & (w > 0)
    w = torch.where(keep, w, 0.0)
    mass = w.cumsum(1)
    all_ = mass[:, -1:]
    token = (mass <= s["uniform"].double()[:, None] * all_).sum(1, keepdim=True)
    last = (keep * rank).amax(1, keepdim=True)
    token = torch.minimum(token, last)
    prob = w.gather(1, token) / all_
    entropy = all_.log() - (w * torch.where(keep, y, 0.0)).sum(1, keepdim=True) / all_
    s["token"].copy_(torch.where(empty, -1, token)[:, 0])
    s["prob"].copy_(torch.where(empty, 0.0, prob)[:, 0])
    s["entropy"].copy_(torch.where(empty, 0.0, entropy)[:, 0])


# ---------------------------------------------------------------------- work
def work(case):
    if case["op"] == "tables":
        total, new = _lengths(case)
        rows, taken = sum(new), sum(_pages(t) - _pages(t - n) for t, n in zip(total, new))
        # lengths in, offsets and totals out; a free page in and a table entry out; three numbers a row out, a table entry in per page
        return {"bytes": case["batch"] * 16 + taken * 8 + rows * 16 + sum(1 for n in new if n) * 4, "flops": rows * 4}
    if case["op"] == "append":
        T, H, kv, d = case["rows"], case["heads"], case["kv"], case["dim"]
        return {"bytes": T * ((H + 2 * kv) * d * 8 + 12) + min(T, case["positions"]) * d * 4, "flops": T * (H + kv) * d * 3}
    if case["op"] == "attend":
        H, kv, d = case["heads"], case["kv"], case["dim"]
        total, new = _lengths(case)
        live = [(t, n) for t, n in zip(total, new) if n]
        pairs = sum(n * (t - n) + n * (n + 1) // 2 for t, n in live)
        return {"bytes": 8 * H * d * sum(new) + sum(t for t, _ in live) * kv * d * 8 + sum(_pages(t) for t, _ in live) * 4, "flops": 4 * d * H * pairs}
    return {"bytes": case["rows"] * (case["vocab"] * 4 + 32), "flops": case["rows"] * case["vocab"] * 4}


# ------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)


def _exact_tables(s):
    return None  # whole numbers only


def _exact_append(s):
    T, kv, d, H = s["q"].shape[0], s["kv"], s["d"], s["H"]
    cs = s["rope"].double()[s["row_pos"].long()]
    turn = torch.view_as_complex(cs.contiguous())[:, None]
    rotate = lambda x: torch.view_as_real(torch.view_as_complex(x.double().reshape(T, -1, d // 2, 2).contiguous()) * turn).reshape(T, -1, d)  # noqa: E731
    pool = s["pool"].double()
    rows = (s["row_slot"] >= 0).nonzero()[:, 0]
    page, token = s["row_slot"][rows] // PAGE, s["row_slot"][rows] % PAGE
    pool[page, LAYER, 0, :, token] = rotate(s["k"])[rows]
    pool[page, LAYER, 1, :, token] = s["v"].double().reshape(T, kv, d)[rows]
    return {"q_out": rotate(s["q"]).reshape(T, H * d), "pool": pool}


def _exact_attend(s):
    H, kv, d = s["H"], s["kv"], s["d"]
    G = H // kv
    offsets, total, table = s["row_offsets"].tolist(), s["total"].tolist(), s["table"].cpu().numpy()
    out = torch.zeros(s["q"].shape[0], H, d, dtype=torch.float64, device="cuda")
    for b, L in enumerate(total):
        a, e = offsets[b], offsets[b + 1]
        if a == e:
            continue
        ids = torch.from_numpy(table[b, : _pages(L)].astype(np.int64)).cuda()
        pages = s["pool"][ids.clamp(min=0), LAYER].double() * (ids >= 0)[:, None, None, None, None]  # [pages, 2, kv, 16, d]
        limit = torch.arange(L - (e - a), L, device="cuda")
        later = torch.arange(L, device="cuda")[None] > limit[:, None]
        for h in range(kv):
            k, v = (pages[:, c, h].reshape(-1, d)[:L] for c in (0, 1))
            for j in range(h * G, h * G + G):
                score = (s["q"][a:e, j * d : (j + 1) * d].double() @ k.T) * d**-0.5
                score[later] = -math.inf
                out[a:e, j] = torch.softmax(score, 1) @ v
    return {"out": out.reshape(-1, H * d)}


def _exact_sample(s):
    x = s["logits"].cpu().numpy().astype(np.float64)
    u, temp, top_k, top_p, min_p = (s[n].cpu().numpy() for n in ("uniform", "temperature", "top_k", "top_p", "min_p"))
    prob, entropy = np.zeros(len(x)), np.zeros(len(x))
    for i, row in enumerate(x):
        held = np.flatnonzero(row > -math.inf)
        if not held.size:
            continue
        if temp[i] == 0:
            prob[i] = 1.0
            continue
        held = held[np.argsort(-row[held], kind="stable")]
        if top_k[i] > 0:
            held = held[: top_k[i]]
        w = np.exp((row[held] - row[held[0]]) / np.float64(temp[i]))
        if top_p[i] < 1:
            held = held[: max(1, int(np.searchsorted(np.cumsum(w), np.float64(top_p[i]) * w.sum())) + 1)]
            w = w[: held.size]
        held = held[w >= np.float64(min_p[i])]
        w = w[w >= np.float64(min_p[i])]
        at = np.argsort(held)
        p = (w / w.sum())[at]
        prob[i] = p[min(int(np.searchsorted(np.cumsum(p), np.float64(u[i]), side="right")), p.size - 1)]
        entropy[i] = -(p[p > 0] * np.log(p[p > 0])).sum()
    return {"token": None, "prob": prob, "entropy": entropy}
