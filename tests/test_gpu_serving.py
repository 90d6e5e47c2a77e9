"""The operators of a serving step (tinybrain_b200.serving) against plain 64-bit
restatements of their definitions in include/tinybrain_cuda.h.

Tolerances, from the arithmetic:
 - page tables, slots, tokens: whole numbers, equal.
 - RoPE: the kernel's three roundings are written out in float32 below: equal.
 - attention: a score's products are carried to 3 * 2^-22 of |q_i k_i| and
   summed in fp32; with q, k ~ N(0, 1) the sum of |q_i k_i| / sqrt(d) is about
   0.64 sqrt(d) <= 7.3, so a score is off by at most 5.2e-6, a weight by as much
   relative to itself, and the result's sums and division add a few 2^-22:
   relative L2 <= 1e-5, the bar of the decode attention's tests.
 - probability and entropy: fp64 inside, one rounding to fp32 (2^-24) and the
   fp64 sums' few 1e-16: 2^-23 of max(1, value).
"""
import numpy as np
import pytest

from tests.helpers import rel_l2

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
PAGE = 16
ATTN_TOL = 1e-5
STAT_TOL = 2.0 ** -23


@pytest.fixture(scope="module")
def serving(ctx):
    from tinybrain_b200 import serving
    serving.check_device()  # nothing left by another test
    return serving


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def pages_of(n):
    return -(-np.asarray(n) // PAGE)


# ------------------------------------------------------------ page tables --
def tables_case(seed, batch, most, longest, slack=3):
    g = np.random.default_rng(seed)
    new = g.integers(0, most + 1, batch)
    cached = g.integers(0, longest + 1, batch)
    stride = int(pages_of(cached + new).max()) + 1
    held, need = int(pages_of(cached).sum()), int((pages_of(cached + new) - pages_of(cached)).sum())
    order = g.permutation(held + need + slack).astype(np.int32)
    table = np.full((batch, stride), -1, np.int32)
    k = 0
    for s, n in enumerate(pages_of(cached)):
        table[s, :n] = order[k:k + n]
        k += n
    if batch > 2 and cached[0] >= PAGE:
        table[0, (cached[0] - 1) // PAGE] = -1  # the page that is written next is evicted
    return cached.astype(np.int32), new.astype(np.int32), order[held:], table


def tables_numpy(cached, new, free, table):
    table = table.copy()
    seq, pos, slot, taken = [], [], [], 0
    for s, (c, n) in enumerate(zip(cached.tolist(), new.tolist())):
        for lp in range(-(-c // PAGE), -(-(c + n) // PAGE)):
            table[s, lp] = free[taken]
            taken += 1
        for p in range(c, c + n):
            seq.append(s)
            pos.append(p)
            page = int(table[s, p // PAGE])
            slot.append(-1 if page < 0 else page * PAGE + p % PAGE)
    return table, np.concatenate([[0], np.cumsum(new)]), cached + new, seq, pos, slot, taken


def tables_device(serving, cached, new, free, table, room):
    batch = len(cached)
    o = dict(table=dev(table), offsets=torch.full((batch + 1,), -7, dtype=torch.int32, device="cuda"),
             total=torch.full((batch,), -7, dtype=torch.int32, device="cuda"))
    for n, t in (("seq", torch.int32), ("pos", torch.int32), ("slot", torch.int64)):
        o[n] = torch.full((room,), -7, dtype=t, device="cuda")
    o["info"] = torch.full((4,), -7, dtype=torch.int32, device="cuda")
    o["inputs"] = (dev(cached), dev(new), dev(free))
    serving.build_page_tables(*o["inputs"], o["table"], o["offsets"], o["total"], o["seq"], o["pos"], o["slot"],
                              o["info"])
    return o


@pytest.mark.parametrize("batch,most,longest,room", [
    (1, 1, 0, 0), (1, 0, 5, 0), (1, 40, 0, 2), (3, 17, 33, 0), (64, 1, 300, 7), (513, 5, 40, 1), (2048, 3, 20, 0),
    (2049, 3, 20, 5), (4500, 9, 100, 0), (2, 3000, 100, 0), (7, 1024, 15, 1)])
def test_page_tables(serving, batch, most, longest, room):
    cached, new, free, table = tables_case(batch + most, batch, most, longest)
    want_table, off, total, seq, pos, slot, taken = tables_numpy(cached, new, free, table)
    rows = len(seq)
    o = tables_device(serving, cached, new, free, table, rows + room)
    assert o["info"].tolist() == [rows, taken, serving.PAGES_OK, -1]
    assert np.array_equal(o["table"].cpu().numpy(), want_table)
    assert o["offsets"].tolist() == off.tolist() and o["total"].tolist() == total.tolist()
    for name, want in (("seq", seq), ("pos", pos), ("slot", slot)):
        assert o[name][:rows].tolist() == want, name
        assert (o[name][rows:] == -7).all(), name  # behind the last row


@pytest.mark.parametrize("cut", [(1, 0), (0, 3), (2, 1)])
def test_page_tables_from_lengths_at_any_address(serving, cut):
    cached, new, free, table = tables_case(8, 2100, 7, 60)
    want_table, off, total, *_ = tables_numpy(cached, new, free, table)
    lens = [torch.cat([torch.zeros(k, dtype=torch.int32, device="cuda"), dev(x)])[k:] for k, x in zip(cut, (cached, new))]
    o = tables_device(serving, cached, new, free, table, int(new.sum()))
    again = {n: torch.full_like(o[n], -7) for n in ("offsets", "total", "seq", "pos", "slot", "info")}
    t = dev(table)
    serving.build_page_tables(*lens, dev(free), t, *again.values())
    assert all(torch.equal(again[n], o[n]) for n in again) and torch.equal(t, o["table"])
    assert o["offsets"].tolist() == off.tolist() and np.array_equal(t.cpu().numpy(), want_table)


@pytest.mark.parametrize("fault", ["pages", "rows", "negative", "negative_new", "long"])
def test_page_tables_that_do_not_fit_take_nothing(serving, fault):
    cached, new, free, table = tables_case(5, 300, 30, 60, slack=0)
    rows = int(new.sum())
    status, who, room = serving.PAGES_BAD_LENGTH, 123, rows
    if fault == "pages":
        free, status, who = free[:-1], serving.PAGES_EXHAUSTED, -1
    elif fault == "rows":
        room, status, who = rows - 1, serving.PAGES_ROWS_EXCEEDED, -1
    elif fault == "negative":
        cached[123] = -1
    elif fault == "negative_new":
        new[123], new[200] = -5, -1
    else:
        cached[123] = 2 ** 31 - 2
    o = tables_device(serving, cached, new, free, table, room)
    assert o["info"].tolist() == [0, 0, status, who]
    assert (o["offsets"] == 0).all() and o["total"].tolist() == cached.tolist()
    assert np.array_equal(o["table"].cpu().numpy(), table)
    assert all((o[n] == -7).all() for n in ("seq", "pos", "slot"))


def test_page_tables_fill_the_table_exactly(serving):
    o = tables_device(serving, np.array([15], np.int32), np.array([17], np.int32), np.array([9], np.int32),
                      np.array([[4, -1]], np.int32), 17)
    assert o["table"].tolist() == [[4, 9]] and o["info"].tolist() == [17, 1, 0, -1]
    assert o["slot"].tolist() == [4 * 16 + 15] + list(range(144, 160))


# ------------------------------------------------------------------ append --
def rotate32(x, cs):
    a, b, c, s = x[..., 0::2], x[..., 1::2], cs[..., 0], cs[..., 1]
    out = np.empty_like(x)
    out[..., 0::2] = a * c - b * s
    out[..., 1::2] = a * s + b * c
    return out


def append_case(seed, rows, H, kv, d, lead=0, positions=50, pages=None):
    g = np.random.default_rng(seed)
    pages = pages or rows // PAGE + 2
    slots = g.permutation(pages * PAGE)[:rows].astype(np.int64)
    if rows > 2:
        slots[1] = -1
    return dict(qkv=g.standard_normal((rows, lead + (H + 2 * kv) * d)).astype(np.float32), slots=slots,
                pos=g.integers(0, positions, rows).astype(np.int32),
                rope=g.standard_normal((positions, d // 2, 2)).astype(np.float32),
                pool=g.standard_normal((pages, 3, 2, kv, PAGE, d)).astype(np.float32), lead=lead)


def append_numpy(c, H, kv, d, layer, rows):
    qkv = c["qkv"][:rows, c["lead"]:]
    cs = c["rope"][c["pos"][:rows]][:, None]
    q = rotate32(qkv[:, :H * d].reshape(rows, H, d), cs).reshape(rows, H * d)
    k = rotate32(qkv[:, H * d:(H + kv) * d].reshape(rows, kv, d), cs)
    v = qkv[:, (H + kv) * d:].reshape(rows, kv, d)
    pool = c["pool"].copy()
    for r, s in enumerate(c["slots"][:rows]):
        if s >= 0:
            pool[s // PAGE, layer, 0, :, s % PAGE] = k[r]
            pool[s // PAGE, layer, 1, :, s % PAGE] = v[r]
    return q, pool


def split(t, lead, H, kv, d):
    return t[:, lead:lead + H * d], t[:, lead + H * d:lead + (H + kv) * d], t[:, lead + (H + kv) * d:]


@pytest.mark.parametrize("rows,H,kv,d,lead", [
    (1, 32, 4, 64, 0), (64, 32, 4, 64, 0), (5, 32, 32, 128, 4), (17, 4, 4, 16, 0), (9, 8, 2, 32, 1), (33, 6, 2, 6, 0),
    (3, 3, 1, 10, 3), (300, 8, 8, 128, 0)])
def test_rope_append(serving, rows, H, kv, d, lead):
    c = append_case(rows + d, rows, H, kv, d, lead)
    q, k, v = split(dev(c["qkv"]), lead, H, kv, d)
    pool = dev(c["pool"])
    out = torch.full((rows, H * d + 4), -7.0, device="cuda")
    serving.rope_append(q, k, v, dev(c["pos"]), dev(c["slots"]), dev(c["rope"]), pool, out[:, :H * d], layer=1)
    want_q, want_pool = append_numpy(c, H, kv, d, 1, rows)
    assert np.array_equal(out[:, :H * d].cpu().numpy(), want_q)
    assert np.array_equal(pool.cpu().numpy(), want_pool)
    assert (out[:, H * d:] == -7).all()
    serving.check_device()


@pytest.mark.parametrize("active", [0, 1, 5, 9])
def test_rope_append_device_row_count_and_in_place(serving, active):
    H, kv, d, rows = 8, 2, 32, 9
    c = append_case(3, rows, H, kv, d)
    t = dev(c["qkv"])
    q, k, v = split(t, 0, H, kv, d)
    pool = dev(c["pool"])
    n = torch.tensor([4, active], dtype=torch.int32, device="cuda")
    serving.rope_append(q, k, v, dev(c["pos"]), dev(c["slots"]), dev(c["rope"]), pool, q, layer=2, num_rows=n[-1:])
    want_q, want_pool = append_numpy(c, H, kv, d, 2, active)
    assert np.array_equal(q[:active].cpu().numpy(), want_q) and np.array_equal(pool.cpu().numpy(), want_pool)
    assert np.array_equal(t[active:].cpu().numpy(), c["qkv"][active:])


@pytest.mark.parametrize("what", ["slot", "position", "negative"])
def test_rope_append_reports_what_lies_outside(serving, what):
    H, kv, d, rows = 4, 2, 16, 6
    c = append_case(8, rows, H, kv, d)
    skip = c["slots"].copy()
    if what == "slot":
        c["slots"][3] = len(c["pool"]) * PAGE
    else:
        c["pos"][3] = 50 if what == "position" else -1
    q, k, v = split(dev(c["qkv"]), 0, H, kv, d)
    pool, out = dev(c["pool"]), torch.full((rows, H * d), -7.0, device="cuda")
    serving.rope_append(q, k, v, dev(c["pos"]), dev(c["slots"]), dev(c["rope"]), pool, out, layer=0)
    from tinybrain_b200 import TinyBrainError
    with pytest.raises(TinyBrainError):
        serving.check_device()
    serving.check_device()  # cleared
    skip[3] = -1
    c["slots"], c["pos"][3] = skip, c["pos"][3] % 50
    want_q, want_pool = append_numpy(c, H, kv, d, 0, rows)
    if what != "slot":
        want_q[3] = -7.0
    assert np.array_equal(out.cpu().numpy(), want_q) and np.array_equal(pool.cpu().numpy(), want_pool)


# --------------------------------------------------------------- attention --
def attend_case(seed, total, new, H, kv, d, evict=(), layers=2, extra_rows=0, scale=1.0):
    g = np.random.default_rng(seed)
    total, new = np.asarray(total, np.int32), np.asarray(new, np.int32)
    count = pages_of(np.maximum(total, 0))
    stride = max(1, int(count.max())) + 1
    pages = int(count.sum()) + 2
    order = g.permutation(pages).astype(np.int32)
    table = np.full((len(total), stride), -1, np.int32)
    k = 0
    for s, n in enumerate(count):
        table[s, :n] = order[k:k + n]
        k += n
    for s, lp in evict:
        table[s, lp] = -1
    rows = int(new.sum()) + extra_rows
    return dict(q=(scale * g.standard_normal((rows, H * d))).astype(np.float32), H=H, kv=kv, d=d, total=total, new=new,
                pool=g.standard_normal((pages, layers, 2, kv, PAGE, d)).astype(np.float32), table=table,
                offsets=np.concatenate([[0], np.cumsum(new)]).astype(np.int32), layer=layers - 1)


def attend_numpy(c):
    H, kv, d, G = c["H"], c["kv"], c["d"], c["H"] // c["kv"]
    out = np.zeros((int(c["offsets"][-1]), H, d))
    with np.errstate(all="ignore"):
        for s, (L, n) in enumerate(zip(c["total"].tolist(), c["new"].tolist())):
            if not n:
                continue
            pos = np.arange(max(L, 0))
            pg = c["table"][s, pos // PAGE]
            rows = c["pool"][np.maximum(pg, 0), c["layer"], :, :, pos % PAGE].astype(np.float64)  # [L, 2, kv, d]
            rows[pg < 0] = 0.0
            for h in range(H):
                K, V = rows[:, 0, h // G], rows[:, 1, h // G]
                q = c["q"][c["offsets"][s]:c["offsets"][s] + n, h * d:(h + 1) * d].astype(np.float64)
                for i in range(n):
                    e = L - n + i + 1
                    if e <= 0:
                        continue
                    sc = K[:e] @ q[i] / np.sqrt(d)
                    p = np.exp(sc - sc.max())
                    out[c["offsets"][s] + i, h] = (p / p.sum()) @ V[:e]
    return out.reshape(-1, H * d)


def attend_device(serving, c, out=None, max_new=None, max_len=None, q=None, **kw):
    q = dev(c["q"]) if q is None else q
    t = [dev(c[n]) for n in ("offsets", "total", "pool", "table")]
    out = torch.full(q.shape, -7.0, device="cuda") if out is None else out
    serving.paged_attention_chunk(q, *t, out, layer=c["layer"], max_new=max_new or max(1, int(c["new"].max())),
                                  max_len=max_len or max(1, int(c["total"].max())), **kw)
    return out


def check_attend(serving, c, **kw):
    out = attend_device(serving, c, **kw).cpu().numpy()
    n = int(c["offsets"][-1])
    want = attend_numpy(c)
    assert rel_l2(out[:n], want) <= ATTN_TOL
    # every row and head by itself, so that a small one cannot hide behind the others
    a, b = out[:n].reshape(-1, c["d"]), want.reshape(-1, c["d"])
    big = np.linalg.norm(b, axis=1)
    off = np.linalg.norm(a - b, axis=1)
    assert np.all(off <= 4 * ATTN_TOL * np.maximum(big, 0.05))
    assert (out[n:] == -7).all()
    serving.check_device()


HEADS = [(32, 4, 64), (8, 8, 128), (16, 4, 32), (4, 4, 16), (8, 1, 128), (8, 1, 64), (6, 2, 64), (16, 1, 16), (3, 1, 32)]


@pytest.mark.parametrize("H,kv,d", HEADS)
@pytest.mark.parametrize("total,new", [
    ([1], [1]), ([129], [1]), ([16], [16]), ([200], [200]), ([7, 16, 17, 300, 129], [1, 16, 3, 77, 0]),
    ([640, 1, 64, 33], [64, 1, 64, 1])])
def test_chunk_attention(serving, H, kv, d, total, new):
    check_attend(serving, attend_case(len(total) + H + d, total, new, H, kv, d, extra_rows=2))


@pytest.mark.parametrize("H,kv,d,total,new", [
    (8, 1, 64, [200, 90], [1, 1]), (8, 1, 64, [4100, 90], [1, 1]), (8, 2, 128, [300, 1500], [70, 3]),
    (16, 2, 64, [900], [300])])
def test_chunk_attention_may_write_over_its_queries(serving, H, kv, d, total, new):
    c = attend_case(H + d, total, new, H, kv, d)
    q = dev(c["q"])
    apart = attend_device(serving, c)
    assert torch.equal(attend_device(serving, c, out=q, q=q), apart)


@pytest.mark.parametrize("H,kv,d", [(16, 2, 64), (8, 4, 128), (4, 4, 16), (32, 4, 32)])
@pytest.mark.parametrize("hint", [None, 1])
def test_chunk_attention_of_few_tokens_over_few_pages(serving, H, kv, d, hint):
    # one CTA a unit: from no position to two pages a warp; with `hint` more units than the bounds tell
    total = [1, 16, 17, 129, 255, 256, 3, 0, 200, 90]
    new = [1, 0, 1, 1, 1, 1, 3, 0, 1, 1] if hint is None else [1, 0, 8, 5, 1, 3, 3, 0, 1, 7]
    c = attend_case(d, total, new, H, kv, d, evict=[(3, 0), (3, 8), (8, 12)], extra_rows=2)
    check_attend(serving, c, max_new=hint, max_len=hint and 256)
    serving.check_device()


@pytest.mark.parametrize("H,kv,d,total,new", [
    (4, 4, 64, [2100], [1100]), (4, 4, 128, [1500], [1069]), (16, 2, 64, [2049, 300, 1025], [203, 5, 180]),
    (8, 4, 128, [700, 1300], [520, 581]), (4, 4, 32, [1700], [1041]), (8, 8, 16, [1100], [1100]),
    (8, 2, 128, [1500], [701])])
def test_chunk_attention_of_long_prompts(serving, H, kv, d, total, new):
    # many row tiles to a sequence, the last one of some rows, in several calls
    c = attend_case(d + H, total, new, H, kv, d, evict=[(0, 3)])
    for _ in range(3):
        check_attend(serving, c)
    serving.check_device()


@pytest.mark.parametrize("H,kv,d", [(32, 4, 64), (8, 8, 128), (16, 4, 32)])
def test_chunk_attention_long_and_ragged(serving, H, kv, d):
    g = np.random.default_rng(d)
    total = [4224, 1, 2049, 15, 0, 700] + g.integers(1, 500, 20).tolist()
    new = [1, 1, 300, 15, 0, 129] + [int(min(t, n)) for t, n in zip(total[6:], g.integers(0, 40, 20))]
    check_attend(serving, attend_case(d, total, new, H, kv, d, evict=[(0, 0), (0, 5), (2, 0), (2, 1), (5, 43)]))


def test_chunk_attention_decode_batch(serving):
    g = np.random.default_rng(4)
    total = g.integers(1, 3000, 70).tolist()
    check_attend(serving, attend_case(1, total, [1] * 70, 32, 4, 64))


def test_chunk_attention_many_sequences(serving):
    g = np.random.default_rng(6)
    total = g.integers(0, 40, 1300).tolist()
    new = [int(min(t, n)) for t, n in zip(total, g.integers(0, 3, 1300))]
    check_attend(serving, attend_case(2, total, new, 4, 4, 16))


def test_chunk_attention_everything_evicted(serving):
    # scores of 0 over rows of zeros: zeros
    c = attend_case(3, [40, 20], [3, 20], 8, 2, 64, evict=[(0, 0), (0, 1), (0, 2)])
    check_attend(serving, c)
    assert (attend_device(serving, c)[:3] == 0).all()


def test_chunk_attention_rows_without_a_position(serving):
    # more new tokens than the length holds: the first rows see nothing
    c = attend_case(4, [3, 0], [5, 2], 8, 2, 64)
    out = attend_device(serving, c).cpu().numpy()
    want = attend_numpy(c)
    assert (out[:2] == 0).all() and (out[5:] == 0).all()
    assert rel_l2(out[2:5], want[2:5]) <= ATTN_TOL


@pytest.mark.parametrize("H,kv,d", [(32, 4, 64), (8, 8, 128)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 3e38])
def test_chunk_attention_ignores_what_is_masked(serving, H, kv, d, value):
    # the rest of the last page, unused pages, and an evicted page's old memory
    total, new = [37, 250], [1, 100]
    c = attend_case(5, total, new, H, kv, d, evict=[(1, 2)])
    want = attend_numpy(c)
    used = set(c["table"][c["table"] >= 0].tolist())
    for p in range(len(c["pool"])):
        if p not in used:
            c["pool"][p] = value
    for s, L in enumerate(total):
        c["pool"][c["table"][s, L // PAGE], :, :, :, L % PAGE:] = value
    c["pool"][:, 0] = value  # another layer
    out = attend_device(serving, c).cpu().numpy()
    assert rel_l2(out, want) <= ATTN_TOL


@pytest.mark.parametrize("H,kv,d", [(32, 4, 64), (8, 8, 128)])
@pytest.mark.parametrize("value", [np.nan, np.inf, 3e30])
def test_chunk_attention_later_tokens_do_not_reach_earlier_rows(serving, H, kv, d, value):
    c = attend_case(6, [300, 40], [150, 40], H, kv, d)
    want = attend_numpy(c)
    for s, t in ((0, 220), (1, 17)):  # a token of the chunk itself
        c["pool"][c["table"][s, t // PAGE], 1, :, :, t % PAGE] = value
    out = attend_device(serving, c).cpu().numpy()
    for s, t in ((0, 220), (1, 17)):
        a = int(c["offsets"][s])
        first = t - (int(c["total"][s]) - int(c["new"][s]))  # the first row that sees it
        assert rel_l2(out[a:a + first], want[a:a + first]) <= ATTN_TOL
        if not np.isfinite(value):
            assert not np.isfinite(out[a + first:a + int(c["new"][s])]).any()


@pytest.mark.parametrize("scale", [1e-3, 30.0, 1e4])
def test_chunk_attention_magnitudes(serving, scale):
    # large scores make the softmax a maximum, small ones an average; the keys shrink
    # as the queries grow, so the scores' own error keeps its bound times 30
    c = attend_case(7, [400, 64], [70, 1], 8, 2, 64, scale=scale)
    c["pool"][:, :, 0] /= np.float32(max(1.0, scale / 3))
    c["pool"][:, :, 1] *= np.float32(1e-5)
    want = attend_numpy(c)
    out = attend_device(serving, c).cpu().numpy()
    assert rel_l2(out, want) <= 3 * ATTN_TOL


def test_chunk_attention_tokens_of_very_different_size(serving):
    # an attention sink: one token with a large key and next to no value, others
    # whose values differ by 1e6
    c = attend_case(8, [500], [30], 8, 2, 64)
    c["pool"][c["table"][0, 0], 1, 0, :, 0] *= 12
    c["pool"][c["table"][0, 0], 1, 1, :, 0] *= 1e-6
    c["pool"][c["table"][0, 3], 1, 1] *= 1e-5
    c["pool"][c["table"][0, 9], 1, 1] *= 30
    want = attend_numpy(c)
    assert rel_l2(attend_device(serving, c).cpu().numpy(), want) <= 2 * ATTN_TOL


@pytest.mark.parametrize("max_new,max_len", [(1, 1), (1, 300), (4000, 100000)])
def test_chunk_attention_bounds_only_shape_the_launch(serving, max_new, max_len):
    c = attend_case(9, [900, 300, 20], [1, 140, 20], 32, 4, 64)
    check_attend(serving, c, max_new=max_new, max_len=max_len)


@pytest.mark.parametrize("H,kv,d", [(12, 4, 64), (16, 8, 64), (8, 8, 128), (8, 2, 128)])
@pytest.mark.parametrize("value", [np.nan, np.inf, 3e30])
def test_chunk_attention_of_long_prompts_with_values_out_of_range(serving, H, kv, d, value):
    # a token of the chunk, an evicted page's old memory and what lies behind the last token; three query heads to a
    # KV head leave rows of a tile empty
    total, new, t = [1503], [700], 1100
    c = attend_case(11, total, new, H, kv, d, evict=[(0, 9)])
    want = attend_numpy(c)
    c["pool"][list(set(range(len(c["pool"]))) - set(c["table"][c["table"] >= 0].tolist()))] = value
    c["pool"][c["table"][0, 1503 // PAGE], :, :, :, 1503 % PAGE:] = value
    c["pool"][c["table"][0, t // PAGE], 1, :, :, t % PAGE] = value
    out = attend_device(serving, c).cpu().numpy()
    first = t - (1503 - 700)
    assert rel_l2(out[:first], want[:first]) <= ATTN_TOL
    if not np.isfinite(value):
        assert not np.isfinite(out[first:]).any()
    serving.check_device()


@pytest.mark.parametrize("max_len", [1, 1000, 5000])
def test_chunk_attention_of_long_prompts_beyond_their_bounds(serving, max_len):
    c = attend_case(12, [1503], [700], 16, 8, 64)
    check_attend(serving, c, max_len=max_len)
    q, out = (torch.zeros(701, 1024 + k, device="cuda") for k in (3, 1))  # rows at any address
    q[:700, 3:] = dev(c["q"])
    attend_device(serving, c, out=out[:, 1:], q=q[:, 3:], max_len=max_len)
    assert rel_l2(out[:700, 1:].cpu().numpy(), attend_numpy(c)) <= ATTN_TOL
    assert (out[700:] == 0).all() and (out[:, 0] == 0).all()


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_chunk_attention_of_few_tokens_ignores_what_is_masked(serving, value):
    c = attend_case(13, [37, 1, 250, 16], [1, 1, 1, 1], 16, 2, 64, evict=[(2, 2)])
    want = attend_numpy(c)
    c["pool"][list(set(range(len(c["pool"]))) - set(c["table"][c["table"] >= 0].tolist()))] = value
    for s, L in enumerate((37, 1, 250)):
        c["pool"][c["table"][s, L // PAGE], :, :, :, L % PAGE:] = value
    assert rel_l2(attend_device(serving, c).cpu().numpy(), want) <= ATTN_TOL
    c["pool"][c["table"][2, 5], 1, 1, 0, 3] = value  # visible to one KV head of one sequence
    out = attend_device(serving, c).cpu().numpy().reshape(4, 16, 64)
    hit = np.zeros((4, 16, 64), bool)
    hit[2, :8] = True
    assert not np.isfinite(out[hit]).any()
    assert rel_l2(np.where(hit, 0, out), np.where(hit, 0, want.reshape(4, 16, 64))) <= ATTN_TOL


def test_chunk_attention_strided_rows(serving):
    c = attend_case(10, [90, 33], [40, 1], 8, 2, 64)
    wide = torch.zeros(41, 3 * 512 + 1, device="cuda")
    q, out = wide[:, 3:515], wide[:, 1024:1536]  # a base that is only 4-byte aligned
    q.copy_(dev(c["q"]))
    attend_device(serving, c, out=out, q=q)
    assert rel_l2(out.cpu().numpy(), attend_numpy(c)) <= ATTN_TOL
    assert (wide[:, 515:1024] == 0).all() and (wide[:, 1536:] == 0).all()


def test_chunk_attention_bad_pages_are_reported(serving):
    from tinybrain_b200 import TinyBrainError
    c = attend_case(11, [80, 50], [20, 1], 8, 2, 64)
    bad = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in c.items()}
    bad["table"][0, 1] = len(c["pool"])
    out = attend_device(serving, bad).cpu().numpy()
    with pytest.raises(TinyBrainError):
        serving.check_device()
    c["table"][0, 1] = -1  # it reads as an evicted page
    assert rel_l2(out, attend_numpy(c)) <= ATTN_TOL
    long = {**c, "total": np.array([80, 5000], np.int32)}  # longer than its table row
    attend_device(serving, long)
    with pytest.raises(TinyBrainError):
        serving.check_device()
    serving.check_device()


def test_chunk_attention_offsets_beyond_32_bits(serving):
    kv, d, pages = 32, 128, 20000  # 2^18 floats a page: 5.2e9 in all
    pool = torch.empty(pages, 2, 2, kv, PAGE, d, device="cuda")
    c = attend_case(12, [100], [20], 32, kv, d)
    ids = [pages - 1 - 17 * i for i in range(7)]
    for i, p in enumerate(ids):
        pool[p] = dev(c["pool"][c["table"][0, i]])
    table = torch.full((1, 8), -1, dtype=torch.int32, device="cuda")
    table[0, :7] = torch.tensor(ids, dtype=torch.int32)
    want = attend_numpy(c)
    out = serving.paged_attention_chunk(dev(c["q"]), dev(c["offsets"]), dev(c["total"]), pool, table, layer=1,
                                        max_new=20, max_len=100)
    assert rel_l2(out.cpu().numpy(), want) <= ATTN_TOL
    # and the write side, to the last slot
    q = torch.randn(1, 32 * d, device="cuda")
    k, v = torch.randn(1, kv * d, device="cuda"), torch.randn(1, kv * d, device="cuda")
    rope = torch.zeros(1, d // 2, 2, device="cuda")
    rope[..., 0] = 1
    slot = torch.tensor([pages * PAGE - 1], device="cuda")
    serving.rope_append(q, k, v, torch.zeros(1, dtype=torch.int32, device="cuda"), slot, rope, pool, layer=1)
    assert torch.equal(pool[-1, 1, 0, :, -1].reshape(-1), k[0]) and torch.equal(pool[-1, 1, 1, :, -1].reshape(-1), v[0])
    serving.check_device()


def test_chunk_attention_matches_the_decode_entry(serving, ctx):
    # the same batch through tb_paged_attention_dev_noalloc
    import ctypes as C
    from tinybrain_b200 import _lib
    c = attend_case(13, [500, 1, 77, 2000], [1, 1, 1, 1], 32, 4, 64)
    t = {n: dev(c[n]) for n in ("q", "pool", "table", "total")}
    ref = torch.empty(4, 32 * 64, device="cuda")
    p = lambda x: C.c_void_p(x.data_ptr())  # noqa: E731
    _lib.call("tb_paged_attention_dev_noalloc", torch.cuda.current_stream().cuda_stream, p(t["q"]), 4, p(t["pool"]),
              p(t["table"]), c["table"].shape[1], p(t["total"]), 2000, 1, 2, 32, 4, 64, p(ref))
    assert rel_l2(attend_device(serving, c).cpu().numpy(), ref.cpu().numpy()) <= 2 * ATTN_TOL


# ------------------------------------------------------------------ sample --
def sample_numpy(x, u, t, k, p, m):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    idx = np.flatnonzero(x > -np.inf)
    if not idx.size:
        return -1, 0.0, 0.0
    order = idx[np.argsort(-x[idx], kind="stable")]
    top = x[order[0]]
    if not t > 0:
        return int(order[0]), 1.0, 0.0
    with np.errstate(all="ignore"):
        e = np.where(x[order] == top, 0.0, (x[order] - top) / np.float64(t))
    if k > 0:
        order, e = order[:k], e[:k]
    w = np.exp(e)
    if not p >= 1:
        n = int(np.searchsorted(np.cumsum(w), np.float64(p) * w.sum())) + 1
        order, w, e = order[:max(1, n)], w[:max(1, n)], e[:max(1, n)]
    keep = (w >= min(max(np.float64(m), 0.0), 1.0)) & (w > 0)
    order, w, e = order[keep], w[keep], e[keep]
    at = np.argsort(order)
    order, w, e = order[at], w[at], e[at]
    i = min(int(np.searchsorted(np.cumsum(w), np.float64(u) * w.sum(), side="right")), w.size - 1)
    pr = w / w.sum()
    return int(order[i]), pr[i], -(pr * np.log(pr)).sum()


def check_sample(serving, x, u, t=None, k=None, p=None, m=None, pad=0):
    rows, V = x.shape
    full = torch.full((rows, V + pad), 1e9, device="cuda")
    full[:, :V] = dev(x)
    cast = lambda v, ty: None if v is None else dev(np.broadcast_to(np.asarray(v, ty), rows).copy())  # noqa: E731
    token, prob, ent = serving.sample_rows(full[:, :V], cast(u, np.float32), temperature=cast(t, np.float32),
                                           top_k=cast(k, np.int32), top_p=cast(p, np.float32),
                                           min_p=cast(m, np.float32))
    token, prob, ent = token.cpu().numpy(), prob.cpu().numpy(), ent.cpu().numpy()
    at = lambda v, i, d, ty: d if v is None else np.broadcast_to(np.asarray(v, ty), rows)[i]  # noqa: E731
    for i in range(rows):
        want = sample_numpy(x[i], at(u, i, 0, np.float32), at(t, i, 1.0, np.float32), at(k, i, 0, np.int32),
                            at(p, i, 1.0, np.float32), at(m, i, 0.0, np.float32))
        assert token[i] == want[0], (i, token[i], want)
        assert abs(prob[i] - want[1]) <= STAT_TOL and abs(ent[i] - want[2]) <= STAT_TOL * max(1.0, want[2]), (i, want)
    return token


def rows_like_a_model(seed, rows, V):
    g = np.random.default_rng(seed)
    x = (2 * g.standard_normal((rows, V))).astype(np.float32)
    for r in range(rows):
        x[r, g.integers(0, V, min(V, 20))] += (10 * g.random(min(V, 20))).astype(np.float32)
    return x, g.random(rows).astype(np.float32)


SETTINGS = [dict(), dict(t=0.0), dict(t=0.7, k=40), dict(k=1), dict(p=0.9), dict(t=1.3, p=0.95), dict(m=0.05),
            dict(t=0.8, k=50, p=0.9, m=0.02), dict(k=7, p=0.3), dict(p=0.0), dict(p=0.9999999), dict(k=10 ** 6, m=1.0),
            dict(t=0.01, p=0.5), dict(t=50.0, p=0.5), dict(t=1e-30), dict(t=np.inf, p=0.5)]


@pytest.mark.parametrize("rows,V,pad", [(1, 32000, 0), (9, 4096, 0), (5, 4097, 3), (3, 33, 1), (2, 1, 0), (40, 1000, 7),
                                        (2, 131072, 1)])
@pytest.mark.parametrize("s", range(len(SETTINGS)))
def test_sample_rows(serving, rows, V, pad, s):
    x, u = rows_like_a_model(V + s, rows, V)
    check_sample(serving, x, u, pad=pad, **SETTINGS[s])


def test_sample_settings_by_row_and_batch_invariance(serving):
    rows, V = 200, 2500
    g = np.random.default_rng(2)
    x, u = rows_like_a_model(1, rows, V)
    s = dict(t=g.choice([0.0, 0.5, 1.0, 2.0], rows), k=g.choice([0, 1, 3, 40, 5000], rows),
             p=g.choice([1.0, 0.9, 0.2], rows), m=g.choice([0.0, 0.1], rows))
    got = check_sample(serving, x, u, **s)
    for r in (0, 17, 199):  # a row alone runs on other launch shapes
        assert check_sample(serving, x[r:r + 1], u[r:r + 1], **{k: v[r:r + 1] for k, v in s.items()})[0] == got[r]


@pytest.mark.parametrize("s", [dict(), dict(k=5), dict(p=0.5), dict(k=700, p=0.7), dict(k=3, p=0.4, m=0.5), dict(p=0.0)])
@pytest.mark.parametrize("kind", ["equal", "two values", "zeros of both signs", "few values"])
def test_sample_ties_go_to_the_lowest_index(serving, s, kind):
    V, rows = 2049, 6
    g = np.random.default_rng(3)
    x = {"equal": np.full((rows, V), 3.5), "two values": g.choice([1.0, 2.0], (rows, V)),
         "zeros of both signs": g.choice([0.0, -0.0], (rows, V)),
         "few values": g.choice([-1.0, 0.25, 4.0, -np.inf], (rows, V))}[kind].astype(np.float32)
    check_sample(serving, x, np.array([0.0, 0.1, 0.5, 0.77, 0.9, 0.999], np.float32), **s)


@pytest.mark.parametrize("s", [dict(), dict(t=0.0), dict(k=3), dict(p=0.9), dict(k=2, p=0.5, m=0.1)])
def test_sample_masked_and_infinite_values(serving, s):
    V, low, inf = 300, np.finfo(np.float32).min, np.inf
    x = np.full((10, V), -inf, np.float32)
    x[1, 7] = low                      # one token, at the type's lowest value
    x[2] = low                         # all of them: equal
    x[3, ::2] = np.nan
    x[3, 5] = 1.0
    x[4] = np.nan                      # nothing
    x[5] = 0.5
    x[5, [40, 90]] = inf               # they share the mass
    x[6] = np.random.default_rng(0).standard_normal(V)
    x[6, 100:] = low
    x[7, 250:] = 88.0
    x[8] = np.linspace(-3e38, 3e38, V)
    x[9, [0, V - 1]] = [2.0, 2.0]
    check_sample(serving, x, np.linspace(0, 0.99, 10).astype(np.float32), **s)


@pytest.mark.parametrize("V", [5000, 40001, 400000])
@pytest.mark.parametrize("s", [dict(k=1777), dict(p=0.6), dict(k=2500, p=0.3), dict(k=2500, p=0.9999), dict(k=4900, p=1e-4),
                               dict(t=np.inf, p=0.5), dict(t=1e-30, k=40, p=0.9), dict(t=3.0, k=4000, m=0.999)])
@pytest.mark.parametrize("kind", ["dense", "steps", "far below"])
def test_sample_boundary_among_many_like_values(serving, kind, s, V):
    # thousands of elements within a few hundredths of a nat, apart from one another,
    # in a few equal steps, or so far below one maximum that they have no mass
    g = np.random.default_rng(V)
    x = {"dense": g.random((3, V)) / 50, "steps": g.integers(0, 4, (3, V)) / 100.0,
         "far below": -60 + g.random((3, V))}[kind].astype(np.float32)
    if kind == "far below":
        x[:, V // 3] = 5.0
    check_sample(serving, x, np.array([0.0, 0.4, 0.97], np.float32), **s)


def test_sample_settings_that_are_no_numbers(serving):
    x, _ = rows_like_a_model(5, 6, 700)
    nan = np.float32(np.nan)
    top = np.where(np.isnan(x), -np.inf, x).argmax(1).tolist()
    f = lambda v: dev(np.full(6, v, np.float32))  # noqa: E731
    assert serving.sample_rows(dev(x), f(0.9), temperature=f(nan))[0].tolist() == top  # not above 0: the maximum
    assert serving.sample_rows(dev(x), f(0.9), temperature=f(-1.0))[0].tolist() == top
    assert serving.sample_rows(dev(x), f(0.9), top_p=f(nan))[0].tolist() == top  # the shortest prefix
    assert serving.sample_rows(dev(x), f(0.9), min_p=f(7.0))[0].tolist() == top
    first = check_sample(serving, x, np.zeros(6, np.float32))
    assert serving.sample_rows(dev(x), f(nan))[0].tolist() == first.tolist()
    assert serving.sample_rows(dev(x), f(-3.0), min_p=f(nan))[0].tolist() == first.tolist()


def test_sample_the_largest_vocabulary(serving):
    V = 1 << 24
    x = torch.zeros(2, V, device="cuda")
    x[0, V - 1], x[1, 5] = 20.0, 30.0
    z = torch.tensor([0.999, 0.5], device="cuda")
    assert serving.sample_rows(x, z)[0].tolist() == [V - 1, 5]
    k = torch.tensor([3, 1000], dtype=torch.int32, device="cuda")  # ties of zeros: the lowest indices
    p = torch.tensor([1.0, 0.9999999], device="cuda")
    t = torch.tensor([1e6, 1e6], device="cuda")
    assert serving.sample_rows(x, z, top_k=k, top_p=p, temperature=t)[0].tolist() == [V - 1, 499]


def test_sample_ends_of_the_unit_interval(serving):
    x = np.full((4, 50), -np.inf, np.float32)
    x[:, [3, 9, 47]] = 0.0
    got = check_sample(serving, x, np.array([0.0, 0.33, 0.67, 1 - 2.0 ** -24], np.float32))
    assert got.tolist() == [3, 3, 47, 47]


def test_sample_without_optional_outputs(serving):
    import ctypes as C
    from tinybrain_b200 import _lib
    x, u = rows_like_a_model(4, 3, 500)
    a, b, token = dev(x), dev(u), torch.full((3,), -7, dtype=torch.int32, device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    _lib.call("tb_sample_rows_dev", torch.cuda.current_stream().cuda_stream, p(a), 500, 3, 500, None, None, None, None,
              p(b), p(token), None, None)
    assert token.tolist() == [sample_numpy(x[i], u[i], 1, 0, 1, 0)[0] for i in range(3)]


# ------------------------------------------------------- a step, and use ----
class Step:
    """One layer's step over fixed buffers: the four operators one after the other."""

    def __init__(self, serving, seed, batch, room, H=8, kv=2, d=64, V=300, stride=24):
        self.s, self.H, self.kv, self.d, self.stride = serving, H, kv, d, stride
        g = np.random.default_rng(seed)
        z = lambda n, t=torch.int32: torch.zeros(n, dtype=t, device="cuda")  # noqa: E731
        self.cached, self.new, self.table = z(batch), z(batch), torch.full((batch, stride), -1, dtype=torch.int32,
                                                                           device="cuda")
        self.free = dev(g.permutation(batch * stride).astype(np.int32))
        self.offsets, self.total, self.seq, self.pos = z(batch + 1), z(batch), z(room), z(room)
        self.slot, self.info = z(room, torch.int64), z(4)
        self.qkv = torch.zeros(room, (H + 2 * kv) * d, device="cuda")
        self.pool = torch.zeros(batch * stride, 1, 2, kv, PAGE, d, device="cuda")
        self.rope = serving.rope_table(stride * PAGE, d, "cuda")
        self.q, self.out = torch.zeros(room, H * d, device="cuda"), torch.zeros(room, H * d, device="cuda")
        self.head = dev((g.standard_normal((H * d, V)) / 8).astype(np.float32))
        self.uniform, self.temperature = torch.zeros(room, device="cuda"), torch.full((room,), 0.8, device="cuda")
        self.token, self.prob, self.entropy = z(room), torch.zeros(room, device="cuda"), torch.zeros(room, device="cuda")
        self.logits = torch.zeros(room, V, device="cuda")

    def run(self):
        s, H, kv, d = self.s, self.H, self.kv, self.d
        s.build_page_tables(self.cached, self.new, self.free, self.table, self.offsets, self.total, self.seq, self.pos,
                            self.slot, self.info)
        s.rope_append(self.qkv[:, :H * d], self.qkv[:, H * d:(H + kv) * d], self.qkv[:, (H + kv) * d:], self.pos,
                      self.slot, self.rope, self.pool, self.q, layer=0, num_rows=self.offsets[-1:])
        s.paged_attention_chunk(self.q, self.offsets, self.total, self.pool, self.table, self.out, layer=0,
                                max_new=len(self.q), max_len=self.stride * PAGE)
        torch.matmul(self.out, self.head, out=self.logits)
        s.sample_rows(self.logits, self.uniform, self.token, self.prob, self.entropy, temperature=self.temperature)

    def feed(self, g, cached, new):
        self.cached.copy_(dev(np.asarray(cached, np.int32)))
        self.new.copy_(dev(np.asarray(new, np.int32)))
        self.qkv.copy_(dev(g.standard_normal(tuple(self.qkv.shape)).astype(np.float32)))
        self.uniform.copy_(dev(g.random(len(self.uniform)).astype(np.float32)))


def replay_numpy(history, H, kv, d, rope):
    """Attention outputs of the last step of every sequence from all its q, k, v so far."""
    outs = []
    for steps in history:
        if not steps or not len(steps[-1]):
            continue
        x = np.concatenate(steps).astype(np.float32)
        cs = rope[np.arange(len(x))][:, None]
        q = rotate32(x[:, :H * d].reshape(-1, H, d), cs).astype(np.float64)
        k = rotate32(x[:, H * d:(H + kv) * d].reshape(-1, kv, d), cs).astype(np.float64)
        v = x[:, (H + kv) * d:].reshape(-1, kv, d).astype(np.float64)
        for i in range(len(x) - len(steps[-1]), len(x)):
            o = np.empty((H, d))
            for h in range(H):
                sc = k[:i + 1, h * kv // H] @ q[i, h] / np.sqrt(d)
                p = np.exp(sc - sc.max())
                o[h] = (p / p.sum()) @ v[:i + 1, h * kv // H]
            outs.append(o.reshape(-1))
    return np.array(outs)


@pytest.mark.parametrize("captured", [False, True])
def test_steps_of_a_growing_batch(serving, captured):
    plan = [[40, 0, 5, 17], [1, 33, 1, 1], [1, 1, 1, 0], [64, 1, 0, 1], [1, 1, 1, 1]]
    st = Step(serving, 1, 4, 70)
    g = np.random.default_rng(9)
    graph = None
    if captured:
        st.run()  # an empty step
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st.run()
    cached, history, taken = [0] * 4, [[] for _ in range(4)], 0
    order = st.free.clone()
    rope = st.rope.cpu().numpy()
    for new in plan:
        st.feed(g, cached, new)
        st.free.copy_(torch.cat([order[taken:], order[:taken]]))
        x, row = st.qkv.cpu().numpy(), 0
        for s, n in enumerate(new):
            history[s].append(x[row:row + n])
            row += n
        graph.replay() if captured else st.run()
        info = st.info.tolist()
        assert info[0] == row and info[2] == serving.PAGES_OK
        taken += info[1]
        want = replay_numpy([h for h, n in zip(history, new) if n], st.H, st.kv, st.d, rope)
        assert rel_l2(st.out[:row].cpu().numpy(), want) <= ATTN_TOL
        logits, u = st.logits.cpu().numpy(), st.uniform.cpu().numpy()
        assert st.token[:row].tolist() == [sample_numpy(logits[i], u[i], np.float32(0.8), 0, 1, 0)[0] for i in range(row)]
        cached = [c + n for c, n in zip(cached, new)]
    serving.check_device()


def test_two_streams_at_once(serving):
    # two steps over their own buffers, in flight together, many times
    a, b = Step(serving, 2, 3, 40), Step(serving, 3, 5, 64)
    for st, seed, new in ((a, 5, [20, 1, 3]), (b, 6, [1, 9, 30, 0, 2])):
        st.feed(np.random.default_rng(seed), [0] * len(new), new)
        st.run()
    want = [(st.out.clone(), st.token.clone(), st.pool.clone()) for st in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, stream in zip((a, b), streams):
            with torch.cuda.stream(stream):
                st.run()
    torch.cuda.synchronize()
    for st, (out, token, pool) in zip((a, b), want):
        assert torch.equal(st.out, out) and torch.equal(st.token, token) and torch.equal(st.pool, pool)
    serving.check_device()


def test_attention_repeats_bit_for_bit(serving):
    c = attend_case(14, [3000, 700, 50], [1, 200, 50], 32, 4, 64)
    first = attend_device(serving, c)
    assert all(torch.equal(first, attend_device(serving, c)) for _ in range(3))


def test_workspace_is_checked_and_may_be_the_callers(serving):
    c = attend_case(15, [900], [1], 32, 4, 64)
    need = serving.paged_attention_chunk_workspace(1, 1, 1, 900, 32, 4, 64)
    w = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN bits: nothing is taken as zero
    check_attend(serving, c, workspace=w)
    if need:
        from tinybrain_b200 import TinyBrainError
        with pytest.raises(TinyBrainError):
            attend_device(serving, c, workspace=w[:need - 1])
        with pytest.raises(TinyBrainError):
            attend_device(serving, c, workspace=w[1:])


def test_wrappers_refuse_wrong_tensors(serving):
    c = attend_case(16, [40], [2], 8, 2, 64)
    q, off, tot, pool, table = (dev(c[n]) for n in ("q", "offsets", "total", "pool", "table"))
    kw = dict(layer=0, max_new=2, max_len=40)
    for bad in (dict(layer=2), dict(layer=-1), dict(max_new=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            serving.paged_attention_chunk(q, off, tot, pool, table, **{**kw, **bad})
    for args in ((q.half(), off, tot, pool, table), (q[:, :500], off, tot, pool, table), (q, off.long(), tot, pool, table),
                 (q, off[:1], tot, pool, table), (q, off, tot, pool.half(), table), (q, off, tot, pool[..., :32], table),
                 (q, off, tot, pool, table.t()), (q.cpu(), off, tot, pool, table), (q.t().contiguous().t(), off, tot, pool, table)):
        with pytest.raises(ValueError):
            serving.paged_attention_chunk(*args, **kw)
    with pytest.raises(ValueError):
        serving.paged_attention_chunk(q, off, tot, pool, table, torch.empty(1, 512, device="cuda"), **kw)
    x = torch.zeros(2, 10, device="cuda")
    u = torch.zeros(2, device="cuda")
    for bad in (dict(top_k=u), dict(temperature=u[:1]), dict(min_p=u.double())):
        with pytest.raises(ValueError):
            serving.sample_rows(x, u, **bad)
    with pytest.raises(ValueError):
        serving.sample_rows(x, u.cpu())
    with pytest.raises(ValueError):
        serving.rope_append(q, q[:, :128], q[:, :64], tot, tot.long(), torch.zeros(4, 32, 2, device="cuda"), pool, layer=0)
    with pytest.raises(ValueError):
        serving.rope_append(q, q[:, :128], q[:, :128], tot, tot.long(), torch.zeros(4, 32, 2, device="cuda"), pool, layer=0)


def test_capture_as_the_first_call_of_a_process(serving):
    # a fresh process whose first use of every entry is inside a capture
    import subprocess
    import sys
    code = """
import sys, torch, numpy as np
sys.path.insert(0, %r)
import tests.test_gpu_serving as t
from tinybrain_b200 import serving
st = t.Step(serving, 1, 2, 8)
st.feed(np.random.default_rng(1), [0, 0], [3, 5])
torch.matmul(st.out, st.head, out=st.logits)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st.run()
g.replay(); torch.cuda.synchronize()
a = st.out.clone()
st.out.zero_(); st.run(); torch.cuda.synchronize()
assert torch.equal(a, st.out) and a.abs().sum() > 0
""" % (__import__("os").path.dirname(__import__("os").path.dirname(__file__)),)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
