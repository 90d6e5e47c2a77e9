"""Chunk attention where its tiles, scales and masks can go wrong.

The reference is the definition in 64 bits (include/tinybrain_cuda.h).  Tolerance:
a score is off by 5.2e-6 at most for q, k ~ N(0, 1) (test_gpu_serving.py's bound),
a weight by as much relative to itself, and the sums add a few 2^-22: 1e-5 in
relative L2, over the call and, four times that, over every row and head by itself.
Nothing in that depends on the size of the values, so rows are held to their own norm.
"""
import numpy as np
import pytest

from tests.helpers import rel_l2
from tests.test_gpu_serving import ATTN_TOL, PAGE, attend_case, attend_device, dev, serving  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def attend_exact(c):
    """The definition in 64 bits, a sequence and head at a time; rows without a position are zeros."""
    H, kv, d = c["H"], c["kv"], c["d"]
    q, pool = dev(c["q"]).double(), dev(c["pool"])[:, c["layer"]].double()
    out = torch.zeros(int(c["offsets"][-1]), H, d, dtype=torch.float64, device="cuda")
    for s, (L, n) in enumerate(zip(c["total"].tolist(), c["new"].tolist())):
        if not n or L <= 0:
            continue
        ids = dev(c["table"][s, :-(-L // PAGE)].astype(np.int64))
        pages = torch.where((ids >= 0)[:, None, None, None, None], pool[ids.clamp(min=0)], 0.0)  # [pages, 2, kv, 16, d]
        K, V = (pages[:, x].transpose(0, 1).reshape(kv, -1, d)[:, :L] for x in (0, 1))
        a, z = int(c["offsets"][s]), max(n - L, 0)  # the first z rows have no position
        limit = torch.arange(L - n + z, L, device="cuda")
        later = torch.arange(L, device="cuda")[None] > limit[:, None]
        for h in range(H):
            sc = (q[a + z:a + n, h * d:(h + 1) * d] @ K[h * kv // H].T) / d ** 0.5
            out[a + z:a + n, h] = torch.softmax(sc.masked_fill(later, -np.inf), 1) @ V[h * kv // H]
    return out.reshape(-1, H * d).cpu().numpy()


def check(serving, c, tol=ATTN_TOL, **kw):  # noqa: F811
    out = attend_device(serving, c, **kw).cpu().numpy()
    n, want = int(c["offsets"][-1]), attend_exact(c)
    assert np.isfinite(out[:n]).all()
    assert rel_l2(out[:n], want) <= tol
    a, b = (x.reshape(-1, c["d"]).astype(np.float64) for x in (out[:n], want))
    big = np.linalg.norm(b, axis=1)
    off = np.linalg.norm(a - b, axis=1)
    assert np.all(off <= 4 * tol * np.maximum(big, 0.02 * big.max())), (off / np.maximum(big, 0.02 * big.max())).max()
    assert (out[n:] == -7).all()
    serving.check_device()
    return out


def cut(G, k, kv=1):
    """k row tiles of whole tokens and one token more."""
    return k * (128 // G) + 1


# Before these were right, the smallest of them walked out of the lengths and the table.
@pytest.mark.parametrize("H,kv,d,total,new", [
    (7, 1, 64, [73], [73]), (28, 4, 128, [512], [512]), (28, 4, 128, [343], [343]), (40, 8, 64, [201], [201]),
    (24, 8, 64, [2048], [2048]), (12, 2, 32, [1100], [cut(6, 30)]), (24, 2, 16, [900], [cut(12, 40)]),
    (14, 2, 64, [900], [577]), (20, 1, 64, [400], [cut(20, 22)]), (100, 1, 32, [200], [200]), (11, 1, 128, [300], [cut(11, 20)]),
    (28, 4, 128, [8192], [2048])])
def test_head_groups_that_do_not_divide_a_tile(serving, H, kv, d, total, new):  # noqa: F811
    check(serving, attend_case(H + d, total, new, H, kv, d, extra_rows=2))


@pytest.mark.parametrize("G,kv,d", [(3, 4, 64), (5, 2, 64), (6, 2, 32), (7, 4, 64), (12, 1, 128), (20, 2, 16), (48, 1, 64)])
def test_head_groups_that_do_not_divide_a_tile_ragged(serving, G, kv, d):  # noqa: F811
    g = np.random.default_rng(G)
    new = [cut(G, int(k)) for k in g.integers(1, 9, 16)]
    new[3], new[7] = 0, 1
    total = [n + int(h) for n, h in zip(new, g.integers(0, 400, 16))]
    check(serving, attend_case(G, total, new, G * kv, kv, d, evict=[(0, 0)], extra_rows=1))


@pytest.mark.parametrize("G", [9, 10, 11, 13, 15, 17, 21, 25, 31, 33, 43, 50, 65, 90, 127, 128])
@pytest.mark.parametrize("beforehand", [False, True])
@pytest.mark.parametrize("more", [-1, 1])
def test_large_head_groups_about_a_tile_end(serving, G, beforehand, more):  # noqa: F811
    d, kv, per = [16, 32, 64][G % 3], 4, 128 // G
    n = 41 * per + more
    total = n + 500
    need = lambda bound: serving.paged_attention_chunk_workspace(n, 1, n, bound, G * kv, kv, d)  # noqa: E731
    tiles = -(-total // 128)
    assert need(total) - need(1) >= 8 * kv * tiles * 128 * d  # its operands: both ways are run
    check(serving, attend_case(G, [total], [n], G * kv, kv, d, evict=[(0, 2)]), max_len=None if beforehand else 1)


@pytest.mark.parametrize("G,kv,d", [(3, 4, 64), (5, 2, 32), (6, 2, 128), (7, 4, 64)])
@pytest.mark.parametrize("max_new,max_len", [(1, 1), (1, 4096), (2, 500)])
def test_head_groups_with_more_tokens_than_the_bounds_tell(serving, G, kv, d, max_new, max_len):  # noqa: F811
    for total, new in (([40], [9]), ([300, 5, 77], [63, 5, 3]), ([30] * 16, list(range(16)))):
        check(serving, attend_case(G + len(new), total, new, G * kv, kv, d), max_new=max_new, max_len=max_len)


@pytest.mark.parametrize("H,kv,d,total,new", [
    (8, 2, 64, [300, 40], [150, 40]), (16, 2, 128, [200], [33]), (4, 4, 32, [500], [500]), (8, 8, 64, [1500], [1100]),
    (32, 4, 64, [300, 17], [1, 1])])
@pytest.mark.parametrize("q,k", [(1e-20, 1e-20), (1e-30, 1e-30), (1e-12, 1e-25), (0.0, 1e-30), (0.0, 0.0), (1e10, 1e-10),
                                 (1e-16, 1e16), (1e15, 1e-15)])
def test_queries_and_keys_of_any_size(serving, H, kv, d, total, new, q, k):  # noqa: F811
    # the scores keep their bound (their size is that of q times k); of next to none the result is the mean
    c = attend_case(d, total, new, H, kv, d)
    c["q"] *= np.float32(q)
    c["pool"][:, :, 0] *= np.float32(k)
    check(serving, c)


TILE = {16: 8, 32: 8, 64: 8, 128: 4}  # pages of a tile


@pytest.mark.parametrize("H,kv,d,total,new", [
    (8, 2, 64, [1000], [30]), (8, 4, 128, [1000], [100]), (16, 1, 16, [1000], [64]), (8, 8, 64, [1500], [1100]),
    (2, 2, 128, [2100], [2000]), (32, 4, 64, [1000], [1])])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-5, 1e-12, 1e-30, 1e5])
@pytest.mark.parametrize("where", ["first", "later", "tile", "most"])
@pytest.mark.parametrize("how", ["evicted", "zeros", "zero values"])
def test_pages_of_zeros_beside_values_of_any_size(serving, H, kv, d, total, new, size, where, how):  # noqa: F811
    c = attend_case(d + H, total, new, H, kv, d)
    c["pool"][:, :, 1] *= np.float32(size)
    n = total[0] // PAGE
    at = {"first": [0], "later": [TILE[d] + 3, n - 2], "tile": list(range(2 * TILE[d], 3 * TILE[d])),
          "most": list(range(n - 1))}[where]
    if how == "evicted":
        c["table"][0, at] = -1
    else:
        c["pool"][c["table"][0, at], :, (0 if how == "zeros" else 1):] = 0
    check(serving, c)


@pytest.mark.parametrize("max_len", [1, None])
def test_a_long_context_of_zero_values(serving, max_len):  # noqa: F811
    # scores that rise to just below what moves the reference maximum, over pages without
    # values: the row sums grow as far as they can.  Operands made beforehand, or not.
    d, L, n = 16, 40000, 4736
    c = attend_case(3, [L], [n], 4, 4, d)
    c["q"][:] = 1.0
    c["pool"][:, :, 0] = np.float32(5.45 / 4)  # d = 16: 5.45 nats, 2^7.86
    c["pool"][c["table"][0, :8], :, 0] = 0
    c["pool"][c["table"][0, :-60], :, 1] = 0
    c["pool"][:, :, 1] *= np.float32(1e-3)
    check(serving, c, max_len=max_len)


@pytest.mark.parametrize("H,kv,d,total,new", [
    (8, 1, 64, [8192, 0], [2048, 64]), (8, 1, 64, [0, 8192, 30], [300, 2048, 200]), (4, 4, 128, [0, 4000], [40, 3200]),
    (4, 2, 32, [2000, 0, 0], [2000, 1, 700]), (8, 1, 64, [300, 0], [70, 64]), (8, 1, 64, [300, 0], [1, 1])])
@pytest.mark.parametrize("fill", [0, 0xFF, 0x7F])
def test_rows_without_a_position_are_zeros_whatever_the_workspace_holds(serving, H, kv, d, total, new, fill):  # noqa: F811
    c = attend_case(d, total, new, H, kv, d)
    need = serving.paged_attention_chunk_workspace(sum(new), len(new), max(new), max(total), H, kv, d)
    w = torch.full((need,), fill, dtype=torch.uint8, device="cuda")
    out = check(serving, c, workspace=w)
    for s, (L, n) in enumerate(zip(total, new)):
        a = int(c["offsets"][s])
        assert (out[a:a + max(n - L, 0)] == 0).all()


def test_rows_without_operands_over_a_long_context(serving):  # noqa: F811
    # bounds of one token launch one CTA; its first unit is summed in fp32 for longer than its other warps'
    # limit of 2 s, and a second unit follows.  (What makes it so is a key of 2^21, which the queries do not see.)
    c = attend_case(5, [131072], [9], 16, 1, 128, layers=1)
    c["q"].reshape(9, 16, 128)[:, :, 0] = 0
    c["pool"][c["table"][0, 0], 0, 0, 0, 0, 0] = 2.0 ** 21
    check(serving, c, max_new=1, max_len=1)
