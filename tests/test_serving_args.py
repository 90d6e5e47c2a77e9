"""Refusals of the serving-step entries that need no GPU: the C entries check
their arguments before they touch the device, and tinybrain_b200.serving checks
its tensors before it calls them."""
import ctypes as C

import numpy as np
import pytest

from tinybrain_b200 import _lib

INVALID = 1
P = C.c_void_p(64)  # never dereferenced: every call below is refused first


def _status(name, *args):
    st = getattr(_lib.load(), name)(*args)
    assert st == 0 or _lib.last_error()
    return st


def tables(**kw):
    a = dict(cached=P, new=P, batch=2, free=P, num_free=4, table=P, stride=8, max_rows=16, offsets=P, total=P, seq=P,
             pos=P, slot=P, info=P)
    a.update(kw)
    return _status("tb_page_tables_build_dev", None, a["cached"], a["new"], a["batch"], a["free"], a["num_free"],
                   a["table"], a["stride"], a["max_rows"], a["offsets"], a["total"], a["seq"], a["pos"], a["slot"],
                   a["info"])


def append(**kw):
    a = dict(q=P, ld_q=256, k=P, ld_k=64, v=P, ld_v=64, rows=4, n=None, pos=P, slot=P, rope=P, positions=8, layer=0,
             layers=2, H=8, Hkv=2, d=32, pool=P, pages=4, out=P, ld_out=256)
    a.update(kw)
    return _status("tb_rope_append_paged_dev", None, *a.values())


def attend(**kw):
    a = dict(q=P, ld_q=256, rows=4, offsets=P, total=P, batch=2, pool=P, pages=4, table=P, stride=8, max_new=4,
             max_len=64, layer=0, layers=2, H=8, Hkv=2, d=32, out=P, ld_out=256, ws=P, ws_bytes=1 << 40)
    a.update(kw)
    return _status("tb_paged_attention_chunk_dev", None, *a.values())


def sample(**kw):
    a = dict(logits=P, ld=100, rows=2, V=100, t=None, k=None, p=None, m=None, u=P, token=P, prob=None, entropy=None)
    a.update(kw)
    return _status("tb_sample_rows_dev", None, *a.values())


@pytest.mark.parametrize("call,kw", [
    (tables, dict(cached=None)), (tables, dict(info=None)), (tables, dict(batch=0)), (tables, dict(stride=0)),
    (tables, dict(stride=1 << 28)), (tables, dict(num_free=-1)), (tables, dict(free=None)), (tables, dict(max_rows=-1)),
    (tables, dict(slot=None)),
    (append, dict(q=None)), (append, dict(rope=None)), (append, dict(rows=-1)), (append, dict(layer=2)),
    (append, dict(layer=-1)), (append, dict(d=31)), (append, dict(d=0)), (append, dict(H=7)), (append, dict(Hkv=0)),
    (append, dict(ld_q=255)), (append, dict(ld_k=63)), (append, dict(ld_v=0)), (append, dict(ld_out=255)),
    (append, dict(pages=0)), (append, dict(positions=0)), (append, dict(H=1 << 20, ld_q=1 << 40, ld_out=1 << 40)),
    (attend, dict(q=None)), (attend, dict(table=None)), (attend, dict(rows=-1)), (attend, dict(batch=0)),
    (attend, dict(layer=2)), (attend, dict(H=9)), (attend, dict(ld_q=255)), (attend, dict(ld_out=10)),
    (attend, dict(max_new=0)), (attend, dict(max_len=0)), (attend, dict(stride=0)), (attend, dict(pages=0)),
    (sample, dict(logits=None)), (sample, dict(u=None)), (sample, dict(token=None)), (sample, dict(V=0)),
    (sample, dict(ld=99)), (sample, dict(rows=-1)), (sample, dict(V=(1 << 24) + 1, ld=1 << 25)),
    (sample, dict(rows=(1 << 31) - 1)),
])
def test_c_entries_refuse_bad_arguments(call, kw):
    assert call(**kw) == INVALID


def test_lengths_may_not_be_written_while_they_are_read():
    at = lambda n: C.c_void_p(4096 + n)  # noqa: E731
    apart = dict(cached=at(0), new=at(8), offsets=at(16), total=at(32))  # two sequences: 8, 8, 12 and 8 bytes
    for clash in (dict(total=at(0)), dict(total=at(4)), dict(total=at(12)), dict(offsets=at(8)), dict(offsets=at(-8))):
        assert tables(**{**apart, **clash}) == INVALID
        assert "overlap" in _lib.last_error()
    assert tables(**apart) != 0 and "overlap" not in _lib.last_error()  # no device here, or not device memory


def test_unsupported_geometry_is_refused():
    assert attend(d=48, H=8, ld_q=384, ld_out=384) == 4
    assert attend(H=258, Hkv=2, ld_q=1 << 20, ld_out=1 << 20) == 4


def test_the_workspace_is_asked_for_where_it_is_used():
    few, many = dict(rows=1, batch=1, max_new=1, max_len=64), dict(rows=1, batch=1, max_new=1, max_len=1 << 20)

    def need(rows, batch, max_new, max_len):
        n = C.c_int64(-1)
        _lib.call("tb_paged_attention_chunk_workspace", rows, batch, max_new, max_len, 8, 2, 32, C.byref(n))
        return n.value

    assert need(**few) == 0 and need(**many) > 0
    assert attend(**few, ws=None, ws_bytes=0) != 0 and "workspace" not in _lib.last_error()  # no device here
    assert attend(**many, ws=None, ws_bytes=0) == INVALID and "workspace" in _lib.last_error()
    assert attend(**many, ws_bytes=need(**many) - 1) == INVALID and "workspace" in _lib.last_error()
    assert attend(**many, ws=C.c_void_p(72)) == INVALID and "workspace" in _lib.last_error()


def test_no_rows_is_no_work():
    assert append(rows=0) == 0 and attend(rows=0) == 0 and sample(rows=0) == 0


def test_host_memory_is_refused_before_any_launch():
    buf = np.zeros(4096, np.float32)
    st = sample(logits=buf.ctypes.data_as(C.c_void_p))
    assert st != 0  # no device here, or not device memory


def test_rope_table_is_the_reference_formula():
    d, n = 64, 40
    got = np.empty((n, d // 2, 2), np.float32)
    _lib.call("tb_rope_table", n, d, got.ctypes.data_as(C.c_void_p))
    i = np.arange(0, d, 2)
    angle = np.arange(n)[:, None] * (10000.0 ** (-i / d))[None]
    # the fp32 angle is off by at most 3 half steps of its own size (theta, its power, the product)
    tol = 3 * 2.0 ** -24 * np.maximum(angle, 1) * 4
    assert np.all(np.abs(got[..., 0] - np.cos(angle)) <= tol)
    assert np.all(np.abs(got[..., 1] - np.sin(angle)) <= tol)
    assert _lib.load().tb_rope_table(4, 63, got.ctypes.data_as(C.c_void_p)) == INVALID
    assert _lib.load().tb_rope_table(0, 64, got.ctypes.data_as(C.c_void_p)) == INVALID


def test_python_wrappers_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from tinybrain_b200 import serving
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        serving.build_page_tables(i32, i32, i32, torch.zeros(2, 4, dtype=torch.int32), i32, i32, i32, i32, i32, i32)
    x = torch.zeros(2, 64)
    pool = torch.zeros(4, 1, 2, 1, 16, 64)
    with pytest.raises(ValueError):
        serving.rope_append(x, x, x, i32, i32.long(), torch.zeros(8, 32, 2), pool, layer=0)
    with pytest.raises(ValueError):
        serving.paged_attention_chunk(x, i32, i32, pool, torch.zeros(2, 4, dtype=torch.int32), layer=0, max_new=1,
                                      max_len=1)
    with pytest.raises(ValueError):
        serving.sample_rows(x, torch.zeros(2))
