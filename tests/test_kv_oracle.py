"""The oracle of the operators on the paged cache (oracle/qk_oracle_kv.py), pinned by what the definitions fix and by the older oracle of
the one-sequence forms; and what the library refuses, with its messages, without a device."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

import kv_cases as KC

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "oracle"))
import qk_oracle_attn as OA  # noqa: E402
import qk_oracle_kv as OK  # noqa: E402


def slot_cache(rng, n_seq=2, hkv=2, cap=40, dh=256):
    return OK.Cache(rng.standard_normal((1, n_seq, hkv, cap, dh)).astype(np.float32), rng.standard_normal((1, n_seq, hkv, cap, dh)).astype(np.float32), None)


def test_one_axis_is_the_older_prep():
    """With one axis, ungrouped rows and a slot cache: the restatement of the reference's mixer."""
    rng = np.random.default_rng(0)
    c = slot_cache(rng)
    qf, kin, vin = rng.standard_normal((3, 4, 512)).astype(np.float32), rng.standard_normal((3, 2, 256)).astype(np.float32), rng.standard_normal((3, 2, 256)).astype(np.float32)
    qn, kn, rope = np.ones(256, np.float32) * 1.5, np.ones(256, np.float32) * 0.5, OA.rope_table(40, 64)
    rows = list(OK.runs(3, [0, 2, 3], [1, 0], [5, 9], c, 3))
    kc, vc = c.k[0].copy(), c.v[0].copy()
    pos = np.array([[at for _, _, at, _, _ in rows]], np.int32)
    got = OK.prep_axes(c, 0, rows, qf, kin, vin, qn, kn, rope, [0] * 32, pos, 256, 1e-6)
    att = OK.attend(c, 0, rows, got.astype(np.float32), qf)
    for r, (row, s, at, _, _) in enumerate(rows):
        want = OA.prep(qf[row], kin[row], vin[row], qn, kn, rope, at, kc[s], vc[s], 64)
        assert np.allclose(got[row], want, atol=2e-6)
    assert np.array_equal(c.v[0], vc) and np.allclose(c.k[0], kc, atol=2e-6)
    for row, s, at, _, _ in rows:
        assert np.allclose(att[row], OA.attend(got[row].astype(np.float32), kc[s], vc[s], qf[row], at), atol=1e-5)


def test_axes_are_independent():
    """A pair is turned by its own axis only; all axes alike is one axis; position 0 turns nothing."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 1, 128)).astype(np.float32)
    ones, rope = np.ones(128, np.float32), OA.rope_table(30, 64)
    run = lambda axis, pos: OK.prep_axes(slot_cache(rng, 1, 1, 4, 128), 0, [(0, 0, 0, 0, 0)], x, x, x, ones, ones, rope, axis, np.array(pos, np.int32)[:, None], 128, 0.0)[0, 0]  # noqa: E731
    axis = OK.rope_axes((12, 10, 10), True)
    a, b, c = run(axis, [7, 0, 0]), run(axis, [7, 3, 0]), run(axis, [0, 0, 0])
    same = np.array(axis) != 1
    assert np.array_equal(a[:32][same], b[:32][same]) and not np.allclose(a[:32][~same], b[:32][~same])
    assert np.allclose(run(axis, [7, 7, 7]), run([0] * 32, [7, 1, 2]))
    assert np.allclose(c, x[0, 0] / np.sqrt((x.astype(np.float64) ** 2).mean()))


def test_sections():
    assert OK.rope_axes((2, 1, 1), False) == [0, 0, 1, 2] and OK.rope_axes((3, 1, 0), True) == [0, 1, 0, 0]


def test_a_chain_is_the_packed_form_and_a_page_table_changes_nothing():
    rng = np.random.default_rng(2)
    c = slot_cache(rng, 1, 2, 32, 128)
    q = rng.standard_normal((6, 4, 128)).astype(np.float32)
    rows = list(OK.runs(6, [0, 6], [0], [11], c, 6))
    packed = OK.attend(c, 0, rows, q)
    assert np.array_equal(packed, OK.attend(c, 0, rows, q, parent=[-1, 0, 1, 2, 3, 4]))
    order = [3, 1]
    k, v = (np.zeros((1, 4, 2, 16, 128), np.float32) for _ in range(2))
    for b, p in enumerate(order):
        k[0, p], v[0, p] = c.k[0, 0, :, 16 * b:16 * b + 16], c.v[0, 0, :, 16 * b:16 * b + 16]
    assert np.array_equal(packed, OK.attend(OK.Cache(k, v, [order]), 0, rows, q))
    one = OK.attend(c, 0, list(OK.runs(1, [0, 1], [0], [0], c, 1)), q[:1])
    assert np.allclose(one[0, 0], c.v[0, 0, 0, 0]) and np.allclose(one[0, 3], c.v[0, 0, 1, 0])   # one key: its value row


def test_siblings_do_not_see_each_other():
    rng = np.random.default_rng(3)
    c = slot_cache(rng, 1, 1, 16, 128)
    q = rng.standard_normal((3, 1, 128)).astype(np.float32)
    rows = list(OK.runs(3, [0, 3], [0], [2], c, 3))
    a = OK.attend(c, 0, rows, q, parent=[-1, 0, 0])
    c.v[0, 0, 0, 3] = 99   # the first sibling's value row
    b = OK.attend(c, 0, rows, q, parent=[-1, 0, 0])
    assert np.array_equal(a[[0, 2]], b[[0, 2]]) and not np.allclose(a[1], b[1])


def test_books_of_the_oracle():
    """Two that share grow at once: each gets a copy, the shared page is free again; what is freed is taken lowest first."""
    rng = np.random.default_rng(4)
    c = OK.Cache(rng.standard_normal((1, 6, 1, 16, 128)).astype(np.float32), rng.standard_normal((1, 6, 1, 16, 128)).astype(np.float32),
                 [[-1] * 3 for _ in range(3)], [0] * 6, [0] * 3)
    assert OK.resize(c, [20, -1, 0]) == 0 and c.table[0] == [0, 1, -1] and c.ref[:2] == [1, 1]
    assert OK.fork(c, [0], [1]) == 0 and c.table[1] == [0, 1, -1] and c.ref[:2] == [2, 2]
    assert OK.fork(c, [0], [1]) == -1 and OK.fork(c, [0, 0], [2, 2]) == -1
    old = c.k[0, 1].copy()
    assert OK.resize(c, [21, 33, -1]) == 0
    assert c.table[0] == [0, 2, -1] and c.table[1] == [0, 3, 4] and c.ref == [2, 0, 1, 1, 1, 0] and np.array_equal(c.k[0, 2, :, :4], old[:, :4])
    assert OK.resize(c, [-1, -1, 48]) == 1 and c.length == [21, 33, 0]
    assert OK.resize(c, [0, -1, 16]) == 0 and c.table[2][0] == 1 and c.ref[0] == 1
    assert OK.resize(c, [49, 0, 0]) == -1 and c.length == [0, 33, 16]


# ---- what the library refuses --------------------------------------------------------------------------------------------

def cache_struct(qk, **change):
    """A valid paged cache with addresses that are never followed."""
    f = dict(type=qk.F32, n_layer=2, n_page=8, n_kv=2, page_rows=16, dh=128, n_seq=3, seq_pages=4, k=4096, v=8192, table=256, ref=512, len=1024)
    f.update(change)
    return qk.capi._KvCache(*[f[n] for n, _ in qk.capi._KvCache._fields_])


def runs_struct(qk, **change):
    f = dict(n_rows=5, n_run=2, max_run=3, start=64, seq=128, pos=192)
    f.update(change)
    return qk.capi._KvRuns(*[f[n] for n, _ in qk.capi._KvRuns._fields_])


CACHES = [
    (dict(k=None), -1, "null"), (dict(type=8), -3, "cache type"), (dict(dh=64), -2, "head size"), (dict(k=4100), -1, "aligned"),
    (dict(n_kv=0), -1, "zero"), (dict(n_page=0), -1, "zero"), (dict(n_seq=0), -1, "zero"), (dict(seq_pages=0), -1, "zero"),
    (dict(page_rows=24), -2, "power of two"), (dict(page_rows=8), -2, "power of two"), (dict(page_rows=1 << 17), -2, "power of two"),
    (dict(table=None), -2, "slot cache"), (dict(table=None, seq_pages=1, n_seq=9), -2, "slot cache"),
    (dict(table=None, seq_pages=1, page_rows=1 << 25), -2, "slot cache"), (dict(n_kv=5000), -2, "too large"),
    (dict(seq_pages=1 << 20, page_rows=1 << 16), -2, "2^30"), (dict(table=258), -1, "aligned"),
]


def last(qk):
    return qk.lib().qkk_last_error().decode()


@pytest.mark.parametrize("change,code,text", CACHES)
def test_cache_is_checked_by_every_call(qk, change, code, text):
    L, c, r = qk.lib(), C.byref(cache_struct(qk, **change)), C.byref(runs_struct(qk))
    big = 1 << 40
    calls = [lambda: L.qkk_attn_prep_axes(c, 0, r, 16, 16, 16, 16, 16, 16, 4, 16, 1, 16, 16, 4, 8, 0, 1e-6, None),
             lambda: L.qkk_attn_packed(c, 0, r, 16, None, 16, 256, big, 4, None), lambda: L.qkk_attn_tree(c, 0, r, 16, 16, None, 16, 256, big, 4, None),
             lambda: L.qkk_kv_resize(c, 16, 16, 256, big, None), lambda: L.qkk_kv_fork(c, 16, 16, 1, 16, 256, big, None),
             lambda: L.qkk_kv_compact(c, 16, 16, 16, 16, 1, 4, None)]
    for call in calls:
        assert call() == code and text in last(qk), last(qk)


def test_other_arguments_are_checked(qk):
    L, big = qk.lib(), 1 << 40
    c, r = C.byref(cache_struct(qk)), C.byref(runs_struct(qk))
    prep = lambda **k: L.qkk_attn_prep_axes(k.get("c", c), k.get("layer", 0), k.get("r", r), k.get("q", 16), 16, 16, 16, 16, 16, k.get("rope_rows", 4), 16,  # noqa: E731
                                            k.get("n_axis", 1), 16, k.get("qhat", 16), k.get("hq", 4), k.get("n_rot", 8), 0, k.get("eps", 1e-6), None)
    for change, code, text in [(dict(q=None), -1, "null"), (dict(q=20), -1, "aligned"), (dict(layer=2), -2, "layer"), (dict(hq=0), -2, "query heads"),
                               (dict(n_rot=7), -2, "n_rot"), (dict(n_rot=130), -2, "n_rot"), (dict(n_rot=0), -2, "n_rot"), (dict(n_axis=0), -2, "axes"),
                               (dict(n_axis=9), -2, "axes"), (dict(rope_rows=0), -2, "rope_rows"), (dict(eps=-1.0), -1, "eps"), (dict(eps=float("nan")), -1, "eps"),
                               (dict(r=None), -1, "null"), (dict(r=C.byref(runs_struct(qk, pos=None))), -1, "null"),
                               (dict(r=C.byref(runs_struct(qk, n_rows=1 << 21))), -2, "2^20"), (dict(c=None), -1, "null")]:
        assert prep(**change) == code and text in last(qk), (change, last(qk))
    tree = lambda **k: L.qkk_attn_tree(c, 0, k.get("r", r), k.get("parent", 16), k.get("q", 16), k.get("gate", None), 16, k.get("ws", 256), k.get("n", big), k.get("hq", 4), None)  # noqa: E731
    for change, code, text in [(dict(parent=None), -1, "null"), (dict(hq=3), -2, "query heads"), (dict(hq=1), -2, "query heads"), (dict(hq=8192), -2, "query heads"),
                               (dict(q=24), -1, "aligned"), (dict(gate=24), -1, "aligned"), (dict(ws=128), -1, "aligned"), (dict(n=16), -5, "workspace"),
                               (dict(r=C.byref(runs_struct(qk, n_rows=300, max_run=257))), -2, "nodes")]:
        assert tree(**change) == code and text in last(qk), (change, last(qk))
    assert L.qkk_kv_resize(c, None, 16, 256, big, None) == -1 and L.qkk_kv_resize(c, 16, None, 256, big, None) == -1
    assert L.qkk_kv_resize(c, 16, 16, 256, 8, None) == -5 and L.qkk_kv_resize(c, 16, 16, 260, big, None) == -1
    assert L.qkk_kv_resize(C.byref(cache_struct(qk, ref=None)), 16, 16, 256, big, None) == -1
    assert L.qkk_kv_resize(C.byref(cache_struct(qk, len=None)), 16, 16, 256, big, None) == -1
    assert L.qkk_kv_fork(c, 16, 16, 4, 16, 256, big, None) == -2 and L.qkk_kv_fork(c, None, 16, 1, 16, 256, big, None) == -1
    assert L.qkk_kv_compact(c, 16, 16, 16, 16, 4, 4, None) == -2 and L.qkk_kv_compact(c, 16, 16, 16, 16, 1, 257, None) == -2
    assert L.qkk_kv_compact(c, 16, 16, None, 16, 1, 4, None) == -1
    axes = (C.c_uint8 * 64)()
    sec = lambda *v: (C.c_uint32 * len(v))(*v)  # noqa: E731
    assert L.qkk_rope_axes(axes, 8, sec(2, 1), 2, 0) == -2 and L.qkk_rope_axes(axes, 7, sec(3), 1, 0) == -2 and L.qkk_rope_axes(axes, 8, sec(4), 0, 0) == -2
    assert L.qkk_rope_axes(None, 8, sec(4), 1, 0) == -1 and L.qkk_rope_axes(axes, 8, sec(*[1] * 9), 9, 0) == -2
    assert L.qkk_attn_runs_workspace_bytes(None, r, 4) == 0 and L.qkk_attn_runs_workspace_bytes(c, r, 1) == 0 and L.qkk_kv_workspace_bytes(None) == 0


def test_no_device_is_an_error(qk):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    c, r = C.byref(cache_struct(qk)), C.byref(runs_struct(qk))
    assert qk.lib().qkk_attn_packed(c, 0, r, 16, None, 16, 256, 1 << 40, 4, None) == -4 and "no HIP device" in last(qk)


def test_binding_checks_tensors():
    """Types, shapes, strides and devices are compared before an address leaves Python."""
    import torch

    import __graft_entry__ as entry
    qk = entry.load_package()
    k = torch.zeros(1, 4, 2, 16, 128)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="float32 or float16"):
        qk.KvCache(k.double(), k.double())
    with pytest.raises(ValueError, match="v must be"):
        qk.KvCache(k, k.half())
    with pytest.raises(ValueError, match="strided"):
        qk.KvCache(k.transpose(3, 4).contiguous().transpose(3, 4), k)
    with pytest.raises(ValueError, match="ref must be"):
        qk.KvCache(k, k, table=torch.zeros(2, 2, dtype=torch.int32), ref=i32(0, 0, 0))
    with pytest.raises(ValueError, match="table must be"):
        qk.KvCache(k, k, table=torch.zeros(2, 2, dtype=torch.int64))
    with pytest.raises(ValueError, match="start must be"):
        qk.KvRuns(3, i32(0, 3, 3), i32(0), i32(0))
    cache, runs = qk.KvCache(k, k), qk.KvRuns(3, i32(0, 3), i32(0), i32(0))
    assert (cache.n_seq, cache.seq_pages) == (4, 1)
    q, ws = torch.zeros(3, 4, 128), torch.zeros(256, dtype=torch.uint8)
    for bad in (q[:2], q.half(), torch.zeros(3, 4, 256), torch.zeros(3, 128, 4).transpose(1, 2)):
        with pytest.raises(ValueError, match="qhat must be"):
            qk.attn_packed(cache, 0, runs, bad, ws)
    with pytest.raises(ValueError, match="qfull must be"):
        qk.attn_packed(cache, 0, runs, q, ws, qfull=q)
    with pytest.raises(ValueError, match="parent"):
        qk.attn_tree(cache, 0, runs, None, q, ws)
    with pytest.raises(ValueError, match="parent must be"):
        qk.attn_tree(cache, 0, runs, i32(-1, 0), q, ws)
    with pytest.raises(ValueError, match="len_new must be"):
        qk.kv_resize(cache, i32(1, 2), ws)
    with pytest.raises(ValueError, match="path must be"):
        qk.kv_compact(cache, i32(0), i32(0), i32(0, 1), i32(2))
    with pytest.raises(ValueError, match="axis_pos"):
        qk.attn_prep_axes(cache, 0, runs, q, q[:, :2], q[:, :2], q[0, 0], q[0, 0], torch.zeros(8, 4, 2), torch.zeros(4, dtype=torch.uint8), i32(0, 1, 2))


def test_bounds_of_the_checks_hold_for_the_oracle():
    """The comparison itself: an oracle with one weight wrong by 1e-3 is outside the bound (the mistake is planted here)."""
    rng = np.random.default_rng(5)
    c = slot_cache(rng, 1, 1, 64, 128)
    q = rng.standard_normal((4, 2, 128)).astype(np.float32)
    rows = list(OK.runs(4, [0, 4], [0], [40], c, 4))
    want = OK.attend(c, 0, rows, q)
    tol = KC.bound(c, 0, rows, q)
    KC.check_att(want.astype(np.float32), want, tol, rows)
    wrong = OK.attend(OK.Cache(c.k * np.float32(1.001), c.v, None), 0, rows, q)
    with pytest.raises(AssertionError):
        KC.check_att(wrong.astype(np.float32), want, tol, rows)


@pytest.mark.parametrize("change", [dict(seq_pages=1 << 31, page_rows=1 << 16), dict(seq_pages=0xFFFFFFFF, page_rows=0xFFFFFFFF), dict(seq_pages=1 << 20, page_rows=1 << 16),
                                    dict(dh=1 << 20)])
def test_workspace_of_a_cache_that_the_calls_refuse(qk, change):
    """Sizes whose ranges of keys do not fit 32 bits ended the process in a division by zero; 0 bytes are asked for."""
    c, r = cache_struct(qk, **change), runs_struct(qk)
    assert qk.lib().qkk_attn_runs_workspace_bytes(C.byref(c), C.byref(r), 4) == 0
    assert qk.lib().qkk_attn_packed(C.byref(c), 0, C.byref(r), 16, None, 16, 256, 1 << 40, 4, None) == -2


@pytest.mark.parametrize("change,hq", [(dict(n_rows=(1 << 20) + 1), 4), (dict(n_run=(1 << 20) + 1), 4), (dict(n_rows=0xFFFFFFFF, max_run=0xFFFFFFFF), 4), (dict(), 8192)])
def test_workspace_of_runs_that_the_calls_refuse(qk, change, hq):
    c, r = cache_struct(qk), runs_struct(qk, **change)
    assert qk.lib().qkk_attn_runs_workspace_bytes(C.byref(c), C.byref(r), hq) == 0
    assert qk.lib().qkk_attn_packed(C.byref(c), 0, C.byref(r), 16, None, 16, 256, 1 << 40, hq, None) == -2


def test_host_tensors_do_not_reach_a_device(monkeypatch):
    """A cache in host memory is consistent in itself, but its addresses are none of a device's: refused in front of the launch.  (Without a
    device the library itself refuses; here torch is made to say that there is one.)"""
    import torch

    import __graft_entry__ as entry
    qk = entry.load_package()
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(qk.capi, "_stream", lambda: None)
    k, i32 = torch.zeros(1, 4, 2, 16, 128), lambda *v: torch.tensor(v, dtype=torch.int32)
    cache, runs = qk.KvCache(k, k.clone(), len=i32(0, 0, 0, 0)), qk.KvRuns(3, i32(0, 3), i32(0), i32(0))
    raw = torch.zeros(1 << 16, dtype=torch.uint8)
    ws, q, kv, w = raw[-raw.data_ptr() % 256:], torch.zeros(3, 4, 128), torch.zeros(3, 2, 128), torch.zeros(128)
    calls = [lambda: qk.attn_packed(cache, 0, runs, q, ws), lambda: qk.attn_tree(cache, 0, runs, i32(-1, 0, 0), q, ws), lambda: qk.kv_resize(cache, i32(1, 1, 1, 1), ws),
             lambda: qk.kv_fork(cache, i32(0), i32(1), ws), lambda: qk.kv_compact(cache, i32(0), i32(0), i32(0, 1).view(1, 2), i32(2)),
             lambda: qk.attn_prep_axes(cache, 0, runs, q, kv, kv, w, w, torch.zeros(8, 4, 2), torch.zeros(4, dtype=torch.uint8), i32(0, 1, 2).view(1, 3))]
    for call in calls:
        with pytest.raises(ValueError, match="host memory"):
            call()
