"""Refusals of the serving operators: bad calls come back with a status before anything is launched, so they need no GPU."""
import ctypes as C

import pytest

from bpd_substrate_b200 import capi

P = 1 << 20          # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def paged(**changes):
    d = dict(heads=8, kv_heads=2, dim=64, act_type=capi.TYPE_BF16, kv_type=capi.TYPE_BF16, page=16, n_pages=40, batch=3, max_pages=10, page_stride=0, k=P, v=P,
             page_table=P, length=P, seq_start=P)
    d.update(changes)
    return capi.PagedKv(**d)


BAD_CACHES = [
    (dict(k=None), -1), (dict(v=None), -1), (dict(page_table=None), -1), (dict(length=None), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(kv_heads=3), -1),
    (dict(dim=0), -1), (dict(n_pages=0), -1), (dict(max_pages=0), -1), (dict(batch=-1), -1), (dict(page_stride=2 * 16 * 64 - 8), -1),
    (dict(act_type=capi.TYPE_F32), -1), (dict(act_type=capi.TYPE_F16), -1), (dict(kv_type=capi.TYPE_F32), -1), (dict(act_type=3, kv_type=3), -1), (dict(act_type=-1, kv_type=-1), -1),
    (dict(page=4), -3), (dict(page=24), -3), (dict(page=512), -3), (dict(dim=60), -3), (dict(dim=136), -3), (dict(batch=2049), -3), (dict(max_pages=1 << 27), -3),
    (dict(k=P + 8), -2), (dict(v=P + 2), -2), (dict(page_stride=2 * 16 * 64 + 4), -2), (dict(seq_start=None, batch=6), -1),
]


def append(lib, kv, q=P, ld_q=512, q_out=P, ld_q_out=512, k=P, ld_k=128, v=P, ld_v=128, n=5, rot=64, neighbours=0, freq=P):
    return lib.bpd_paged_append_cuda(C.byref(kv) if kv else None, q, ld_q, q_out, ld_q_out, k, ld_k, v, ld_v, n, rot, neighbours, freq, None)


def attention(lib, kv, q=P, ld_q=512, o=P, ld_o=512, n=5, scale=0.1, cap=0.0, groups=None):
    return lib.bpd_paged_attention_cuda(C.byref(kv) if kv else None, q, ld_q, o, ld_o, n, scale, cap, groups, None)


@pytest.mark.parametrize("changes,status", BAD_CACHES)
def test_bad_caches(lib, changes, status):
    kv = paged(**changes)
    assert append(lib, kv) == status
    assert attention(lib, kv) == status
    assert lib.bpdq_paged_attention_workspace_bytes(C.byref(kv), 5, None) == 0
    assert lib.bpd_paged_attention_ws_cuda(C.byref(kv), P, 512, P, 512, 5, 0.1, 0.0, None, P, 1 << 30, None) == status
    lib.bpdq_clear_status()


@pytest.mark.parametrize("changes", [dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(ld_q=511), dict(ld_q_out=8), dict(ld_k=127), dict(ld_v=0), dict(n=-1),
                                     dict(rot=66), dict(rot=7), dict(rot=-2), dict(freq=None)])
def test_bad_appends(lib, changes):
    assert append(lib, paged(), **changes) == -1
    lib.bpdq_clear_status()


@pytest.mark.parametrize("name", ["q", "q_out", "k", "v"])
def test_misaligned_appends(lib, name):
    assert append(lib, paged(), **{name: P + 1}) == -2
    assert append(lib, paged(act_type=capi.TYPE_F32, kv_type=capi.TYPE_F16), **{name: P + 2}) == -2
    lib.bpdq_clear_status()


@pytest.mark.parametrize("changes,status", [(dict(q=None), -1), (dict(o=None), -1), (dict(ld_q=504), -1), (dict(ld_o=0), -1), (dict(n=-1), -1), (dict(cap=-1.0), -1),
                                            (dict(cap=float("nan")), -1), (dict(cap=float("inf")), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1),
                                            (dict(q=P + 8), -2), (dict(o=P + 2), -2), (dict(ld_q=516), -2), (dict(ld_o=513), -2)])
def test_bad_attention(lib, changes, status):
    assert attention(lib, paged(), **changes) == status
    lib.bpdq_clear_status()


@pytest.mark.parametrize("n,start,pages", [(-1, P, P), (4, P, P), (1, None, P), (1, P, None)])
def test_bad_groups(lib, n, start, pages):
    g = capi.PagedGroups(n, start, pages)
    assert attention(lib, paged(), groups=C.byref(g)) == -1
    assert lib.bpdq_paged_attention_workspace_bytes(C.byref(paged()), 5, C.byref(g)) == 0
    lib.bpdq_clear_status()


@pytest.mark.parametrize("changes", [dict(heads=258, kv_heads=2), dict(batch=1280, max_pages=1 << 21), dict(batch=1281)])
def test_attention_beyond_its_range(lib, changes):
    kv = paged(**changes)
    assert attention(lib, kv, ld_q=258 * 64, ld_o=258 * 64) == -3
    assert lib.bpdq_paged_attention_workspace_bytes(C.byref(kv), 5, None) == 0
    lib.bpdq_clear_status()


def test_more_products_than_are_counted(lib):
    """Four million tokens against two million positions: units of work are counted in 32 bits."""
    kv = paged(max_pages=1 << 17)
    assert lib.bpdq_paged_attention_workspace_bytes(C.byref(kv), 1 << 17, None) > 0
    assert attention(lib, kv, n=1 << 22) == -3
    assert lib.bpdq_paged_attention_workspace_bytes(C.byref(kv), 1 << 22, None) == 0
    lib.bpdq_clear_status()


def test_no_descriptor_and_no_workspace(lib):
    assert append(lib, None) == -1 and attention(lib, None) == -1
    assert lib.bpdq_paged_attention_workspace_bytes(None, 5, None) == 0
    assert lib.bpd_paged_attention_ws_cuda(C.byref(paged()), P, 512, P, 512, 5, 0.1, 0.0, None, None, 1 << 30, None) == -1
    lib.bpdq_clear_status()


def test_nothing_to_do_is_no_error(lib):
    for kv in (paged(), paged(batch=0), paged(batch=0, seq_start=None)):
        assert append(lib, kv, n=0) == 0 and attention(lib, kv, n=0) == 0
    assert append(lib, paged(batch=0)) == 0 and attention(lib, paged(batch=0)) == 0
    assert lib.bpd_sample_cuda(P, 0, 32, 0, 32, None, None, None, None, P, P, None, None) == 0


@pytest.mark.parametrize("changes,status", [(dict(logits=None), -1), (dict(u=None), -1), (dict(token=None), -1), (dict(rows=-1), -1), (dict(vocab=0), -1), (dict(ld=31), -1),
                                            (dict(type=-1), -1), (dict(type=3), -1), (dict(vocab=262145, ld=262145), -3), (dict(logits=P + 2), -2), (dict(logits=P + 1, type=2), -2)])
def test_bad_samples(lib, changes, status):
    a = dict(logits=P, type=0, ld=32, rows=2, vocab=32, u=P, token=P)
    a.update(changes)
    assert lib.bpd_sample_cuda(a["logits"], a["type"], a["ld"], a["rows"], a["vocab"], None, None, None, None, a["u"], a["token"], None, None) == status
    lib.bpdq_clear_status()


@pytest.mark.parametrize("batch,n,seq_start", [(0, 0, P), (0, 5, P), (3, 0, P), (0, 0, None), (0, 5, None)])
@pytest.mark.parametrize("types", [(capi.TYPE_BF16, capi.TYPE_BF16), (capi.TYPE_F32, capi.TYPE_F16)])
def test_scratch_of_an_empty_step(lib, batch, n, seq_start, types):
    """Its size can be asked for, and a workspace of that size (or any other) does."""
    kv = paged(batch=batch, seq_start=seq_start, act_type=types[0], kv_type=types[1])
    size = lib.bpdq_paged_attention_workspace_bytes(C.byref(kv), n, None)
    assert size > 0
    g = capi.PagedGroups(0, None, None)
    assert lib.bpdq_paged_attention_workspace_bytes(C.byref(kv), n, C.byref(g)) == size
    for given in (size, 16):
        assert lib.bpd_paged_attention_ws_cuda(C.byref(kv), P, 512, P, 512, n, 0.1, 0.0, None, P, given, None) == 0


def test_in_place_only_row_by_row(lib):
    """Results in the place of the queries with other distances between rows would overwrite queries that are still to be read."""
    kv = paged()
    assert append(lib, kv, ld_q=512, ld_q_out=640) == -1 and append(lib, kv, ld_q=640, ld_q_out=512) == -1
    assert attention(lib, kv, ld_q=512, ld_o=640) == -1 and attention(lib, kv, ld_q=640, ld_o=512) == -1
    assert lib.bpd_paged_attention_ws_cuda(C.byref(kv), P, 512, P, 640, 5, 0.1, 0.0, None, P, 1 << 30, None) == -1
    lib.bpdq_clear_status()
