"""Refusals of the paged cache's entry points: every bad argument is turned down before any device work, so these need
no GPU. The pointers are placeholders that nothing reads."""
import ctypes

import pytest
import torch

from yalama_b200 import engine as E

INV, OK = E.Status.INVALID_ARG, E.Status.OK
A = 1 << 24  # placeholder address, 16-byte aligned


def cache(**kw):
    a = dict(k=A, v=2 * A, n_pages=50, page=16, hkv=2)
    a.update(kw)
    return E.paged_cache(**a)


def step(**kw):
    a = dict(row_start=3 * A, length=4 * A, page_table=5 * A, parent=None, n_seq=3, table_ld=9, rows=20, max_rows=8,
             fault=None)
    a.update(kw)
    return E.paged_step(**a)


def append(c=None, st=None, q=8 * A, qs=512, k=9 * A, ks=256, v=10 * A, vs=256, hq=4, qn=None, kn=None, cos=11 * A,
           sin=12 * A, max_pos=100, out=13 * A, os=512):
    return E.lib().ylm_k_paged_append(cache() if c is None else c, step() if st is None else st, q, qs, k, ks, v, vs, hq,
                                      qn, kn, 1e-6, cos, sin, max_pos, out, os, None)


def attend(c=None, st=None, q=8 * A, qs=512, hq=4, out=9 * A, os=512, ws=None, wb=0):
    return E.lib().ylm_k_paged_attention(cache() if c is None else c, step() if st is None else st, q, qs, hq, out, os,
                                         ws, wb, None)


def size(c=None, st=None, hq=4):
    b = ctypes.c_size_t()
    return E.lib().ylm_k_paged_attention_workspace(cache() if c is None else c, step() if st is None else st, hq,
                                                   ctypes.byref(b))


def accept(c=None, st=None, tokens=14 * A, picks=15 * A, layers=2, stride=16 * A, acc=16 * A, n=17 * A, nxt=18 * A,
           new=19 * A):
    return E.lib().ylm_k_paged_accept(cache() if c is None else c, step() if st is None else st, tokens, picks, layers,
                                      stride, acc, n, nxt, new, None)


LAYER_BYTES = 50 * 2 * 16 * 128 * 2  # of the placeholder cache
BAD_CACHES = [dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 2), dict(page=0), dict(page=8), dict(page=48),
              dict(page=256), dict(page=-16), dict(n_pages=0), dict(n_pages=-1), dict(hkv=0), dict(hkv=65536)]
BAD_CACHES += [dict(v=A), dict(v=A + LAYER_BYTES - 16), dict(k=2 * A + 16)]
BAD_STEPS = [dict(row_start=None), dict(length=None), dict(page_table=None), dict(row_start=A + 2), dict(length=A + 1),
             dict(page_table=A + 3), dict(parent=A + 2), dict(fault=A + 1), dict(n_seq=-1), dict(n_seq=65536),
             dict(table_ld=0), dict(table_ld=-3), dict(table_ld=(1 << 26) + 1), dict(table_ld=2 ** 31 - 1), dict(rows=-1),
             dict(max_rows=-1), dict(parent=A, max_rows=129)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches_are_refused_everywhere(bad):
    for call in (append, attend, size, accept):
        assert call(c=cache(**bad)) == INV
        assert E.lib().ylm_last_error() != b""


@pytest.mark.parametrize("bad", BAD_STEPS, ids=str)
def test_bad_steps_are_refused_everywhere(bad):
    for call in (append, attend, size, accept):
        assert call(st=step(**bad)) == INV


def test_null_descriptors_are_refused():
    L, c, st = E.lib(), cache(), step()
    b = ctypes.c_size_t()
    for x, y in ((None, st), (c, None)):
        assert L.ylm_k_paged_append(x, y, A, 512, A, 256, A, 256, 4, None, None, 0.0, None, None, 0, A, 512, None) == INV
        assert L.ylm_k_paged_attention(x, y, A, 512, 4, A, 512, None, 0, None) == INV
        assert L.ylm_k_paged_attention_workspace(x, y, 4, ctypes.byref(b)) == INV
        assert L.ylm_k_paged_accept(x, y, A, A, 1, 0, A, A, A, A, None) == INV
    assert L.ylm_k_paged_attention_workspace(c, st, 4, None) == INV


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=A + 8), dict(k=A + 2),
                                 dict(v=A + 4), dict(out=A + 8), dict(qs=504), dict(qs=516), dict(ks=248), dict(vs=255),
                                 dict(vs=-256), dict(os=256), dict(hq=-1), dict(hq=65536), dict(cos=None),
                                 dict(sin=None), dict(max_pos=0), dict(cos=A + 8), dict(sin=A + 2), dict(qn=A + 2),
                                 dict(kn=A + 8)], ids=str)
def test_append_refuses(bad):
    assert append(**bad) == INV


@pytest.mark.parametrize("bad", [dict(hq=0), dict(hq=3), dict(hq=-2), dict(hq=258), dict(q=None), dict(out=None),
                                 dict(q=A + 8), dict(out=A + 4), dict(qs=511), dict(qs=516), dict(os=504),
                                 dict(ws=A + 8, wb=1 << 40)], ids=str)
def test_attention_refuses(bad):
    assert attend(**bad) == INV


@pytest.mark.parametrize("hq", [0, 3, -2, 258])
def test_attention_workspace_refuses(hq):
    assert size(hq=hq) == INV


Q = 8 * A  # where the queries of append() and attend() lie: 20 rows of 512 halves


# (addresses are bytes: a row of 512 halves is 1024 of them)
@pytest.mark.parametrize("bad", [dict(out=Q, os=520), dict(out=Q + 16), dict(out=Q + 1024), dict(out=Q - 1024),
                                 dict(out=Q + 19 * 1024 + 1008), dict(out=9 * A + 512), dict(out=10 * A + 19 * 512),
                                 # a fused projection of 4 + 2 + 2 heads: the keys' and the values' columns
                                 dict(qs=1024, k=Q + 1024, ks=1024, v=Q + 1536, vs=1024, out=Q + 1024, os=1024),
                                 dict(qs=1024, k=Q + 1024, ks=1024, v=Q + 1536, vs=1024, out=Q + 512, os=1024),
                                 dict(qs=1024, k=Q + 1024, ks=1024, v=Q + 1536, vs=1024, out=Q, os=512),
                                 dict(qs=1024, k=Q + 1024, ks=1024, v=Q + 1536, vs=1024, out=Q + 2048, os=1024)], ids=str)
def test_append_refuses_queries_out_over_other_rows(bad):
    assert append(**bad) == INV
    assert b"overlap" in E.lib().ylm_last_error()


# (what is not refused stops at the device, which is not looked for before every check has passed)
@pytest.mark.parametrize("good", [dict(out=Q), dict(out=Q + 20 * 1024), dict(out=Q - 20 * 1024),
                                  dict(qs=1024, k=Q + 1024, ks=1024, v=Q + 1536, vs=1024, out=Q, os=1024)], ids=str)
@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are placeholders")
def test_append_takes_queries_out_in_place_or_elsewhere(good):
    assert append(**good) not in (INV, OK)


@pytest.mark.parametrize("bad", [dict(out=Q), dict(out=Q + 1024), dict(out=Q, os=520), dict(out=Q - 19 * 1024 - 16),
                                 dict(qs=1024, out=Q + 512, os=1024)], ids=str)
def test_attention_refuses_out_over_the_queries(bad):
    assert attend(**bad) == INV
    assert b"overlap" in E.lib().ylm_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are placeholders")
@pytest.mark.parametrize("good", [dict(out=Q + 20 * 1024), dict(qs=1024, out=Q + 1024, os=1024)], ids=str)
def test_attention_takes_columns_beside_the_queries(good):
    assert attend(**good) not in (INV, OK)


LAYER = 50 * 2 * 16 * 128  # halves of the placeholder cache's layer


@pytest.mark.parametrize("bad", [dict(tokens=None), dict(picks=None), dict(tokens=A + 4), dict(picks=A + 4),
                                 dict(layers=-1), dict(stride=LAYER - 8), dict(stride=LAYER + 4), dict(acc=None),
                                 dict(n=None), dict(nxt=None), dict(new=None), dict(acc=A + 2), dict(n=A + 1),
                                 dict(nxt=A + 4), dict(new=A + 2), dict(new=4 * A), dict(n=4 * A + 8), dict(acc=5 * A),
                                 dict(nxt=14 * A), dict(acc=15 * A + 152), dict(n=3 * A + 12), dict(new=17 * A),
                                 dict(nxt=16 * A + 88)], ids=str)
def test_accept_refuses(bad):
    assert accept(**bad) == INV


def test_accept_refuses_a_layers_keys_over_another_layers_values():
    assert accept(stride=A // 2) == INV  # layer 1's keys lie where layer 0's values do
    assert b"overlap" in E.lib().ylm_last_error()


def test_accept_refuses_results_over_the_parents():
    assert accept(st=step(parent=6 * A), new=6 * A + 76) == INV


@pytest.mark.parametrize("parent", [None, 6 * A])
def test_accept_without_rows_needs_its_results_all_the_same(parent):
    """max_rows entries a request are written, whatever the rows."""
    assert accept(st=step(rows=0, parent=parent), tokens=None, picks=None, acc=None) == INV
    assert b"output" in E.lib().ylm_last_error()


def test_nothing_to_do_is_fine():
    for st in (step(n_seq=0, row_start=None, length=None, page_table=None), step(n_seq=0, rows=0, table_ld=0)):
        assert append(st=st, q=None, k=None, v=None, out=None) == OK
        assert attend(st=st, q=None, out=None) == OK
        assert accept(st=st, tokens=None, picks=None, acc=None, n=None, nxt=None, new=None) == OK
    assert append(st=step(rows=0), q=None, k=None, v=None, out=None) == OK
    assert attend(st=step(rows=0), q=None, out=None) == OK
