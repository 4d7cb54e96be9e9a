"""Refusals of the 8-bit K/V cache's and the log probabilities' entry points: every bad argument is turned down
before any device work, so these need no GPU. The pointers are placeholders that nothing reads."""
import ctypes

import pytest

from yalama_b200 import engine as E

INV, OK = E.Status.INVALID_ARG, E.Status.OK
A = 1 << 20  # placeholder address, 16-byte aligned


def cache(**kw):
    a = dict(k=A, v=2 * A, k_scale=3 * A, v_scale=4 * A, fmt="e4m3", block=32, cap=100, hkv=2)
    a.update(kw)
    c = E.kv8_cache(a["k"], a["v"], a["k_scale"], a["v_scale"], a["fmt"], a["block"], a["cap"], a["hkv"])
    if "format" in kw:
        c.format = kw["format"]
    return c


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(block=8), dict(block=0),
              dict(block=48), dict(block=256), dict(cap=0), dict(cap=-1), dict(hkv=0), dict(hkv=65536),
              dict(k=A + 8), dict(v=2 * A + 4), dict(k_scale=3 * A + 2), dict(v_scale=4 * A + 1), dict(format=2),
              dict(format=-1)]


def store(c=None, k=8 * A, ks=256, v=9 * A, vs=256, t=1, slot=0):
    return E.lib().ylm_k_kv8_store(cache() if c is None else c, k, ks, v, vs, t, slot, None)


def attend(c=None, q=8 * A, qs=512, hq=4, t=1, n=10, mask=None, acc=None, out=9 * A, os=512, ws=None, wb=0):
    return E.lib().ylm_k_kv8_attention(cache() if c is None else c, q, qs, hq, t, n, mask, acc, out, os, ws, wb, None)


def evict(src=None, dst=None, acc=5 * A, acc_dst=15 * A, n=50, keep=20, sink=2, recent=3, kept=16 * A):
    src = cache() if src is None else src
    dst = cache(k=11 * A, v=12 * A, k_scale=13 * A, v_scale=14 * A) if dst is None else dst
    return E.lib().ylm_k_kv8_evict(src, dst, acc, acc_dst, n, keep, sink, recent, kept, None)


def logprobs(x=A, ld=100, rows=1, vocab=100, ids=2 * A, mask=None, n_top=2, lp=3 * A, ent=4 * A, ti=5 * A, tl=6 * A):
    return E.lib().ylm_k_logprobs(x, ld, rows, vocab, ids, mask, n_top, lp, ent, ti, tl, None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches_are_refused_everywhere(bad):
    c = cache(**bad)
    size = ctypes.c_size_t()
    good = cache(k=11 * A, v=12 * A, k_scale=13 * A, v_scale=14 * A)
    assert store(c) == INV
    assert attend(c) == INV
    assert E.lib().ylm_k_kv8_attention_workspace(c, 4, 1, 1, 0, ctypes.byref(size)) == INV
    assert evict(src=c, dst=good) == INV
    assert evict(src=good, dst=c) == INV
    assert E.lib().ylm_last_error() != b""


def test_null_cache_is_refused():
    size = ctypes.c_size_t()
    L = E.lib()
    assert L.ylm_k_kv8_store(None, A, 256, A, 256, 1, 0, None) == INV
    assert L.ylm_k_kv8_attention(None, A, 512, 4, 1, 1, None, None, A, 512, None, 0, None) == INV
    assert L.ylm_k_kv8_attention_workspace(None, 4, 1, 1, 0, ctypes.byref(size)) == INV
    assert L.ylm_k_kv8_attention_workspace(cache(), 4, 1, 1, 0, None) == INV
    assert L.ylm_k_kv8_evict(None, cache(), A, A, 1, 1, 0, 0, A, None) == INV
    assert L.ylm_k_kv8_evict(cache(), None, A, A, 1, 1, 0, 0, A, None) == INV


@pytest.mark.parametrize("bad", [dict(t=-1), dict(slot=-1), dict(slot=101, t=0), dict(slot=100), dict(slot=50, t=51),
                                 dict(slot=2 ** 31 - 1, t=2 ** 31 - 1), dict(k=None), dict(v=None), dict(k=8 * A + 8),
                                 dict(v=9 * A + 2), dict(ks=248), dict(vs=255), dict(ks=260), dict(vs=-256)], ids=str)
def test_store_refuses(bad):
    assert store(**bad) == INV


def test_store_of_nothing_is_fine():
    assert store(t=0, k=None, v=None, slot=100) == OK


@pytest.mark.parametrize("bad", [dict(hq=0), dict(hq=3), dict(hq=-4), dict(hq=258), dict(t=-1), dict(t=11),
                                 dict(n=101), dict(q=None), dict(out=None), dict(q=8 * A + 2), dict(out=9 * A + 8),
                                 dict(qs=511), dict(qs=516), dict(os=256), dict(mask=A + 2), dict(acc=A + 1),
                                 dict(ws=A + 8, wb=1 << 30)], ids=str)
def test_attention_refuses(bad):
    assert attend(**bad) == INV


def test_attention_of_nothing_is_fine():
    assert attend(t=0, q=None, out=None) == OK
    assert attend(t=0, n=0, q=None, out=None) == OK


@pytest.mark.parametrize("bad", [
    dict(dst=cache(k=11 * A, v=12 * A, k_scale=13 * A, v_scale=14 * A, fmt="int8")),
    dict(dst=cache(k=11 * A, v=12 * A, k_scale=13 * A, v_scale=14 * A, block=16)),
    dict(dst=cache(k=11 * A, v=12 * A, k_scale=13 * A, v_scale=14 * A, hkv=1)),
    dict(dst=cache(k=11 * A, v=12 * A, k_scale=13 * A, v_scale=14 * A, cap=19)),
    dict(dst=cache()), dict(dst=cache(v=12 * A, k_scale=13 * A, v_scale=14 * A)),
    dict(dst=cache(k=A + 2 * 100 * 128 - 16, v=12 * A, k_scale=13 * A, v_scale=14 * A)),
    dict(dst=cache(k=11 * A, v=11 * A, k_scale=13 * A, v_scale=14 * A)),
    dict(n=101), dict(n=-1), dict(n=19), dict(keep=-1), dict(sink=-1), dict(recent=-1), dict(sink=10, recent=11),
    dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1), dict(acc=None), dict(acc_dst=None), dict(kept=None),
    dict(acc=5 * A + 2), dict(acc_dst=15 * A + 1), dict(kept=16 * A + 2), dict(acc_dst=5 * A), dict(kept=5 * A),
    dict(kept=15 * A), dict(kept=11 * A)], ids=range(26))
def test_evict_refuses(bad):
    assert evict(**bad) == INV


@pytest.mark.parametrize("bad", [dict(x=None), dict(ld=99), dict(rows=-1), dict(vocab=0), dict(vocab=-5),
                                 dict(vocab=2 ** 31, ld=2 ** 31), dict(vocab=2 ** 30 + 1, ld=2 ** 31), dict(n_top=-1), dict(n_top=65), dict(ids=None),
                                 dict(ti=None), dict(tl=None), dict(lp=None, ent=None, n_top=0), dict(x=A + 1),
                                 dict(ids=2 * A + 4), dict(mask=A + 2), dict(lp=A + 2), dict(ent=A + 1),
                                 dict(ti=A + 4), dict(tl=A + 2)], ids=str)
def test_logprobs_refuses(bad):
    assert logprobs(**bad) == INV


def test_logprobs_of_no_rows_is_fine():
    assert logprobs(rows=0, x=None) == OK


def test_engine_logprobs_refuses_a_null_engine():
    assert E.lib().ylm_logprobs(None, 0, 0, 0, None, None, None, None) == INV


def test_kv8_struct_layout_matches_c(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [f for f, _ in E.KV8Cache._fields_]
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include "yalama_b200.h"\nint main(void) { printf("%zu", sizeof(ylm_kv8_cache));'
                   + "".join(f'printf(" %zu", offsetof(ylm_kv8_cache, {f}));' for f in fields) + "return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(E.KV8Cache)] + [getattr(E.KV8Cache, f).offset for f in fields]


@pytest.mark.parametrize("cap", [2 ** 30 + 1, 2 ** 31 - 4000, 2 ** 31 - 1])
def test_slots_whose_arithmetic_leaves_32_bits_are_refused(cap):
    """More slots than any device holds: block counts, splits and strides over the slots would pass 32 bits."""
    c, size = cache(cap=cap, hkv=1), ctypes.c_size_t()
    good = cache(k=11 * A, v=12 * A, k_scale=13 * A, v_scale=14 * A, hkv=1)
    assert store(c, slot=cap - 1) == INV
    assert attend(c, n=cap) == INV
    assert E.lib().ylm_k_kv8_attention_workspace(c, 4, 1, cap, 1, ctypes.byref(size)) == INV
    assert evict(src=c, dst=good, n=50) == INV
    far = [1 << 52, 1 << 53, 1 << 54, 1 << 55]  # so far apart that nothing overlaps
    big = cache(k=far[0], v=far[1], k_scale=far[2], v_scale=far[3], cap=cap, hkv=1)
    assert evict(src=good, dst=big, acc_dst=1 << 56, kept=1 << 57) == INV
    # the largest that is taken: refused for its slots only, so these reach the device (or its absence)
    c = cache(cap=2 ** 30, hkv=1)
    assert attend(c, n=2 ** 30 + 1) == INV
    assert E.lib().ylm_k_kv8_attention_workspace(c, 4, 1, 2 ** 30, 1, ctypes.byref(size)) != INV
