"""What the 8-bit key/value cache's entry points refuse, before any launch (no device is touched: the context is a blank
block of memory that a refused call never looks into)."""
import ctypes as C

import numpy as np
import pytest

import vrt

_blank = C.create_string_buffer(4096)
CTX = C.addressof(_blank)
A = 1 << 20          # an aligned address nobody reads
ROW = [(0, 0, 5, 0)]


def _cache(**kw):
    d = dict(data=A, bytes=1 << 40, max_seqs=4, max_ctx=96, kv_heads=2, head_dim=64)
    d.update(kw)
    return vrt.Kv8CacheDesc(*[d[n] for n, _ in vrt.Kv8CacheDesc._fields_])


def _rows(r, width=4):
    return np.asarray(r, dtype=np.uint32).reshape(-1, width)


def _refused(rc, match):
    assert rc == vrt.VRT_ERR_INVALID, (rc, vrt.lib().vrt_last_error())
    assert match in vrt.lib().vrt_last_error().decode(), vrt.lib().vrt_last_error()


def _append(cache=None, rows=ROW, ctx=CTX, k=A, v=A, stride=0, n=None):
    r = _rows(rows)
    return vrt.lib().vrt_kv8_append(ctx, C.byref(cache or _cache()), vrt.ptr(r), len(r) if n is None else n, k, v, stride)


def _attend(cache=None, rows=ROW, q=A, out=A, heads=4, window=0, scale=1.0, cap=0.0, win=None, wout=None, ws=A, nws=1 << 40,
            qs=0, os=0):
    r = _rows(rows)
    at = vrt.Kv8Attn(heads, window, scale, cap)
    return vrt.lib().vrt_kv8_attend(CTX, C.byref(cache or _cache()), C.byref(at), vrt.ptr(r), len(r), q, qs, out, os, win, wout, ws,
                                    nws)


def _evict(moves, cache=None, w=A, kept=A, stride=96):
    m = _rows(moves, 5)
    return vrt.lib().vrt_kv8_evict(CTX, C.byref(cache or _cache()), vrt.ptr(m), len(m), w, kept, stride)


@pytest.mark.parametrize("kw,match", [
    (dict(max_seqs=0), "max_seqs"), (dict(max_seqs=65536), "max_seqs"), (dict(max_ctx=0), "max_ctx"),
    (dict(max_ctx=(1 << 26) + 1), "max_ctx"), (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=1025), "kv_heads"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=30), "head_dim"), (dict(head_dim=260), "head_dim")])
def test_cache_sizes(kw, match):
    n = C.c_uint64()
    _refused(vrt.lib().vrt_kv8_cache_bytes(C.byref(_cache(**kw)), C.byref(n)), match)
    _refused(_append(cache=_cache(**kw)), match)
    _refused(_attend(cache=_cache(**kw)), match)


def test_cache_bytes():
    """Two regions, three heads, 70 positions (3 blocks), 40 dims in 64: codes, scales, two blocks' rows in fp32, in pairs of
    halves, and the rows' factors."""
    n = C.c_uint64()
    vrt.check(vrt.lib().vrt_kv8_cache_bytes(C.byref(_cache(max_seqs=2, kv_heads=3, max_ctx=70, head_dim=40)), C.byref(n)))
    up = lambda x: (x + 255) // 256 * 256  # noqa: E731
    assert n.value == up(2 * 3 * 3 * 64 * 64) + up(2 * 3 * 3 * 8) + up(2 * 3 * 128 * 64 * 4) + up(2 * 3 * 128 * 64 * 4) + up(2 * 3 * 128 * 4)


def test_cache_memory():
    n = C.c_uint64()
    vrt.check(vrt.lib().vrt_kv8_cache_bytes(C.byref(_cache()), C.byref(n)))
    _refused(_append(cache=_cache(bytes=n.value - 1)), "too small")
    _refused(_append(cache=_cache(data=None)), "aligned")
    _refused(_append(cache=_cache(data=A + 128)), "aligned")
    _refused(_attend(cache=_cache(data=None)), "aligned")
    _refused(_evict([(0, 1, 5, 3, 1)], cache=_cache(data=None)), "aligned")


@pytest.mark.parametrize("call", [_append, _attend])
def test_rows(call):
    _refused(call(rows=[(4, 0, 1, 0)]), "out of range")
    _refused(call(rows=[(1, 0, 1, 0), (2, 0, 1, 0), (1, 8, 1, 0)]), "twice")
    _refused(call(rows=[(0, 1 << 26, 1, 0)]), "positions past")
    _refused(call(rows=[(0, 5, 0xffffffff, 0)]), "positions past")
    _refused(call(rows=np.zeros((0, 4))), "n_seqs")
    _refused(call(rows=[(i, 0, 1, 0) for i in range(65)], cache=_cache(max_seqs=100)), "n_seqs")


def test_append_arguments():
    _refused(_append(ctx=None), "null context")
    _refused(_append(k=None), "k must be")
    _refused(_append(v=A + 4), "v must be")
    _refused(_append(stride=64), "row stride")        # narrower than a row of 2 heads of 64
    _refused(_append(stride=130), "row stride")
    _refused(_append(rows=[(0, 31, 66, 0)]), "more blocks")   # 31 .. 96: four blocks, a region of three
    _refused(_append(rows=[(0, 0, 97, 0)]), "more blocks")


def test_attend_arguments():
    _refused(_attend(heads=3), "heads")
    _refused(_attend(heads=0), "heads")
    _refused(_attend(scale=float("nan")), "scale")
    _refused(_attend(cap=-1.0), "softcap")
    _refused(_attend(cap=float("inf")), "softcap")
    _refused(_attend(q=A + 8), "q must be")
    _refused(_attend(out=None), "out must be")
    _refused(_attend(qs=252), "row stride")
    _refused(_attend(os=258), "row stride")
    _refused(_attend(win=A), "weights_in without")
    _refused(_attend(wout=A + 2), "weights must be")
    # what a ring has overwritten: 128 positions in blocks of a region of 96, from its first position or within a window
    _refused(_attend(rows=[(0, 127, 1, 0)]), "no longer holds position 0")
    _refused(_attend(rows=[(0, 127, 1, 0)], window=98), "no longer holds position 30")
    _refused(_attend(rows=[(0, 127, 1, 3)], window=10), "no longer holds position 0")
    _refused(_attend(rows=[(0, 100, 5, 0)], window=64, wout=A), "weights need")
    # a workspace that is short, missing or not aligned
    r, n = _rows([(0, 95, 1, 0), (1, 95, 1, 0)]), C.c_uint64()
    at = vrt.Kv8Attn(4, 0, 1.0, 0.0)
    vrt.check(vrt.lib().vrt_kv8_attend_workspace(C.byref(_cache()), C.byref(at), vrt.ptr(r), 2, 1, C.byref(n)))
    assert n.value > 0
    _refused(_attend(rows=r, wout=A, nws=n.value - 1), "workspace")
    _refused(_attend(rows=r, wout=A, ws=None), "workspace")
    _refused(_attend(rows=r, wout=A, ws=A + 64), "workspace")


def test_attend_softcap_has_a_reciprocal():
    _refused(_attend(cap=1e-40), "softcap")
    _refused(_attend(cap=9e-7), "softcap")


def test_attend_grid():
    """Every sequence of a call has as many workgroups as its longest: 64 rows of a head each, fewer than 2^24 in all."""
    big, n = _cache(max_seqs=64, max_ctx=1 << 26), C.c_uint64()
    at = vrt.Kv8Attn(4, 0, 1.0, 0.0)
    rows = lambda m: _rows([(i, 0, m if i == 0 else 0, 0) for i in range(64)])  # noqa: E731
    r = rows(1 << 22)    # 2 heads of 2^17 units, 64 times
    _refused(vrt.lib().vrt_kv8_attend_workspace(C.byref(big), C.byref(at), vrt.ptr(r), 64, 0, C.byref(n)), "too many rows")
    r = rows((1 << 22) - 64)
    vrt.check(vrt.lib().vrt_kv8_attend_workspace(C.byref(big), C.byref(at), vrt.ptr(r), 64, 0, C.byref(n)))
    r = rows(1 << 22)
    vrt.check(vrt.lib().vrt_kv8_attend_workspace(C.byref(big), C.byref(at), vrt.ptr(r), 1, 0, C.byref(n)))


def test_read_arguments():
    def read(rows, lens=None, cache=None, k=A):
        r = _rows(rows)
        n = None if lens is None else np.asarray(lens, dtype=np.uint32)
        return vrt.lib().vrt_kv8_read(CTX, C.byref(cache or _cache()), vrt.ptr(r), len(r), vrt.ptr(n), k, A, 0)
    _refused(read([(0, 0, 5, 0)], [4]), "past its length")
    _refused(read([(0, 0, 5, 0)], [128]), "no longer holds")
    _refused(read([(0, 0, 5, 0)], k=None), "k must be")


def test_evict_arguments():
    _refused(_evict([(0, 4, 5, 3, 1)]), "out of range")
    _refused(_evict([(4, 0, 5, 3, 1)]), "out of range")
    _refused(_evict([(0, 1, 5, 6, 1)]), "recent <= keep")
    _refused(_evict([(0, 1, 5, 3, 4)]), "recent <= keep")
    _refused(_evict([(0, 1, 97, 3, 1)]), "recent <= keep")
    _refused(_evict([(1, 1, 5, 3, 1)]), "source and a destination")
    _refused(_evict([(0, 1, 5, 3, 1), (1, 2, 5, 3, 1)]), "source and a destination")
    _refused(_evict([(0, 2, 5, 3, 1), (1, 2, 5, 3, 1)]), "destination twice")
    _refused(_evict([(0, 1, 5, 3, 1)], stride=2), "kept_stride")
    _refused(_evict([(0, 1, 5, 3, 1)], w=None), "null")
    _refused(_evict([(0, 1, 5, 3, 1)], kept=A + 1), "aligned")
    _refused(_evict([(i, 70 + i, 5, 3, 1) for i in range(65)], cache=_cache(max_seqs=200)), "n must be")
