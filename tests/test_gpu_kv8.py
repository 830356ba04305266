"""The 8-bit key/value cache (vrt_kv8_*) against its definition in 64 bits (kv8_ref.py). What the cache holds and what eviction
keeps are compared bit for bit; attention with a bound derived there."""
import ctypes as C

import numpy as np
import pytest

import kv8_ref as R
import vrt

pytestmark = pytest.mark.gpu


def _values(seed, n, heads, hd):
    r = np.random.default_rng(seed)
    x = r.standard_normal((n, heads, hd)).astype(np.float32)
    x[:, :, 3::29] *= 4.0
    return x


def _same(a, b, what=""):
    a, b = np.asarray(a, np.float32), np.asarray(b, np.float32)
    assert a.shape == b.shape
    assert np.array_equal(np.isnan(a), np.isnan(b)), what
    ok = ~np.isnan(a)
    assert np.array_equal(a[ok], b[ok]), (what, np.argwhere(ok & (a != b))[:4])


def _append(ctx, c, rows, k, v, stride=0):
    kd, vd = ctx.upload(k), ctx.upload(v)
    c.append(rows, kd, vd, stride)
    ctx.sync()


def _read(ctx, c, seq, pos, n, length, kv, hd):
    k, v = ctx.alloc(max(1, n) * kv * hd * 4), ctx.alloc(max(1, n) * kv * hd * 4)
    c.read([(seq, pos, n, 0)], k, v, [length])
    ctx.sync()
    return [b.read(np.float32, n * kv * hd).reshape(n, kv, hd) for b in (k, v)]


def _attend(ctx, c, rows, q, heads, scale, **kw):
    qd, od = ctx.upload(q), ctx.upload(np.full(q.shape, -7.0, np.float32))
    c.attend(rows, qd, od, heads, scale, **kw)
    ctx.sync()
    return od.read(np.float32, q.size).reshape(q.shape)


def _check(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol) & ~(np.isnan(got) & np.isnan(want))
    assert not bad.any(), (what, np.argwhere(bad)[:4], float(np.nanmax(np.abs(got - want) / tol)))


# ---- what the cache holds --------------------------------------------------------------------

@pytest.mark.parametrize("kv,hd", [(1, 4), (3, 20), (1, 32), (2, 64), (2, 100), (1, 128), (1, 252), (1, 256)])
def test_append_and_read(ctx, kv, hd):
    """A sequence in pieces of 1, 30, 2, 31, 64, 5, 40 rows, another in one: the same bits, and the definition's."""
    lens = [1, 30, 2, 31, 64, 5, 40]
    n = sum(lens)
    k, v = _values(1, n, kv, hd), _values(2, n, kv, hd)
    c = vrt.Kv8Cache(ctx, 3, n, kv, hd)
    p = 0
    for m in lens:
        _append(ctx, c, [(2, p, m, 0)], k[p:p + m], v[p:p + m])
        p += m
    _append(ctx, c, [(0, 0, n, 0)], k, v)
    for seq in (2, 0):
        a, b = _read(ctx, c, seq, 0, n, n, kv, hd)
        _same(a, R.stored(k), f"keys of {seq}")
        _same(b, R.stored(v), f"values of {seq}")
    a, b = _read(ctx, c, 2, 37, 90, n, kv, hd)   # some positions in the middle
    _same(a, R.stored(k)[37:127])
    c.close()


def test_append_borders(ctx):
    """Quotients on and next to the border of two codes, blocks of zeros, of denormals, with an infinity, with a NaN in one head."""
    x = np.zeros((32 * 6, 2, 8), np.float32)
    r = np.random.default_rng(3)
    s = np.float32(0.03125)
    x[:32] = (r.integers(-126, 126, (32, 2, 8)) + 0.5).astype(np.float32) * s
    x[0] = 127 * s                                     # the scale is s: every quotient but these is a tie
    t = np.float32(1.7)
    x[32:64] = np.nextafter((r.integers(-126, 126, (32, 2, 8)) + 0.5).astype(np.float32) * t,
                            np.float32(np.inf) * r.choice([-1, 1], (32, 2, 8)).astype(np.float32))
    x[32] = 127 * t
    x[96:128] = r.standard_normal((32, 2, 8)) * 1e-40  # 64..95: zeros
    x[128:160] = r.standard_normal((32, 2, 8))
    x[130, 0, 3] = np.inf
    x[160:] = r.standard_normal((32, 2, 8))
    x[170, 1, 0] = np.nan
    c = vrt.Kv8Cache(ctx, 1, len(x), 2, 8)
    _append(ctx, c, [(0, 0, len(x), 0)], x, x)
    for got in _read(ctx, c, 0, 0, len(x), len(x), 2, 8):
        _same(got, R.stored(x))
    c.close()


def test_append_takes_back(ctx):
    """A sequence taken back inside its last block, inside the one before (no position two blocks on has been written
    since) and to a block's start, then on: as if it had never been longer."""
    kv, hd = 2, 36
    k = _values(4, 200, kv, hd)
    c = vrt.Kv8Cache(ctx, 1, 200, kv, hd)
    other = _values(5, 200, kv, hd)
    _append(ctx, c, [(0, 0, 100, 0)], k[:100], k[:100])
    k = k[:100]
    for back, m in ((98, 50), (130, 5), (99, 40), (64, 10), (70, 20), (68, 33), (90, 1), (32, 60), (60, 3)):
        new = other[back:back + m]
        _append(ctx, c, [(0, back, m, 0)], new, new)
        k = np.concatenate([k[:back], new])
        a, b = _read(ctx, c, 0, 0, back + m, back + m, kv, hd)
        _same(a, R.stored(k), f"back to {back}")
        _same(b, R.stored(k))
    c.close()


def test_many_sequences_strides_and_bystanders(ctx):
    """Rows inside wider ones, zero-length sequences between others; regions, rows and columns that are nobody's stay."""
    kv, hd, stride = 2, 24, 60
    lens = [0, 3, 33, 0, 64, 1]
    seqs = [5, 0, 6, 2, 4, 1]
    x = np.random.default_rng(6).standard_normal((sum(lens), stride)).astype(np.float32)
    c = vrt.Kv8Cache(ctx, 8, 64, kv, hd)
    keep = _values(7, 40, kv, hd)
    for s in (3, 7):
        _append(ctx, c, [(s, 0, 40, 0)], keep, keep)
    rows = [(s, 0, n, 0) for s, n in zip(seqs, lens)]
    _append(ctx, c, rows, x, x, stride)
    out = ctx.upload(np.full((sum(lens) + 1, stride), 9.0, np.float32))
    tmp = ctx.alloc(sum(lens) * stride * 4)
    c.read(rows, out, tmp, stride=stride)
    ctx.sync()
    got = out.read(np.float32, (sum(lens) + 1) * stride).reshape(-1, stride)
    p = 0
    for n in lens:
        _same(got[p:p + n, :kv * hd].reshape(n, kv, hd), R.stored(x[p:p + n, :kv * hd].reshape(n, kv, hd)))
        p += n
    assert np.all(got[:, kv * hd:] == 9.0) and np.all(got[-1] == 9.0)
    for s in (3, 7):
        _same(_read(ctx, c, s, 0, 40, 40, kv, hd)[0], R.stored(keep))
    c.close()


# ---- attention ------------------------------------------------------------------------------

CASES = [
    # heads, kv, hd, [(len, n)], window, cap, prefix
    (1, 1, 4, [(1, 1)], 0, 0.0, 0),
    (4, 1, 64, [(33, 1), (1, 1), (32, 1), (31, 1), (64, 1), (700, 1)], 0, 0.0, 0),
    (4, 1, 256, [(129, 1), (1000, 1)], 0, 0.0, 0),
    (8, 2, 96, [(257, 1), (90, 1), (600, 1)], 64, 0.0, 0),
    (8, 2, 100, [(257, 1), (90, 1), (600, 1)], 50, 30.0, 7),
    (48, 2, 32, [(40, 1), (300, 1)], 0, 0.0, 0),                # 24 heads a group: two row tiles
    (6, 2, 128, [(77, 5), (40, 3), (900, 4)], 0, 50.0, 0),      # a few new positions each
    (4, 1, 128, [(300, 300)], 0, 0.0, 0),                       # a prompt
    (4, 1, 256, [(200, 137)], 0, 0.0, 0),
    (2, 2, 80, [(333, 333), (65, 65), (2, 2)], 40, 0.0, 0),
    (4, 2, 64, [(400, 400)], 0, 0.0, 150),                      # a prefix that sees itself
    (4, 2, 64, [(400, 100), (320, 320)], 33, 20.0, 70),         # a prefix and a window
    (3, 1, 160, [(250, 250)], 1, 0.0, 0),                       # each position sees itself alone
    (2, 1, 192, [(97, 60)], 0, 0.0, 1000),                      # all see all
    (5, 5, 224, [(130, 40)], 100, 0.0, 3),
    (16, 2, 64, [(1200, 515)], 0, 30.0, 0),
    (8, 4, 32, [(1050, 40), (600, 600), (33, 33), (1056, 70), (900, 20)], 0, 0.0, 0),   # 660 blocks' weights
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_attend(ctx, case):
    heads, kv, hd, seqs, window, cap, prefix = CASES[case]
    scale = float(np.float32(1.0 / np.sqrt(hd)))
    n_seq, top = len(seqs), max(n for n, _ in seqs)
    c = vrt.Kv8Cache(ctx, n_seq + 1, top, kv, hd)
    ks = [_values(10 * i + 1, n, kv, hd) for i, (n, _) in enumerate(seqs)]
    vs = [_values(10 * i + 2, n, kv, hd) for i, (n, _) in enumerate(seqs)]
    q = (np.random.default_rng(case).standard_normal((sum(m for _, m in seqs), heads, hd)) * 1.5).astype(np.float32)
    reg = [(i + 1) % (n_seq + 1) for i in range(n_seq)]   # regions in another order than the call's
    for i, (n, _) in enumerate(seqs):
        _append(ctx, c, [(reg[i], 0, n, 0)], ks[i], vs[i])
    rows = [(reg[i], n - m, m, prefix) for i, (n, m) in enumerate(seqs)]
    w0 = np.random.default_rng(99).random((n_seq + 1, kv, top)).astype(np.float32)
    wd, wo = ctx.upload(w0), ctx.upload(np.full(w0.shape, 5.0, np.float32))
    got = _attend(ctx, c, rows, q, heads, scale, softcap=cap, window=window)
    got2 = _attend(ctx, c, rows, q, heads, scale, softcap=cap, window=window, weights_in=wd, weights_out=wo)
    assert np.array_equal(got, got2), "with weights the outputs are the same"
    w = wo.read(np.float32, w0.size).reshape(w0.shape)
    p = 0
    for i, (n, m) in enumerate(seqs):
        want, ww, tol = R.attend(q[p:p + m], R.stored(ks[i]), R.stored(vs[i]), n - m, scale, cap, window, prefix)
        _check(got[p:p + m], want, tol, f"sequence {i}")
        base = w0[reg[i], :, :n].astype(np.float64)
        base[:, n - m:] = 0.0
        # a sum of m heads' weights: each off by the factor 1 + 2 ds, the sum's roundings
        rel = 2 * float(tol.max()) / max(1e-9, float(np.abs(R.stored(vs[i])).max()))
        _check(w[reg[i], :, :n], base + ww, (base + ww) * (rel + 2.0 ** -20) + 1e-30, f"weights of sequence {i}")
        assert np.all(w[reg[i], :, n:] == 5.0), "entries past the length stay"
        p += m
    assert np.all(w[[r for r in range(n_seq + 1) if r not in reg]] == 5.0), "other regions' weights stay"
    c.close()


def test_weights_in_place_and_from_nothing(ctx):
    kv, hd, heads = 2, 64, 4
    k, v = _values(1, 90, kv, hd), _values(2, 90, kv, hd)
    q = _values(3, 1, heads, hd)
    c = vrt.Kv8Cache(ctx, 1, 96, kv, hd)
    _append(ctx, c, [(0, 0, 90, 0)], k, v)
    w0 = np.random.default_rng(4).random((1, kv, 96)).astype(np.float32)
    a, b, z = ctx.upload(w0), ctx.upload(w0), ctx.upload(w0)
    _attend(ctx, c, [(0, 89, 1, 0)], q, heads, 0.125, weights_in=a, weights_out=a)
    _attend(ctx, c, [(0, 89, 1, 0)], q, heads, 0.125, weights_in=ctx.upload(w0), weights_out=b)
    _attend(ctx, c, [(0, 89, 1, 0)], q, heads, 0.125, weights_out=z)
    A, B, Z = (x.read(np.float32, w0.size).reshape(w0.shape) for x in (a, b, z))
    assert np.array_equal(A, B)
    assert np.array_equal(A[:, :, 90:], w0[:, :, 90:])
    assert np.allclose(Z[:, :, :90].sum(axis=2), heads / kv, rtol=1e-5)   # every row's weights sum to 1
    c.close()


@pytest.mark.parametrize("window,hd", [(64, 32), (50, 64), (96, 256)])
def test_ring(ctx, window, hd):
    """Far past the capacity, one position at a time and several, in a region of the window's blocks."""
    kv, heads = 1, 3
    cap = (window + 31) // 32 * 32
    n = 400
    k, v = _values(1, n, kv, hd), _values(2, n, kv, hd)
    q = _values(3, n, heads, hd)
    c = vrt.Kv8Cache(ctx, 2, cap, kv, hd)
    p = 0
    for i, m in enumerate([1, 31, 1, 30] + [1] * 100 + [32] * 4 + [1] * 40):
        _append(ctx, c, [(1, p, m, 0)], k[p:p + m], v[p:p + m])
        if m == 1:
            got = _attend(ctx, c, [(1, p, 1, 0)], q[p:p + 1], heads, 0.2, window=window)
            # the blocks of this length, and the open one in fp32
            want, _, tol = R.attend(q[p:p + 1], R.stored(k[:p + 1]), R.stored(v[:p + 1]), p, 0.2, 0.0, window, 0)
            _check(got, want, tol, f"position {p}")
        p += m
    c.close()


def test_magnitudes(ctx):
    """Blocks of very different scales, values and queries far from 1: what the halves' range could lose."""
    kv, heads, hd, n = 1, 2, 64, 300
    k, v = _values(1, n, kv, hd), _values(2, n, kv, hd)
    q = _values(3, 1, heads, hd)
    for ksc, vsc, qsc in [(1e-6, 1e-20, 1e6), (1e6, 1e20, 1e-6), (1e-18, 1.0, 1e18), (1.0, 1e-37, 1.0), (1e15, 3e30, 1e-15)]:
        steps = np.float32(10.0) ** (np.arange(n) // 32 % 4 * -2.0)     # blocks from 1 to 1e-6
        kk, vv = (k * np.float32(ksc)), (v * np.float32(vsc) * steps[:, None, None]).astype(np.float32)
        qq = (q * np.float32(qsc)).astype(np.float32)
        c = vrt.Kv8Cache(ctx, 1, n, kv, hd)
        _append(ctx, c, [(0, 0, n, 0)], kk, vv)
        got = _attend(ctx, c, [(0, n - 1, 1, 0)], qq, heads, 0.125)
        want, _, tol = R.attend(qq, R.stored(kk), R.stored(vv), n - 1, 0.125)
        _check(got, want, tol, (ksc, vsc, qsc))
        # and where the largest block's weights are next to nothing: a key that all but the first block's positions like
        kk = k.copy()
        kk[32:] += 6.0
        vv = v.copy()
        vv[:32] *= 1e4
        c2 = vrt.Kv8Cache(ctx, 1, n, kv, hd)
        _append(ctx, c2, [(0, 0, n, 0)], kk, vv)
        qp = np.abs(q)
        got = _attend(ctx, c2, [(0, n - 1, 1, 0)], qp, heads, 0.125)
        want, _, tol = R.attend(qp, R.stored(kk), R.stored(vv), n - 1, 0.125)
        _check(got, want, tol)
        c.close()
        c2.close()


def test_large_scores(ctx):
    """Scores of hundreds: one position takes all; capped ones stay apart."""
    kv, heads, hd, n = 1, 4, 128, 200
    k, v, q = _values(1, n, kv, hd), _values(2, n, kv, hd), _values(3, 2, heads, hd) * 20
    c = vrt.Kv8Cache(ctx, 1, n, kv, hd)
    _append(ctx, c, [(0, 0, n, 0)], k, v)
    for cap in (0.0, 15.0):
        got = _attend(ctx, c, [(0, n - 2, 2, 0)], q, heads, 0.5, softcap=cap)
        want, _, tol = R.attend(q, R.stored(k), R.stored(v), n - 2, 0.5, cap)
        _check(got, want, tol, cap)
    c.close()


@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_not_finite(ctx, where, what):
    """A key or value that is not finite: NaN for the queries that see it (a full block's: any of the block), nothing for
    the others, rows of the same tile among them."""
    kv, heads, hd, n, m = 2, 4, 64, 110, 110
    k, v, q = _values(1, n, kv, hd), _values(2, n, kv, hd), _values(3, m, heads, hd)
    (k if where == "key" else v)[103, 1, 5] = what     # in the open block (96..109)
    (k if where == "key" else v)[40, 0, 2] = what      # in a full block (32..63)
    for window in (0, 5):
        c = vrt.Kv8Cache(ctx, 1, n, kv, hd)
        _append(ctx, c, [(0, 0, n, 0)], k, v)
        got = _attend(ctx, c, [(0, 0, n, 0)], q, heads, 0.125, window=window)
        see = R.visible(0, n, window, 0)
        ks, vs = R.stored(k), R.stored(v)
        fk, fv = np.where(np.isfinite(ks), ks, 0), np.where(np.isfinite(vs), vs, 0)
        want, _, tol = R.attend(q, fk, fv, 0, 0.125, 0.0, window)
        want[np.ix_(see[:, 32:64].any(axis=1), [0, 1])] = np.nan
        want[np.ix_(see[:, 103], [2, 3])] = np.nan
        _check(got, want, tol, window)
        c.close()


def test_stale_rows_are_not_seen(ctx):
    """A sequence started again after one whose last rows held NaN."""
    kv, heads, hd = 1, 2, 32
    c = vrt.Kv8Cache(ctx, 1, 64, kv, hd)
    bad = np.full((50, kv, hd), np.nan, np.float32)
    _append(ctx, c, [(0, 0, 50, 0)], bad, bad)
    k, v, q = _values(1, 40, kv, hd), _values(2, 40, kv, hd), _values(3, 1, heads, hd)
    for n in (1, 5, 33, 40):
        _append(ctx, c, [(0, 0, n, 0)], k[:n], v[:n])
        got = _attend(ctx, c, [(0, n - 1, 1, 0)], q, heads, 0.2)
        want, _, tol = R.attend(q, R.stored(k[:n]), R.stored(v[:n]), n - 1, 0.2)
        _check(got, want, tol, n)
    c.close()


def test_attend_strides_and_rows_behind(ctx):
    kv, heads, hd, n = 1, 3, 20, 70
    k, v = _values(1, n, kv, hd), _values(2, n, kv, hd)
    c = vrt.Kv8Cache(ctx, 2, n, kv, hd)
    for s in (0, 1):
        _append(ctx, c, [(s, 0, n, 0)], k, v)
    qs, os = 72, 64
    q = np.random.default_rng(5).standard_normal((9, qs)).astype(np.float32)
    qd, od = ctx.upload(q), ctx.upload(np.full((9, os), 3.0, np.float32))
    rows = [(1, n - 4, 4, 0), (0, n, 0, 0)]
    c.attend(rows, qd, od, heads, 0.2, q_stride=qs, out_stride=os)
    ctx.sync()
    got = od.read(np.float32, 9 * os).reshape(9, os)
    want, _, tol = R.attend(q[:4, :60].reshape(4, heads, hd), R.stored(k), R.stored(v), n - 4, 0.2)
    _check(got[:4, :60].reshape(4, heads, hd), want, tol)
    assert np.all(got[4:] == 3.0) and np.all(got[:, 60:] == 3.0)
    c.close()


# ---- eviction -------------------------------------------------------------------------------

def _evict(ctx, kv, hd, lens, keeps, recents, weights, seed=0):
    n = len(lens)
    top = max(lens)
    c = vrt.Kv8Cache(ctx, 2 * n, top, kv, hd)
    ks = [_values(seed + 3 * i, m, kv, hd) for i, m in enumerate(lens)]
    vs = [_values(seed + 3 * i + 1, m, kv, hd) for i, m in enumerate(lens)]
    w = np.full((2 * n, kv, top), 5.0, np.float32)
    for i, m in enumerate(lens):
        w[2 * i, :, :m] = weights[i]
        if m:
            _append(ctx, c, [(2 * i, 0, m, 0)], ks[i], vs[i])
    wd = ctx.upload(w)
    stride = max(1, max(keeps)) + 3
    kd = ctx.upload(np.full((n, kv, stride), 77, np.uint32))
    c.evict([(2 * i, 2 * i + 1, lens[i], keeps[i], recents[i]) for i in range(n)], wd, kd, stride)
    ctx.sync()
    wn = wd.read(np.float32, w.size).reshape(w.shape)
    kept = kd.read(np.uint32, n * kv * stride).reshape(n, kv, stride)
    for i, m in enumerate(lens):
        for h in range(kv):
            want = R.keep_rule(w[2 * i, h, :m], keeps[i], recents[i])
            assert np.array_equal(kept[i, h, :keeps[i]], want), (i, h)
            assert np.array_equal(wn[2 * i + 1, h, :keeps[i]], w[2 * i, h][want], equal_nan=True)
        assert np.all(kept[i, :, keeps[i]:] == 77) and np.all(wn[2 * i + 1, :, keeps[i]:] == 5.0)
        if keeps[i] == 0:
            continue
        for x, got in zip((ks[i], vs[i]), _read(ctx, c, 2 * i + 1, 0, keeps[i], keeps[i], kv, hd)):
            y = R.stored(x)
            y = np.stack([y[kept[i, h, :keeps[i]], h] for h in range(kv)], axis=1)
            _same(got, R.stored(y), f"move {i}")
    assert np.array_equal(wn[::2], w[::2], equal_nan=True), "the sources' weights stay"
    return c, ks, vs, kept


@pytest.mark.parametrize("kv,hd", [(1, 64), (2, 20), (3, 256)])
def test_evict(ctx, kv, hd):
    """Random weights, ties, all equal, none kept, all kept, the recent alone, a single position."""
    r = np.random.default_rng(kv)
    lens = [300, 257, 64, 100, 90, 33, 1, 2500]
    keeps = [100, 200, 32, 0, 90, 7, 1, 1111]
    recents = [10, 0, 5, 0, 3, 7, 0, 100]
    ws = [r.random((kv, m)).astype(np.float32) ** 8 for m in lens]
    ws[1] = r.integers(0, 4, (kv, lens[1])).astype(np.float32)   # ties
    ws[2][:] = 0.25
    c, *_ = _evict(ctx, kv, hd, lens, keeps, recents, ws)
    c.close()


def test_evict_odd_weights(ctx):
    """Negative ones, both zeros (equal), infinities, NaN (never preferred), more NaN than may go."""
    w = np.array([[np.nan, -1, 0.0, -0.0, np.inf, -np.inf, 3, np.nan, 0.0, -0.0, 1e-40, -1e-40] * 5], np.float32)
    n = w.shape[1]
    for keep in (1, 5, 14, 24, 30, 51, 52, 58, n):
        c, *_ = _evict(ctx, 1, 8, [n], [keep], [min(keep, 1)], [w])
        c.close()


def test_together(ctx):
    """As a service runs them: prompt, steps with weights, eviction, steps on the shorter sequence, against 64 bits all along."""
    kv, heads, hd, ctx_len = 2, 6, 64, 160
    scale = 0.125
    c = vrt.Kv8Cache(ctx, 3, ctx_len, kv, hd)
    wd = ctx.alloc(3 * kv * ctx_len * 4)
    n0, steps = 120, 30
    k, v = _values(1, n0 + 2 * steps, kv, hd), _values(2, n0 + 2 * steps, kv, hd)
    q = _values(3, n0 + 2 * steps, heads, hd)
    weights = np.zeros((kv, ctx_len))

    def run(seq, pos, at, n, ks, vs):
        _append(ctx, c, [(seq, pos, n, 0)], k[at:at + n], v[at:at + n])
        got = _attend(ctx, c, [(seq, pos, n, 0)], q[at:at + n], heads, scale, weights_in=wd, weights_out=wd)
        ks, vs = np.concatenate([ks, k[at:at + n]]), np.concatenate([vs, v[at:at + n]])
        want, w, tol = R.attend(q[at:at + n], R.stored(ks), R.stored(vs), pos, scale)
        _check(got, want, tol, (seq, pos))
        weights[:, pos:pos + n] = 0.0
        weights[:, :pos + n] += w
        return ks, vs

    ks = vs = np.zeros((0, kv, hd), np.float32)
    ks, vs = run(1, 0, 0, n0, ks, vs)
    for i in range(steps):
        ks, vs = run(1, n0 + i, n0 + i, 1, ks, vs)
    n = n0 + steps
    kd = ctx.alloc(kv * 70 * 4)
    c.evict([(1, 2, n, 70, 16)], wd, kd, 70)
    ctx.sync()
    kept = kd.read(np.uint32, kv * 70).reshape(kv, 70)
    w = wd.read(np.float32, 3 * kv * ctx_len).reshape(3, kv, ctx_len)
    assert np.allclose(w[1, :, :n], weights[:, :n], rtol=1e-4, atol=1e-6)
    for h in range(kv):
        assert np.array_equal(kept[h], R.keep_rule(w[1, h, :n], 70, 16))
    # the shorter sequence starts from what the cache stands for
    ks = np.stack([R.stored(ks)[kept[h], h] for h in range(kv)], axis=1)
    vs = np.stack([R.stored(vs)[kept[h], h] for h in range(kv)], axis=1)
    weights[:, :70] = w[2, :, :70]
    for i in range(steps):
        ks, vs = run(2, 70 + i, n + i, 1, ks, vs)
    c.close()


# ---- memory, streams, graphs -----------------------------------------------------------------

def test_offsets_past_32_bits(ctx):
    """A region that starts 4.3 GB into the cache."""
    kv, hd, n = 8, 256, 70
    c = vrt.Kv8Cache(ctx, 2, 1 << 20, kv, hd)
    assert c.desc.bytes > (1 << 33)
    k, v, q = _values(1, n, kv, hd), _values(2, n, kv, hd), _values(3, 1, kv, hd)
    _append(ctx, c, [(1, 0, n, 0)], k, v)
    _same(_read(ctx, c, 1, 0, n, n, kv, hd)[1], R.stored(v))
    got = _attend(ctx, c, [(1, n - 1, 1, 0)], q, kv, 0.0625)
    want, _, tol = R.attend(q, R.stored(k), R.stored(v), n - 1, 0.0625)
    _check(got, want, tol)
    c.close()


def test_two_contexts(ctx):
    """Two contexts' streams on two caches at once: each its own results."""
    other = vrt.Context("")
    kv, heads, hd, n = 2, 8, 128, 2000
    jobs = []
    for i, x in enumerate((ctx, other)):
        c = vrt.Kv8Cache(x, 1, n, kv, hd)
        k, v, q = _values(10 + i, n, kv, hd), _values(20 + i, n, kv, hd), _values(30 + i, 1, heads, hd)
        kd, vd, qd, od = x.upload(k), x.upload(v), x.upload(q), x.alloc(q.nbytes)
        c.append([(0, 0, n, 0)], kd, vd)
        jobs.append((x, c, k, v, q, qd, od, (kd, vd)))
    for _ in range(20):
        for x, c, k, v, q, qd, od, _keep in jobs:
            c.attend([(0, n - 1, 1, 0)], qd, od, heads, 0.1)
    for x, c, k, v, q, qd, od, _keep in jobs:
        x.sync()
        want, _, tol = R.attend(q, R.stored(k), R.stored(v), n - 1, 0.1)
        _check(od.read(np.float32, q.size).reshape(q.shape), want, tol)
        c.close()
    other.close()


def _hip():
    """The HIP runtime that libvrt_hip.so runs on."""
    vrt.lib()
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libamdhip64.so" in line)
    return C.CDLL(path)


def test_captured_and_replayed(ctx):
    """append, attend with weights and eviction in a graph, replayed over new inputs, with eager calls between the replays."""
    hip = _hip()
    kv, heads, hd, n = 1, 4, 64, 600
    c = vrt.Kv8Cache(ctx, 3, n + 1, kv, hd)
    k, v = _values(1, n, kv, hd), _values(2, n, kv, hd)
    _append(ctx, c, [(0, 0, n, 0)], k, v)
    s = C.c_void_p()
    vrt.check(vrt.lib().vrt_stream(ctx.h, C.byref(s)))
    kd, vd, qd = (ctx.alloc(x * hd * 4) for x in (kv, kv, heads))
    od, wi, wo, kept = ctx.alloc(heads * hd * 4), ctx.upload(np.zeros((3, kv, n + 1), np.float32)), ctx.alloc(3 * kv * (n + 1) * 4), ctx.alloc(800)
    ws = ctx.alloc(c.workspace_bytes([(0, n, 1, 0)], heads, 0.125, scored=True))

    def calls():
        c.append([(0, n, 1, 0)], kd, vd)
        c.attend([(0, n, 1, 0)], qd, od, heads, 0.125, weights_in=wi, weights_out=wo, workspace=ws)
        c.evict([(0, 1, n + 1, 200, 20)], wo, kept, 200)

    def results():
        ctx.sync()
        return (od.read(np.float32, heads * hd), wo.read(np.float32, 2 * kv * (n + 1)), kept.read(np.uint32, 200),
                *_read(ctx, c, 1, 0, 200, 200, kv, hd))

    graph, run = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(s, 2) == 0    # hipStreamCaptureModeRelaxed
    calls()
    assert hip.hipStreamEndCapture(s, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for i in range(4):
        x = [_values(50 + 3 * i + j, 1, m, hd) for j, m in enumerate((kv, kv, heads))]
        for d, a in zip((kd, vd, qd), x):
            d.write(a)
        assert hip.hipGraphLaunch(run, s) == 0
        got = results()
        wo.write(np.zeros(2 * kv * (n + 1), np.float32))
        calls()
        for a, b in zip(got, results()):
            assert np.array_equal(a, b), f"replay {i}"
        want, _, tol = R.attend(x[2], R.stored(np.concatenate([k, x[0]])), R.stored(np.concatenate([v, x[1]])), n, 0.125)
        _check(got[0].reshape(1, heads, hd), want, tol)
        _append(ctx, c, [(2, 0, 40, 0)], k[:40], v[:40])   # other work between the replays
    hip.hipGraphExecDestroy(run)
    hip.hipGraphDestroy(graph)
    c.close()
