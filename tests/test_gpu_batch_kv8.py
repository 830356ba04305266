"""Batched decode over 8-bit caches (vrt_g3_batch_create_kv8) and its eviction, against the 64-bit model over the same caches
(model64.py). Logits: the batch's own bound (1e-3 of max|logit|, test_gpu_batch.py), and as much again: a key or value that
the fp32 path has a few 1e-6 off its 64-bit value may lie on the other side of a code's border. One code is 1/127 of its block's
largest entry, at most 0.03 of an entry's usual size; it moves one of 64 products of a score by that, a score by 0.125 x 0.03
x |q| < 0.01, or one of an output's values by 0.03 times its weight."""
import numpy as np
import pytest

import model64
import synth
import vrt

pytestmark = pytest.mark.gpu
TOL = 2e-3


def _rel(a, b):
    return float(np.max(np.abs(a.astype(np.float64) - b)) / np.max(np.abs(b)))


def test_batch_kv8_tiny(ctx, tiny_model):
    """Four sequences that join at different steps, past two windows' rings and three blocks of the global cache."""
    g = vrt.Gemma3(ctx, tiny_model)
    b = vrt.Gemma3Batch(g, 5, 128, kv="i8")
    ids = [synth.uniform_ids(700 + i, 110, 2, 1000) for i in range(4)]
    ms = [model64.Model64(tiny_model) for _ in range(4)]
    starts, lens = [0, 1, 5, 40], [110, 70, 33, 32]
    slots = [4, 0, 2, 1]
    for step in range(110):
        rows = [i for i in range(4) if starts[i] <= step < starts[i] + lens[i]]
        if not rows:
            continue
        toks = [int(ids[i][step - starts[i]]) for i in rows]
        idx, val = b.step([slots[i] for i in rows], toks)
        for r, i in enumerate(rows):
            want = ms[i].step(toks[r])
            if step % 5 == 0 or step - starts[i] in (31, 32, 63, 64):
                assert _rel(b.logits(r), want) <= TOL, (i, step)
            assert abs(float(val[r]) - want.max()) <= TOL * np.abs(want).max()
            assert b.position(slots[i]) == b.length(slots[i]) == ms[i].pos
    b.close()
    g.close()


@pytest.mark.parametrize("window", [True, False])
def test_batch_evicts(ctx, tiny_model, tiny_model_nowindow, window):
    """Caches of 48 entries cut to 20 (5 recent) whenever they are full, to odd numbers too; another sequence in the step is not
    touched; positions go on."""
    path = tiny_model if window else tiny_model_nowindow
    g = vrt.Gemma3(ctx, path)
    b = vrt.Gemma3Batch(g, 2, 48, kv="i8", evict=True)
    m, other = model64.Model64(path), model64.Model64(path)
    ids = synth.uniform_ids(800, 130, 2, 1000)
    cuts = [(20, 5), (33, 0), (48, 3), (7, 7)]
    for p in range(130):
        if b.length(0) == 48:
            with pytest.raises(vrt.VrtError, match="context length"):
                b.step([0], [5])
            keep, recent = cuts.pop(0) if cuts else (20, 5)
            b.evict(0, keep, recent)
            m.evict(keep, recent)
            assert b.length(0) == keep and b.position(0) == p
            if keep == 48:   # all stay: now for real
                b.evict(0, 21, 4)
                m.evict(21, 4)
        both = p < 40
        t = int(ids[p])
        b.step([0, 1] if both else [0], [t, t] if both else [t])
        want = m.step(t)
        if both:
            assert _rel(b.logits(1), other.step(t)) <= TOL, p
        assert _rel(b.logits(0), want) <= TOL, p
    assert b.position(0) == 130 and b.length(1) == b.position(1) == 40
    b.reset(0)
    assert b.length(0) == 0
    m.reset()
    b.step([0], [9])
    assert _rel(b.logits(0), m.step(9)) <= TOL
    b.close()
    g.close()


def test_batch_generate_past_its_caches(ctx, tiny_model):
    """generate() with eviction: sequences of 90 tokens through caches of 32 entries; the same twice."""
    g = vrt.Gemma3(ctx, tiny_model)
    b = vrt.Gemma3Batch(g, 3, 32, kv="i8", evict=True)
    prompts = [synth.uniform_ids(900 + i, 3 + 15 * i, 2, 1000) for i in range(3)]
    first = b.generate(prompts, 90, evict=(16, 4))
    again = b.generate(prompts, 90, evict=(16, 4))
    assert [len(x) for x in first] == [90] * 3
    for a, c in zip(first, again):
        np.testing.assert_array_equal(a, c)
    b.close()
    g.close()


def test_batch_kv8_full_shape(ctx, full_model):
    """The 270M shape: 8-bit caches beside fp32 ones over 70 positions; the logits stay near (8-bit rounding), the first
    blocks' worth of positions (all in fp32) within the batch's own bound."""
    g = vrt.Gemma3(ctx, full_model)
    a, b = vrt.Gemma3Batch(g, 3, 128), vrt.Gemma3Batch(g, 3, 128, kv="i8", evict=True)
    ids = synth.uniform_ids(77, 70, 2, 262144)
    for p, t in enumerate(ids):
        t = int(t)
        a.step([0, 2], [t, (t + 1) % 262144])
        b.step([1, 2], [t, (t + 1) % 262144])
        if p in (5, 30, 40, 69):
            for r in range(2):
                d = _rel(a.logits(r), b.logits(r).astype(np.float64))
                print(f"[kv8] position {p} row {r}: logits {d:.2e} of max apart", flush=True)
                assert d <= (1e-3 if p < 31 else 0.1), (p, r)
    a.close()
    b.close()
    g.close()


def test_batch_kv8_restarts_after_a_failed_step(ctx, tiny_model):
    """Sequences reset by a failed step (a token outside the vocabulary) repeat a fresh batch's results bit for bit."""
    g = vrt.Gemma3(ctx, tiny_model)
    b = vrt.Gemma3Batch(g, 2, 64, kv="i8", evict=True)
    ids = [int(t) for t in synth.uniform_ids(1000, 40, 2, 1000)]
    first = [b.step([0, 1], [t, t])[1].copy() for t in ids]
    with pytest.raises(vrt.VrtError):
        b.step([0, 1], [3, 1000])
    assert b.length(0) == b.length(1) == 0
    again = [b.step([0, 1], [t, t])[1].copy() for t in ids]
    assert np.array_equal(np.array(first), np.array(again))
    b.close()
    g.close()


def test_batch_kv8_refusals(ctx, tiny_model):
    g = vrt.Gemma3(ctx, tiny_model)
    b = vrt.Gemma3Batch(g, 2, 32, kv="i8")
    with pytest.raises(vrt.VrtError, match="not created with eviction"):
        b.evict(0, 1, 1)
    b.close()
    b = vrt.Gemma3Batch(g, 2, 32, kv="i8", evict=True)
    b.step([1], [5])
    for args, match in (((2, 1, 1), "out of range"), ((1, 0, 0), "1 <= keep"), ((1, 2, 0), "1 <= keep"), ((1, 1, 2), "recent"),
                        ((0, 1, 0), "1 <= keep")):
        with pytest.raises(vrt.VrtError, match=match):
            b.evict(*args)
    b.evict(1, 1, 0)
    assert b.length(1) == 1
    with pytest.raises(vrt.VrtError, match="out of range"):
        b.length(2)
    b.close()
    with pytest.raises(ValueError):
        vrt.Gemma3Batch(g, 2, 32, evict=True)
    with pytest.raises(ValueError):
        vrt.Gemma3Batch(g, 2, 32, kv="f64")
    assert vrt.lib().vrt_g3_batch_create_kv8(g.h, 2, 32, 2, vrt.C.byref(vrt.C.c_void_p())) == vrt.VRT_ERR_INVALID
    b = vrt.Gemma3Batch(g, 1, 256, kv="i8", evict=True)   # the context's last position
    for i in range(256):
        b.step([0], [7])
    b.evict(0, 10, 5)
    with pytest.raises(vrt.VrtError, match="context length"):
        b.step([0], [7])
    b.close()
    g.close()
