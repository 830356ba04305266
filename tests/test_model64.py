"""The 64-bit model of the 8-bit batch tests (model64.py), over an exact cache, against the oracle."""
import numpy as np

import model64
import oracle
import synth


def test_model64_is_the_oracles(tiny_model):
    m, o = model64.Model64(tiny_model, kv8=False), oracle.Model(tiny_model)
    for i, t in enumerate(synth.uniform_ids(5, 20, 2, 1000)):
        want = o.decode(int(t), i, want_logits=True, logits=True)["logits"]
        got = m.step(int(t))
        assert np.max(np.abs(got - want)) <= 1e-4 * np.max(np.abs(want)), i
    o.close()
