"""lm_sample over rows whose largest logit is +infinity: those logits alone have weight, whatever the temperature."""
import numpy as np
import pytest

import litemind_amd as lm
import serving_ref as ref
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_sample import run, settings

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


@pytest.mark.parametrize("vocab", [100, 6007, 20011, 102400])
@pytest.mark.parametrize("masked", [0.0, 0.6, 0.97])
@pytest.mark.parametrize("temperature", [1e-30, 1.0, 1e37, 1e38, np.inf])
def test_infinite_logits(ctx, vocab, masked, temperature):
    announce(f"sample: +infinity among {vocab} logits, {masked:.0%} masked, temperature {temperature}")
    rng = np.random.default_rng(vocab)
    sets = settings([(temperature, k, p, m) for k, p, m in ((0, 1.0, 0.0), (1, 1.0, 0.0), (50, 1.0, 0.0), (1000, 1.0, 0.0),
                                                            (3000, 0.8, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.3), (700, 0.6, 0.01),
                                                            (2, 0.4, 1.0))])
    for many in (1, 2, 40):
        x = rng.normal(size=(len(sets), vocab)).astype(np.float32) * np.float32(3)
        x[rng.random(x.shape) < masked] = -np.inf
        for row in x:
            row[rng.choice(vocab, many, replace=False)] = np.inf
        u = rng.random(len(sets)).astype(np.float32)
        t, p = run(ctx, x, sets, u)
        for i in range(len(sets)):
            want, chance, near = ref.sample(x[i], *sets[i], u[i])
            assert near < 1e-9 or t[i] == want, f"row {i}: {t[i]}, not {want} ({sets[i]}, u {u[i]})"
            # one weight over a whole number of them, rounded once
            assert abs(p[i] - chance) <= 2.0 ** -24 * chance
