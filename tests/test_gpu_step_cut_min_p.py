"""mako_step_cut_rows with a min_p that no token's weight reaches: one token is left, however many are equal to it."""
import numpy as np
import pytest

from mako_amd import api, hip, step
from test_gpu_step_cut import check

pytestmark = pytest.mark.gpu

ABOVE_ONE = float(np.nextafter(np.float32(1), np.float32(2)))
WAYS = [dict(min_p=1.5), dict(min_p=ABOVE_ONE), dict(min_p=float("inf")), dict(min_p=1.5, top_k=5000), dict(min_p=1.5, top_k=3), dict(min_p=1.5, top_p=0.5),
        dict(min_p=1.5, temperature=float("inf")), dict(min_p=1.5, temperature=1e-40), dict(min_p=1.0), dict(min_p=1.0, top_k=70)]


@pytest.fixture(scope="module")
def ctx():
    if hip.device_count() < 1:
        pytest.fail("no HIP device: GPU tests need an MI355X")
    hip.set_device(0)
    c = step.StepContext(max_rows=16, max_vocab=50021)
    yield c
    c.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [300, 6144, 6145, 50021])
@pytest.mark.parametrize("kind", ["equal", "many largest", "one largest", "masked"])
def test_no_token_weighs_enough(ctx, vocab, dtype, kind):
    rng = np.random.default_rng([vocab, len(kind)])
    rows, bits = len(WAYS), None
    x = np.full((rows, vocab), -2.5, np.float32)
    if kind == "many largest":
        x = np.where(rng.random((rows, vocab)) < 0.6, 4.0, rng.normal(0, 0.5, (rows, vocab))).astype(np.float32)
    elif kind == "one largest":
        x[:, vocab // 3] = 4.0
    elif kind == "masked":
        bits = rng.random((rows, vocab)) < 0.7
    p = api.make_params(rows)
    for r, way in enumerate(WAYS):
        for f, v in way.items():
            p[f][r] = v
    got = check(ctx, x, p, dtype, bits, probs=True)
    assert (got["n_kept"][:8] == 1).all() and (got["cut_token"][:8] == got["top_token"][:8]).all()
