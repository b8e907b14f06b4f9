"""mako_step_cut_rows against a plain implementation in 64 bits: kept numbers, tokens and cut logits are equal, totals and
probabilities as near as their arithmetic allows."""
import numpy as np
import pytest

from mako_amd import api, hip, step
from step_oracle import FLT_MAX, cut_row, cut_rows, encode, probs_row

pytestmark = pytest.mark.gpu

# A weight is exp(t) with t = (x - max) / T, of rounded numbers: t has an error of 3 half steps (the difference, the reciprocal
# of T, the product), which is 3 |t| 2^-53 of the weight, 3e-14 at t = -90; weights below that are nothing beside the first.
# The kernels' 2^t is within 2.7e-14, exp here within 2^-52.  What a cut leaves is added up in whole units, each token's weight
# off by half of one.  Rows whose weights are summed up beforehand: a unit is at most 2^-62 of that sum, and what a top_p leaves
# at least a twentieth of it here: 2^18 2^-63 / 0.05 = 5.7e-13 of it (with top_p of 0.5 and more, 2^20 tokens 2.3e-13).  Rows of
# a top_k of up to 2500: a unit is at most 2^-50, and a total at least 1: 2500 2^-51 = 1.11e-12.  The sums' own roundings (20
# levels, 2^-53 each) are 2.2e-15.  All together 1.17e-12.
TOTAL = 1.2e-12
# a probability is rounded to fp32: half a step, 2^-24, and below the normal range half of 2^-149
PROB, PROB_LEAST = 2.0**-24 + 1e-11, 2.0**-150


@pytest.fixture(scope="module")
def ctx():
    if hip.device_count() < 1:
        pytest.fail("no HIP device: GPU tests need an MI355X")
    hip.set_device(0)
    c = step.StepContext(max_rows=512, max_vocab=1048576)
    yield c
    c.close()


def check(ctx, x, params, dtype="float32", bits=None, rows_per_params=1, probs=False, **kw):
    got, dense = cut_rows(ctx, x, params, dtype, bits, rows_per_params=rows_per_params, probs=probs, **kw)
    seen = encode(x, dtype)[1]
    for r in range(len(x)):
        mask = None if bits is None else bits[r]
        want, ids, _ = cut_row(seen[r], params[r // rows_per_params], mask)
        for f in ("max_logit", "temperature", "cut_logit", "cut_token", "n_kept", "top_token"):
            assert got[r][f] == want[f], (r, f, got[r], want)
        assert abs(got[r]["total"] - want["total"]) <= TOTAL * want["total"], (r, got[r], want)
        if probs:
            p = probs_row(seen[r], want, mask)
            assert (np.abs(dense[r] - p) <= PROB * p + PROB_LEAST).all(), r
            assert not dense[r][np.setdiff1d(np.arange(x.shape[1]), ids)].any()
    return got


KINDS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=40, top_p=0.95), dict(top_p=0.9), dict(temperature=0.4, top_k=1), dict(top_k=300),
         dict(min_p=0.05), dict(temperature=1.3, min_p=0.001, top_k=500, top_p=0.99), dict(temperature=3.0, top_p=0.5), dict(temperature=0.05, top_k=1000, top_p=0.999)]


def all_kinds(rows):
    p = api.make_params(rows)
    for r in range(rows):
        for f, v in KINDS[r % len(KINDS)].items():
            p[f][r] = v
    return p


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab,pad,offset", [(1, 0, 0), (2, 1, 1), (31, 0, 0), (64, 3, 0), (1000, 0, 1), (1024, 0, 0), (1025, 2, 3), (4097, 0, 0), (32000, 0, 0), (33333, 1, 1)])
def test_sizes_types_and_strides(ctx, dtype, vocab, pad, offset):
    rng = np.random.default_rng([vocab, pad])
    rows = 2 * len(KINDS)
    check(ctx, rng.normal(0, 3, (rows, vocab)), all_kinds(rows), dtype, pad=pad, offset=offset, probs=True)


@pytest.mark.parametrize("share,mask_pad", [(0.5, 0), (0.01, 3), (0.999, 1)])
def test_masks(ctx, share, mask_pad):
    rng = np.random.default_rng(int(1000 * share))
    rows, vocab = 2 * len(KINDS), 20011
    bits = rng.random((rows, vocab)) < share
    bits[3] = False  # a row of nothing
    bits[4] = False
    bits[4, vocab - 1] = True  # and of one token, the last
    bits[7] = False
    bits[7, 5] = True
    got = check(ctx, rng.normal(0, 3, (rows, vocab)), all_kinds(rows), bits=bits, mask_pad=mask_pad, probs=True)
    assert got[3]["n_kept"] == 0 and got[3]["total"] == 0 and got[4]["top_token"] == vocab - 1


@pytest.mark.parametrize("sigma", [0.0, 1e-6, 0.1, 3.0, 30.0])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_flat_and_peaked_rows(ctx, sigma, dtype):
    """sigma 0: nothing but ties, cut in the tokens' order; bf16 has thousands of equal logits everywhere."""
    rng = np.random.default_rng([int(sigma * 10), len(dtype)])
    rows = len(KINDS)
    check(ctx, rng.normal(0, 1, (rows, 50021)) * sigma + 1.5, all_kinds(rows), dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_a_crowd_far_below_one_token(ctx, dtype):
    """One token above everything else, and the cut in a crowd that one bin of the first pass holds."""
    rng = np.random.default_rng(5)
    vocab = 60000
    x = -8.0 + 1e-3 * rng.normal(0, 1, (6, vocab))
    x[:, 4321] = 9.0
    x[2:4] = np.round(x[2:4], 3)  # (with ties)
    x[4, :] = -8.0
    x[4, 77] = 9.0
    p = api.make_params(6, top_k=20001)
    p["top_k"][1::2], p["top_p"][1::2], p["temperature"][1::2] = 0, 0.7, 30.0
    p["top_k"][5] = 45000
    p["top_p"][5] = 1.0
    check(ctx, x, p, dtype)


def test_no_numbers_infinities_and_lowest_values(ctx):
    rng = np.random.default_rng(11)
    rows, vocab = len(KINDS), 5003
    for kind in range(7):
        x = rng.normal(0, 2, (rows, vocab)).astype(np.float32)
        if kind == 0:
            x[:, ::3] = np.nan
        elif kind == 1:
            x[:, 7], x[:, 100:200] = np.inf, -np.inf
        elif kind == 2:  # (two largest: the first of them wins)
            x[:, [4000, 90]] = np.inf
        elif kind == 3:
            x[:, 10:] = np.finfo(np.float32).min
        elif kind == 4:
            x[:] = np.finfo(np.float32).min
        elif kind == 5:
            x[:] = -np.inf
            x[::2] = np.nan
        else:
            x[:, ::2] = -0.0
            x[:, 1::2] = 0.0
        check(ctx, x, all_kinds(rows), probs=True)
    x = rng.normal(0, 2, (rows, vocab)).astype(np.float32)
    x[:, 50:] = -65504.0  # (float16's lowest)
    x[:, 3] = np.inf
    check(ctx, x, all_kinds(rows), "float16", probs=True)
    x[:, 50:] = -3.3895313892515355e38  # (bfloat16's)
    check(ctx, x, all_kinds(rows), "bfloat16")


def test_parameters_at_their_ends(ctx):
    rng = np.random.default_rng(12)
    ends = [dict(top_k=2**32 - 1), dict(top_k=5003), dict(top_k=5002), dict(top_p=0.0), dict(top_p=-1.0), dict(top_p=float(np.float32(1 - 2.0**-24))),
            dict(top_p=float("nan")), dict(min_p=1.0), dict(min_p=1.5), dict(temperature=1e-40), dict(temperature=float("inf"), top_p=0.25),
            dict(temperature=-1.0, top_k=5), dict(temperature=float("nan")), dict(temperature=1e-40, top_p=0.5), dict(temperature=float("inf"), min_p=0.5),
            dict(temperature=1e30, top_k=77)]
    p = api.make_params(len(ends))
    for r, e in enumerate(ends):
        for f, v in e.items():
            p[f][r] = v
    check(ctx, rng.normal(0, 2, (len(ends), 5003)), p, probs=True)


def test_parameters_of_several_rows(ctx):
    rng = np.random.default_rng(13)
    check(ctx, rng.normal(0, 2, (35, 3001)), all_kinds(7), rows_per_params=5)


@pytest.mark.parametrize("vocab", [129280, 151553, 262144, 1048576])
def test_large_vocabularies(ctx, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 3, (len(KINDS), vocab)).astype(np.float32)
    x[::2, rng.integers(0, vocab, 50)] += 10
    check(ctx, x, all_kinds(len(KINDS)))


def test_wide_nuclei_of_flat_rows(ctx):
    rng = np.random.default_rng(15)
    x = rng.normal(0, 0.1, (6, 151552)).astype(np.float32)
    p = api.make_params(6, top_p=0.9)
    p["top_p"][1], p["top_k"][2], p["top_k"][3], p["top_p"][4], p["min_p"][5] = 0.99, 100000, 5000, 0.05, 0.6
    check(ctx, x, p)
    check(ctx, x, p, "bfloat16")


def test_a_row_does_not_depend_on_its_batch(ctx):
    rng = np.random.default_rng(16)
    x = rng.normal(0, 3, (300, 40009)).astype(np.float32)
    x[::3, :50] += 10
    p = all_kinds(300)
    whole, _ = cut_rows(ctx, x, p)
    for r in (0, 1, 2, 3, 7, 150, 299):
        alone, _ = cut_rows(ctx, x[r:r + 1], p[r:r + 1])
        assert alone.tobytes() == whole[r:r + 1].tobytes(), r
    again, _ = cut_rows(ctx, x, p)
    assert again.tobytes() == whole.tobytes()


def test_lowest_cut_is_a_finite_number(ctx):
    """A cut among logits of the lowest finite value keeps those of the first tokens."""
    x = np.full((1, 3000), -FLT_MAX, np.float32)
    got = check(ctx, x, api.make_params(1, top_k=1234))
    assert got[0]["cut_token"] == 1233 and got[0]["cut_logit"] == -FLT_MAX


@pytest.mark.parametrize("vocab", [6143, 6144, 6145, 6200])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_that_are_held_whole_and_the_next_larger(ctx, vocab, dtype):
    rng = np.random.default_rng(vocab)
    rows = 2 * len(KINDS)
    p = all_kinds(rows)
    p["top_k"][1], p["temperature"][1] = vocab - 1, 2.0
    p["top_k"][11], p["temperature"][11], p["top_p"][11] = 5000, 2.0, 0.99
    x = rng.normal(0, 3, (rows, vocab))
    x[::2] *= 0.01
    check(ctx, x, p, dtype)


def odd_rows(kind, rows, vocab, rng):
    x = rng.normal(0, 3, (rows, vocab)).astype(np.float32)
    if kind == "falling":
        x = -np.sort(-x, axis=1)
    elif kind == "rising":
        x = np.sort(x, axis=1)
    elif kind == "outlier":
        x[:, 77] = 1000.0
    elif kind == "heavy":
        x = (x / rng.normal(0, 1, (rows, vocab))).astype(np.float32)
    elif kind == "two":
        x[:, rng.random(vocab) < 0.5] -= 500.0
    elif kind == "narrow":
        x = (20.0 + 0.01 * x).astype(np.float32)
    elif kind == "together":
        x[:, 5000:9000] += 12.0
    elif kind == "ends":
        x[:, -1] = 30.0
        x[:, 0] = 30.0
    return x


@pytest.mark.parametrize("kind", ["falling", "rising", "outlier", "heavy", "two", "narrow", "together", "ends"])
def test_rows_that_no_sample_and_no_list_fits(ctx, kind):
    """Where samples mislead and lists overflow: tokens in order or together, one far above, two crowds far apart."""
    rng = np.random.default_rng(len(kind) * 100 + ord(kind[0]))
    ways = [dict(top_p=0.9), dict(top_p=0.5), dict(temperature=50.0, top_p=0.9), dict(top_k=40), dict(top_k=1000, top_p=0.9), dict(top_k=1250), dict(top_k=1300),
            dict(top_k=2500, top_p=0.99), dict(top_k=2501), dict(top_k=3500), dict(top_k=20000, top_p=0.9), dict(top_k=70000), dict(min_p=0.05),
            dict(min_p=1e-4, top_p=0.95), dict(min_p=1e-30), dict(temperature=0.05, top_p=0.99)]
    p = api.make_params(len(ways))
    for r, w in enumerate(ways):
        for f, v in w.items():
            p[f][r] = v
    check(ctx, odd_rows(kind, len(ways), 80021, rng), p)


def test_more_rows_than_workgroups():
    """More rows with a cut beyond their lists than the kernels for these have workgroups: 50 rows over and over."""
    rng = np.random.default_rng(31)
    p = api.make_params(50, top_p=0.8)
    p["top_k"][::5], p["top_p"][::5] = 2000, 1.0
    p["temperature"][1::5] = 0.0
    p["top_p"][2::5], p["min_p"][2::5] = 1.0, 0.2
    x = rng.normal(0, 0.5, (50, 8192)).astype(np.float32)
    c = step.StepContext(max_rows=5000, max_vocab=8192)
    few = check(c, x, p, "float16")
    many, _ = cut_rows(c, np.tile(x, (100, 1)), np.tile(p, 100), "float16")
    assert many.tobytes() == few.tobytes() * 100
    c.close()


def test_as_many_rows_as_there_may_be():
    rng = np.random.default_rng(32)
    x = rng.normal(0, 3, (51, 40)).astype(np.float32)
    p = all_kinds(51)
    c = step.StepContext(max_rows=step.MAX_ROWS, max_vocab=40)
    few = check(c, x, p, probs=True)
    _, few_probs = cut_rows(c, x, p, probs=True)
    many, many_probs = cut_rows(c, np.tile(x, (1285, 1)), np.tile(p, 1285), probs=True)
    assert len(many) == step.MAX_ROWS
    assert many.tobytes() == few.tobytes() * 1285 and many_probs.tobytes() == few_probs.tobytes() * 1285
    c.close()
