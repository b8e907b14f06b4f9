"""mako_step_verify_drafts against a plain implementation in 64 bits: accepted drafts, drawn tokens and lengths are equal."""
import numpy as np
import pytest

from mako_amd import api, hip, step
from step_oracle import Buffers, cut_row, encode, probs_row, verify_desc, verify_request

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    if hip.device_count() < 1:
        pytest.fail("no HIP device: GPU tests need an MI355X")
    hip.set_device(0)
    c = step.StepContext(max_rows=65535, max_vocab=151553)
    yield c
    c.close()


def params_of(n, rng):
    p = api.make_params(n)
    kinds = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=40, top_p=0.95), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.3, top_k=500)]
    for r in range(n):
        for f, v in kinds[rng.integers(len(kinds))].items():
            p[f][r] = v
    return p


def run(ctx, case):
    """The device's outputs and the plain ones of a case (keyword arguments of verify_desc)."""
    b = Buffers()
    seq = case.get("seq_len")
    desc, out = verify_desc(b, **case)
    ctx.verify_drafts(desc)
    hip.synchronize()
    got = {f: a.download() for f, a in out.items()}
    tokens, u, n_drafts = case["tokens"], np.asarray(case["u"], np.float32), case.get("n_drafts")
    n, k = tokens.shape
    want = dict(tokens=np.full((n, k + 1), -77, np.int32), accepted=np.full(n, -77, np.int32))
    if seq is not None:
        want["seq_len"] = np.array(seq, np.int32)
    target = encode(case["target"], case.get("target_type", "float32"))[1]
    draft = case.get("draft")
    draft = None if draft is None else encode(draft, case.get("draft_type", "float32"))[1]

    def rows(x, cuts, bits, first):
        return lambda j: probs_row(x[first + j], None if cuts is None else cuts[first + j], None if bits is None else bits[first + j])

    for r in range(n):
        drafts = k if n_drafts is None else min(int(n_drafts[r]), k)
        if drafts < 0:
            continue
        p = rows(target, case.get("target_cuts"), case.get("target_bits"), r * (k + 1))
        q = None if draft is None else rows(draft, case.get("draft_cuts"), case.get("draft_bits"), r * k)
        given, accepted = verify_request(p, q, tokens[r], drafts, u[r], k)
        want["tokens"][r] = given + [-1] * (k + 1 - len(given))
        want["accepted"][r] = accepted
        if seq is not None:
            want["seq_len"][r] += len(given)
    for f in want:
        assert np.array_equal(got[f], want[f]), (f, np.argwhere(got[f] != want[f])[:5], got[f][got[f] != want[f]][:5], want[f][got[f] != want[f]][:5])
    return got


def make(rng, n, k, vocab, kind, dtype="float32", draft_type=None, mask=0.0):
    """kind: "logits", "probs" (the drafter's distributions; the target's are of the same form), "point", "mixed" (target
    logits, drafter's probabilities)."""
    base = rng.normal(0, 2.5, (n, k + 1, vocab)).astype(np.float32)
    near = (base[:, :k] + rng.normal(0, 0.7, (n, k, vocab))).astype(np.float32).reshape(n * k, vocab)
    target = base.reshape(n * (k + 1), vocab)
    bits = None if not mask else rng.random((n * (k + 1), vocab)) < mask
    case = dict(u=rng.random((n, k + 1)).astype(np.float32), seq_len=rng.integers(0, 1000, n))
    p = np.repeat(params_of(n, rng), k + 1)
    seen = encode(target, dtype)[1]
    cuts = np.array([cut_row(seen[r], p[r], None if bits is None else bits[r])[0] for r in range(len(target))], step.CUT_DTYPE)
    draft_type = draft_type or dtype
    seen_draft = encode(near, draft_type)[1]
    draft_cuts = np.array([cut_row(x, api.make_params(1, temperature=0.9, top_k=200)[0])[0] for x in seen_draft], step.CUT_DTYPE)
    q = np.array([probs_row(seen_draft[r], draft_cuts[r]) for r in range(n * k)]).reshape(n * k, vocab)
    tokens = np.array([rng.choice(vocab, p=row / row.sum()) for row in q], np.int32).reshape(n, k)
    if kind == "probs":
        probs = np.array([probs_row(seen[r], cuts[r], None if bits is None else bits[r]) for r in range(len(target))]).astype(np.float32)
        case.update(target=probs, target_cuts=None, draft=q.astype(np.float32), draft_cuts=None)
    else:
        case.update(target=target, target_cuts=cuts, target_type=dtype, target_bits=bits)
        if kind == "logits":
            case.update(draft=near, draft_cuts=draft_cuts, draft_type=draft_type)
        elif kind == "mixed":
            case.update(draft=q.astype(np.float32), draft_cuts=None)
    case["tokens"] = tokens
    return case


@pytest.mark.parametrize("kind", ["logits", "probs", "point", "mixed"])
@pytest.mark.parametrize("n,k,vocab", [(1, 1, 1), (3, 2, 7), (40, 4, 513), (5, 8, 4096), (9, 3, 4099), (2, 2, 32003)])
def test_forms_and_sizes(ctx, kind, n, k, vocab):
    rng = np.random.default_rng([n, k, vocab, len(kind)])
    got = run(ctx, make(rng, n, k, vocab, kind))
    if kind != "point" and n * k >= 20:  # (that both ends of a chain occur; a draft without a distribution has just p(d))
        assert 0 < got["accepted"].sum() < n * k


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("draft_type", ["float32", "bfloat16", "float16"])
def test_types(ctx, dtype, draft_type):
    rng = np.random.default_rng([len(dtype), len(draft_type)])
    run(ctx, make(rng, 12, 3, 2003, "logits", dtype, draft_type))


def test_masks(ctx):
    rng = np.random.default_rng(3)
    case = make(rng, 12, 3, 3001, "point", mask=0.3)
    run(ctx, case)
    # rows whose masks leave nothing give no token, and their drafts are not accepted
    case["target_bits"][::3] = False
    for r in range(0, len(case["target"]), 3):
        case["target_cuts"][r] = cut_row(case["target"][r], api.make_params(1)[0], case["target_bits"][r])[0]
    case["u"][:, :] = 0.0
    got = run(ctx, case)
    assert (got["tokens"] == -1).all(1).any()
    # the drafter's own masks
    case = make(rng, 12, 3, 3001, "logits")
    bits = rng.random(case["draft"].shape) < 0.5
    bits[np.arange(36), case["tokens"].reshape(-1)] = True
    case["draft_bits"] = bits
    case["draft_cuts"] = np.array([cut_row(x, api.make_params(1)[0], m)[0] for x, m in zip(case["draft"], bits)], step.CUT_DTYPE)
    run(ctx, case)


def test_ragged_batches_leave_the_rest_alone(ctx):
    rng = np.random.default_rng(4)
    case = make(rng, 30, 5, 1025, "logits")
    case["n_drafts"] = rng.integers(-1, 8, 30)
    case["n_drafts"][-4:] = -1
    got = run(ctx, case)
    assert (got["tokens"][-4:] == -77).all() and (got["accepted"][-4:] == -77).all()


def test_no_drafts_at_all(ctx):
    rng = np.random.default_rng(5)
    case = make(rng, 20, 1, 5000, "point")
    keep = np.arange(0, 40, 2)
    case.update(tokens=np.zeros((20, 0), np.int32), target=case["target"][keep], target_cuts=case["target_cuts"][keep], u=case["u"][:, :1])
    run(ctx, case)


def test_as_many_drafts_as_there_may_be(ctx):
    rng = np.random.default_rng(6)
    case = make(rng, 3, step.MAX_DRAFTS, 67, "logits")
    case["u"][0, :-1] = 0.0
    run(ctx, case)
    # (with nothing cut off the target's rows all drafts of the first request are kept)
    for r in range(step.MAX_DRAFTS + 1):
        case["target_cuts"][r] = cut_row(case["target"][r], api.make_params(1)[0])[0]
    assert run(ctx, case)["accepted"][0] == step.MAX_DRAFTS


def test_uniforms_at_their_ends(ctx):
    rng = np.random.default_rng(7)
    for kind in ("logits", "point"):
        case = make(rng, 20, 3, 4100, kind)
        for u in (0.0, 1.0 - 2.0**-24):
            case["u"][:] = u
            run(ctx, case)


def test_drafts_that_are_no_tokens(ctx):
    rng = np.random.default_rng(8)
    for kind in ("logits", "point", "probs"):
        case = make(rng, 12, 2, 300, kind)
        case["u"][:, :2] = 0.0
        case["tokens"][::3, 0] = -1
        case["tokens"][1::3, 1] = 300
        case["tokens"][2::3, 1] = 2**31 - 1
        got = run(ctx, case)
        assert (got["accepted"][::3] == 0).all()


def test_probabilities_that_are_none(ctx):
    """NaN, infinities and negative values count as 0; a q above p everywhere leaves nothing but p; a p of zeros gives nothing."""
    rng = np.random.default_rng(9)
    case = make(rng, 24, 2, 999, "probs")
    t = case["target"]
    t[::5, 3], t[1::5, 4], t[2::5, 5] = np.nan, np.inf, -1.0
    case["draft"][::7, 6] = np.nan
    case["draft"][6 * 2:8 * 2] = 0.9
    t[9 * 3:10 * 3] = 0.0
    case["u"][6:8, :2] = 0.99
    got = run(ctx, case)
    assert (got["tokens"][9] == -1).all() and got["accepted"][9] == 0
    assert (got["accepted"][6:8] == 0).all() and (got["tokens"][6:8, 0] >= 0).all()


@pytest.mark.parametrize("kind", ["logits", "point"])
def test_large_vocabulary(ctx, kind):
    rng = np.random.default_rng(10)
    run(ctx, make(rng, 3, 2, 151553, kind, "bfloat16"))


def test_offsets_beyond_31_bits(ctx):
    """Rows far apart: the last begins more than 2^31 elements (of 2 bytes) behind the first."""
    rng = np.random.default_rng(11)
    vocab, n = 128, 3
    stride = 2**30 + 64
    x = rng.normal(0, 2, (n, vocab)).astype(np.float32)
    raw, seen = encode(x, "bfloat16")
    room = hip.DeviceArray((n - 1) * stride + vocab, np.uint16)
    for r in range(n):
        hip.check(hip.lib().hipMemcpy(room.ptr + 2 * r * stride, np.ascontiguousarray(raw[r]).ctypes.data, 2 * vocab, hip.hipMemcpyHostToDevice))
    cuts = np.array([cut_row(s, api.make_params(1, top_k=50)[0])[0] for s in seen], step.CUT_DTYPE)
    u = rng.random((n, 1))
    b = Buffers()
    d, out = verify_desc(b, seen, cuts, np.zeros((n, 0), np.int32), u, "bfloat16")
    d.target, d.target_stride = room.ptr, stride
    ctx.verify_drafts(d)
    c = step.CutDesc()
    found = b.out(np.zeros(n * 32, np.uint8))
    c.logits, c.logits_type, c.logits_stride, c.n_rows, c.n_vocab = room.ptr, step.LOGITS_BF16, stride, n, vocab
    c.params, c.out_cuts = b.up(api.make_params(n, top_k=50)), found.ptr
    ctx.cut_rows(c)
    hip.synchronize()
    far = out["tokens"].download()
    records = found.download().view(step.CUT_DTYPE)
    for f in ("n_kept", "cut_token", "top_token"):
        assert np.array_equal(records[f], cuts[f])
    d, out = verify_desc(b, seen, cuts, np.zeros((n, 0), np.int32), u, "bfloat16")
    ctx.verify_drafts(d)
    hip.synchronize()
    assert np.array_equal(out["tokens"].download(), far)


def test_tokens_are_distributed_as_the_targets(ctx):
    """60 000 requests of one distribution: the first token given out has the target's probabilities, whatever the drafter's."""
    rng = np.random.default_rng(12)
    n, vocab = 60000, 8
    p = np.array([0.3, 0.05, 0.2, 0.0, 0.15, 0.1, 0.15, 0.05])
    q = np.array([0.05, 0.3, 0.1, 0.1, 0.05, 0.2, 0.1, 0.1])
    tokens = rng.choice(vocab, n, p=q).astype(np.int32)
    b = Buffers()
    d, out = verify_desc(b, np.tile(p, (2 * n, 1)), None, tokens[:, None], rng.random((n, 2)), draft=np.tile(q, (n, 1)))
    ctx.verify_drafts(d)
    hip.synchronize()
    got = np.bincount(out["tokens"].download()[:, 0], minlength=vocab) / n
    sigma = np.sqrt(p * (1 - p) / n)
    assert (np.abs(got - p) <= 5 * sigma + 1e-9).all(), (got, p)
    rate = out["accepted"].download().mean()
    want = np.minimum(p, q).sum()
    assert abs(rate - want) <= 5 * np.sqrt(want * (1 - want) / n)


def test_as_many_requests_as_there_may_be():
    rng = np.random.default_rng(33)
    few, times = 257, step.MAX_ROWS // 257
    c = step.StepContext(max_rows=step.MAX_ROWS, max_vocab=30)
    case = make(rng, few, 2, 30, "probs")
    got = run(c, case)
    b = Buffers()
    many = {f: np.tile(a, (times,) + (1,) * (a.ndim - 1)) if isinstance(a, np.ndarray) else a for f, a in case.items()}
    desc, out = verify_desc(b, **many)
    c.verify_drafts(desc)
    hip.synchronize()
    for f, a in out.items():
        assert np.array_equal(a.download(), np.tile(got[f], (times,) + (1,) * (got[f].ndim - 1))), f
    c.close()
