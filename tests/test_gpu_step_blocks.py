"""mako_step_assign_blocks against a plain implementation, request by request: everything is equal."""
import numpy as np
import pytest

from mako_amd import hip, step
from step_oracle import Buffers, assign_blocks

pytestmark = pytest.mark.gpu
OUT = ("table", "free", "n_blocks", "n_free", "status", "start", "slots", "positions", "request")


@pytest.fixture(scope="module")
def ctx():
    if hip.device_count() < 1:
        pytest.fail("no HIP device: GPU tests need an MI355X")
    hip.set_device(0)
    c = step.StepContext(max_rows=65535, max_vocab=1)
    yield c
    c.close()


def call(ctx, s, size, max_blocks, max_tokens, in_place=False, optional=True, repeat=1):
    """The device's outputs.  s: dict of seq, new, have, table, stack, n_free."""
    b = Buffers()
    n = len(s["seq"])
    table, stack = b.out(s["table"]), b.out(s["stack"])
    have, free = b.out(np.asarray(s["have"], np.int32)), b.out(np.array([s["n_free"]], np.int32))
    # (room behind every output, to be left alone)
    outs = dict(n_blocks=have if in_place else b.out(np.full(n + 2, -55, np.int32)), n_free=free if in_place else b.out(np.full(2, -55, np.int32)),
                status=b.out(np.full(n + 2, -55, np.int32)), start=b.out(np.full(n + 3, -55, np.int32)), slots=b.out(np.full(max_tokens + 2, -55, np.int64)),
                positions=b.out(np.full(max_tokens + 2, -55, np.int32)), request=b.out(np.full(max_tokens + 2, -55, np.int32)))
    d = step.BlocksDesc()
    d.n_requests, d.block_size, d.max_tokens = n, size, max_tokens
    d.seq_len, d.new_len = b.up(np.asarray(s["seq"], np.int32)), b.up(np.asarray(s["new"], np.int32))
    d.block_table, d.table_stride, d.max_blocks = table.ptr, s["table"].shape[1], max_blocks
    d.n_blocks, d.out_n_blocks = have.ptr, outs["n_blocks"].ptr
    d.free_blocks, d.free_capacity, d.n_free, d.out_n_free = stack.ptr, len(s["stack"]), free.ptr, outs["n_free"].ptr
    d.out_start, d.out_status, d.out_slots = outs["start"].ptr, outs["status"].ptr, outs["slots"].ptr
    if optional:
        d.out_positions, d.out_request = outs["positions"].ptr, outs["request"].ptr
    for _ in range(repeat):
        ctx.assign_blocks(d)
    hip.synchronize()
    got = {f: a.download() for f, a in outs.items()}
    for f, a in got.items():
        if not (in_place and f in ("n_blocks", "n_free")):
            assert (a[-2 if f != "n_free" else -1:] == -55).all(), "written behind " + f
            got[f] = a[:-2 if f != "n_free" else -1]
    got["table"], got["free"] = table.download(), stack.download()
    return got


def check(ctx, s, size, max_blocks, max_tokens, **kw):
    want = assign_blocks(s["seq"], s["new"], s["have"], s["table"], s["stack"], s["n_free"], size, max_blocks, max_tokens)
    got = call(ctx, s, size, max_blocks, max_tokens, **kw)
    for f in OUT:
        if kw.get("optional", True) or f not in ("positions", "request"):
            assert np.array_equal(got[f], want[f]), (f, np.argwhere(got[f] != want[f])[:5])
    return want


def batch(rng, n, size, max_blocks, free, longest_new=9, ended=0.1, absent=0.1):
    seq = rng.integers(0, max_blocks * size * 3 // 4 + 1, n)
    have = np.minimum((seq + rng.integers(0, 3 * size, n) + size - 1) // size, max_blocks)
    seq = np.where(rng.random(n) < ended, 0, seq)
    new = np.where(seq == 0, 0, rng.integers(0, longest_new + 1, n))
    seq = np.where(rng.random(n) < absent, -1, seq)
    ids = rng.permutation(n * max_blocks + free).astype(np.int32)
    table = np.full((n, max_blocks + 3), -9, np.int32)
    table[:, :max_blocks] = ids[:n * max_blocks].reshape(n, max_blocks)
    stack = np.full(n * max_blocks + free, -3, np.int32)
    stack[:free] = ids[n * max_blocks:]
    return dict(seq=seq, new=new, have=have, table=table, stack=stack, n_free=free)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 1024, 1025, 3000])
@pytest.mark.parametrize("size", [1, 16, 24])
def test_batches(ctx, n, size):
    rng = np.random.default_rng([n, size])
    s = batch(rng, n, size, 12, 4 * n + 7)
    want = check(ctx, s, size, 12, 9 * n)
    assert n < 60 or (want["status"] == 0).all() or (want["status"] == step.BLOCKS_WIDE).any()
    check(ctx, s, size, 12, 9 * n, in_place=True)
    check(ctx, s, size, 12, 9 * n, optional=False)


@pytest.mark.parametrize("n", [2047, 2048, 2049, 5000])
def test_many_requests(ctx, n):
    """Plans in LDS and in device memory."""
    rng = np.random.default_rng(n)
    s = batch(rng, n, 16, 6, 3 * n)
    check(ctx, s, 16, 6, 9 * n)
    check(ctx, s, 16, 6, 9 * n, in_place=True)
    s = batch(rng, n, 4, 6, n // 2)
    want = check(ctx, s, 4, 6, 3 * n, in_place=True)
    assert (want["status"] != 0).any()


def test_prefill_chunks(ctx):
    rng = np.random.default_rng(1)
    s = batch(rng, 40, 16, 700, 3000, longest_new=2000)
    check(ctx, s, 16, 700, 60000)


@pytest.mark.parametrize("free", [0, 1, 5, 40])
def test_too_few_blocks(ctx, free):
    rng = np.random.default_rng(free)
    s = batch(rng, 200, 4, 16, free, longest_new=12, ended=0.01)
    s["have"] = np.minimum(s["have"], (np.maximum(s["seq"], 0) + 3) // 4)  # (nobody has any to spare)
    want = check(ctx, s, 4, 16, 4000)
    assert (want["status"] == step.BLOCKS_SHORT).any() and (want["status"] == step.BLOCKS_OK).any()


def test_too_few_tokens_and_table_entries(ctx):
    rng = np.random.default_rng(2)
    s = batch(rng, 300, 4, 10, 900, longest_new=40)
    want = check(ctx, s, 4, 10, 500)
    assert {step.BLOCKS_OK, step.BLOCKS_WIDE, step.BLOCKS_TOKENS} <= set(want["status"].tolist())
    check(ctx, s, 4, 10, 0)


def test_everything_is_given_back(ctx):
    rng = np.random.default_rng(3)
    s = batch(rng, 50, 16, 300, 10)
    s["seq"][:], s["new"][:] = 0, 0
    want = check(ctx, s, 16, 300, 64)
    assert want["n_free"][0] == 10 + s["have"].sum()


def test_values_out_of_their_ranges(ctx):
    """Numbers of blocks below 0 or above the table's, and of free ones beyond the list; lengths whose sum has 32 bits; a list
    with no room for what is given back."""
    rng = np.random.default_rng(4)
    s = batch(rng, 64, 8, 10, 30)
    s["have"][::4], s["have"][1::4] = -5, 99
    check(ctx, s, 8, 10, 700)
    for n_free in (-4, 10**6, len(s["stack"]) - 3):
        check(ctx, dict(s, n_free=n_free), 8, 10, 700)
    s["seq"][3], s["new"][3] = 2**31 - 1, 1
    s["seq"][5], s["new"][5] = 2**31 - 1, 2**31 - 1
    s["seq"][7], s["new"][7] = 0, 2**31 - 1
    check(ctx, s, 65536, 10, 700)


def test_slots_beyond_31_bits(ctx):
    s = dict(seq=[70000, 0], new=[3, 2], have=[2, 0], table=np.array([[2**31 - 1, 2**31 - 2], [0, 0]], np.int32), stack=np.array([2**31 - 5, 9], np.int32), n_free=1)
    want = check(ctx, s, 65536, 2, 8)
    assert want["slots"].max() > 2**46


def test_the_same_call_again(ctx):
    """Where the numbers go to arrays of their own, a second call on the same inputs finds and gives the same."""
    rng = np.random.default_rng(5)
    check(ctx, batch(rng, 500, 16, 20, 900), 16, 20, 4500, repeat=3)


def test_no_block_is_lost_or_given_twice(ctx):
    """200 steps of a serving loop in place: requests come, grow by what was verified, and end."""
    rng = np.random.default_rng(6)
    n, size, max_blocks, blocks = 96, 8, 40, 1500
    s = dict(seq=np.full(n, 0), new=np.zeros(n, int), have=np.zeros(n, int), table=np.zeros((n, max_blocks), np.int32),
             stack=rng.permutation(blocks).astype(np.int32), n_free=blocks)
    for step_no in range(200):
        ends = rng.random(n) < 0.02
        s["seq"] = np.where(ends, 0, s["seq"])
        s["new"] = np.where(ends, 0, np.where(s["seq"] == 0, rng.integers(1, 60, n), 5))
        got = call(ctx, s, size, max_blocks, 2048, in_place=True)
        if step_no % 40 == 0:
            want = assign_blocks(s["seq"], s["new"], s["have"], s["table"], s["stack"], s["n_free"], size, max_blocks, 2048)
            assert all(np.array_equal(got[f], want[f]) for f in OUT)
        s.update(table=got["table"], stack=got["free"], have=got["n_blocks"], n_free=int(got["n_free"][0]))
        held = np.concatenate([s["table"][b, :s["have"][b]] for b in range(n)] + [s["stack"][:s["n_free"]]])
        assert np.array_equal(np.sort(held), np.arange(blocks)), step_no
        granted = got["status"] == 0
        new = np.where(granted, s["new"], 0)
        kept = np.where(s["new"] == 5, rng.integers(1, 6, n), s["new"])
        s["seq"] = np.where(granted, s["seq"] + np.minimum(kept, new), 0)
