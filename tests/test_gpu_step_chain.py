"""The operators of include/mako_step.h one after the other, as a serving loop has them: eagerly and as a graph that is
replayed, on streams of their own, with two contexts at once."""
import numpy as np
import pytest

from mako_amd import api, hip, step
from step_oracle import assign_blocks, cut_row, probs_row, verify_request

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def device():
    if hip.device_count() < 1:
        pytest.fail("no HIP device: GPU tests need an MI355X")
    torch.cuda.set_device(0)


class On:
    """A torch stream as the calls take it."""

    def __init__(self, stream):
        self.ptr = stream.cuda_stream


class Loop:
    """A serving loop's state on the device: logits come in, tokens, lengths and the next step's blocks go out."""

    def __init__(self, n, k, vocab, seed, size=8, max_blocks=64):
        self.n, self.k, self.vocab, self.size, self.max_blocks = n, k, vocab, size, max_blocks
        rng = np.random.default_rng(seed)
        blocks = n * max_blocks
        dev = "cuda"
        i32 = torch.int32
        self.params_host = api.make_params(n, temperature=0.8, top_p=0.95)
        self.params_host["top_k"][::2] = 50
        self.params = torch.from_numpy(self.params_host.view(np.uint8).copy()).to(dev)
        self.draft_params = torch.from_numpy(api.make_params(n * k, temperature=0.9).view(np.uint8).copy()).to(dev)
        self.target = torch.zeros(n * (k + 1), vocab, dtype=torch.bfloat16, device=dev)
        self.draft = torch.zeros(n * k, vocab, dtype=torch.bfloat16, device=dev)
        self.tokens = torch.zeros(n, k, dtype=i32, device=dev)
        self.u = torch.zeros(n, k + 1, device=dev)
        self.cuts = torch.zeros(n * (k + 1), 32, dtype=torch.uint8, device=dev)
        self.draft_cuts = torch.zeros(n * k, 32, dtype=torch.uint8, device=dev)
        self.out = torch.zeros(n, k + 1, dtype=i32, device=dev)
        self.accepted = torch.zeros(n, dtype=i32, device=dev)
        self.seq = torch.from_numpy(rng.integers(1, 40, n).astype(np.int32)).to(dev)
        self.new = torch.full((n,), k + 1, dtype=i32, device=dev)
        have = (self.seq.cpu().numpy() + k + 1 + size - 1) // size
        ids = rng.permutation(blocks).astype(np.int32)
        table = np.zeros((n, max_blocks), np.int32)
        at = 0
        for b in range(n):
            table[b, :have[b]] = ids[at:at + have[b]]
            at += have[b]
        self.table = torch.from_numpy(table).to(dev)
        stack = np.zeros(blocks, np.int32)
        stack[:blocks - at] = ids[at:]
        self.stack = torch.from_numpy(stack).to(dev)
        self.n_free = torch.tensor([blocks - at], dtype=i32, device=dev)
        self.have = torch.from_numpy(have.astype(np.int32)).to(dev)
        self.status = torch.zeros(n, dtype=i32, device=dev)
        self.start = torch.zeros(n + 1, dtype=i32, device=dev)
        self.slots = torch.zeros(n * (k + 1) + 5, dtype=torch.int64, device=dev)
        self.positions = torch.zeros(n * (k + 1) + 5, dtype=i32, device=dev)
        self.ctx = step.StepContext(max_rows=n * (k + 1), max_vocab=vocab)
        self.bind()

    def bind(self):
        c = self.cut = step.CutDesc()
        c.logits, c.logits_type, c.logits_stride, c.n_rows, c.n_vocab = self.target.data_ptr(), step.LOGITS_BF16, self.vocab, self.n * (self.k + 1), self.vocab
        c.params, c.rows_per_params, c.out_cuts = self.params.data_ptr(), self.k + 1, self.cuts.data_ptr()
        q = self.cut_draft = step.CutDesc()
        q.logits, q.logits_type, q.logits_stride, q.n_rows, q.n_vocab = self.draft.data_ptr(), step.LOGITS_BF16, self.vocab, self.n * self.k, self.vocab
        q.params, q.out_cuts = self.draft_params.data_ptr(), self.draft_cuts.data_ptr()
        v = self.verify = step.VerifyDesc()
        v.n_requests, v.max_drafts, v.n_vocab = self.n, self.k, self.vocab
        v.target, v.target_type, v.target_stride, v.target_cuts = self.target.data_ptr(), step.LOGITS_BF16, self.vocab, self.cuts.data_ptr()
        v.draft, v.draft_type, v.draft_stride, v.draft_cuts = self.draft.data_ptr(), step.LOGITS_BF16, self.vocab, self.draft_cuts.data_ptr()
        v.draft_tokens, v.u, v.seq_len, v.out_seq_len = self.tokens.data_ptr(), self.u.data_ptr(), self.seq.data_ptr(), self.seq.data_ptr()
        v.out_tokens, v.out_accepted = self.out.data_ptr(), self.accepted.data_ptr()
        b = self.blocks = step.BlocksDesc()
        b.n_requests, b.block_size, b.max_tokens = self.n, self.size, self.slots.numel()
        b.seq_len, b.new_len = self.seq.data_ptr(), self.new.data_ptr()
        b.block_table, b.table_stride, b.max_blocks = self.table.data_ptr(), self.max_blocks, self.max_blocks
        b.n_blocks = b.out_n_blocks = self.have.data_ptr()
        b.free_blocks, b.free_capacity = self.stack.data_ptr(), self.stack.numel()
        b.n_free = b.out_n_free = self.n_free.data_ptr()
        b.out_start, b.out_status, b.out_slots, b.out_positions = self.start.data_ptr(), self.status.data_ptr(), self.slots.data_ptr(), self.positions.data_ptr()

    def feed(self, gen):
        """New logits, drafts and uniforms, by ordinary torch work on the current stream."""
        x = 3 * torch.randn(self.n, self.k + 1, self.vocab, generator=gen, device="cuda")
        self.target.copy_(x.view(-1, self.vocab))
        q = x[:, :self.k] + 0.5 * torch.randn(self.n, self.k, self.vocab, generator=gen, device="cuda")
        self.draft.copy_(q.reshape(-1, self.vocab))
        noise = -torch.log(-torch.log(torch.rand(self.n * self.k, self.vocab, generator=gen, device="cuda")))
        self.tokens.copy_((self.draft.float() / 0.9 + noise).argmax(1).view(self.n, self.k))
        self.u.copy_(torch.rand(self.n, self.k + 1, generator=gen, device="cuda"))

    def calls(self, stream):
        s = On(stream)
        self.ctx.cut_rows(self.cut_draft, s)
        self.ctx.cut_rows(self.cut, s)
        self.ctx.verify_drafts(self.verify, s)
        self.ctx.assign_blocks(self.blocks, s)

    FIELDS = ("out", "accepted", "seq", "have", "table", "stack", "n_free", "status", "start", "slots", "positions", "cuts")

    def state(self):
        return {f: getattr(self, f).cpu().numpy().copy() for f in self.FIELDS}

    def expected(self, before):
        """What a step has to leave, from the state before it, in 64 bits on the host."""
        target = self.target.float().cpu().numpy()
        draft = self.draft.float().cpu().numpy()
        u, tokens = self.u.cpu().numpy(), self.tokens.cpu().numpy()
        q_params = api.make_params(1, temperature=0.9)[0]
        out, accepted, seq = np.full((self.n, self.k + 1), -1, np.int32), np.zeros(self.n, np.int32), before["seq"].copy()
        for r in range(self.n):
            def p_row(j):
                x = target[r * (self.k + 1) + j]
                return probs_row(x, cut_row(x, self.params_host[r])[0])

            def q_row(j):
                x = draft[r * self.k + j]
                return probs_row(x, cut_row(x, q_params)[0])

            got, accepted[r] = verify_request(p_row, q_row, tokens[r], self.k, u[r], self.k)
            out[r, :len(got)] = got
            seq[r] += len(got)
        blocks = assign_blocks(seq, np.full(self.n, self.k + 1), before["have"], before["table"], before["stack"], before["n_free"][0], self.size,
                               self.max_blocks, self.slots.numel())
        return dict(out=out, accepted=accepted, seq=seq, have=blocks["n_blocks"], table=blocks["table"], stack=blocks["free"], n_free=blocks["n_free"],
                    status=blocks["status"], start=blocks["start"], slots=blocks["slots"], positions=blocks["positions"])


def same(got, want):
    for f in want:
        assert np.array_equal(got[f], want[f]), f


def test_steps_of_a_serving_loop():
    loop, gen = Loop(24, 3, 5003, seed=1), torch.Generator(device="cuda").manual_seed(1)
    stream = torch.cuda.Stream()
    for _ in range(6):
        with torch.cuda.stream(stream):
            loop.feed(gen)
            stream.synchronize()
            before = loop.state()
            loop.calls(stream)
            stream.synchronize()
            same(loop.state(), loop.expected(before))


def test_a_captured_step_replayed():
    """One graph of the whole step, replayed on new inputs between ordinary torch work: every replay is what eager calls give."""
    loop, eager = Loop(16, 4, 30011, seed=2), Loop(16, 4, 30011, seed=2)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        eager.feed(torch.Generator(device="cuda").manual_seed(9))
        eager.calls(stream)  # (kernels are loaded outside the capture)
        stream.synchronize()
    eager = Loop(16, 4, 30011, seed=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        loop.calls(torch.cuda.current_stream())
    for i in range(5):
        loop.feed(torch.Generator(device="cuda").manual_seed(100 + i))
        eager.feed(torch.Generator(device="cuda").manual_seed(100 + i))
        torch.cuda.synchronize()
        graph.replay()
        junk = torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        torch.cuda.synchronize()
        assert torch.isfinite(junk).all()
        eager.calls(torch.cuda.current_stream())
        torch.cuda.synchronize()
        same(loop.state(), eager.state())
    assert (loop.state()["accepted"] > 0).any()


def test_two_contexts_at_once():
    """Two loops on streams of their own, their calls interleaved without a wait, give what each gives alone."""
    loops = [Loop(16, 3, 20011, seed=s) for s in (5, 6)]
    alone = [Loop(16, 3, 20011, seed=s) for s in (5, 6)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for pair in (loops, alone):
        for i, loop in enumerate(pair):
            loop.feed(torch.Generator(device="cuda").manual_seed(50 + i))
    torch.cuda.synchronize()
    for _ in range(4):
        for loop, stream in zip(loops, streams):
            loop.calls(stream)
    torch.cuda.synchronize()
    for loop in alone:
        for _ in range(4):
            loop.calls(torch.cuda.current_stream())
        torch.cuda.synchronize()
    for a, b in zip(loops, alone):
        same(a.state(), b.state())


def test_the_current_device_is_left_alone():
    before = torch.cuda.current_device()
    loop = Loop(2, 1, 64, seed=3)
    loop.calls(torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert torch.cuda.current_device() == before


def test_refused_calls_say_why():
    ctx = step.StepContext(max_rows=4, max_vocab=100)
    with pytest.raises(api.MakoError, match="empty vocabulary"):
        ctx.cut_rows(step.CutDesc())
    with pytest.raises(api.MakoError, match="max_rows"):
        d = step.CutDesc(logits=4096, n_rows=5, n_vocab=100, logits_stride=100, params=4096, out_cuts=4096)
        ctx.cut_rows(d)
    with pytest.raises(api.MakoError, match="probabilities are fp32"):
        d = step.VerifyDesc(n_requests=4, n_vocab=100, target=4096, target_type=step.LOGITS_BF16, target_stride=100, u=4096, out_tokens=4096, out_accepted=4096)
        ctx.verify_drafts(d)
    with pytest.raises(api.MakoError, match="no requests"):
        ctx.assign_blocks(step.BlocksDesc(block_size=16))
    ctx.cut_rows(step.CutDesc(n_vocab=100))  # (no rows: nothing to do)
