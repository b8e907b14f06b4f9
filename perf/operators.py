"""The operators of a speculative decode step, as an engine calls them: cases for timing, with their inputs, their plain
forms and the calls.

A step verifies each request's drafted tokens against the target model and makes room for the tokens of the next step:

  cut     every row of logits gets its cut: what temperature, min_p, top_k and top_p leave of it (the weights' total, the
          last logit and token kept, their number), and with "probs" the row as fp32 probabilities
  verify  drafted tokens are kept while u q(d) < p(d); the first that is not, or the end of the drafts, has a token drawn
          from what max(0, p - q) leaves of the target's row there
  blocks  from the requests' lengths: blocks that they no longer need go back to the free list, blocks that the next
          step's tokens need come from it into the requests' block tables, and every new token gets its cache slot, its
          position and its request

A case is a dict of plain values:
  op            "cut", "verify" or "blocks"
  dtype         of the logits: "float32", "bfloat16", "float16"; verify alone: "probs", rows of fp32 probabilities
  rows, vocab   of cut; pad: elements between a row's end and the next row; logits and params: row_logits(), row_params()
  requests, drafts, vocab   of verify; draft: "logits" / "probs" (a drafter with a distribution), "point" (one without);
                ragged: requests have 0 to `drafts` drafts and some have none in flight (padding of the batch)
  mask          share of the vocabulary that a row's mask allows, 0: no mask
  requests, tokens, block, context   of blocks: the next step's tokens in all, the block size, the longest context; kind:
                "decode" (every request the same few tokens) or "mixed" (some requests a chunk of their prompt)

Weights are in 64 bits here and there: cuts and draws are whole numbers, and a sum in 32 bits would move them.
"""
import ctypes
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "probs": torch.float32}
MOST_LOGITS = 512 * 129280  # of the largest batch of rows
FLT_MAX = torch.finfo(torch.float32).max
PARAMS = ("temperature", "top_k", "top_p", "min_p")


def cut(name, rows, vocab, dtype, params, logits="spiked", pad=0, mask=0.0, probs=False):
    return dict(name=name, op="cut", rows=rows, vocab=vocab, dtype=dtype, params=params, logits=logits, pad=pad, mask=mask, probs=probs)


def verify(name, requests, drafts, vocab, dtype, draft, params, logits="spiked", mask=0.0, ragged=False):
    return dict(name=name, op="verify", requests=requests, drafts=drafts, vocab=vocab, dtype=dtype, draft=draft, params=params,
                logits=logits, mask=mask, ragged=ragged)


def blocks(name, requests, tokens, block, context, kind):
    return dict(name=name, op="blocks", requests=requests, tokens=tokens, block=block, context=context, kind=kind)


def listed():
    return [
        # one sequence on one's own machine: its next row, cut to a nucleus
        cut("cut_1", 1, 151552, "float32", "nucleus", "normal"),
        # a server's decode batch, every request with parameters of its own
        cut("cut_64", 64, 129280, "float32", "serving"),
        # a vocabulary that is a multiple of nothing, rows that are not aligned, all kinds of requests under a grammar's masks
        cut("cut_ragged_24", 24, 151553, "float16", "any", "normal", pad=1, mask=0.5),
        # full-vocabulary nuclei, on rows as peaked and as flat as they come
        cut("cut_nucleus_256", 256, 151552, "float32", "nucleus", "stress"),
        # 64 requests of eight positions each, as the target model's head leaves them
        cut("cut_512", 512, 129280, "bfloat16", "serving"),
        # a draft model's rows as probabilities, for a program that keeps its distributions
        cut("probs_128", 128, 32000, "bfloat16", "temperature", probs=True),
        # one sequence with four drafts
        verify("verify_1", 1, 4, 151552, "float32", "logits", "top_p"),
        # 64 requests of four drafts by a draft model
        verify("verify_64", 64, 4, 129280, "bfloat16", "logits", "serving"),
        # drafts looked up in the text so far, under masks; the batch is padded
        verify("verify_lookup_32", 32, 7, 129280, "float32", "point", "top_k", mask=0.5, ragged=True),
        # rows of probabilities, a large batch of a small vocabulary
        verify("verify_probs_256", 256, 3, 32000, "probs", "probs", "temperature", "normal", ragged=True),
        # the next step of 64 requests of five positions each
        blocks("blocks_64", 64, 320, 16, 8192, "decode"),
        # a large batch where some requests bring chunks of their prompts
        blocks("blocks_1024", 1024, 131072, 64, 131072, "mixed"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _vocab(rng):
    v = _spread(rng, 8000, 160000)
    return (v + 63) // 64 * 64 if rng.random() < 0.6 else v  # most vocabularies are padded, the others as they come


def draw(rng):
    op = rng.choice(("cut", "cut", "verify", "verify", "blocks"))
    if op == "blocks":
        requests, block = _spread(rng, 1, 1024), rng.choice((16, 16, 24, 32, 64, 128))
        if rng.random() < 0.5:
            return dict(op=op, requests=requests, tokens=requests * rng.randint(1, 8), block=block, context=_spread(rng, 64, 32768), kind="decode")
        return dict(op=op, requests=requests, tokens=requests + _spread(rng, 64, 130000), block=max(block, requests // 16), context=_spread(rng, 256, 131072), kind="mixed")
    vocab, logits = _vocab(rng), rng.choice(("spiked", "spiked", "normal", "stress"))
    mask = rng.choice((0.0, 0.0, 0.01, 0.5, 0.9))
    params = rng.choice(("greedy", "top_k", "nucleus", "serving", "temperature", "min_p", "wide_top_k", "any"))
    if op == "cut":
        dtype, probs = rng.choice(("float32", "bfloat16", "float16")), rng.random() < 0.25
        rows = _spread(rng, 1, MOST_LOGITS // vocab // (4 if probs or dtype == "float32" else 1))
        return dict(op=op, rows=min(rows, 512), vocab=vocab, dtype=dtype, params=params, logits=logits, pad=rng.choice((0, 0, 0, 64, 1)), mask=mask, probs=probs)
    dtype = rng.choice(("float32", "bfloat16", "float16", "probs"))
    drafts = rng.randint(1, 8)
    requests = min(256, _spread(rng, 1, MOST_LOGITS // 4 // vocab // (drafts + 1)))
    draft = rng.choice(("point", "probs" if dtype == "probs" else "logits"))
    return dict(op=op, requests=requests, drafts=drafts, vocab=vocab, dtype=dtype, draft=draft, params=params, logits=logits,
                mask=0.0 if dtype == "probs" else mask, ragged=rng.random() < 0.3)


# ---- inputs ----

def row_params(kind, n, gen):
    """{field: [n]} of the rows' parameters."""
    def full(v, dtype=torch.float32):
        return torch.full((n,), v, dtype=dtype, device="cuda")

    def uniform(low, high):
        return torch.rand(n, generator=gen, device="cuda") * (high - low) + low

    def choice(values, dtype):
        at = torch.randint(0, len(values), (n,), generator=gen, device="cuda")
        return torch.tensor(values, dtype=dtype, device="cuda")[at]

    p = dict(temperature=full(1.0), top_k=full(0, torch.int32), top_p=full(1.0), min_p=full(0.0))
    if kind == "greedy":
        p["temperature"] = full(0.0)
    elif kind == "top_k":
        p.update(temperature=full(0.7), top_k=full(40, torch.int32), top_p=full(0.95))
    elif kind == "nucleus":
        p["top_p"] = full(0.9)
    elif kind == "top_p":
        p.update(temperature=full(0.8), top_p=full(0.95))
    elif kind == "serving":  # a server's batch: every request has its own
        p.update(temperature=uniform(0.3, 1.2), top_k=choice([0, 20, 50, 100], torch.int32), top_p=uniform(0.8, 1.0).clamp(max=1.0 - 2.0**-24))
    elif kind == "temperature":
        p["temperature"] = uniform(0.5, 1.2)
    elif kind == "min_p":
        p["min_p"] = choice([0.02, 0.05, 0.1], torch.float32)
    elif kind == "wide_top_k":
        p.update(top_k=choice([200, 500, 1000], torch.int32), top_p=full(0.95))
    elif kind == "any":  # each row one of the kinds
        kinds = ("greedy", "top_k", "nucleus", "serving", "temperature", "min_p", "wide_top_k")
        parts = [row_params(k, n, gen) for k in kinds]
        which = torch.randperm(n, generator=gen, device="cuda") % len(kinds)
        for f in PARAMS:
            p[f] = torch.stack([q[f] for q in parts]).gather(0, which[None])[0]
    else:
        raise ValueError(kind)
    return p


def row_logits(kind, rows, vocab, stride, gen):
    """fp32 [rows, stride]: "spiked": N(0, 3^2) with up to 50 tokens of each row raised by 10, "normal": N(0, 3^2), "stress":
    half the rows Student-t(3) * 4, half N(0, 0.1^2)."""
    x = torch.randn(rows, stride, generator=gen, device="cuda")
    if kind == "stress":
        half = rows // 2
        if half:
            z = torch.randn(3, half, stride, generator=gen, device="cuda")
            x[:half] *= 4.0 / (z.square_().sum(0) / 3.0).sqrt_()
        x[half:] *= 0.1
        return x
    x *= 3.0
    if kind == "spiked":
        at = torch.randint(0, vocab, (rows, 50), generator=gen, device="cuda")
        n = torch.randint(1, 51, (rows, 1), generator=gen, device="cuda")
        x.scatter_add_(1, at, torch.where(torch.arange(50, device="cuda") < n, 10.0, 0.0))
    return x


def row_masks(rows, vocab, share, gen):
    """uint32 words as int32 [rows, ceil(vocab / 32)]: bit i & 31 of word i >> 5 allows token i."""
    words = (vocab + 31) // 32
    bits = torch.rand(rows, words * 32, generator=gen, device="cuda") < share
    bits[:, vocab:] = False
    bits[:, 0] = True
    weight = (1 << torch.arange(32, device="cuda")).to(torch.int64)
    out = torch.empty(rows, words, dtype=torch.int32, device="cuda")
    for r in range(0, rows, 64):
        v = (bits[r:r + 64].view(-1, words, 32) * weight).sum(2)
        out[r:r + 64] = torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32)
    return out


def mask_bits(mask, vocab):
    """bool [rows, vocab] of row_masks()'s words."""
    at = torch.arange(32, device=mask.device, dtype=torch.int32)
    return ((mask[:, :, None] >> at) & 1).view(mask.shape[0], -1)[:, :vocab].bool()


def packed_params(p):
    """The rows' parameters as the entry points take them: 28 bytes a row, the penalties neutral."""
    n = p["temperature"].shape[0]
    one, zero = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    cols = [p["temperature"], p["top_k"].view(torch.float32), p["top_p"], p["min_p"], zero, zero, one]
    return torch.stack([c.view(torch.int32) for c in cols], 1).contiguous()


def packed_cuts(c):
    """Cuts as the entry points take them: 32 bytes a row."""
    total = c["total"].view(torch.int32).view(-1, 2)
    cols = [c["max"].view(torch.int32), c["temperature"].view(torch.int32), c["cut"].view(torch.int32), c["cut_token"], c["n_kept"], c["top_token"]]
    return torch.cat([total, torch.stack(cols, 1)], 1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "blocks":
        return prepare_blocks(case, gen, s)
    vocab = case["vocab"]
    if case["op"] == "cut":
        rows, stride = case["rows"], vocab + case["pad"]
        s["params"] = row_params(case["params"], rows, gen)
        s["logits"] = row_logits(case["logits"], rows, vocab, stride, gen).to(DTYPES[case["dtype"]])
        s["mask"] = row_masks(rows, vocab, case["mask"], gen) if case["mask"] else None
        s["packed"] = packed_params(s["params"])
        s["out"] = dict(cuts=torch.zeros(rows, 8, dtype=torch.int32, device="cuda"))
        if case["probs"]:
            s["out"]["probs"] = torch.empty(rows, vocab, device="cuda")
        return s
    n, k = case["requests"], case["drafts"]
    one = row_params(case["params"], n, gen)
    dtype = DTYPES[case["dtype"]]
    target = row_logits(case["logits"], n * (k + 1), vocab, vocab, gen)
    near = target.view(n, k + 1, vocab)[:, :k].reshape(n * k, vocab)
    draft = near + 0.7 * torch.randn(n * k, vocab, generator=gen, device="cuda") if case["draft"] != "point" else near
    target, draft = target.to(dtype), draft.to(dtype)
    s["mask"] = row_masks(n * (k + 1), vocab, case["mask"], gen) if case["mask"] else None
    # (the drafter samples from its own distribution at the request's temperature, under the masks of the same positions)
    at = torch.arange(n, device="cuda")
    cuts = plain_cuts(target, s["mask"], {f: v[at.repeat_interleave(k + 1)] for f, v in one.items()})
    warm = {f: v[at.repeat_interleave(k)] for f, v in row_params("temperature", n, gen).items()}
    s["draft_mask"] = None if s["mask"] is None else s["mask"].view(n, k + 1, -1)[:, :k].reshape(n * k, -1).contiguous()
    draft_cuts = plain_cuts(draft, s["draft_mask"], warm)
    q = plain_probs(draft, s["draft_mask"], draft_cuts, slice(None))
    cdf = q.cumsum(1)
    u = torch.rand(n * k, 1, dtype=torch.float64, generator=gen, device="cuda") * cdf[:, -1:]
    tokens = torch.searchsorted(cdf, u, right=True).clamp(max=vocab - 1)[:, 0]
    s["tokens"] = tokens.to(torch.int32).view(n, k)
    s["n_drafts"] = None
    if case["ragged"]:  # some requests have fewer drafts, and an eighth of the batch is padding
        s["n_drafts"] = torch.randint(0, k + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)
        s["n_drafts"][n - n // 8:] = -1
    if case["dtype"] == "probs":
        s["target"] = plain_probs(target, s["mask"], cuts, slice(None)).float()
        s["cuts"], s["draft_cuts"] = None, None
        s["draft"] = q.float()
    else:
        s["target"], s["cuts"], s["draft"], s["draft_cuts"] = target, cuts, draft, draft_cuts
    if case["draft"] == "point":
        s["draft"], s["draft_cuts"], s["draft_mask"] = None, None, None
    s["packed"] = {f: packed_cuts(s[f]) for f in ("cuts", "draft_cuts") if s[f] is not None}
    s["u"] = torch.rand(n, k + 1, generator=gen, device="cuda")
    s["seq_len"] = torch.randint(16, 32768, (n,), generator=gen, device="cuda", dtype=torch.int32)
    s["out"] = dict(tokens=torch.full((n, k + 1), -1, dtype=torch.int32, device="cuda"), accepted=torch.zeros(n, dtype=torch.int32, device="cuda"),
                    seq_len=s["seq_len"].clone())
    return s


def prepare_blocks(case, gen, s):
    n, size = case["requests"], case["block"]
    every = case["tokens"] // n
    longest = max(case["context"], 2)
    seq_len = torch.exp(torch.rand(n, generator=gen, device="cuda") * math.log(longest)).to(torch.int32)
    if case["kind"] == "decode":
        new_len = torch.full((n,), every, dtype=torch.int32, device="cuda")
    else:  # one token each, and the rest of the step's tokens in chunks of an eighth of the requests
        chunks = max(1, n // 8)
        new_len = torch.ones(n, dtype=torch.int32, device="cuda")
        at = torch.randperm(n, generator=gen, device="cuda")[:chunks]
        new_len[at] += (case["tokens"] - n) // chunks
    # a sixteenth of the requests have ended, the others hold what the last step had needed: a few tokens that were rejected
    ended = torch.rand(n, generator=gen, device="cuda") < 1 / 16
    rejected = torch.randint(0, 8, (n,), generator=gen, device="cuda", dtype=torch.int32)
    held = (seq_len + rejected + size - 1) // size
    seq_len, new_len = torch.where(ended, 0, seq_len), torch.where(ended, 0, new_len)
    # (the free list, the tables' rows and the step's tokens have the same sizes whatever the seed)
    widest = (longest + 8 + case["tokens"] + size - 1) // size
    free = 2 * n + case["tokens"] // size + 64
    in_tables = torch.arange(widest, device="cuda") < held[:, None]
    ids = torch.randperm(n * widest + free, generator=gen, device="cuda").to(torch.int32)
    table = torch.where(in_tables, ids[:n * widest].view(n, widest), -1).contiguous()
    stack = torch.full((n * widest + free,), -1, dtype=torch.int32, device="cuda")
    stack[:free] = ids[n * widest:]
    s.update(seq_len=seq_len, new_len=new_len, n_blocks=held.to(torch.int32), table=table, free=stack,
             n_free=torch.tensor([free], dtype=torch.int32, device="cuda"))
    most = case["tokens"]
    s["out"] = dict(n_blocks=torch.zeros(n, dtype=torch.int32, device="cuda"), n_free=torch.zeros(1, dtype=torch.int32, device="cuda"),
                    status=torch.zeros(n, dtype=torch.int32, device="cuda"), start=torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
                    slots=torch.zeros(most, dtype=torch.int64, device="cuda"), positions=torch.zeros(most, dtype=torch.int32, device="cuda"),
                    request=torch.zeros(most, dtype=torch.int32, device="cuda"))
    return s


# ---- the plain forms ----

def allowed_logits(x, mask):
    """fp32 logits; -inf where the mask has no bit, for NaN too; +inf as the largest finite value."""
    x = x.float()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=FLT_MAX)
    return x if mask is None else torch.where(mask_bits(mask, x.shape[1]), x, -math.inf)


def plain_cuts(logits, mask, p):
    """What temperature, min_p, top_k and top_p (in this order) leave of every row: a prefix of its tokens in the order of
    falling logits, equal ones by token."""
    x, ids = torch.sort(allowed_logits(logits, mask), dim=1, descending=True, stable=True)
    there = x > -math.inf
    top = x[:, :1]
    greedy = ~(p["temperature"] > 0)
    t = torch.where(greedy, 1.0, p["temperature"])[:, None].double()
    w = torch.where(there, torch.exp((x.double() - torch.where(there[:, :1], top, 0.0).double()) / t), 0.0)
    n = (there & (w >= p["min_p"][:, None].double())).sum(1)
    n = torch.maximum(n, there[:, 0].long())
    n = torch.where(p["top_k"] > 0, torch.minimum(n, p["top_k"].long()), n)
    n = torch.where(greedy, there[:, 0].long(), n)
    mass = w.cumsum(1)
    last = (n - 1).clamp(min=0)[:, None]
    under = (mass < p["top_p"][:, None].double() * mass.gather(1, last)).sum(1) + 1
    n = torch.where(p["top_p"] < 1, torch.minimum(n, under), n)
    last = (n - 1).clamp(min=0)[:, None]
    none, whole = n == 0, n == there.sum(1)  # (where nothing is cut off, the cut lies below every logit)
    return dict(total=torch.where(none, 0.0, mass.gather(1, last)[:, 0]), max=top[:, 0], temperature=torch.where(greedy, 0.0, p["temperature"]),
                cut=torch.where(whole, -math.inf, x.gather(1, last)[:, 0]), cut_token=torch.where(whole, -1, ids.gather(1, last)[:, 0]).to(torch.int32),
                n_kept=n.to(torch.int32), top_token=torch.where(none, -1, ids[:, 0]).to(torch.int32))


def plain_probs(logits, mask, c, rows):
    """fp64 probabilities of some rows under their cuts (None: the rows are probabilities; what is not positive and finite is 0)."""
    if c is None:
        p = logits[rows].double()
        return torch.where(torch.isfinite(p) & (p > 0), p, 0.0)
    c = {f: v[rows][:, None] for f, v in c.items()}
    x = allowed_logits(logits[rows], None if mask is None else mask[rows])
    at = torch.arange(x.shape[1], device=x.device)
    kept = (x > c["cut"]) | ((x == c["cut"]) & (at <= c["cut_token"]))
    t = torch.where(c["temperature"] > 0, c["temperature"], 1.0).double()
    return torch.where(kept & (c["n_kept"] > 0), torch.exp((x.double() - c["max"].double()) / t) / c["total"], 0.0)


def plain_one(logits, mask, c, rows, token):
    """... and of one token of each of them."""
    inside = (token >= 0) & (token < logits.shape[1])
    token = token.clamp(0, logits.shape[1] - 1)
    x = logits[rows, token].float()
    if c is None:
        x = x.double()
        return torch.where(inside & torch.isfinite(x) & (x > 0), x, 0.0)
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=FLT_MAX)
    if mask is not None:
        x = torch.where((mask[rows, token >> 5] >> (token & 31).to(torch.int32)) & 1 != 0, x, -math.inf)
    c = {f: v[rows] for f, v in c.items()}
    kept = (x > c["cut"]) | ((x == c["cut"]) & (token <= c["cut_token"]))
    t = torch.where(c["temperature"] > 0, c["temperature"], 1.0).double()
    return torch.where(inside & kept & (c["n_kept"] > 0), torch.exp((x.double() - c["max"].double()) / t) / c["total"], 0.0)


def plain_verify(s):
    n, k = s["tokens"].shape
    at = torch.arange(n, device="cuda")
    drafts = torch.full((n,), k, device="cuda") if s["n_drafts"] is None else s["n_drafts"].clamp(max=k)
    here = drafts >= 0
    step = torch.arange(k, device="cuda")
    d = s["tokens"].long()
    p = plain_one(s["target"], s["mask"], s["cuts"], (at[:, None] * (k + 1) + step).view(-1), d.view(-1)).view(n, k)
    if s["draft"] is None:
        q = torch.ones_like(p)
    else:
        q = plain_one(s["draft"], s["draft_mask"], s["draft_cuts"], (at[:, None] * k + step).view(-1), d.view(-1)).view(n, k)
    kept = (s["u"][:, :k].double() * q < p) & (step < drafts[:, None])
    accepted = kept.long().cumprod(1).sum(1)
    rejected = accepted < drafts
    token = d.gather(1, accepted.clamp(max=k - 1)[:, None])
    left = p_row = plain_probs(s["target"], s["mask"], s["cuts"], at * (k + 1) + accepted)
    if s["draft"] is None:
        at_draft = torch.arange(p_row.shape[1], device="cuda") == token
        left = torch.where(at_draft & rejected[:, None], 0.0, p_row)
    else:
        q_row = plain_probs(s["draft"], s["draft_mask"], s["draft_cuts"], at * k + accepted.clamp(max=k - 1))
        left = torch.where(rejected[:, None], (p_row - q_row).clamp(min=0), p_row)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, p_row)
    cdf = left.cumsum(1)
    total = cdf[:, -1:]
    u = s["u"].gather(1, torch.full((n, 1), k, device="cuda")).double()
    drawn = torch.searchsorted(cdf, u * total, right=True)[:, 0]
    last = torch.where(left > 0, torch.arange(left.shape[1], device="cuda"), -1).amax(1)
    drawn = torch.where(total[:, 0] > 0, torch.minimum(drawn, last), -1)
    place = torch.arange(k + 1, device="cuda")
    tokens = torch.where(place < accepted[:, None], torch.cat([d, d[:, :1]], 1), torch.where(place == accepted[:, None], drawn[:, None], -1))
    tokens = torch.where(here[:, None], tokens, s["out"]["tokens"]).to(torch.int32)
    count = accepted + (drawn >= 0)
    return dict(tokens=tokens, accepted=torch.where(here, accepted, s["out"]["accepted"]).to(torch.int32),
                seq_len=torch.where(here, s["seq_len"] + count, s["out"]["seq_len"]).to(torch.int32))


def plain_blocks(s):
    size, widest, most = s["case"]["block"], s["table"].shape[1], s["out"]["slots"].shape[0]
    seq, new, have = s["seq_len"].long(), s["new_len"].long(), s["n_blocks"].long().clamp(0, widest)
    here = (seq >= 0) & (new >= 0)
    want = torch.where(here, (seq + new + size - 1) // size, have)
    wide = want > widest
    want = torch.where(wide, have, want)
    # blocks that are no longer needed go onto the stack, request by request
    column = torch.arange(widest, device="cuda")
    back = (column >= want[:, None]) & (column < have[:, None])
    place = s["n_free"] + back.view(-1).long().cumsum(0) - 1
    stack = s["free"].clone()
    spare = torch.cat([stack, stack[:1]])
    spare[torch.where(back.view(-1), place, stack.shape[0])] = s["table"].view(-1)
    stack = spare[:-1]
    n_free = s["n_free"] + back.sum()
    # and those that are needed come off it in the requests' order, as far as they go
    need = (want - have).clamp(min=0)
    short = (need > 0) & (need.cumsum(0) > n_free)
    count = torch.where(here & ~wide & ~short, new, 0)
    full = count.cumsum(0) > most
    full &= count > 0
    count = torch.where(full, 0, count)
    need = torch.where(short | full, 0, need)
    first = need.cumsum(0) - need
    taken = column - have[:, None]
    gets = (taken >= 0) & (taken < need[:, None])
    source = (n_free - 1 - first[:, None] - taken).clamp(min=0)
    table = torch.where(gets, stack[source], s["table"])
    held = torch.where(want < have, want, have + need)
    start = torch.cat([count.new_zeros(1), count.cumsum(0)])
    token = torch.arange(most, device="cuda")
    request = torch.searchsorted(start, token, right=True) - 1
    inside = request < len(seq)
    request = request.clamp(max=len(seq) - 1)
    position = seq[request] + token - start[request]
    slot = table[request, (position // size).clamp(0, widest - 1)].long() * size + position % size
    status = torch.where(wide, 2, torch.where(short, 1, torch.where(full, 3, 0)))
    i32 = torch.int32
    return dict(table=table.to(i32), free=stack, n_blocks=held.to(i32), n_free=(n_free - need.sum()).to(i32), status=status.to(i32),
                start=start.to(i32), slots=torch.where(inside, slot, -1), positions=torch.where(inside, position, 0).to(i32),
                request=torch.where(inside, request, -1).to(i32))


# ---- the framework's operators ----

_contexts = {}  # the one in use: a program keeps its context for all its steps


def context(rows, vocab):
    from mako_amd import step
    key = (rows, vocab)
    if key not in _contexts:
        _contexts.clear()
        _contexts[key] = step.StepContext(max_rows=rows, max_vocab=vocab)
    return _contexts[key]


def bind(s):
    """The call of a state: (context, entry point, descriptor)."""
    from mako_amd import step
    case, out = s["case"], s["out"]

    def at(t):
        return None if t is None else t.data_ptr()

    if case["op"] == "cut":
        d = step.CutDesc()
        d.logits, d.logits_type, d.logits_stride = at(s["logits"]), step.LOGITS_TYPES[case["dtype"]], s["logits"].shape[1]
        d.n_rows, d.n_vocab, d.params = case["rows"], case["vocab"], at(s["packed"])
        if s["mask"] is not None:
            d.mask, d.mask_stride = at(s["mask"]), s["mask"].shape[1]
        d.out_cuts = at(out["cuts"])
        if case["probs"]:
            d.out_probs, d.probs_stride = at(out["probs"]), case["vocab"]
        ctx = context(case["rows"], case["vocab"])
        return ctx, ctx.cut_rows, d
    if case["op"] == "verify":
        n, k, vocab = case["requests"], case["drafts"], case["vocab"]
        kind = step.LOGITS_TYPES["float32" if case["dtype"] == "probs" else case["dtype"]]
        d = step.VerifyDesc()
        d.n_requests, d.max_drafts, d.n_vocab = n, k, vocab
        d.target, d.target_type, d.target_stride, d.target_cuts = at(s["target"]), kind, vocab, at(s["packed"].get("cuts"))
        if s["mask"] is not None:
            d.target_mask, d.target_mask_stride = at(s["mask"]), s["mask"].shape[1]
        if s["draft"] is not None:
            d.draft, d.draft_type, d.draft_stride, d.draft_cuts = at(s["draft"]), kind, vocab, at(s["packed"].get("draft_cuts"))
            if s["draft_mask"] is not None:
                d.draft_mask, d.draft_mask_stride = at(s["draft_mask"]), s["draft_mask"].shape[1]
        d.draft_tokens, d.n_drafts, d.u, d.seq_len = at(s["tokens"]), at(s["n_drafts"]), at(s["u"]), at(s["seq_len"])
        d.out_tokens, d.out_accepted, d.out_seq_len = at(out["tokens"]), at(out["accepted"]), at(out["seq_len"])
        ctx = context(n, vocab)
        return ctx, ctx.verify_drafts, d
    d = step.BlocksDesc()
    d.n_requests, d.block_size, d.max_tokens = case["requests"], case["block"], out["slots"].shape[0]
    d.seq_len, d.new_len = at(s["seq_len"]), at(s["new_len"])
    d.block_table, d.table_stride, d.max_blocks = at(s["table"]), s["table"].shape[1], s["table"].shape[1]
    d.n_blocks, d.out_n_blocks = at(s["n_blocks"]), at(out["n_blocks"])
    d.free_blocks, d.free_capacity, d.n_free, d.out_n_free = at(s["free"]), s["free"].shape[0], at(s["n_free"]), at(out["n_free"])
    d.out_start, d.out_status = at(out["start"]), at(out["status"])
    d.out_slots, d.out_positions, d.out_request = at(out["slots"]), at(out["positions"]), at(out["request"])
    ctx = context(case["requests"], 1)
    return ctx, ctx.assign_blocks, d


def cut_fields(cuts):
    """A row's cut as its fields (views of the records)."""
    f = cuts.view(torch.float32)
    return dict(total=cuts[:, :2].view(torch.float64)[:, 0], max=f[:, 2], temperature=f[:, 3], cut=f[:, 4], cut_token=cuts[:, 5], n_kept=cuts[:, 6],
                top_token=cuts[:, 7])


def run(s):
    op = s["case"]["op"]
    if own:
        if "call" not in s:
            s["call"] = bind(s)
        _, call, desc = s["call"]
        call(desc)
        if op == "blocks":
            return dict(s["out"], table=s["table"], free=s["free"])
        return s["out"] if op == "verify" else dict(cut_fields(s["out"]["cuts"]), **{f: s["out"][f] for f in s["out"] if f == "probs"})
    if op == "blocks":
        return plain_blocks(s)
    if op == "verify":
        return plain_verify(s)
    c = plain_cuts(s["logits"][:, :s["case"]["vocab"]], s["mask"], s["params"])
    if s["case"]["probs"]:
        c["probs"] = plain_probs(s["logits"][:, :s["case"]["vocab"]], s["mask"], c, slice(None)).float()
    return c


def work(case):
    """Each input read once and each output written once; of a verification the one row that a token is drawn from, and
    the drafter's beside it.  An exponential counts as one operation."""
    if case["op"] == "blocks":
        n, t = case["requests"], case["tokens"]
        return dict(bytes=n * (4 * 6) + 16 * t + 4 * t // case["block"] * 2, flops=4 * t)
    size = DTYPES[case["dtype"]].itemsize
    words = (case["vocab"] + 31) // 32 * 4 if case["mask"] else 0
    if case["op"] == "cut":
        row = case["vocab"] * (size + (4 if case["probs"] else 0)) + words + 28 + 32
        return dict(bytes=case["rows"] * row, flops=case["rows"] * case["vocab"] * 4)
    row = (case["vocab"] * size + words) * (1 if case["draft"] == "point" else 2) + (case["drafts"] + 1) * 100
    return dict(bytes=case["requests"] * row, flops=case["requests"] * case["vocab"] * 8)


# ---- the definitions in 64 bits ----

def exact_weights(x, mask, t):
    """(weights in 64 bits, the logits as 64-bit numbers)."""
    x = x.to(torch.float64)
    x = torch.nan_to_num(x, nan=-math.inf, posinf=FLT_MAX, neginf=-math.inf)
    if mask is not None:
        token = torch.arange(x.shape[1], device=x.device)
        x = x.masked_fill(torch.bitwise_and(torch.bitwise_right_shift(mask.long()[:, token // 32], token % 32), 1) == 0, -math.inf)
    m = x.amax(1, keepdim=True)
    w = torch.where(torch.isfinite(x), torch.exp((x - torch.where(torch.isfinite(m), m, 0.0)) / t[:, None]), 0.0)
    return w, x


def exact_cut(x, mask, temperature, top_k, top_p, min_p):
    """(one row's kept tokens in falling order, all tokens' weights, whether tokens were cut off)."""
    w, x = exact_weights(x[None], mask if mask is None else mask[None], torch.tensor([temperature if temperature > 0 else 1.0], dtype=torch.float64, device=x.device))
    w, x = w[0], x[0]
    order = torch.argsort(x, descending=True, stable=True)
    order = order[:int(torch.isfinite(x).sum())]
    if not len(order):
        return order, w, False
    if not temperature > 0:
        return order[:1], w, len(order) > 1
    keep = len(order)
    if min_p > 0:
        keep = max(1, int((w >= min_p).sum()))
    if top_k > 0:
        keep = min(keep, top_k)
    if top_p < 1:
        run_ = torch.cumsum(w[order[:keep]], 0)
        keep = min(keep, int(torch.searchsorted(run_, (top_p * run_[-1]).view(1))) + 1)
    return order[:keep], w, keep < len(order)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "blocks":
        return exact_blocks(case, s)
    if case["op"] == "cut":
        p = {f: s["params"][f].double().tolist() for f in PARAMS}
        found = []
        probs = torch.zeros(case["rows"], case["vocab"], dtype=torch.float64, device="cuda") if case["probs"] else None
        for r in range(case["rows"]):
            x = s["logits"][r, :case["vocab"]]
            kept, w, off = exact_cut(x, None if s["mask"] is None else s["mask"][r], p["temperature"][r], int(p["top_k"][r]), p["top_p"][r], p["min_p"][r])
            total = w[kept].sum()
            t = max(p["temperature"][r], 0.0)
            last = (float(x[kept[-1]].double().clamp(max=FLT_MAX)), int(kept[-1])) if off else (-math.inf, -1)
            first = (float(x[kept[0]].double().clamp(max=FLT_MAX)), int(kept[0])) if len(kept) else (-math.inf, -1)
            found.append([float(total), first[0], t, *last, len(kept), first[1]])
            if probs is not None and len(kept):
                probs[r, kept] = w[kept] / total
        f = torch.tensor(found, dtype=torch.float64).T
        out = dict(total=f[0], max=f[1], temperature=f[2], cut=f[3], cut_token=f[4].to(torch.int32), n_kept=f[5].to(torch.int32), top_token=f[6].to(torch.int32))
        if probs is not None:
            out["probs"] = probs
        return out
    return exact_verify(case, s)


def exact_row(s, which, row):
    """A row's probabilities in 64 bits, from its cut."""
    logits, mask, c = s[which], s["mask" if which == "target" else "draft_mask"], s["cuts" if which == "target" else "draft_cuts"]
    if c is None:
        return torch.nan_to_num(logits[row].double(), nan=0.0, posinf=0.0).clamp(min=0)
    c = {f: v[row] for f, v in c.items()}
    t = c["temperature"].double()
    w, x = exact_weights(logits[row][None], None if mask is None else mask[row][None], torch.where(t > 0, t, 1.0)[None])
    w, x = w[0], x[0]
    below = (x < c["cut"].double()) | ((x == c["cut"].double()) & (torch.arange(len(x), device=x.device) > c["cut_token"]))
    return w.masked_fill(below, 0.0) / c["total"]


def exact_verify(case, s):
    n, k = s["tokens"].shape
    tokens, accepted, seq_len = (s["out"][f].clone() for f in ("tokens", "accepted", "seq_len"))
    us, ds = s["u"].double().tolist(), s["tokens"].tolist()
    for b in range(n):
        drafts = k if s["n_drafts"] is None else int(s["n_drafts"][b])
        if drafts < 0:
            continue
        j, left = 0, None
        while True:
            p = exact_row(s, "target", b * (k + 1) + j)
            if j == drafts:
                left = p
                break
            d = ds[b][j]
            q = None if s["draft"] is None else exact_row(s, "draft", b * k + j)
            if us[b][j] * (1.0 if q is None else float(q[d])) < float(p[d]):
                j += 1
                continue
            left = p.clone()
            if q is None:
                left[d] = 0.0
            else:
                left = torch.relu(p - q)
            if not float(left.sum()) > 0:
                left = p
            break
        run_ = torch.cumsum(left, 0)
        got = ds[b][:j]
        if float(run_[-1]) > 0:
            got = got + [min(int((run_ <= us[b][k] * run_[-1]).sum()), int(torch.nonzero(left)[-1]))]
        accepted[b] = j
        seq_len[b] = s["seq_len"][b] + len(got)
        tokens[b] = torch.tensor(got + [-1] * (k + 1 - len(got)), dtype=torch.int32)
    return dict(tokens=tokens, accepted=accepted, seq_len=seq_len)


def exact_blocks(case, s):
    """Request by request, on the host."""
    size, most = case["block"], case["tokens"]
    table, widest = s["table"].cpu().numpy().copy(), s["table"].shape[1]
    stack, n_free = s["free"].cpu().numpy().copy(), int(s["n_free"])
    seq, new, have = s["seq_len"].tolist(), s["new_len"].tolist(), s["n_blocks"].tolist()
    n = len(seq)
    status, want, held = [0] * n, [0] * n, list(have)
    for b in range(n):
        want[b] = -(-(seq[b] + new[b]) // size) if seq[b] >= 0 and new[b] >= 0 else have[b]
        if want[b] > widest:
            status[b] = 2
            continue
        for i in range(want[b], have[b]):
            stack[n_free] = table[b, i]
            n_free += 1
        held[b] = min(have[b], want[b])
    asked, available, start, tokens = 0, n_free, [0], 0
    slots, positions, request = [], [], []
    for b in range(n):
        need = 0 if status[b] == 2 else max(0, want[b] - held[b])
        asked += need
        count = max(new[b], 0) if seq[b] >= 0 and status[b] == 0 else 0
        if need and asked > available:
            status[b], count, need = 1, 0, 0
        tokens += count
        if count and tokens > most:
            status[b], count, need = 3, 0, 0
        for _ in range(need):
            n_free -= 1
            table[b, held[b]] = stack[n_free]
            held[b] += 1
        for i in range(count):
            at = seq[b] + i
            slots.append(int(table[b, at // size]) * size + at % size)
            positions.append(at)
            request.append(b)
        start.append(len(slots))
    pad = most - len(slots)

    def whole(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype)

    return dict(table=torch.from_numpy(table), free=torch.from_numpy(stack), n_blocks=whole(held), n_free=whole([n_free]), status=whole(status),
                start=whole(start), slots=whole(slots + [-1] * pad, torch.int64), positions=whole(positions + [0] * pad), request=whole(request + [-1] * pad))
