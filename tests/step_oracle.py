"""Plain restatements in 64 bits (numpy, row by row) of the operators of include/mako_step.h, and what their tests share."""
import ctypes

import numpy as np

from mako_amd import api, hip, step

FLT_MAX = np.finfo(np.float32).max


# ---- types ----

def to_bf16(x):
    """fp32 -> the bits of bfloat16, to nearest even (NaN stays NaN)."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def encode(x, dtype):
    """(the array a call gets, the same values as fp32)."""
    if dtype == "bfloat16":
        b = to_bf16(x)
        return b, (b.astype(np.uint32) << 16).view(np.float32)
    if dtype == "float16":
        with np.errstate(over="ignore"):
            h = np.asarray(x, np.float16)
        return h, h.astype(np.float32)
    x = np.ascontiguousarray(x, np.float32)
    return x, x


def pack_mask(bits):
    """bool [rows, V] -> uint32 words [rows, ceil(V / 32)]."""
    rows, v = bits.shape
    b = np.zeros((rows, (v + 31) // 32 * 32), np.uint8)
    b[:, :v] = bits
    return np.packbits(b, axis=1, bitorder="little").view(np.uint32)


# ---- definitions ----

def token_logits(x, bits=None):
    """fp64 logits, -inf for what is no token."""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, float(FLT_MAX))
    if bits is not None:
        x[~bits] = -np.inf
    return x


def cut_row(x, p, bits=None):
    """(record, kept ids in falling order, their weights) of one row."""
    x = token_logits(x, bits)
    ids = np.lexsort((np.arange(len(x)), -x))
    ids = ids[x[ids] > -np.inf]
    out = np.zeros((), step.CUT_DTYPE)
    t = float(p["temperature"])
    greedy = not t > 0
    out["temperature"] = 0 if greedy else p["temperature"]
    out["max_logit"], out["cut_logit"], out["cut_token"], out["top_token"] = -np.inf, -np.inf, -1, -1
    if not len(ids):
        return out, ids, np.zeros(0)
    with np.errstate(over="ignore", under="ignore"):
        w = np.exp((x[ids] - x[ids[0]]) / (1.0 if greedy else t))
    n = 1 if greedy else len(ids)
    if not greedy:
        if p["min_p"] > 0:
            n = max(1, int((w >= float(p["min_p"])).sum()))
        if p["top_k"] > 0:
            n = min(n, int(p["top_k"]))
        if p["top_p"] < 1:
            mass = np.cumsum(w[:n])
            n = min(n, int(np.searchsorted(mass, float(p["top_p"]) * mass[-1])) + 1)
    out["total"], out["max_logit"], out["n_kept"], out["top_token"] = w[:n].sum(), x[ids[0]], n, ids[0]
    if n < len(ids):
        out["cut_logit"], out["cut_token"] = x[ids[n - 1]], ids[n - 1]
    return out, ids[:n], w[:n]


def probs_row(x, cut, bits=None):
    """A row's probabilities in 64 bits: under its cut, or (cut None) as they are."""
    if cut is None:
        x = np.asarray(x, np.float64)
        return np.where(np.isfinite(x) & (x > 0), x, 0.0)
    x = token_logits(x, bits)
    kept = (x > cut["cut_logit"]) | ((x == cut["cut_logit"]) & (np.arange(len(x)) <= cut["cut_token"]))
    kept &= x > -np.inf
    t = float(cut["temperature"]) or 1.0
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        return np.where(kept, np.exp((x - float(cut["max_logit"])) / t) / cut["total"], 0.0) if cut["n_kept"] else np.zeros(len(x))


def verify_request(p_row, q_row, tokens, drafts, u, max_drafts):
    """(tokens given out, accepted drafts); p_row(j), q_row(j): the distributions at place j (q_row None: no drafter's)."""
    j = 0
    while True:
        p = p_row(j)
        left = p
        if j == drafts:
            break
        d = int(tokens[j])
        inside = 0 <= d < len(p)
        q = None if q_row is None else q_row(j)
        qd = 1.0 if q is None else (q[d] if inside else 0.0)
        if float(u[j]) * qd < (p[d] if inside else 0.0):
            j += 1
            continue
        if q is None:
            left = p.copy()
            if inside:
                left[d] = 0.0
        else:
            left = np.maximum(p - q, 0.0)
        if not left.sum() > 0:
            left = p
        break
    got = [int(t) for t in tokens[:j]]
    run = np.cumsum(left)
    if run[-1] > 0:
        got.append(min(int(np.searchsorted(run, float(u[max_drafts]) * run[-1], side="right")), int(np.nonzero(left)[0][-1])))
    return got, j


def assign_blocks(seq, new, have, table, stack, n_free, size, max_blocks, max_tokens):
    """(table, stack, blocks held, n_free, status, start, slots, positions, request), request by request."""
    table, stack = table.copy(), stack.copy()
    n, capacity = len(seq), len(stack)
    n_free = min(max(int(n_free), 0), capacity)
    have = [min(max(int(h), 0), max_blocks) for h in have]
    status, held, need, count = [0] * n, list(have), [0] * n, [0] * n
    for b in range(n):
        if seq[b] < 0 or new[b] < 0:
            continue
        total = int(seq[b]) + int(new[b])
        want = -(-total // size)
        if want > max_blocks or total > 2**31 - 1:
            status[b] = step.BLOCKS_WIDE
            continue
        count[b], need[b] = int(new[b]), max(0, want - have[b])
        for i in range(want, have[b]):
            if n_free < capacity:
                stack[n_free] = table[b, i]
                n_free += 1
        held[b] = min(have[b], want)
    asked, tokens, available, start = 0, 0, n_free, [0]
    slots, positions, request = [], [], []
    for b in range(n):
        if status[b] == step.BLOCKS_WIDE:
            count[b] = need[b] = 0
        asked += need[b]
        if need[b] and asked > available:
            status[b], count[b], need[b] = step.BLOCKS_SHORT, 0, 0
        tokens += count[b]
        if count[b] and tokens > max_tokens:
            status[b], count[b], need[b] = step.BLOCKS_TOKENS, 0, 0
        for _ in range(need[b]):
            n_free -= 1
            table[b, held[b]] = stack[n_free]
            held[b] += 1
        for i in range(count[b]):
            at = int(seq[b]) + i
            slots.append(int(table[b, at // size]) * size + at % size)
            positions.append(at)
            request.append(b)
        start.append(len(slots))
    pad = max_tokens - len(slots)
    return dict(table=table, free=stack, n_blocks=np.array(held, np.int32), n_free=np.array([n_free], np.int32), status=np.array(status, np.int32),
                start=np.array(start, np.int32), slots=np.array(slots + [-1] * pad, np.int64), positions=np.array(positions + [0] * pad, np.int32),
                request=np.array(request + [-1] * pad, np.int32))


# ---- calls ----

class Buffers:
    """Device copies of host arrays, kept until the call is over."""

    def __init__(self):
        self.keep = []

    def up(self, a):
        if a is None:
            return None
        d = hip.DeviceArray.from_host(np.ascontiguousarray(a))
        self.keep.append(d)
        return d.ptr

    def out(self, a):
        d = hip.DeviceArray.from_host(np.ascontiguousarray(a))
        self.keep.append(d)
        return d


def cut_rows(ctx, x, params, dtype="float32", bits=None, pad=0, offset=0, rows_per_params=1, probs=False, mask_pad=0, stream=None):
    """(records, probabilities or None) of the device path; `offset`: elements before the first row, `pad`: behind each."""
    rows, v = x.shape
    raw, _ = encode(x, dtype)
    room = np.zeros(offset + rows * (v + pad), raw.dtype)
    if pad or offset:
        room[:] = encode(np.full(1, 1e4, np.float32), dtype)[0][0]  # (what lies between rows would win)
    room[offset:].reshape(rows, v + pad)[:, :v] = raw
    b = Buffers()
    d = step.CutDesc()
    d.logits = b.up(room) + offset * raw.dtype.itemsize
    d.logits_type, d.logits_stride, d.n_rows, d.n_vocab = step.LOGITS_TYPES[dtype], v + pad, rows, v
    d.params, d.rows_per_params = b.up(np.ascontiguousarray(params, api.PARAMS_DTYPE)), rows_per_params
    if bits is not None:
        words = pack_mask(bits)
        words = np.concatenate([words, np.full((rows, mask_pad), 0xFFFFFFFF, np.uint32)], 1)
        d.mask, d.mask_stride = b.up(words), words.shape[1]
    cuts = b.out(np.full(rows * step.CUT_DTYPE.itemsize, 0xA5, np.uint8))
    d.out_cuts = cuts.ptr
    if probs:
        dense = b.out(np.full((rows, v + 3), 7.0, np.float32))
        d.out_probs, d.probs_stride = dense.ptr, v + 3
    ctx.cut_rows(d, stream)
    hip.synchronize()
    got = cuts.download().view(step.CUT_DTYPE)
    if not probs:
        return got, None
    p = dense.download()
    assert (p[:, v:] == 7.0).all(), "written behind the rows"
    return got, p[:, :v]


def verify_desc(b, target, target_cuts, tokens, u, target_type="float32", target_bits=None, draft=None, draft_cuts=None, draft_type="float32",
                draft_bits=None, n_drafts=None, seq_len=None):
    """A VerifyDesc over device copies in `b`, and its outputs' arrays."""
    n, k = tokens.shape
    d = step.VerifyDesc()
    d.n_requests, d.max_drafts, d.n_vocab = n, k, target.shape[1]
    raw = encode(target, target_type)[0]
    d.target, d.target_type, d.target_stride, d.target_cuts = b.up(raw), step.LOGITS_TYPES[target_type], raw.shape[1], b.up(target_cuts)
    if target_bits is not None:
        words = pack_mask(target_bits)
        d.target_mask, d.target_mask_stride = b.up(words), words.shape[1]
    if draft is not None:
        raw = encode(draft, draft_type)[0]
        d.draft, d.draft_type, d.draft_stride, d.draft_cuts = b.up(raw), step.LOGITS_TYPES[draft_type], raw.shape[1], b.up(draft_cuts)
        if draft_bits is not None:
            words = pack_mask(draft_bits)
            d.draft_mask, d.draft_mask_stride = b.up(words), words.shape[1]
    d.draft_tokens = b.up(tokens.astype(np.int32)) if k else None
    d.n_drafts = b.up(None if n_drafts is None else np.asarray(n_drafts, np.int32))
    d.u = b.up(u.astype(np.float32))
    out = dict(tokens=b.out(np.full((n, k + 1), -77, np.int32)), accepted=b.out(np.full(n, -77, np.int32)))
    d.out_tokens, d.out_accepted = out["tokens"].ptr, out["accepted"].ptr
    if seq_len is not None:
        out["seq_len"] = b.out(np.asarray(seq_len, np.int32))
        d.seq_len = d.out_seq_len = out["seq_len"].ptr  # (in place)
    return d, out


def call_raw(ctx, name, desc):
    """The C call itself: (status, text)."""
    rc = getattr(ctx.lib, name)(ctx.ptr, ctypes.byref(desc), None)
    return rc, ctx.last_error()
