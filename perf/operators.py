"""The prompt operators: the cases that stand for their use, their plain forms and their definitions in 64 bits.

Three operators carry a prompt through the two kinds of attention layer of a
Kimi-Linear decoder, each over one sequence, a batch of equal ones, or
sequences of different lengths packed one behind the other:

* ``conv`` -- the width-4 causal convolutions with SiLU before a KDA layer,
  ``kernels.short_conv_prefill_triple``;
* ``scan`` -- the KDA recurrence with its carried state,
  ``kernels.kda_prefill``;
* ``attention`` -- causal attention with grouped heads, over the prompt alone
  or over the prompt behind a prefix whose keys are already there,
  ``kernels.attention_prefill``.

Layouts are those of the decoder: 32 KDA heads of 128 (convolutions of 4096
channels), full attention with 192-wide queries and keys (128 + 64) and
128-wide values; grouped heads and other widths are generic.
"""

from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
WIDTH = 4  # taps of the short convolutions


# ---------------------------------------------------------------------------
# the cases
#
# "tokens" is the whole call's; "sequences" of them are packed, ragged where
# "ragged", else a batch of equal lengths. "prefix" is the longest prefix whose
# keys (attention) lie before a sequence's own.


def listed() -> list[dict]:
    return [
        # a short chat turn's convolutions in one decoder layer: launch latency
        {"name": "conv_turn", "op": "conv", "tokens": 19, "sequences": 1, "ragged": False,
         "channels": 4096, "dtype": "bfloat16"},
        # the prompts that a serving step packs together, some continued from earlier pieces
        {"name": "conv_packed", "op": "conv", "tokens": 4096, "sequences": 23, "ragged": True,
         "channels": 4096, "dtype": "bfloat16"},
        # a long prompt, fp16 activations, a channel count of no large power of two
        {"name": "conv_long", "op": "conv", "tokens": 16384, "sequences": 1, "ragged": False,
         "channels": 2304, "dtype": "float16"},
        # a short chat turn through the recurrence: latency
        {"name": "scan_turn", "op": "scan", "tokens": 19, "sequences": 1, "ragged": False,
         "heads": 32, "d_k": 128, "d_v": 128, "dtype": "bfloat16"},
        # prompts of different lengths packed into one call
        {"name": "scan_packed", "op": "scan", "tokens": 4096, "sequences": 11, "ragged": True,
         "heads": 32, "d_k": 128, "d_v": 128, "dtype": "bfloat16"},
        # one long prompt: its steps follow one another
        {"name": "scan_long", "op": "scan", "tokens": 8192, "sequences": 1, "ragged": False,
         "heads": 32, "d_k": 128, "d_v": 128, "dtype": "bfloat16"},
        # a batch of equal prompts in fp32 with small heads
        {"name": "scan_batch_fp32", "op": "scan", "tokens": 2000, "sequences": 4, "ragged": False,
         "heads": 16, "d_k": 64, "d_v": 96, "dtype": "float32"},
        # a short chat turn's full attention: latency
        {"name": "attention_turn", "op": "attention", "tokens": 19, "sequences": 1, "ragged": False,
         "prefix": 0, "heads": 32, "kv_heads": 32, "d_qk": 192, "d_v": 128, "dtype": "bfloat16"},
        # prompts of different lengths packed into one call
        {"name": "attention_packed", "op": "attention", "tokens": 4096, "sequences": 11,
         "ragged": True, "prefix": 0, "heads": 32, "kv_heads": 32, "d_qk": 192, "d_v": 128,
         "dtype": "bfloat16"},
        # the next pieces of prompts whose earlier keys are in hand
        {"name": "attention_continued", "op": "attention", "tokens": 777, "sequences": 3,
         "ragged": True, "prefix": 6000, "heads": 32, "kv_heads": 32, "d_qk": 192, "d_v": 128,
         "dtype": "bfloat16"},
        # grouped heads in fp16, two prompts of one length
        {"name": "attention_grouped", "op": "attention", "tokens": 4096, "sequences": 2,
         "ragged": False, "prefix": 0, "heads": 32, "kv_heads": 8, "d_qk": 128, "d_v": 128,
         "dtype": "float16"},
        # one long prompt
        {"name": "attention_long", "op": "attention", "tokens": 8192, "sequences": 1,
         "ragged": False, "prefix": 0, "heads": 32, "kv_heads": 32, "d_qk": 192, "d_v": 128,
         "dtype": "bfloat16"},
    ]


def _log_int(rng, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    op = rng.choice(["conv", "scan", "scan", "attention", "attention"])
    tokens = _log_int(rng, 1, 8192)
    sequences = 1 if rng.random() < 0.4 else min(tokens, _log_int(rng, 2, 48))
    ragged = sequences > 1 and rng.random() < 0.75
    if not ragged:
        tokens -= tokens % sequences
    case = {"op": op, "tokens": tokens, "sequences": sequences, "ragged": ragged}
    if op == "conv":
        return {**case, "channels": rng.choice([4096, 2304, 512, rng.randrange(1, 4096)]),
                "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    if op == "scan":
        d_k, d_v = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128),
                               (rng.randrange(1, 33) * 4, rng.randrange(1, 129))])
        return {**case, "heads": rng.choice([32, 16, rng.randrange(1, 32)]), "d_k": d_k,
                "d_v": d_v, "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (16, 2), (8, 1), (6, 3), (5, 5)])
    d_qk, d_v = rng.choice([(192, 128), (192, 128), (128, 128), (64, 64),
                            (rng.randrange(1, 25) * 8, rng.randrange(1, 17) * 8)])
    prefix = _log_int(rng, 1, 4096) if tokens <= 2048 and rng.random() < 0.5 else 0
    return {**case, "prefix": prefix, "heads": heads, "kv_heads": kv_heads, "d_qk": d_qk,
            "d_v": d_v, "dtype": rng.choice(["bfloat16", "bfloat16", "float16"])}


def _lengths(case: dict) -> list[int]:
    """Tokens of each sequence. Ragged ones are cut at places drawn from the
    sizes alone (some sequences come out empty or with one token)."""
    tokens, n = case["tokens"], case["sequences"]
    if not case["ragged"]:
        return [tokens // n] * n
    rng = random.Random(tokens * 131 + n)
    cuts = sorted(rng.randint(0, tokens) for _ in range(n - 1))
    return [b - a for a, b in zip([0, *cuts], [*cuts, tokens])]


def _prefixes(case: dict) -> list[int]:
    if not case.get("prefix"):
        return [0] * case["sequences"]
    if not case["ragged"]:
        return [case["prefix"]] * case["sequences"]
    rng = random.Random(case["prefix"] * 131 + case["sequences"])
    return [case["prefix"], *(rng.randint(0, case["prefix"]) for _ in range(case["sequences"] - 1))]


# ---------------------------------------------------------------------------
# inputs


def _offsets(lengths) -> list[int]:
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _inputs(case: dict, seed: int) -> dict:
    """The operands alone, from the seed (shared by prepare and exact)."""
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 29)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=DEV).mul_(std).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=DEV)

    op, t, n = case["op"], case["tokens"], case["sequences"]
    lengths = _lengths(case)
    rows = (1, t) if case["ragged"] else (n, t // n)
    dtype = getattr(torch, case["dtype"])
    # every second sequence goes on from an earlier piece, the others start afresh
    carried = (torch.arange(n, device=DEV) % 2).float()
    d = {"op": op, "lengths": lengths}
    if op == "conv":
        c = case["channels"]
        d["in"] = [normal(*rows, c, dtype=dtype) for _ in range(3)]
        d["state"] = [(normal(n, c, WIDTH) * carried[:, None, None]).to(dtype) for _ in range(3)]
        d["weight"] = [normal(c, 1, WIDTH, std=0.5, dtype=dtype) for _ in range(3)]
        return d
    if op == "scan":
        h, dk, dv = case["heads"], case["d_k"], case["d_v"]
        # what the gates of a KDA layer give: unit keys and queries, a log
        # decay -exp(a_log) softplus(x + bias) with rates of 1 to 16 and steps of 0.001 to 0.1
        # about the bias, and beta a sigmoid
        for name in ("q", "k"):
            x = normal(*rows, h, dk)
            d[name] = x * torch.rsqrt(x.square().sum(-1, keepdim=True) + 1e-6)
        step = torch.exp(uniform(h, dk) * math.log(100.0) + math.log(1e-3))
        bias = step + torch.log(-torch.expm1(-step))
        rate = 1.0 + 15.0 * uniform(h, 1)
        d["decay"] = -rate * torch.nn.functional.softplus(normal(*rows, h, dk) + bias)
        d["beta"] = torch.sigmoid(normal(*rows, h))
        d["v"] = normal(*rows, h, dv, dtype=dtype)
        d["state"] = normal(n, h, dk, dv, std=0.1) * carried[:, None, None, None]
        d["scale"] = dk ** -0.5
        return d
    prefixes = _prefixes(case)
    keys = [a + b for a, b in zip(lengths, prefixes)]
    key_rows = (1, sum(keys)) if case["ragged"] else (n, keys[0])
    d["q"] = normal(*rows, case["heads"], case["d_qk"], dtype=dtype)
    d["k"] = normal(*key_rows, case["kv_heads"], case["d_qk"], dtype=dtype)
    d["v"] = normal(*key_rows, case["kv_heads"], case["d_v"], dtype=dtype)
    d["scale"] = case["d_qk"] ** -0.5
    d["key_lengths"] = keys
    return d


def prepare(case: dict, seed: int):
    """The call's operands, and what a serving step keeps beside them: the
    offsets of packed sequences and the buffers that take the next states (the
    states read are a shared prefix's and stay as they are)."""
    d = _inputs(case, seed)
    d["cu_seqlens"] = d["cu_seqlens_k"] = None
    if case["ragged"]:
        d["cu_seqlens"] = torch.tensor(_offsets(d["lengths"]), dtype=torch.int32, device=DEV)
        if case.get("prefix"):
            d["cu_seqlens_k"] = torch.tensor(_offsets(d["key_lengths"]), dtype=torch.int32,
                                             device=DEV)
    if d["op"] == "conv":
        d["state_out"] = [torch.empty_like(s) for s in d["state"]]
    elif d["op"] == "scan":
        d["state_out"] = torch.empty_like(d["state"])
    return d


# ---------------------------------------------------------------------------
# one pass


def _rows_of(cu, lengths, tokens):
    """Sequence and position of every token of the flattened rows."""
    dev = torch.device(DEV)
    if cu is None:
        at = torch.arange(tokens, device=dev)
        return at // max(1, lengths[0]), at % max(1, lengths[0])
    at = torch.arange(tokens, device=dev)
    seq = (at[:, None] >= cu[None, 1:]).sum(1)
    return seq, at - cu.long()[seq]


def _plain_conv(s):
    outs, states = [], []
    x0 = s["in"][0]
    tokens, channels = x0.shape[0] * x0.shape[1], x0.shape[2]
    seq, pos = _rows_of(s["cu_seqlens"], s["lengths"], tokens)
    n = len(s["lengths"])
    length = torch.bincount(seq, minlength=n)
    start = torch.cumsum(length, 0) - length
    tap = torch.arange(WIDTH, device=x0.device)
    # rows of a table that holds the tokens first, then each sequence's four state rows
    back = pos[:, None] + tap - (WIDTH - 1)
    window = torch.where(back >= 0, start[seq][:, None] + back,
                         tokens + seq[:, None] * WIDTH + WIDTH + back)
    last = length[:, None] + tap - WIDTH
    kept = torch.where(last >= 0, start[:, None] + last,
                       tokens + torch.arange(n, device=x0.device)[:, None] * WIDTH + WIDTH + last)
    for x, state, weight, out in zip(s["in"], s["state"], s["weight"], s["state_out"]):
        table = torch.cat((x.reshape(tokens, channels),
                           state.transpose(1, 2).reshape(n * WIDTH, channels)))
        y = (table[window].float() * weight[:, 0, :].float().t()).sum(1)
        outs.append((y / (1.0 + torch.exp(-y))).to(x.dtype).reshape(x.shape))
        out.copy_(table[kept].transpose(1, 2))
        states.append(out)
    return outs + states


def _plain_scan(s):
    # the recurrence itself, a step for each position, all sequences and heads at once
    v = s["v"]
    tokens, (heads, dv), dk = v.shape[0] * v.shape[1], v.shape[2:], s["q"].shape[-1]
    seq, pos = _rows_of(s["cu_seqlens"], s["lengths"], tokens)
    n, longest = len(s["lengths"]), max(s["lengths"])

    def padded(x, width):
        p = torch.zeros((longest, n, heads, width), dtype=torch.float32, device=x.device)
        p[pos, seq] = x.reshape(tokens, heads, width).float()
        return p

    q, k, vp = padded(s["q"] * s["scale"], dk), padded(s["k"], dk), padded(v, dv)
    keep, beta = torch.exp(padded(s["decay"], dk)), padded(s["beta"], 1)
    state = s["state"].clone()
    out = torch.empty((longest, n, heads, dv), dtype=torch.float32, device=v.device)
    for t in range(longest):
        state.mul_(keep[t].unsqueeze(-1))
        delta = beta[t] * (vp[t] - (state * k[t].unsqueeze(-1)).sum(-2))
        state.addcmul_(k[t].unsqueeze(-1), delta.unsqueeze(-2))
        torch.sum(state * q[t].unsqueeze(-1), dim=-2, out=out[t])
    s["state_out"].copy_(state)
    return [out[pos, seq].to(v.dtype).reshape(v.shape), s["state_out"]]


def _plain_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    heads, kv_heads, dv = q.shape[2], k.shape[2], v.shape[3]
    if s["cu_seqlens"] is None:  # a batch of equal sequences
        pos = torch.arange(q.shape[1], device=q.device) + (k.shape[1] - q.shape[1])
        seen = torch.arange(k.shape[1], device=q.device)[None, :] <= pos[:, None]
    else:
        cu_k = s["cu_seqlens"] if s["cu_seqlens_k"] is None else s["cu_seqlens_k"]
        seq, pos = _rows_of(s["cu_seqlens"], s["lengths"], q.shape[1])
        seq_k, pos_k = _rows_of(cu_k, s["key_lengths"], k.shape[1])
        ahead = torch.diff(cu_k.long()) - torch.diff(s["cu_seqlens"].long())
        seen = (seq[:, None] == seq_k) & (pos_k <= (pos + ahead[seq])[:, None])
    kh, vh = (x.float().permute(0, 2, 1, 3).repeat_interleave(heads // kv_heads, dim=1)
              for x in (k, v))
    score = torch.matmul(q.float().permute(0, 2, 1, 3) * s["scale"],
                         kh.transpose(-1, -2).contiguous())
    score.masked_fill_(~seen, -math.inf)
    peak = score.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    p = score.sub_(peak).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, vh) / torch.where(total > 0, total, 1.0)
    return out.permute(0, 2, 1, 3).to(v.dtype).reshape(*q.shape[:3], dv)


@torch.no_grad()
def run(state):
    s, op = state, state["op"]
    if not own:
        return {"conv": _plain_conv, "scan": _plain_scan, "attention": _plain_attention}[op](s)
    from local_kimi_amd import kernels

    if op == "conv":
        outs = kernels.short_conv_prefill_triple(*s["in"], *s["state"], *s["weight"],
                                                 cu_seqlens=s["cu_seqlens"],
                                                 conv_states_out=tuple(s["state_out"]))
        return [*outs, *s["state_out"]]
    if op == "scan":
        out = kernels.kda_prefill(s["state"], s["q"], s["k"], s["v"], s["decay"], s["beta"],
                                  scale=s["scale"], cu_seqlens=s["cu_seqlens"],
                                  state_out=s["state_out"])
        return [out, s["state_out"]]
    return kernels.attention_prefill(s["q"], s["k"], s["v"], scale=s["scale"],
                                     cu_seqlens=s["cu_seqlens"], cu_seqlens_k=s["cu_seqlens_k"])


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case: dict) -> dict:
    op, t, n = case["op"], case["tokens"], case["sequences"]
    size = 4 if case["dtype"] == "float32" else 2
    if op == "conv":
        c = case["channels"]
        return {"bytes": 3 * size * c * (2 * t + 2 * WIDTH * n + WIDTH),
                "flops": 3.0 * t * c * (2 * WIDTH + 4)}
    if op == "scan":
        h, dk, dv = case["heads"], case["d_k"], case["d_v"]
        # decay, prediction, update and output of each step's state
        return {"bytes": t * h * (4 * (3 * dk + 1) + 2 * size * dv) + 2 * 4 * n * h * dk * dv,
                "flops": 7.0 * t * h * dk * dv}
    lengths, prefixes = _lengths(case), _prefixes(case)
    h, hk, dqk, dv = case["heads"], case["kv_heads"], case["d_qk"], case["d_v"]
    keys = sum(lengths) + sum(prefixes)
    pairs = sum(a * (a + 1) // 2 + a * b for a, b in zip(lengths, prefixes))
    return {"bytes": size * (t * h * (dqk + dv) + keys * hk * (dqk + dv)),
            "flops": 2.0 * pairs * h * (dqk + dv)}


# ---------------------------------------------------------------------------
# the same in 64 bits, a sequence at a time


def _cut(x, lengths):
    """The rows of each sequence, in 64 bits."""
    flat = x.reshape(-1, *x.shape[2:]).double()
    return torch.split(flat, lengths)


def _exact_conv(d):
    outs, states = [], []
    for x, state, weight in zip(d["in"], d["state"], d["weight"]):
        w = weight[:, 0].double()
        ys, kept = [], []
        for rows, st in zip(_cut(x, d["lengths"]), state.double()):
            line = torch.cat((st.t(), rows))
            y = sum(line[j + 1:j + 1 + rows.shape[0]] * w[:, j] for j in range(WIDTH))
            ys.append(y * torch.sigmoid(y))
            kept.append(line[line.shape[0] - WIDTH:].t())
        outs.append(torch.cat(ys).reshape(x.shape))
        states.append(torch.stack(kept))
    return outs + states


def _exact_scan(d, block=16):
    """The recurrence over blocks of positions: with G the running sum of the
    log decay within a block and S the state before it, the corrections u of
    its positions solve (I + A) u = v - (k e^G) S, A_ij = beta_j sum k_i k_j
    e^(G_i - G_j) for j < i; outputs and the next state follow from u."""
    outs, finals = [], []
    cut = [_cut(d[name], d["lengths"]) for name in ("q", "k", "v", "decay", "beta")]
    for q, k, v, decay, beta, s in zip(*cut, d["state"].double()):
        ys = []
        for at in range(0, q.shape[0], block):
            qb, kb, vb, gb = (x[at:at + block].transpose(0, 1) for x in (q, k, v, decay))
            bb = beta[at:at + block].t()
            run_sum = torch.cumsum(gb, 1)
            c = qb.shape[1]
            low = torch.tril(torch.ones((c, c), dtype=torch.bool, device=q.device))
            gap = run_sum[:, :, None] - run_sum[:, None]
            pair = torch.exp(torch.where(low[:, :, None], gap, -math.inf)) * kb[:, None]
            a = (kb[:, :, None] * pair).sum(-1) * bb[:, None]
            p = (qb[:, :, None] * pair).sum(-1) * bb[:, None]
            a = torch.tril(a, -1) + torch.eye(c, dtype=a.dtype, device=a.device)
            fade = torch.exp(run_sum)
            u = torch.linalg.solve_triangular(a, vb - (kb * fade) @ s, upper=False)
            ys.append((((qb * fade) @ s + p @ u) * d["scale"]).transpose(0, 1))
            left = torch.exp(run_sum[:, -1:] - run_sum) * kb * bb[..., None]
            s = fade[:, -1, :, None] * s + left.transpose(1, 2).contiguous() @ u
        outs.extend(ys)
        finals.append(s)
    return [torch.cat(outs).reshape(d["v"].shape), torch.stack(finals)]


def _exact_attention(d):
    q, k, v = d["q"], d["k"], d["v"]
    group = q.shape[2] // k.shape[2]
    ys = []
    for qs, ks, vs in zip(_cut(q, d["lengths"]), _cut(k, d["key_lengths"]),
                          _cut(v, d["key_lengths"])):
        a, b = qs.shape[0], ks.shape[0]
        unseen = torch.triu(torch.ones((a, b), dtype=torch.bool, device=q.device), b - a + 1)
        y = torch.zeros((a, q.shape[2], v.shape[3]), dtype=torch.float64, device=q.device)
        for h in range(q.shape[2] if a else 0):
            score = (qs[:, h] @ ks[:, h // group].t().contiguous()) * d["scale"]
            y[:, h] = torch.softmax(score.masked_fill_(unseen, -math.inf), -1) @ vs[:, h // group]
        ys.append(y)
    return torch.cat(ys).reshape(*q.shape[:3], v.shape[3])


@torch.no_grad()
def exact(case: dict, seed: int):
    d = _inputs(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "attention": _exact_attention}[d["op"]](d)
