"""The operators over rows of logits whose speed this library is judged by,
next to the calls in cases.py: processed logits (penalties, biases, grammar
masks), log-probabilities with the best alternatives, and distillation from a
teacher's top logits, forward, backward and both as a training step. With `own` set, each
pass is the call a user makes through the Python binding, with tables, scratch
and argument records made beforehand, as an engine or a trainer keeps them;
otherwise the same results come from plain torch operations in 32 bits."""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
LOWEST = 3.402823466e38
# Presence, frequency and repetition penalties of a batch's rows in turn.
PENALTIES = [dict(repetition=1.1, presence=0.5, frequency=0.3),
             dict(presence=0.8, frequency=0.1), dict(repetition=1.3), dict()]


def listed():
    def process(name, rows, vocab, dtype, out, history, biases, masked, pad=0):
        return dict(name=name, kind="process", rows=rows, vocab=vocab, dtype=dtype, out=out,
                    history=history, biases=biases, masked=masked, pad=pad)

    def logprobs(name, rows, vocab, dtype, top, rank, tempered=False, pad=0):
        return dict(name=name, kind="logprobs", rows=rows, vocab=vocab, dtype=dtype, top=top,
                    rank=rank, tempered=tempered, pad=pad)

    def distill(name, rows, vocab, dtype, top, direction, normalize, temperature, pad=0):
        return dict(name=name, kind="distill", rows=rows, vocab=vocab, dtype=dtype, top=top,
                    direction=direction, normalize=normalize, temperature=temperature, pad=pad)
    return [
        # One user's row: a repetition penalty over the prompt, a few biases.
        process("process_1", 1, 151936, "f32", "f32", 256, 8, 0.0),
        # A ragged batch: every other row constrained, an odd vocabulary, so
        # that rows start unaligned.
        process("process_24_odd", 24, 100003, "f32", "f32", 512, 30, 0.5),
        # A batch of chats: bf16 logits widened for a sampler elsewhere, the
        # longest bias lists that a request may carry.
        process("process_64", 64, 151936, "bf16", "f32", 2048, 300, 0.0),
        # A large constrained offline batch, long histories.
        process("process_256", 256, 248320, "bf16", "bf16", 8192, 0, 1.0),
        # One user's chosen token with its rank and five alternatives.
        logprobs("logprobs_1", 1, 151936, "f32", 5, True),
        # A batch of chats that ask for twenty alternatives, each request at
        # its own temperature.
        logprobs("logprobs_64", 64, 151936, "f32", 20, True, tempered=True),
        # A teacher's lists for distillation, a large and odd vocabulary.
        logprobs("teacher_lists_256", 256, 248319, "bf16", 64, False),
        # Prompt scoring: every token of a prompt, no alternatives.
        logprobs("prompt_2048", 2048, 151936, "bf16", 0, False),
        # The draft model's seven positions of four requests, evaluated.
        distill("distill_28", 28, 151936, "f32", 16, "forward", True, 1.0),
        # A validation batch.
        distill("distill_1024", 1024, 151936, "bf16", 64, "forward", True, 2.0),
        # The backward pass of a small fp32 batch, an odd vocabulary, the
        # teacher's log-probabilities as they are.
        distill("distill_backward_96_odd", 96, 100003, "f32", 20, "backward", False, 1.0),
        # A training step over a packed batch of sequences: loss and gradient.
        distill("distill_step_2048", 2048, 151936, "bf16", 64, "step", True, 2.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["process", "logprobs", "distill"])
    vocab = _log_uniform(rng, 32000, 262144)
    if rng.random() < 0.5:
        vocab -= vocab % 64
    dtype = rng.choice(["f32", "bf16"])
    # Room between rows, as where logits are a view of a wider buffer.
    pad = rng.choice([0, 0, 0, 1, 64, 1000])
    size = 4 if dtype == "f32" else 2
    if kind == "process":
        rows = min(_log_uniform(rng, 1, 256), int(250e6 / (vocab * 2 * size)))
        return dict(kind=kind, rows=max(1, rows), vocab=vocab, dtype=dtype,
                    out=rng.choice([dtype, "f32"]), history=rng.choice([0, 100, 512, 2048, 8192]),
                    biases=rng.choice([0, 0, 1, 30, 300]), masked=rng.choice([0.0, 0.0, 0.3, 1.0]),
                    pad=pad)
    rows = max(1, min(_log_uniform(rng, 1, 2048), int(600e6 / (vocab * size))))
    if kind == "logprobs":
        top = rng.choice([0, 1, 5, 20, 64, 128])
        if top:
            # Lists are asked for by serving batches and teachers' micro-batches.
            rows = min(rows, int(130e6 / (vocab * size)))
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, top=top,
                    rank=rng.random() < 0.5, tempered=rng.random() < 0.5, pad=pad)
    return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, top=_log_uniform(rng, 1, 128),
                direction=rng.choice(["forward", "backward", "step"]),
                normalize=rng.random() < 0.5,
                temperature=rng.choice([0.5, 1.0, 2.0, 4.0]), pad=pad)


# ---- inputs ------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _torch_type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _rows_of(rows, vocab, pad, dtype):
    """Empty rows of logits with `pad` elements between them."""
    return torch.empty((rows, vocab + pad), dtype=dtype, device=DEV)[:, :vocab]


def _logits(g, rows, vocab, pad, dtype):
    """Rows whose r-th most likely token has about probability r^-a, a drawn
    per row from 1.1 (thousands of tokens matter) to 2.2 (a handful do); every
    64 rows get a temporary of their own."""
    out = _rows_of(rows, vocab, pad, dtype)
    for r in range(0, rows, 64):
        n = min(64, rows - r)
        a = torch.rand((n, 1), generator=g, device=DEV) * 1.1 + 1.1
        x = torch.rand((n, vocab), generator=g, device=DEV)
        x = -a * torch.log1p(x * vocab)
        out[r:r + n] = x + 0.25 * torch.randn((n, vocab), generator=g, device=DEV) + 12.0
    return out


def _allowed(g, rows, vocab):
    """Admitted tokens of a grammar's states: runs of up to 40 ids, about 2%
    of the vocabulary, and some single ids."""
    n = max(4, int(0.001 * vocab))
    start = torch.randint(0, vocab, (rows, n), generator=g, device=DEV)
    length = torch.randint(1, 41, (rows, n), generator=g, device=DEV)
    edge = torch.zeros((rows, vocab + 64), dtype=torch.int32, device=DEV)
    one = torch.ones_like(start, dtype=torch.int32)
    edge.scatter_add_(1, start, one)
    edge.scatter_add_(1, start + length, -one)
    allowed = edge.cumsum(1)[:, :vocab] > 0
    single = torch.randint(0, vocab, (rows, 20), generator=g, device=DEV)
    return allowed.scatter_(1, single, True)


def _mask_words(allowed):
    rows, vocab = allowed.shape
    words = (vocab + 31) // 32
    bits = torch.zeros((rows, words * 32), dtype=torch.int64, device=DEV)
    bits[:, :vocab] = allowed
    w = (bits.view(rows, words, 32) << torch.arange(32, device=DEV)).sum(2)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32).contiguous()


def _process_inputs(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    rows, vocab, history, biases = case["rows"], case["vocab"], case["history"], case["biases"]
    i = dict(x=_logits(g, rows, vocab, case["pad"], _torch_type(case["dtype"])))
    # The first half of a history is the prompt.
    i["history"] = rng.integers(0, vocab, (rows, history), dtype=np.int64).astype(np.uint32)
    i["penalties"] = [PENALTIES[r % 4] if history else {} for r in range(rows)]
    # Distinct tokens a row: bans and values of a request's range.
    i["bias_ids"] = np.stack([rng.choice(vocab, biases, replace=False) for _ in range(rows)])
    values = rng.uniform(-10, 10, (rows, biases)).astype(np.float32)
    i["bias_values"] = np.where(rng.random((rows, biases)) < 0.1, np.float32(-100), values)
    i["masked"] = [bool(case["masked"]) and r % round(1 / case["masked"]) == 0
                   for r in range(rows)] if case["masked"] else [False] * rows
    i["masks"] = _mask_words(_allowed(g, rows, vocab)) if case["masked"] else None
    return i


def _entries(case, i):
    """Every row's distinct tokens of its history: (token, generated count,
    whether the prompt marks it), padded to the longest row's with its first."""
    got = []
    for r in range(case["rows"]):
        h, half = i["history"][r].astype(np.int64), case["history"] - case["history"] // 2
        tokens = np.unique(h)
        counts = np.zeros(tokens.size, np.int64)
        np.add.at(counts, np.searchsorted(tokens, h[half:]), 1)
        marked = np.isin(tokens, h[:half]) & (i["penalties"][r].get("repetition", 1.0) != 1.0)
        keep = (counts > 0) | marked
        got.append((tokens[keep], counts[keep]))
    width = max(t.size for t, _ in got)
    tokens, counts = np.zeros((2, case["rows"], width), np.int64)
    for r, (t, c) in enumerate(got):
        tokens[r], counts[r] = t[0], c[0]
        tokens[r, :t.size], counts[r, :t.size] = t, c
    return torch.from_numpy(tokens).to(DEV), torch.from_numpy(counts).to(DEV)


def _distill_inputs(case, seed):
    """A student's logits near the teacher's; the teacher's list holds its
    best tokens in order, some rows a shorter one, every 16th row none (the
    padding of a packed batch)."""
    g = _gen(seed)
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    z = _logits(g, rows, vocab, case["pad"], _torch_type(case["dtype"]))
    ids = torch.empty((rows, top), dtype=torch.int64, device=DEV)
    values = torch.empty((rows, top), dtype=torch.float32, device=DEV)
    for r in range(0, rows, 64):
        part = z[r:r + 64].float()
        teacher = part + 0.8 * torch.randn(part.shape, generator=g, device=DEV)
        best, at = torch.topk(teacher, top, dim=1)
        if not case["normalize"]:
            best = best / case["temperature"] - torch.logsumexp(
                teacher / case["temperature"], 1, keepdim=True)
        ids[r:r + 64], values[r:r + 64] = at, best
    length = torch.randint(1, top + 1, (rows, 1), generator=g, device=DEV)
    length = torch.where(torch.rand((rows, 1), generator=g, device=DEV) < 0.7, top, length)
    row = torch.arange(rows, device=DEV)[:, None]
    length = torch.where(row % 16 == 15, 0, length)
    ids = torch.where(torch.arange(top, device=DEV) < length, ids, -1)
    i = dict(z=z, ids=ids.to(torch.int32), values=values)
    if case["direction"] != "forward":
        # A mean over the rows that have a list, as a trainer weighs them.
        i["grad_loss"] = torch.full((rows,), 1.0 / max(1, rows - rows // 16), device=DEV)
    return i


def _logprob_inputs(case, seed):
    g = _gen(seed)
    rows, vocab = case["rows"], case["vocab"]
    x = _logits(g, rows, vocab, case["pad"], _torch_type(case["dtype"]))
    tokens = torch.randint(0, vocab, (rows, 1), generator=g, device=DEV)
    # Most chosen tokens are likely ones.
    best = torch.cat([x[r:r + 64].argmax(1, keepdim=True) for r in range(0, rows, 64)])
    tokens = torch.where(torch.rand((rows, 1), generator=g, device=DEV) < 0.6, best, tokens)
    temperatures = 0.5 + torch.rand(rows, generator=g, device=DEV) if case["tempered"] else None
    return dict(x=x, tokens=tokens.to(torch.int32), temperatures=temperatures)


# ---- preparation -------------------------------------------------------------


def _binding():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "justfit-llm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import jf_sampler
    return jf_sampler


def _prepare_process(case, seed):
    i = _process_inputs(case, seed)
    rows, vocab = case["rows"], case["vocab"]
    x, masked = i["x"], i["masked"]
    if not own:
        state = dict(x=x, out=_torch_type(case["out"]), entries=None, biases=None, masks=i["masks"])
        if case["history"]:
            column = lambda name, none: torch.tensor(  # noqa: E731
                [[p.get(name, none)] for p in i["penalties"]], dtype=torch.float32, device=DEV)
            state.update(entries=_entries(case, i), repetition=column("repetition", 1.0),
                         presence=column("presence", 0.0), frequency=column("frequency", 0.0))
        if case["biases"]:
            state["biases"] = (torch.from_numpy(i["bias_ids"]).to(DEV),
                               torch.from_numpy(i["bias_values"]).to(DEV))
        state["masked"] = torch.tensor(masked, device=DEV)[:, None]
        return state
    J = _binding()
    kw = {}
    if case["history"]:
        table = J.PenaltyTable(vocab, rows, case["history"])
        for r, p in enumerate(i["penalties"]):
            table.rebuild(r, i["history"][r], case["history"] // 2, None,
                          p.get("repetition", 1.0) != 1.0)
        kw.update(penalties=table, penalty_rows=list(range(rows)))
    if case["biases"]:
        table = J.BiasTable(vocab, rows, case["biases"])
        for r in range(rows):
            table.set(r, i["bias_ids"][r], i["bias_values"][r])
        kw.update(biases=table, bias_rows=list(range(rows)))
    if i["masks"] is not None:
        kw["masks"] = i["masks"]
    out = _rows_of(rows, vocab, case["pad"], _torch_type(case["out"]))
    s = J.Scorer(vocab, rows)
    policies = [J.policy(constrained=c, **p) for c, p in zip(masked, i["penalties"])]
    args, keep = s.process_args(x, policies, out, **kw)
    return dict(scorer=s, args=args, out=dict(logits=out), hold=(keep, kw, x))


def _prepare_logprobs(case, seed):
    i = _logprob_inputs(case, seed)
    if not own:
        return dict(i, top=case["top"], rank=case["rank"])
    J = _binding()
    rows, top = case["rows"], case["top"]
    out = dict(lse=torch.empty(rows, device=DEV), logprobs=torch.empty((rows, 1), device=DEV))
    if case["rank"]:
        out["ranks"] = torch.empty(rows, dtype=torch.int32, device=DEV)
    if top:
        out.update(top_ids=torch.empty((rows, top), dtype=torch.int32, device=DEV),
                   top_logprobs=torch.empty((rows, top), device=DEV))
    s = J.Scorer(case["vocab"], rows)
    args = s.logprobs_args(i["x"], tokens=i["tokens"], temperatures=i["temperatures"], **out)
    return dict(scorer=s, args=args, out=out, hold=i)


def _prepare_distill(case, seed):
    i = _distill_inputs(case, seed)
    kw = dict(temperature=case["temperature"], normalize=case["normalize"])
    direction, rows = case["direction"], case["rows"]
    if not own:
        state = dict(i, direction=direction, **kw)
        if direction == "backward":
            # What the forward pass keeps: each row's maximum and sum, and the
            # teacher's probabilities.
            state["saved"] = _plain_forward(state)[0]
        return state
    J = _binding()
    s = J.Scorer(case["vocab"], rows)
    out = dict(loss=torch.empty(rows, device=DEV), lse=torch.empty(rows, device=DEV))
    if direction == "backward":
        kw["saved"] = torch.empty((rows, 2 + case["top"]), device=DEV)
        s.launch_distill(s.distill_args(i["z"], i["ids"], i["values"], **out, **kw))
        out = {}
    if direction != "forward":
        out["grad"] = _rows_of(rows, case["vocab"], case["pad"], i["z"].dtype)
        kw["grad_loss"] = i["grad_loss"]
    args = s.distill_args(i["z"], i["ids"], i["values"], **out, **kw)
    return dict(scorer=s, args=args, out=out, direction=direction, hold=(i, kw))


def prepare(case, seed):
    state = {"process": _prepare_process, "logprobs": _prepare_logprobs,
             "distill": _prepare_distill}[case["kind"]](case, seed)
    state["kind"] = case["kind"]
    return state


# ---- the passes --------------------------------------------------------------


def _plain_process(s):
    x = s["x"].float()
    if s["entries"] is not None:
        tokens, counts = s["entries"]
        v = x.gather(1, tokens)
        v = v * torch.where(v > 0, 1.0 / s["repetition"], s["repetition"])
        lowered = v - (s["frequency"] * counts + s["presence"])
        v = torch.where(counts > 0, lowered, v).clamp(-LOWEST, LOWEST)
        x = x.scatter(1, tokens, v)
    if s["biases"] is not None:
        x = x.scatter_add(1, *s["biases"])
    if s["masks"] is not None:
        bits = (s["masks"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        admitted = bits.view(x.shape[0], -1)[:, :x.shape[1]] > 0
        x = torch.where(admitted | ~s["masked"], x, -math.inf)
    return dict(logits=x.to(s["out"]))


def _plain_logprobs(s):
    x = s["x"].float()
    rows, vocab = x.shape
    at = s["tokens"].long()
    scale = 1.0 if s["temperatures"] is None else (1.0 / s["temperatures"])[:, None]
    maximum = x.amax(1, keepdim=True)
    log_sum = torch.exp((x - maximum) * scale).sum(1, keepdim=True).log()
    logprob = lambda v: (v - maximum) * scale - log_sum  # noqa: E731
    chosen = x.gather(1, at)
    out = dict(lse=(maximum * scale + log_sum)[:, 0], logprobs=logprob(chosen))
    if s["rank"]:
        earlier = torch.arange(vocab, device=DEV) < at
        ahead = (x > chosen) | ((x == chosen) & earlier)
        out["ranks"] = (ahead.sum(1) + 1).to(torch.int32)
    if s["top"]:
        # The largest (logit, -id) pairs, each pair as one 64-bit number.
        bits = x.view(torch.int32).long()
        key = torch.where(bits < 0, -2 ** 31 - bits, bits)
        pair = key * 2 ** 32 + (vocab - 1 - torch.arange(vocab, device=DEV))
        best = torch.topk(pair, s["top"], dim=1).values
        ids = vocab - 1 - (best & 0xFFFFFFFF)
        out.update(top_ids=ids.to(torch.int32), top_logprobs=logprob(x.gather(1, ids)))
    return out


def _plain_forward(s):
    """What the backward pass takes, with the exponentials, and the outputs."""
    z, scale = s["z"].float(), 1.0 / s["temperature"]
    listed_ = s["ids"] >= 0
    at = s["ids"].long().clamp(min=0)
    maximum = z.amax(1, keepdim=True)
    e = torch.exp((z - maximum) * scale)
    total = e.sum(1, keepdim=True)
    log_q = (z.gather(1, at) - maximum) * scale - total.log()
    log_p = torch.where(listed_, s["values"], -math.inf)
    if s["normalize"]:
        log_p = log_p * scale
        log_p = log_p - log_p.amax(1, keepdim=True).clamp(min=-LOWEST)
        log_p = log_p - torch.exp(log_p).sum(1, keepdim=True).log()
    p = torch.where(listed_, torch.exp(log_p), 0.0)
    loss = torch.where(p > 0, p * (log_p - log_q), 0.0).sum(1)
    lse = (maximum * scale + total.log())[:, 0]
    return (maximum, total, p), e, dict(loss=loss, lse=lse)


def _plain_backward(s, saved, e):
    _, total, p = saved
    g = s["grad_loss"][:, None] * (1.0 / s["temperature"])
    grad = e * (g * p.sum(1, keepdim=True) / total)
    return grad.scatter_add_(1, s["ids"].long().clamp(min=0), -g * p).to(s["z"].dtype)


def _plain_distill(s):
    if s["direction"] == "backward":
        e = torch.exp((s["z"].float() - s["saved"][0]) * (1.0 / s["temperature"]))
        return dict(grad=_plain_backward(s, s["saved"], e))
    saved, e, out = _plain_forward(s)
    if s["direction"] == "step":
        out["grad"] = _plain_backward(s, saved, e)
    return out


def run(state):
    if not own:
        return {"process": _plain_process, "logprobs": _plain_logprobs,
                "distill": _plain_distill}[state["kind"]](state)
    s, a = state["scorer"], state["args"]
    if state["kind"] == "process":
        s.launch_process(a)
    elif state["kind"] == "logprobs":
        s.launch_logprobs(a)
    elif state["direction"] == "backward":
        s.launch_distill_backward(a)
    elif state["direction"] == "step":
        s.launch_distill_step(a)
    else:
        s.launch_distill(a)
    return state["out"]


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    size = 4 if case["dtype"] == "f32" else 2
    read = rows * vocab * size
    if case["kind"] == "process":
        # 8 bytes a penalized or biased token, a bit a token of a masked row.
        tables = rows * 8 * (case["history"] + case["biases"])
        mask = rows * case["masked"] * vocab / 8
        return {"bytes": read + rows * vocab * (4 if case["out"] == "f32" else 2) + tables + mask,
                "flops": rows * 4 * (case["history"] + case["biases"])}
    if case["kind"] == "logprobs":
        # A maximum, a difference, its scale, an exponential and a sum a token.
        return {"bytes": read + rows * (12 + 8 * case["top"]), "flops": 5 * rows * vocab}
    direction = case["direction"]
    return {"bytes": read * (1 if direction == "forward" else 2) + rows * (8 + 8 * case["top"]),
            "flops": {"forward": 5, "backward": 4, "step": 8}[direction] * rows * vocab}


# ---- the definitions in 64 bits ------------------------------------------------


def _exact_process(case, seed):
    i = _process_inputs(case, seed)
    rows, vocab, history = case["rows"], case["vocab"], case["history"]
    out = []
    for r in range(rows):
        y = i["x"][r].double()
        p = i["penalties"][r]
        if p:
            repetition = float(np.float32(p.get("repetition", 1.0)))
            h = torch.from_numpy(i["history"][r].astype(np.int64)).to(DEV)
            count = torch.bincount(h[history - history // 2:], minlength=vocab)
            seen = count > 0
            if repetition != 1.0:
                seen[h[:history - history // 2]] = True
            pushed = torch.where(y > 0, y / repetition, y * repetition)
            pushed = pushed - (count > 0) * (float(np.float32(p.get("presence", 0.0)))
                                             + float(np.float32(p.get("frequency", 0.0))) * count)
            y = torch.where(seen, pushed, y)
        if case["biases"]:
            ids = torch.from_numpy(i["bias_ids"][r]).to(DEV)
            y[ids] = y[ids] + torch.from_numpy(i["bias_values"][r]).to(DEV).double()
        if i["masked"][r]:
            token = torch.arange(vocab, device=DEV)
            word = i["masks"][r].long()[token // 32]
            y = y.masked_fill((word >> (token % 32)) % 2 == 0, -math.inf)
        out.append(y)
    return dict(logits=torch.stack(out))


def _exact_logprobs(case, seed):
    i = _logprob_inputs(case, seed)
    rows = case["rows"]
    out = dict(lse=[], logprobs=[], top_logprobs=[])
    for r in range(rows):
        y = i["x"][r].double()
        if i["temperatures"] is not None:
            y = y / i["temperatures"][r].double()
        lse = torch.logsumexp(y, 0)
        y = y - lse
        out["lse"].append(lse)
        out["logprobs"].append(y[i["tokens"][r].long()])
        if case["top"]:
            out["top_logprobs"].append(torch.topk(y, case["top"]).values)
    got = {k: torch.stack(v) if v else None for k, v in out.items()}
    # Ids and ranks are no computed numbers.
    for name, here in (("top_logprobs", case["top"]), ("top_ids", case["top"]),
                       ("ranks", case["rank"])):
        if not here:
            got.pop(name, None)
        else:
            got.setdefault(name, None)
    return got


def _exact_distill(case, seed):
    i = _distill_inputs(case, seed)
    t = case["temperature"]
    losses, lses = [], []
    direction = case["direction"]
    grads = torch.empty(i["z"].shape, dtype=torch.float64, device=DEV) \
        if direction != "forward" else None
    for r in range(case["rows"]):
        ids, u = i["ids"][r].long(), i["values"][r].double()
        ids, u = ids[ids >= 0], u[i["ids"][r] >= 0]
        log_q = i["z"][r].double() / t
        lses.append(torch.logsumexp(log_q, 0))
        log_q = log_q - lses[-1]
        log_p = torch.log_softmax(u / t, 0) if case["normalize"] else u
        p = log_p.exp()
        losses.append((p * (log_p - log_q[ids])).sum())
        if grads is not None:
            # The mass on the list pulls every token's probability down, each
            # listed token's own pushes it up.
            d = log_q.exp() * p.sum()
            d[ids] -= p
            grads[r] = d * (float(i["grad_loss"][r]) / t)
    if direction == "backward":
        return dict(grad=grads)
    out = dict(loss=torch.stack(losses), lse=torch.stack(lses))
    if direction == "step":
        out["grad"] = grads
    return out


def exact(case, seed):
    return {"process": _exact_process, "logprobs": _exact_logprobs,
            "distill": _exact_distill}[case["kind"]](case, seed)
