"""Plain implementations in 64 bits of processed logits, log-probabilities and
distillation, for the tests of the operators over rows of logits, with bounds
of the fp32 operators' errors derived from their steps, and rows of logits at
any element's alignment on the device."""
import numpy as np

NO = 0xFFFFFFFF
U = 2.0 ** -24        # half an ulp of fp32, relative
LOWEST = float(np.finfo(np.float32).max)


def bf16(x):
    """The nearest bf16 of each value (ties to even), as float32. Keeps NaN."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def device_rows(x, dtype, pad=0, lead=0):
    """A [rows, V] device tensor of x with `pad` elements between its rows and
    the first row `lead` elements into its buffer; every element around the
    rows holds a value that no result may follow (a huge logit). Returns the
    tensor and its buffer."""
    import torch
    kind = torch.bfloat16 if dtype == "bf16" else torch.float32
    rows, V = x.shape
    buf = torch.full((lead + rows * (V + pad) + 8,), 3e38, dtype=torch.float32).to(kind).cuda()
    t = buf[lead:lead + rows * (V + pad)].view(rows, V + pad)[:, :V]
    t.copy_(torch.from_numpy(np.ascontiguousarray(x, np.float32)))
    return t, buf


def excess(got, want, bound, dtype):
    """How far stored values lie outside of what a result within `bound` of
    `want` rounds to in its type, in units of the bound: at most 1 is right. A
    bf16 result is the nearest bf16 of some such value, exactly."""
    if dtype == "f32":
        return np.abs(got - want) / (bound + U * np.abs(want))
    with np.errstate(over="ignore"):
        lo = bf16((want - bound).astype(np.float32))
        hi = bf16((want + bound).astype(np.float32))
    return np.where((got >= lo) & (got <= hi), 0.0, np.abs(got - want) / bound + 1)


def host(t):
    return t.float().cpu().numpy()


# ---- processed logits ----------------------------------------------------------


def process_plain(x, policy, words=None, extra=(), bias=None, mask=None, stops=()):
    """One row in 64 bits: (values, whether edited, the magnitude that its
    roundings scale with). words: the penalty words; bias: {token: value};
    mask: admitted tokens as booleans; stops: excluded tokens."""
    y = x.astype(np.float64)
    edited = np.zeros(len(x), bool)
    size = np.abs(np.where(np.isfinite(y), y, 0))
    if words is not None:
        counts = (words & 0x7FFFFFFF).astype(np.int64)
        seen = words != 0
        for t in extra:
            if t < len(x):
                counts[t] += 1
                seen[t] = True
        f = lambda v: float(np.float32(v))  # noqa: E731
        with np.errstate(invalid="ignore", over="ignore"):
            p = np.where(y > 0, y / f(policy.repetition), y * f(policy.repetition))
            lowered = f(policy.presence) + f(policy.frequency) * counts
            p = np.where(counts > 0, p - lowered, p)
        size = np.where(seen, np.abs(np.where(np.isfinite(p), p, 0)) + 2 * np.abs(lowered), size)
        # A NaN saturates to the lowest value, as in the selection.
        p = np.where(np.isnan(p), -LOWEST, np.clip(p, -LOWEST, LOWEST))
        y = np.where(seen, p, y)
        edited |= seen
    for t, b in (bias or {}).items():
        b = float(np.float32(b))
        y[t] = b if b == -np.inf else y[t] + b
        size[t] += abs(b) if np.isfinite(b) else 0
        edited[t] = True
    if mask is not None:
        y = np.where(mask, y, -np.inf)
        edited |= ~mask
    for t in stops:
        if t < len(x):
            y[t] = -np.inf
            edited[t] = True
    return y, edited, size


def process_bound(size):
    """An edited value takes at most six roundings (the inverse, the product,
    the scaled frequency, its sum, the difference, the bias), each of a number
    no larger than twice `size`."""
    return 12 * U * size + 1e-44


# ---- log-probabilities ----------------------------------------------------------


def sum_bound(d, terms):
    """Relative error of the fp32 sum of exp(d_v), d_v <= 0: each exponent is
    a difference, its scale (a rounded constant over a rounded temperature) and
    a product, 4 roundings of |d|, and the exponential is good to 2 ulp; a sum
    of `terms` numbers by threads, waves and blocks, each partial rescaled at
    most 9 times on the way with an exponent within |d| too."""
    far = min(float(np.max(np.abs(d[np.isfinite(d)]), initial=0.0)), 104.0)
    return U * (terms + 9 * (4 + 4 * far) + 4 + 4 * far)


def adds(V):
    """Additions a term goes through at most: a thread's 32 a chunk, then
    waves, the block and segments."""
    return 32 * ((V + 8191) // 8192) + 6 + 2 + 6 + 8


def score_plain(x, T=1.0):
    """(m, log-probabilities, lse, bound of the errors of a log-probability
    and of lse) of one row in 64 bits."""
    y = x.astype(np.float64)
    m = y.max() if len(y) and not np.isnan(y).any() else np.nan
    if m == -np.inf:
        return m, np.full(len(y), -np.inf), m, np.zeros(len(y)), 0.0
    with np.errstate(invalid="ignore"):
        d = (y - m) / T
        log_sum = np.log(np.exp(d).sum())
        lp = d - log_sum
        rel = sum_bound(d, adds(len(y)))
        # The logarithm is good to 2 ulp; then a difference, a scale (2
        # roundings) and a difference again.
        lp_bound = rel + U * (3 * abs(log_sum) + 4 * np.where(np.isfinite(d), np.abs(d), 0)) + \
            U * np.where(np.isfinite(lp), np.abs(lp), 0) + 1e-38
        lse = m / T + log_sum
        lse_bound = rel + U * (3 * abs(log_sum) + 3 * abs(m / T) + abs(lse)) + 1e-38
    return m, lp, lse, lp_bound, lse_bound


def order(x):
    """Token ids by (logit down, id up), NaN and -infinity left out."""
    x = x.astype(np.float64)
    ids = np.flatnonzero(x > -np.inf)
    return ids[np.lexsort((ids, -x[ids]))]


def rank_of(x, token):
    x = x.astype(np.float64)
    t = x[token]
    with np.errstate(invalid="ignore"):
        return 1 + int((x > t).sum()) + int((x[:token] == t).sum())


# ---- distillation ----------------------------------------------------------------


def distill_plain(z, ids, values, T, normalize):
    """(loss, gradient for a loss gradient of 1, bounds of both) of one row in
    64 bits."""
    z = z.astype(np.float64)
    V = len(z)
    used, seen = np.zeros(len(ids), bool), set()
    for k, i in enumerate(ids):
        i = int(i) & NO
        used[k] = i < V and i not in seen
        seen.add(i)
    at, u = ids[used].astype(np.int64), values[used].astype(np.float64)
    grad = np.zeros(V)
    with np.errstate(invalid="ignore", divide="ignore"):
        _, log_q, _, q_bound, _ = score_plain(z, T)
        log_p = u / T if normalize else u.copy()
        if normalize and len(u):
            top = log_p.max()
            top = top if np.isfinite(top) else 0.0
            total = np.exp(log_p - top).sum()
            log_p = log_p - top - (np.log(total) if total else 0.0)
        p = np.exp(log_p)
        terms = np.where(p == 0, 0.0, p * (log_p - log_q[at]))
        loss = terms.sum()
        mass = p.sum()
        if not mass > 0:
            return loss, grad, 0.0, np.zeros(V)
        q = np.exp(log_q)
        grad = q * mass
        grad[at] -= p
        grad /= T
        # p: an exponential of a difference (2 ulp and the exponent's error),
        # over a sum of K of them; a term: two more roundings; then a sum.
        size = np.where(np.isfinite(log_p), np.abs(log_p), 0)
        spread = np.abs(u / T).max(initial=0.0) if normalize else 0.0
        p_rel = U * (8 + 4 * size + 6 * min(spread, 1e4) + 24)
        finite = np.where(np.isfinite(terms), np.abs(terms), 0)
        gap = np.where(np.isfinite(log_q[at]), np.abs(log_q[at]), 0)
        loss_bound = (p * (q_bound[at] + p_rel + U * (size + gap))).sum() + \
            (finite * (p_rel + 24 * U)).sum() + 1e-37
        rel = sum_bound((z - z.max()) / T, adds(V))
        far = np.minimum(np.where(np.isfinite(log_q), np.abs(log_q), 0), 200)
        worst_p = p_rel.max(initial=0.0)
        grad_bound = q * mass * (rel + worst_p + U * (16 + 8 * far))
        grad_bound[at] += p * (worst_p + 6 * U)
        grad_bound = grad_bound / T + 1e-37
    return loss, grad, loss_bound, grad_bound


