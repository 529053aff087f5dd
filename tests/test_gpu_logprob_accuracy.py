"""How far the losses' log-probabilities are off, as a whole: their error's mean and
standard deviation over drawn tokens of peaked rows, in every form that takes a row's sums.
A bound of each step's worst case is a thousand times as wide, and would pass sums that lose
bits to the order they are taken in.

What is stored is rounded to fp32; the error before that is seen through small differences.
A sequence of one token has its log-probability less the reference's for a score; a KL term
e^c - c - 1 of c near 1e-3 tells c to 2^-24 of 5e-7 / 1e-3.

Limits. The scale c = log2(e) / T is rounded, and the token's exponent is by the same c, so
its share weighs the token's distance from the row's mean exponent, which is 0 on the average
of drawn tokens: it has no part in the mean, and its part in the deviation is worked out
here. The deviation at T = 1 is that of the same fp32 steps done one by one on a CPU with
correctly rounded exponentials, over 1500 and more such rows (standing beside each form); 12%
more is allowed for: three deviations of both samples' own (2.3% together), and 5% for the
exponential's instruction. Sums joined in 32 bits are at 7.5e-8 for 32,000 tokens and 7.9
to 9.5e-8 beyond in the same steps. The mean may be half a step of the exponential, 2^-24, one
way: by the steps it is below 2e-8, and where a row's tokens are added in one chain 1.4e-7 to
5e-7, or with the token's exponent by 1 / T alone 2.2e-7 at T = 1.33."""
import functools

import pytest

import jf_sampler as J
from scoring_cases import U

pytestmark = pytest.mark.gpu

ROWS = 2048


@functools.lru_cache(maxsize=1)
def drawn(V, dtype, T):
    """Rows whose r-th most likely token has about probability r^-a, a from 1.1 to 2.2, a
    token drawn from each, its log-probability in 64 bits, and its exponent's distance from
    the row's mean one."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(V)
    T = float(torch.tensor(T))  # temperatures are fp32
    x = torch.empty((ROWS, V), dtype=torch.bfloat16 if dtype == "bf16" else torch.float32,
                    device="cuda")
    tokens = torch.empty(ROWS, dtype=torch.int32, device="cuda")
    lp, distance = torch.empty((2, ROWS), dtype=torch.float64, device="cuda")
    for r in range(0, ROWS, 64):
        a = torch.rand((64, 1), generator=g, device="cuda") * 1.1 + 1.1
        rank = torch.rand((64, V), generator=g, device="cuda") * V
        x[r:r + 64] = 12 - a * torch.log1p(rank) + \
            0.25 * torch.randn((64, V), generator=g, device="cuda")
        y = x[r:r + 64].double() / T
        noise = torch.rand((64, V), generator=g, device="cuda").clamp(1e-12, 1 - 1e-7).double()
        at = (y - torch.log(-torch.log(noise))).argmax(1, keepdim=True)
        log_q = torch.log_softmax(y, 1)
        tokens[r:r + 64] = at[:, 0]
        lp[r:r + 64] = log_q.gather(1, at)[:, 0]
        distance[r:r + 64] = (y.gather(1, at) - (log_q.exp() * y).sum(1, keepdim=True))[:, 0]
    return x, tokens, lp, distance


def preference_errors(s, call, x, tokens, lp, T):
    import torch
    n = len(tokens)
    reference, scores = lp.float(), torch.empty(n, device="cuda")
    kw = dict(grad=torch.empty_like(x), grad_loss=torch.ones(n // 2, device="cuda")) \
        if call == "step" else {}
    a = s.preference_args(x, tokens, torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                          reference_logprobs=reference, temperature=T, scores=scores,
                          loss=torch.empty(n // 2, device="cuda"),
                          saved=torch.empty((n, 4), device="cuda"), **kw)
    (s.launch_preference_step if call == "step" else s.launch_preference)(a)
    return scores.double() - (lp - reference.double())


def clipped_errors(s, call, x, tokens, lp, T):
    import torch
    n = len(tokens)
    reference, kl = lp.float() + 1e-3, torch.empty(n, device="cuda")
    kw = dict(grad=torch.empty_like(x), grad_loss=torch.ones(n, device="cuda"),
              saved=torch.empty((n, 4), device="cuda")) if call == "step" else {}
    a = s.clipped_args(x, tokens, torch.ones(n, device="cuda"), reference_logprobs=reference,
                       temperature=T, kl=kl, loss=torch.empty(n, device="cuda"), **kw)
    (s.launch_clipped_step if call == "step" else s.launch_clipped)(a)
    c = reference.double() - lp
    return -(kl.double() - (torch.expm1(c) - c)) / torch.expm1(c)


# Loss, call, rows of a call, vocabulary, type, and the deviation by steps at T = 1, 1e-8.
FORMS = [
    ("preference", "forward", 256, 32000, "f32", 5.94),     # rows whole, 512 threads
    ("preference", "step", 128, 32000, "f32", 5.84),        # chunks, joined by the pairs' launch
    ("clipped", "step", 16, 32000, "f32", 5.94),            # blocks that share a row
    ("preference", "forward", 2048, 32000, "bf16", 6.33),   # rows whole, 256 threads
    ("clipped", "forward", 2048, 32000, "bf16", 6.33),
    ("clipped", "step", 512, 32000, "bf16", 5.88),          # a block of 512 threads a row
    ("clipped", "forward", 64, 100003, "f32", 5.67),        # chunks, joined by their launch
    ("clipped", "forward", 256, 100003, "f32", 6.33),       # rows whole, 512 threads
    ("clipped", "step", 16, 100003, "f32", 5.67),           # chunks, joined by the gradient's
    ("clipped", "forward", 256, 100003, "bf16", 6.24),
    ("preference", "forward", 2048, 151936, "f32", 5.84),   # chunks of 8 vectors
    ("clipped", "step", 256, 151936, "f32", 6.07),          # a block of 1024 threads a row
    ("preference", "step", 2048, 151936, "bf16", 5.93),     # chunks of 4
    ("clipped", "step", 256, 151936, "bf16", 6.73),         # a block of 512 threads a row
    ("clipped", "step", 16, 151936, "bf16", 6.03),          # chunks of 2, by the gradient's
]


@pytest.mark.parametrize("T", [1.0, 1.33])  # at 1.33 the scale is off by 6.4e-8 of itself
@pytest.mark.parametrize("loss,call,rows,V,dtype,deviation", FORMS)
def test_log_probabilities(loss, call, rows, V, dtype, deviation, T):
    import torch
    print(f"accuracy {loss} {call} {rows} x {V} {dtype} T {T}", flush=True)
    x, tokens, lp, distance = drawn(V, dtype, T)
    s = J.Scorer(V, rows)
    errors = preference_errors if loss == "preference" else clipped_errors
    e = torch.cat([errors(s, call, x[r:r + rows], tokens[r:r + rows], lp[r:r + rows], T)
                   for r in range(0, ROWS, rows)])
    t = torch.tensor(T)
    scale = float(torch.tensor(1.44269504088896341) / t)
    share = abs(scale * 0.693147180559945309417 * float(t) - 1)
    by_scale = share * float(distance.std())
    mean, off = float(e.mean()), float(e.std())
    print(f"  mean {mean:.2e} deviation {off:.2e}, by the scale {by_scale:.2e}")
    assert abs(mean) <= U + 3 * off / ROWS ** 0.5
    assert off <= 1.12e-8 * deviation + (by_scale if T != 1.0 else 0.0)
    s.close()
