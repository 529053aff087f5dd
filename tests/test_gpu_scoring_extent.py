"""The operators over rows of logits at the ends of their extents: rows whose
offsets pass 32 bits, more rows than one launch takes, the largest and the
smallest vocabulary."""
import numpy as np
import pytest

import jf_sampler as J
from scoring_cases import (U, bf16, device_rows, distill_plain, excess, host, order, rank_of,
                           score_plain)

pytestmark = pytest.mark.gpu


def test_row_offsets_past_32_bits():
    """Two rows 2^32 + 2 elements apart, in and out."""
    import torch
    V, K, apart = 9001, 5, 2 ** 32 + 2
    rng = np.random.default_rng(1)
    x = bf16(rng.normal(0, 3, (2, V)).astype(np.float32))
    buf = torch.empty(apart + V, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(apart + V, dtype=torch.bfloat16, device="cuda")
    t, y = (b.as_strided((2, V), (apart, 1)) for b in (buf, out))
    t.copy_(torch.from_numpy(x))
    y.zero_()
    s = J.Scorer(V, 2)
    bias = J.BiasTable(V, 2, 1)
    bias.set(1, [V - 1], [2.5])
    s.process(t, [J.policy()] * 2, y, biases=bias, bias_rows=[0, 1])
    want = x.copy()
    want[1, V - 1] = bf16(np.float32([x[1, V - 1] + np.float32(2.5)]))[0]
    np.testing.assert_array_equal(host(y), want)
    lse = torch.zeros(2, device="cuda")
    ids, lps = torch.zeros((2, 9), dtype=torch.int32).cuda(), torch.zeros((2, 9)).cuda()
    tokens = torch.tensor([[7], [V - 1]], dtype=torch.int32).cuda()
    ranks, chosen = torch.zeros(2, dtype=torch.int32).cuda(), torch.zeros((2, 1)).cuda()
    s.logprobs(t, tokens=tokens, logprobs=chosen, ranks=ranks, lse=lse, top_ids=ids,
               top_logprobs=lps)
    for r in range(2):
        _, lp, want_lse, lp_bound, lse_bound = score_plain(x[r])
        assert abs(float(lse[r]) - want_lse) <= lse_bound
        token = int(tokens[r, 0])
        assert abs(float(chosen[r, 0]) - lp[token]) <= lp_bound[token]
        assert int(ranks[r]) == rank_of(x[r], token)
        np.testing.assert_array_equal(ids[r].cpu().numpy(), order(x[r])[:9])
    teacher = order(x[1])[:K].astype(np.uint32)
    t_ids = torch.from_numpy(np.stack([teacher, teacher]).view(np.int32)).cuda()
    values = torch.zeros((2, K)).cuda()
    loss, g = torch.zeros(2).cuda(), torch.ones(2).cuda()
    s.launch_distill_step(s.distill_args(t, t_ids, values, loss=loss, grad_loss=g, grad=y))
    grad = host(y)
    for r in range(2):
        want_loss, want_grad, loss_bound, grad_bound = distill_plain(
            x[r], teacher, np.zeros(K, np.float32), 1.0, True)
        assert abs(float(loss[r]) - want_loss) <= loss_bound + U * abs(want_loss)
        bound = grad_bound + 4 * U * np.abs(want_grad) + 1e-37
        assert np.all(excess(grad[r], want_grad, bound, "bf16") <= 1)
    s.close()
    del buf, out, t, y
    torch.cuda.empty_cache()


def test_more_rows_than_a_launch():
    """1.1 million rows of 3 tokens: calls of several launches."""
    import torch
    rows, V = 1100000, 3
    rng = np.random.default_rng(2)
    x = rng.normal(0, 2, (rows, V)).astype(np.float32)
    t, _ = device_rows(x, "f32")
    tokens = rng.integers(0, V, (rows, 1)).astype(np.int32)
    lse, chosen = torch.zeros(rows).cuda(), torch.zeros((rows, 1)).cuda()
    ranks = torch.zeros(rows, dtype=torch.int32).cuda()
    s = J.Scorer(V, rows)
    s.logprobs(t, tokens=torch.from_numpy(tokens).cuda(), lse=lse, logprobs=chosen, ranks=ranks)
    y = x.astype(np.float64)
    m = y.max(1, keepdims=True)
    want = (m + np.log(np.exp(y - m).sum(1, keepdims=True)))[:, 0]
    # Three exponentials, their sum, a logarithm and a sum: values of at most 16.
    assert np.abs(lse.cpu().numpy() - want).max() <= 64 * U * 16
    picked = np.take_along_axis(y, tokens.astype(np.int64), 1)
    assert np.abs(chosen.cpu().numpy() - (picked - want[:, None])).max() <= 64 * U * 16
    ahead = (y > picked) | ((y == picked) & (np.arange(V) < tokens))
    np.testing.assert_array_equal(ranks.cpu().numpy(), ahead.sum(1) + 1)
    # A list of one token: cross entropy.
    loss, grad = torch.zeros(rows).cuda(), torch.zeros_like(t)
    g = torch.ones(1).cuda().expand(rows)
    values, ids = torch.zeros((rows, 1)).cuda(), torch.from_numpy(tokens).cuda()
    s.launch_distill_step(s.distill_args(t, ids, values, loss=loss, grad_loss=g, grad=grad))
    assert np.abs(loss.cpu().numpy() - (want[:, None] - picked)[:, 0]).max() <= 64 * U * 16
    q = np.exp(y - want[:, None])
    np.put_along_axis(q, tokens.astype(np.int64), np.take_along_axis(q, tokens.astype(np.int64), 1) - 1, 1)
    assert np.abs(host(grad) - q).max() <= 64 * U * 16
    s.close()


@pytest.mark.parametrize("rows", [1, 2, 140, 410])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_largest_vocabulary(rows, dtype):
    """524,288 tokens: few rows by chunks, many by whole rows."""
    import torch
    V, K = 524288, 200
    rng = np.random.default_rng(3)
    z = rng.normal(0, 2, (2, V)).astype(np.float32)
    if dtype == "bf16":
        z = bf16(z)
    kind = torch.bfloat16 if dtype == "bf16" else torch.float32
    t = torch.from_numpy(z).to(kind).cuda()[torch.arange(rows) % 2].contiguous()
    ids = np.stack([rng.choice(V, K, replace=False), np.argsort(-z[1])[:K]]).astype(np.uint32)
    values = rng.normal(0, 2, (2, K)).astype(np.float32)
    pick = np.arange(rows) % 2
    loss, grad = torch.zeros(rows).cuda(), torch.zeros_like(t)
    g = torch.ones(1).cuda().expand(rows)
    s = J.Scorer(V, rows)
    d_ids = torch.from_numpy(ids[pick].view(np.int32)).cuda()
    d_values = torch.from_numpy(values[pick]).cuda()
    s.launch_distill_step(s.distill_args(t, d_ids, d_values, loss=loss, grad_loss=g, grad=grad,
                                         temperature=2.0))
    for r in {0, min(1, rows - 1), rows - 1}:
        want_loss, want, loss_bound, bound = distill_plain(z[r % 2], ids[r % 2], values[r % 2],
                                                           2.0, True)
        assert abs(float(loss[r]) - want_loss) <= loss_bound + U * abs(want_loss)
        got = host(grad[r:r + 1])[0]
        assert np.all(excess(got, want, bound + 4 * U * np.abs(want) + 1e-37, dtype) <= 1)
    s.close()


def test_host_tensors_are_refused():
    """A host address would fault the device: every tensor is asked for."""
    import torch
    V, rows = 64, 2
    t = torch.zeros((rows, V), device="cuda")
    ids, values = (torch.zeros((rows, 3), dtype=d, device="cuda")
                   for d in (torch.int32, torch.float32))
    each = torch.zeros(rows, device="cuda")
    masks = torch.zeros((rows, 2), dtype=torch.int32, device="cuda")
    s = J.Scorer(V, rows)
    pol = [J.policy()] * rows
    process = dict(logits=t, policies=pol, out=t, masks=masks, extra_tokens=masks)
    logprobs = dict(logits=t, tokens=ids, temperatures=each, lse=each, logprobs=values,
                    ranks=masks[:, 0].contiguous(), top_ids=ids, top_logprobs=values)
    distill = dict(logits=t, teacher_ids=ids, teacher_values=values, loss=each, lse=each,
                   saved=torch.zeros((rows, 5), device="cuda"), grad_loss=each, grad=t)
    for build, kw in ((s.process_args, process), (s.logprobs_args, logprobs),
                      (s.distill_args, distill)):
        build(**kw)
        for name, value in kw.items():
            if torch.is_tensor(value):
                with pytest.raises(ValueError, match="not on the GPU"):
                    build(**dict(kw, **{name: value.cpu()}))
    with pytest.raises(ValueError):
        s.process_args(**dict(process, mask_rows=[0, -1]))
    s.close()
