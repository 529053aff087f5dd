"""The torch loss (jf_sampler.train.distill_loss) as trainers use it: list buffers
filled anew between a forward pass and its backward pass, empty batches."""
import numpy as np
import pytest

import jf_sampler as J
from scoring_cases import U, device_rows, distill_plain, excess, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("refill", ["library", "torch"])
@pytest.mark.parametrize("kind", ["int32", "uint32"])
def test_list_buffers_may_be_filled_anew_before_the_backward_pass(normalize, refill, kind):
    """Two micro-batches through the same list buffers, as Scorer.logprobs fills
    them, their losses added up before one backward pass."""
    import torch
    from jf_sampler.train import distill_loss
    rng = np.random.default_rng(1)
    rows, V, K = 5, 9000, 12
    z = rng.normal(0, 2, (2, rows, V)).astype(np.float32)
    teacher = rng.normal(0, 3, (2, rows, V)).astype(np.float32)
    s = J.Scorer(V, rows)
    ids = torch.zeros((rows, K), dtype=torch.int32).cuda()
    lps = torch.zeros((rows, K)).cuda()
    leaves, total, want = [], 0.0, []
    for n in range(2):
        t, _ = device_rows(teacher[n], "f32")
        s.logprobs(t, top_ids=ids, top_logprobs=lps)
        leaf = torch.from_numpy(z[n]).cuda().requires_grad_(True)
        with torch.no_grad():
            again = distill_loss(s, leaf, ids, lps, temperature=1.5, normalize=normalize)
        loss = distill_loss(s, leaf, ids.view(getattr(torch, kind)), lps, temperature=1.5,
                            normalize=normalize)
        assert torch.equal(again, loss) and not again.requires_grad
        total = total + loss.sum()
        leaves.append(leaf)
        want.append((loss.detach(), ids.cpu().numpy().copy(), lps.cpu().numpy().copy()))
    if refill == "torch":
        ids.fill_(-1)
        lps.fill_(float("nan"))
    total.backward()
    for n in range(2):
        got, (loss, i, v) = host(leaves[n].grad), want[n]
        for r in range(rows):
            want_loss, grad, loss_bound, bound = distill_plain(z[n][r], i[r].astype(np.uint32),
                                                               v[r], 1.5, normalize)
            assert abs(float(loss[r]) - want_loss) <= loss_bound + U * abs(want_loss)
            assert np.all(excess(got[r], grad, bound + 4 * U * np.abs(grad) + 1e-37, "f32") <= 1)
    s.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_an_empty_batch_has_no_losses_and_an_empty_gradient(dtype):
    """A packed batch none of whose tokens is trained on."""
    import torch
    from jf_sampler.train import distill_loss
    V, K = 500, 4
    s = J.Scorer(V, 8)
    leaf = torch.randn((3, V), device="cuda", dtype=getattr(torch, dtype)).requires_grad_(True)
    ids, values = torch.zeros((0, K), dtype=torch.int32).cuda(), torch.zeros((0, K)).cuda()
    loss = distill_loss(s, leaf[:0], ids, values)
    assert loss.shape == (0,) and loss.dtype == torch.float32 and loss.is_cuda
    loss.sum().backward()
    assert leaf.grad.shape == (3, V) and leaf.grad.dtype == leaf.dtype and not leaf.grad.any()
    # Its tensors are looked at all the same.
    for bad in ((leaf[:0, :9], ids, values), (leaf[:1], ids, values), (leaf[:0], ids.long(), values),
                (leaf[:0], ids, values[:, :2]), (leaf[:0], ids[:, :0], values[:, :0])):
        with pytest.raises(ValueError):
            distill_loss(s, *bad)
    s.close()
