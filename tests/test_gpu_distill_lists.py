"""The teacher's side of the distillation: a list's probabilities, as the forward
pass saves them, against 64 bits, whatever the values' common offset and however
small the temperature."""
import numpy as np
import pytest

import jf_sampler as J
from scoring_cases import U, device_rows, distill_plain, excess, host

pytestmark = pytest.mark.gpu


def list_plain(values, T):
    """(probabilities of softmax(values / T), their errors' bound) in 64 bits."""
    u, T = values.astype(np.float64), float(np.float32(T))
    d = (u - u.max()) / T
    e = np.exp(d)
    log_sum = np.log(e.sum())
    log_p = d - log_sum
    # An exponent is a difference, a rounded inverse and a product: 3 roundings of
    # |d|; an exponential is good to 2 ulp, which are 4 U, and so is the logarithm.
    # A sum goes through 4 slots of a lane and 6 steps of the wave, then log_p is a
    # difference and p an exponential.
    far = np.minimum(np.abs(d), 200.0)  # past that the exponential is 0
    total = 14 + 3 * (e * far).sum() / e.sum()
    bound = U * (3 * far + total + 4 * log_sum + np.minimum(np.abs(log_p), 200.0) + 4)
    return np.exp(log_p), bound


def run(z, ids, values, T, mode):
    """(losses, probabilities, gradients for loss gradients of T), each row's."""
    import torch
    rows, V = z.shape
    K = values.shape[1]
    t, _ = device_rows(z, "f32")
    loss, saved = torch.full((rows,), 7.0).cuda(), torch.full((rows, 2 + K), 7.0).cuda()
    grad = torch.full((rows, V), 7.0).cuda()
    d_ids = torch.from_numpy(ids.astype(np.int32)).cuda()
    d_values, g = torch.from_numpy(values).cuda(), torch.full((rows,), T).cuda()
    s = J.Scorer(V, rows)
    kw = dict(temperature=T, normalize=True, saved=saved)
    if mode == "step":
        s.launch_distill_step(s.distill_args(t, d_ids, d_values, loss=loss, grad_loss=g, grad=grad,
                                             **kw))
    else:
        s.launch_distill(s.distill_args(t, d_ids, d_values, loss=loss, **kw))
        s.launch_distill_backward(s.distill_args(t, d_ids, None, grad_loss=g, grad=grad, **kw))
    got = host(loss), host(saved)[:, 2:], host(grad)
    s.close()
    return got


@pytest.mark.parametrize("K", [1, 7, 64, 65, 256])
@pytest.mark.parametrize("T", [0.0625, 0.1, 1.0, 4.0])
@pytest.mark.parametrize("mode", ["separate", "step"])
def test_a_common_offset_costs_the_probabilities_nothing(K, T, mode):
    rng = np.random.default_rng(K)
    V, offsets = 3000, np.float32([0, 30, -30, 1e4, -1e4, 1e6])[:, None]
    z = rng.normal(0, 3, (6, V)).astype(np.float32)
    values = (rng.normal(0, 2, (6, K)).astype(np.float32) + offsets).astype(np.float32)
    ids = np.stack([rng.choice(V, K, replace=False) for _ in range(6)])
    loss, p, _ = run(z, ids, values, T, mode)
    for r in range(6):
        want, bound = list_plain(values[r], T)
        assert np.all(np.abs(p[r] - want) <= bound * want + 1e-38), (r, np.abs(p[r] - want).max())
        want_loss, _, loss_bound, _ = distill_plain(z[r], ids[r], values[r], float(np.float32(T)),
                                                    True)
        assert abs(loss[r] - want_loss) <= loss_bound + U * abs(want_loss)


@pytest.mark.parametrize("K", [2, 64, 200])
@pytest.mark.parametrize("T", [float(np.finfo(np.float32).tiny), 1e-37])
@pytest.mark.parametrize("mode", ["separate", "step"])
def test_values_past_the_range_at_a_small_temperature(K, T, mode):
    """u / T overflows fp32 for every value: equal values share the mass, one
    ahead of the others has it. The student's logits are equal, so a loss is
    ln V - ln K or ln V, and T times a gradient is 1 / V - p."""
    V, T = 3000, float(np.float32(T))
    values = np.repeat(np.float32([300, -300, 3e38, -3e38, 300, -300])[:, None], K, 1)
    values[4, 1:] = 299
    values[5, 1:] = -3e38
    want = np.full((6, K), 1 / K)
    want[4:] = 0
    want[4:, 0] = 1
    ids = np.stack([np.arange(K) * 13 for _ in range(6)])
    loss, p, grad = run(np.zeros((6, V), np.float32), ids, values, T, mode)
    assert np.all(np.abs(p - want) <= 32 * U * want)
    losses = np.log(V) - np.where(np.arange(6) < 4, np.log(K), 0.0)
    assert np.all(np.abs(loss - losses) <= 64 * U * np.log(V))
    pulled = np.full((6, V), 1 / V)
    np.put_along_axis(pulled, ids, 1 / V - want, 1)
    assert np.all(excess(grad, pulled, 64 * U * (1 / V + 1 / K + np.abs(pulled)), "f32") <= 1)


def test_lists_without_mass():
    """Values of -infinity are no probability; a NaN reaches the row."""
    values = np.float32([[-np.inf, -np.inf], [-np.inf, -1e30], [np.nan, 0.0]])
    ids = np.tile([4, 9], (3, 1))
    loss, p, grad = run(np.zeros((3, 50), np.float32), ids, values, 0.5, "step")
    assert loss[0] == 0 and not p[0].any() and not grad[0].any()
    np.testing.assert_array_equal(p[1], [0, 1])
    assert abs(loss[1] - np.log(50)) <= 64 * U * np.log(50)
    assert np.isnan(loss[2]) and np.isnan(grad[2]).all()


@pytest.mark.parametrize("V", [3000, 80003])
@pytest.mark.parametrize("g", [np.nan, np.inf, -np.inf, 2.0])
@pytest.mark.parametrize("mode", ["separate", "step"])
def test_tokens_without_probability_have_no_share_of_the_loss_gradient(V, g, mode):
    """No slot of rows 0 and 1 has probability: no gradient, whatever comes in. In
    row 2 one has: the others' gradients are g / T times q, as any token's.
    Short rows by whole rows, long ones by chunks."""
    rng = np.random.default_rng(4)
    z = rng.normal(0, 1, (3, V)).astype(np.float32)
    ids = np.tile([5, 70, V - 1], (3, 1))
    values = np.float32([[-np.inf] * 3, [-np.inf, -300, -np.inf], [-1, -np.inf, -np.inf]])
    import torch
    t, _ = device_rows(z, "f32")
    loss, saved = torch.full((3,), 7.0).cuda(), torch.full((3, 5), 7.0).cuda()
    grad, gl = torch.full((3, V), 7.0).cuda(), torch.full((3,), g).cuda()
    d_ids, d_values = torch.from_numpy(ids.astype(np.int32)).cuda(), torch.from_numpy(values).cuda()
    s = J.Scorer(V, 3)
    kw = dict(normalize=False, saved=saved)
    if mode == "step":
        s.launch_distill_step(s.distill_args(t, d_ids, d_values, loss=loss, grad_loss=gl,
                                             grad=grad, **kw))
    else:
        s.launch_distill(s.distill_args(t, d_ids, d_values, loss=loss, **kw))
        s.launch_distill_backward(s.distill_args(t, d_ids, None, grad_loss=gl, grad=grad, **kw))
    got = host(grad)
    assert not host(loss)[:2].any() and not got[:2].any()
    if g == 2.0:
        _, want, _, bound = distill_plain(z[2], ids[2], values[2], 1.0, False)
        assert np.all(np.abs(got[2] - 2 * want) <= 2 * bound + 8 * U * np.abs(want))
    else:
        # The listed token takes g (q - p), inf - inf in the order it is worked out in.
        np.testing.assert_array_equal(np.delete(got[2], 5), np.full(V - 1, g))
    s.close()
