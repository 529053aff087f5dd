"""The plain 64-bit implementations that the operators over rows of logits are
tested against, themselves against differences and small closed forms, and the
refusals that need no GPU."""
import ctypes

import numpy as np
import pytest

import jf_sampler as J
from scoring_cases import NO, bf16, distill_plain, order, process_plain, rank_of, score_plain


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T", [1.0, 2.5])
def test_distillation_gradient_is_the_losses_difference(normalize, T):
    rng = np.random.default_rng(1)
    z = rng.normal(0, 2, 40)
    ids = np.uint32([3, 39, NO, 7, 3, 40])
    values = np.float32([-1.0, -2.0, 9.0, -1.5, 5.0, 5.0])
    loss, grad, _, _ = distill_plain(z, ids, values, T, normalize)
    for j in range(40):
        step = np.zeros(40)
        step[j] = 1e-5
        hi = distill_plain(z + step, ids, values, T, normalize)[0]
        lo = distill_plain(z - step, ids, values, T, normalize)[0]
        assert abs((hi - lo) / 2e-5 - grad[j]) < 1e-8
    assert abs(grad.sum()) < 1e-12 and loss > 0 or not normalize


def test_distillation_of_one_token_is_cross_entropy():
    z = np.random.default_rng(2).normal(0, 2, 30)
    loss, grad, _, _ = distill_plain(z, np.uint32([4]), np.float32([12.0]), 1.0, True)
    q = np.exp(z) / np.exp(z).sum()
    assert abs(loss + np.log(q[4])) < 1e-12
    q[4] -= 1
    np.testing.assert_allclose(grad, q, atol=1e-14)


def test_scores_order_and_ranks():
    x = np.float32([1.0, np.nan, 3.0, -np.inf, 3.0, -0.0, 0.0])
    np.testing.assert_array_equal(order(x), [2, 4, 0, 5, 6])
    assert [rank_of(x, t) for t in (2, 4, 0, 6)] == [1, 2, 3, 5]
    _, lp, lse, _, _ = score_plain(np.log(np.float64([1, 2, 5])), 1.0)
    np.testing.assert_allclose(np.exp(lp), [0.125, 0.25, 0.625], rtol=1e-12)
    assert abs(lse - np.log(8)) < 1e-12
    _, lp, lse, _, _ = score_plain(np.full(4, -np.inf))
    assert np.isneginf(lp).all() and np.isneginf(lse)


def test_processed_values():
    p = J.policy(repetition=2.0, presence=0.5, frequency=0.25)
    words = np.uint32([0, 0x80000000, 2, 0x80000001, 0])
    y, edited, _ = process_plain(np.float32([1, 1, 1, -1, 1]), p, words, extra=[4, 4, 2, NO],
                                 bias={0: 3.0, 2: -np.inf}, mask=np.array([1, 1, 1, 0, 1], bool),
                                 stops=(1, NO))
    np.testing.assert_allclose(y, [4.0, -np.inf, -np.inf, -np.inf, 0.5 - 0.5 - 0.5])
    assert edited.all()


def test_bf16_rounding():
    x = np.float32([1.0, 1.00390625, 1.01171875, 3.4e38, -1e-45, np.nan])
    np.testing.assert_array_equal(bf16(x), np.float32([1.0, 1.0, 1.015625, np.inf, -0.0, np.nan]))


def test_refusals_before_any_device_call():
    h = ctypes.c_void_p()
    for fn, args, message in (
            ("jf_scorer_create", (0, 1), "geometry"),
            ("jf_scorer_create", (524289, 1), "524288 tokens"),
            ("jf_scorer_create", (10, 0), "1..4194304"),
            ("jf_scorer_create", (10, (1 << 22) + 1), "1..4194304"),
            ("jf_bias_table_create", (0, 1, 1), "geometry"),
            ("jf_bias_table_create", (10, 0, 1), "geometry"),
            ("jf_bias_table_create", (10, 1, 0), "geometry")):
        rc = getattr(J.lib(), fn)(*args, ctypes.byref(h))
        assert rc == J.JF_ERR_INVALID_ARGUMENT and not h.value
        assert message in J.lib().jf_last_error().decode()
    for fn, record in (("jf_process_logits", J.JfProcessArgs()), ("jf_logprobs", J.JfLogprobsArgs()),
                       ("jf_distill", J.JfDistillArgs()), ("jf_distill_step", J.JfDistillArgs()),
                       ("jf_distill_backward", J.JfDistillArgs())):
        assert getattr(J.lib(), fn)(None, ctypes.byref(record), None) == J.JF_ERR_INVALID_ARGUMENT
        assert "null scorer" in J.lib().jf_last_error().decode()
    assert J.lib().jf_bias_table_set(None, 0, None, None, 0, None) == J.JF_ERR_INVALID_ARGUMENT
    assert J.lib().jf_scorer_destroy(None) == 0 and J.lib().jf_bias_table_destroy(None) == 0
