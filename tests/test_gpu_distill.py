"""Distillation (jf_distill, jf_distill_backward, jf_distill_step and the torch
loss over them) against a plain implementation in 64 bits and against
differences of the losses."""
import numpy as np
import pytest

import jf_sampler as J
from scoring_cases import U, bf16, device_rows, distill_plain, excess, host, score_plain

pytestmark = pytest.mark.gpu

NO = 0xFFFFFFFF


def _ids(ids):
    import torch
    return torch.from_numpy(np.ascontiguousarray(ids, np.uint32).view(np.int32)).cuda()


def lists(rng, z, K, normalize, T):
    """Teacher lists near the rows' best tokens; a list may be short, hold
    absent slots anywhere, repeat a token, or be empty."""
    rows, V = z.shape
    teacher = z + rng.normal(0, 1, z.shape)
    ids = np.full((rows, K), NO, np.uint32)
    values = np.full((rows, K), np.nan, np.float32)
    for r in range(rows):
        n = min(K, V)
        best = np.argsort(-teacher[r], kind="stable")[:n]
        u = teacher[r][best]
        if not normalize:
            u = u / T - np.log(np.exp((teacher[r] - teacher[r].max()) / T).sum()) \
                - teacher[r].max() / T
        at = rng.permutation(K)[:n]
        ids[r, at], values[r, at] = best, u
        if r % 4 == 1:
            gone = rng.random(K) < 0.4
            ids[r, gone] = rng.choice([NO, V, V + 5], int(gone.sum()))
        if r % 4 == 2 and K > 2:
            ids[r, K - 1], values[r, K - 1] = ids[r, 0], 3.0
        if r % 8 == 7:
            ids[r] = NO
    return ids, values


def check(z, ids, values, T, normalize, g, dtype, got):
    for r in range(len(z)):
        loss, grad, loss_bound, grad_bound = distill_plain(z[r], ids[r], values[r], T, normalize)
        if "loss" in got:
            bound = loss_bound + U * abs(loss)
            assert abs(got["loss"][r] - loss) <= bound, (r, got["loss"][r], loss, bound)
        if "lse" in got:
            _, _, lse, _, lse_bound = score_plain(z[r], T)
            assert abs(got["lse"][r] - lse) <= lse_bound
        if "grad" in got:
            want = grad * float(np.float32(g[r]))
            bound = (grad_bound + 4 * U * np.abs(grad)) * abs(g[r]) + 1e-37
            over = excess(got["grad"][r], want, bound, dtype)
            assert np.all(over <= 1), (r, int(np.argmax(over)), over.max())


def run(z, ids, values, T, normalize, g, dtype, mode="separate", pad=0, lead=0):
    """Host results; mode: separate calls, the step, or the step in place."""
    import torch
    rows, V = z.shape
    K = ids.shape[1]
    t, buf = device_rows(z, dtype, pad, lead)
    grad, grad_buf = (t, buf) if mode == "in place" else \
        device_rows(np.ones_like(z), dtype, (pad + 1) % 3, lead)
    around = grad_buf.clone()
    loss, lse = torch.full((rows,), 7.0).cuda(), torch.full((rows,), 7.0).cuda()
    gl = torch.from_numpy(np.asarray(g, np.float32)).cuda()
    s = J.Scorer(V, rows)
    kw = dict(temperature=T, normalize=normalize, loss=loss, lse=lse)
    d_ids, d_values = _ids(ids), torch.from_numpy(values).cuda()
    if mode == "separate":
        saved = torch.full((rows, 2 + K), 7.0).cuda()
        s.launch_distill(s.distill_args(t, d_ids, d_values, saved=saved, **kw))
        d_values.fill_(float("nan"))  # the backward pass reads none
        s.launch_distill_backward(s.distill_args(t, d_ids, d_values, temperature=T, saved=saved,
                                                 grad_loss=gl, grad=grad))
    else:
        s.launch_distill_step(s.distill_args(t, d_ids, d_values, grad_loss=gl, grad=grad, **kw))
    torch.cuda.synchronize()
    inside = torch.zeros_like(grad_buf, dtype=torch.bool)
    inside[lead:lead + rows * grad.stride(0)].view(rows, -1)[:, :V] = True
    assert torch.equal(grad_buf[~inside], around[~inside])
    s.close()
    return dict(loss=loss.cpu().numpy(), lse=lse.cpu().numpy(), grad=host(grad))


@pytest.mark.parametrize("V", [1, 2, 7, 65, 1000, 8191, 8192, 8193, 20011])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("normalize,T", [(True, 1.0), (True, 2.5), (False, 0.7)])
def test_losses_and_gradients(V, dtype, normalize, T):
    for K, mode in ((1, "separate"), (9, "step"), (64, "in place"), (256, "separate")):
        rng = np.random.default_rng(V + K)
        print(f"distill V={V} {dtype} normalize={normalize} T={T} K={K} {mode}", flush=True)
        z = rng.normal(0, 4, (9, V)).astype(np.float32)
        if dtype == "bf16":
            z = bf16(z)
        ids, values = lists(rng, z, K, normalize, T)
        g = rng.normal(0, 1, 9).astype(np.float32)
        g[3] = 0.0
        got = run(z, ids, values, T, normalize, g, dtype, mode, pad=V % 3, lead=V % 2)
        check(z, ids, values, T, normalize, g, dtype, got)
        assert not got["grad"][3].any() and not got["grad"][7].any() and got["loss"][7] == 0


# Lists of which most or all slots repeat a token, and of tokens apart by
# multiples of powers of two.
@pytest.mark.parametrize("K", [2, 63, 64, 65, 200, 256])
@pytest.mark.parametrize("mode", ["separate", "step"])
def test_a_token_counts_at_its_first_slot(K, mode):
    rng = np.random.default_rng(K)
    V, rows = 70001, 6
    z = rng.normal(0, 3, (rows, V)).astype(np.float32)
    ids = np.stack([np.full(K, 17), rng.integers(0, 3, K), rng.integers(0, max(2, K // 2), K),
                    rng.integers(0, 68, K) * 1024, rng.choice(V, K, replace=False),
                    np.repeat(rng.choice(V, K, replace=False), 2)[:K]]).astype(np.uint32)
    ids[3, K // 2] = NO
    values = rng.normal(0, 1, (rows, K)).astype(np.float32)
    g = np.ones(rows, np.float32)
    for normalize in (True, False):
        v = values if normalize else values - 8
        check(z, ids, v, 1.5, normalize, g, "f32", run(z, ids, v, 1.5, normalize, g, "f32", mode))


# Rows that start anywhere in a line, over more tokens than a block holds; the
# gradient's rows start elsewhere than the logits' but in place.
@pytest.mark.parametrize("V", [73001, 73727, 65536])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mode", ["step", "in place"])
@pytest.mark.parametrize("K", [5, 70])
def test_whole_rows_at_any_alignment(V, dtype, mode, K):
    rng = np.random.default_rng(V + K)
    z = rng.normal(0, 3, (5, V)).astype(np.float32)
    if dtype == "bf16":
        z = bf16(z)
    ids, values = lists(rng, z, K, True, 2.0)
    ids[:, 0] = 0, 1, V - 1, 2, 70
    g = rng.normal(0, 1, 5).astype(np.float32)
    for pad, lead in ((0, 0), (1, 1), (7, 33)):
        got = run(z, ids, values, 2.0, True, g, dtype, mode, pad, lead)
        check(z, ids, values, 2.0, True, g, dtype, got)


def test_cross_entropy_is_a_list_of_one():
    rng = np.random.default_rng(3)
    z = rng.normal(0, 3, (4, 9001)).astype(np.float32)
    labels = rng.integers(0, 9001, (4, 1)).astype(np.uint32)
    got = run(z, labels, np.zeros((4, 1), np.float32), 1.0, True, np.ones(4), "f32")
    for r in range(4):
        _, lp, _, bound, _ = score_plain(z[r])
        i = int(labels[r, 0])
        assert abs(got["loss"][r] + lp[i]) <= bound[i] + 8 * U * abs(lp[i])
        want = np.exp(lp)
        want[i] -= 1
        assert np.abs(got["grad"][r] - want).max() <= 1e-5


def test_gradients_against_differences():
    """The directional derivative from the gradient against a central
    difference of the losses, f32, a random direction per row: the losses are
    held to about 3e-6 of themselves (their own bound), the step leaves a
    third-order term of at most step^2 |d|^3 / T^3."""
    rng = np.random.default_rng(17)
    V, K, T = 3001, 12, 1.5
    z = rng.normal(0, 2, (6, V)).astype(np.float32)
    ids, values = lists(rng, z, K, True, T)
    d = rng.normal(0, 1, z.shape).astype(np.float32)
    d /= np.abs(d).max(1, keepdims=True)
    step = np.float32(2.0 ** -4)
    ones = np.ones(6)
    grad = run(z, ids, values, T, True, ones, "f32")["grad"].astype(np.float64)
    up, down = (z + step * d).astype(np.float32), (z - step * d).astype(np.float32)
    hi = run(up, ids, values, T, True, ones, "f32")["loss"].astype(np.float64)
    lo = run(down, ids, values, T, True, ones, "f32")["loss"].astype(np.float64)
    moved = (up.astype(np.float64) - down) / 2
    for r in range(6):
        bounds = [distill_plain(v[r], ids[r], values[r], T, True)[2] for v in (up, down)]
        error = sum(bounds) + 2 * U * (hi[r] + lo[r])
        third = 2 * (float(step) / T) ** 3
        assert abs((grad[r] * moved[r]).sum() - (hi[r] - lo[r]) / 2) <= error / 2 + third


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_students(dtype):
    """Masked student rows: a listed token that the mask drops, rows that
    leave nothing, the type's lowest value as a mask."""
    rng = np.random.default_rng(21)
    V, K = 9000, 6
    z = rng.normal(0, 3, (5, V)).astype(np.float32)
    ids = np.stack([rng.choice(V, K, replace=False) for _ in range(5)]).astype(np.uint32)
    values = rng.normal(0, 1, (5, K)).astype(np.float32)
    z[0, ids[0, 2]] = -np.inf
    z[1] = -np.inf
    lowest = np.float32(-3.3895314e38)
    z[2, np.setdiff1d(np.arange(V), ids[2])] = lowest
    z[3] = lowest
    values[4, 3] = -np.inf  # no teacher probability where the student has none
    z[4, ids[4, 3]] = -np.inf
    if dtype == "bf16":
        z = bf16(z)
    got = run(z, ids, values, 1.0, True, np.ones(5), dtype)
    assert np.isposinf(got["loss"][0]) and np.isposinf(got["loss"][1])
    assert np.isneginf(got["lse"][1])
    assert np.all(np.isfinite(got["grad"]))
    # Nothing left: q is 0 everywhere, and the listed tokens pull alone.
    p = np.exp(values[1].astype(np.float64))
    p /= p.sum()
    want = np.zeros(V)
    want[ids[1].astype(int)] = -p
    assert np.all(excess(got["grad"][1], want, 32 * U * np.abs(want) + 1e-37, dtype) <= 1)
    keep = [2, 3, 4]
    check(z[keep], ids[keep], values[keep], 1.0, True, np.ones(3), dtype,
          {k: v[keep] for k, v in got.items()})
    check(z[:1], ids[:1], values[:1], 1.0, True, np.ones(1), dtype, dict(grad=got["grad"][:1]))


def test_rows_with_nan_and_infinity():
    """NaN and +infinity reach their own row's loss and gradient, except where
    the row has no list or its loss gradient is 0."""
    rng = np.random.default_rng(22)
    V = 9000
    z = rng.normal(0, 3, (5, V)).astype(np.float32)
    z[0, 8500], z[1, 3], z[2, 3], z[3, 3] = np.nan, np.inf, np.nan, np.nan
    ids = np.tile(np.uint32([5, 6, 7]), (5, 1))
    ids[2] = NO
    got = run(z, ids, np.zeros((5, 3), np.float32), 1.0, True, [1, 1, 1, 0, 1], "f32")
    assert np.isnan(got["loss"][[0, 1, 3]]).all() and got["loss"][2] == 0
    assert np.isnan(got["grad"][[0, 1]]).all()
    assert not got["grad"][2].any() and not got["grad"][3].any()
    assert np.isfinite(got["grad"][4]).all() and np.isfinite(got["loss"][4])


@pytest.mark.parametrize("rows", [1, 40, 700, 2100])
def test_many_rows(rows):
    rng = np.random.default_rng(rows)
    V, K = 9001, 5
    z = bf16(rng.normal(0, 3, (rows, V)).astype(np.float32))
    ids, values = lists(rng, z, K, True, 2.0)
    g = np.full(rows, 1.0 / rows, np.float32)
    got = run(z, ids, values, 2.0, True, g, "bf16", "step")
    check(z, ids, values, 2.0, True, g, "bf16", got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_torch_loss(dtype):
    """The loss under autograd: a mean's expanded gradient, logits that are a
    view of a wider buffer, two forwards before their backwards."""
    import torch
    from jf_sampler.train import distill_loss
    rng = np.random.default_rng(30)
    rows, V, K = 6, 8500, 8
    z = rng.normal(0, 3, (2, rows, V)).astype(np.float32)
    if dtype == "bf16":
        z = bf16(z)
    s = J.Scorer(V, rows)
    wide, losses, want = [], [], []
    for n in range(2):
        t, _ = device_rows(z[n], dtype, 3)
        leaf = torch.zeros((rows, V + 3), dtype=t.dtype, device="cuda")
        leaf[:, :V] = t
        leaf.requires_grad_(True)
        ids, values = lists(rng, z[n], K, True, 1.0)
        loss = distill_loss(s, leaf[:, :V], _ids(ids), torch.from_numpy(values).cuda())
        wide.append(leaf)
        losses.append(loss)
        want.append((ids, values))
    for n in range(2):
        losses[n].mean().backward()
    for n in range(2):
        g = np.full(rows, np.float32(1) / np.float32(rows), np.float32)
        grad = host(wide[n].grad)
        assert not grad[:, V:].any()
        check(z[n], *want[n], 1.0, True, g, dtype,
              dict(loss=losses[n].detach().cpu().numpy(), grad=grad[:, :V]))
    with pytest.raises(ValueError):
        distill_loss(s, wide[0][:, :V], torch.zeros((rows, 257), dtype=torch.int32).cuda(),
                     torch.zeros((rows, 257)).cuda())
    s.close()


def test_repeats_are_bit_identical_and_replay_under_a_graph():
    import torch
    rng = np.random.default_rng(31)
    rows, V, K = 5, 20011, 10
    z = rng.normal(0, 3, (rows, V)).astype(np.float32)
    ids, values = lists(rng, z, K, True, 1.0)
    t, _ = device_rows(z, "f32")
    grad, loss = torch.zeros_like(t), torch.zeros(rows).cuda()
    s = J.Scorer(V, rows)
    g = torch.ones(1).cuda().expand(rows)
    a = s.distill_args(t, _ids(ids), torch.from_numpy(values).cuda(), loss=loss, grad_loss=g,
                       grad=grad)
    hold = (g, t)
    d_ids, d_values = _ids(ids), torch.from_numpy(values).cuda()
    a.teacher_ids, a.teacher_values = d_ids.data_ptr(), d_values.data_ptr()
    s.launch_distill_step(a)
    want = [host(loss), host(grad)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.launch_distill_step(a)
    for turn in range(4):
        loss.zero_()
        grad.zero_()
        if turn % 2:
            s.launch_distill_step(a)
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(host(loss), want[0])
        np.testing.assert_array_equal(host(grad), want[1])
    del graph, hold
    s.close()


def test_refusals():
    import torch
    V, rows, K = 100, 2, 3
    t, _ = device_rows(np.zeros((rows, V), np.float32), "f32")
    ids, values = torch.zeros((rows, K), dtype=torch.int32).cuda(), torch.zeros((rows, K)).cuda()
    loss, saved = torch.zeros(rows).cuda(), torch.zeros((rows, 2 + K)).cuda()
    grad = torch.zeros_like(t)
    s = J.Scorer(V, rows)

    def refused(message, fn=None, **change):
        a = s.distill_args(t, ids, values, loss=loss, saved=saved, grad_loss=loss, grad=grad)
        for k, v in change.items():
            setattr(a, k, v)
        for f in (fn,) if fn else (s.launch_distill, s.launch_distill_step,
                                   s.launch_distill_backward):
            with pytest.raises(J.JfError) as e:
                f(a)
            assert e.value.code == J.JF_ERR_INVALID_ARGUMENT and message in e.value.message, \
                e.value.message

    refused("batch width", rows=0)
    refused("batch width", rows=3)
    refused("dtype", dtype=2)
    refused("null logits", logits=None)
    refused("aligned", logits=t.data_ptr() + 2)
    refused("stride is below", logits_stride=V - 1)
    refused("1..256", teacher_count=0)
    refused("1..256", teacher_count=257)
    refused("needs ids", teacher_ids=None)
    refused("needs ids", s.launch_distill, teacher_values=None)
    refused("teacher row stride", teacher_stride=2)
    for T in (0.0, -1.0, float("nan"), float("inf"), 1e-39):
        refused("temperature", temperature=T)
    refused("null losses", s.launch_distill, out_loss=None)
    refused("null losses", s.launch_distill_step, out_loss=None)
    refused("null loss gradients", s.launch_distill_step, grad_loss=None)
    refused("saved", s.launch_distill_backward, saved=None)
    refused("null gradients", s.launch_distill_backward, grad=None)
    refused("gradients are not aligned", s.launch_distill_step, grad=grad.data_ptr() + 2)
    refused("gradients row stride", s.launch_distill_step, grad_stride=V - 1)
    refused("in place", s.launch_distill_step, grad=t.data_ptr(), grad_stride=V + 1)
    for bad in (dict(loss=loss[:1]), dict(grad=grad.bfloat16()), dict(grad_loss=loss.double()),
                dict(saved=saved[:, :-1]), dict(grad=grad[:, :50])):
        with pytest.raises(ValueError):
            s.distill_args(t, ids, values, **bad)
    with pytest.raises(ValueError):
        s.distill_args(t, ids.long(), values)
    assert not grad.any() and not loss.any() and not saved.any()
    s.close()


@pytest.mark.parametrize("rows", [6, 200])
def test_a_row_without_a_list_has_no_gradient_whatever_comes_in(rows):
    """NaN and infinite loss gradients of rows with empty lists (few rows by
    chunks, many by whole rows), separate passes and the step."""
    rng = np.random.default_rng(41)
    V = 70000
    z = bf16(rng.normal(0, 2, (rows, V)).astype(np.float32))
    ids = np.tile(np.uint32([5, 6]), (rows, 1))
    ids[:3] = NO
    g = np.ones(rows, np.float32)
    g[0], g[1], g[4] = np.nan, np.inf, np.nan
    for mode in ("separate", "step"):
        got = run(z, ids, np.zeros((rows, 2), np.float32), 1.0, True, g, "bf16", mode)
        assert not got["grad"][:3].any()
        assert np.isnan(got["grad"][4]).all()
        check(z[3:4], ids[3:4], np.zeros((1, 2), np.float32), 1.0, True, g[3:4], "bf16",
              dict(grad=got["grad"][3:4]))
