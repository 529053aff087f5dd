"""Gradients by chunks of a row (jf_distill_backward, and steps of fewer rows than
are taken whole), every element against 64 bits: threads of two and of four
vectors, gradients that start on a line and within one, out of place and over the
logits, lists that are short, empty or repeat a token, listed tokens at the row's
and the chunks' ends."""
import numpy as np
import pytest

import jf_sampler as J
from scoring_cases import U, bf16, device_rows, distill_plain, excess, host
from test_gpu_distill import NO, _ids

pytestmark = pytest.mark.gpu


def edge_lists(rng, rows, V, K):
    """Ids from the row's ends, around the multiples of 2,048 (each chunk's size is
    one) and those less the elements of a line that may come ahead of a row."""
    edges = np.arange(0, V + 2048, 2048)
    near = np.concatenate([edges + d for d in (-65, -64, -63, -33, -32, -31, -2, -1, 0, 1, 2)])
    near = np.unique(near[(near >= 0) & (near < V)])
    ids = np.stack([rng.choice(near, K, replace=False) for _ in range(rows)]).astype(np.uint32)
    ids[:, 0], ids[:, K // 2] = V - 1, 0
    for r in range(rows):
        if r % 5 == 1:
            ids[r, rng.random(K) < 0.5] = rng.choice([NO, V, V + 7])
        if r % 5 == 2:
            ids[r] = ids[r, rng.integers(0, max(1, K // 3), K)]
        if r % 5 == 3:
            ids[r] = NO
    return ids, rng.normal(0, 2, (rows, K)).astype(np.float32)


def grads_of(z, ids, values, T, g, dtype, how, pad, lead, grad_lead):
    """Host losses and gradients; nothing around the gradients is written."""
    import torch
    rows, V = z.shape
    t, buf = device_rows(z, dtype, pad, lead)
    in_place = how.endswith("in place")
    grad, grad_buf = (t, buf) if in_place else \
        device_rows(np.ones_like(z), dtype, pad, grad_lead)
    around, first = grad_buf.clone(), lead if in_place else grad_lead
    loss, gl = torch.full((rows,), 7.0).cuda(), torch.from_numpy(g).cuda()
    saved = torch.full((rows, 2 + ids.shape[1]), 7.0).cuda()
    d_ids, d_values = _ids(ids), torch.from_numpy(values).cuda()
    s = J.Scorer(V, rows)
    kw = dict(temperature=T, loss=loss)
    if how.startswith("backward"):
        s.launch_distill(s.distill_args(t, d_ids, d_values, saved=saved, **kw))
        s.launch_distill_backward(s.distill_args(t, d_ids, None, temperature=T, saved=saved,
                                                 grad_loss=gl, grad=grad))
    else:
        # Saved in the scorer, or in the caller's buffer.
        s.launch_distill_step(s.distill_args(t, d_ids, d_values, grad_loss=gl, grad=grad,
                                             saved=saved if "saved" in how else None, **kw))
    torch.cuda.synchronize()
    inside = torch.zeros_like(grad_buf, dtype=torch.bool)
    inside[first:first + rows * grad.stride(0)].view(rows, -1)[:, :V] = True
    assert torch.equal(grad_buf[~inside], around[~inside])
    got = loss.cpu().numpy(), host(grad)
    s.close()
    return got


HOWS = ["backward", "backward in place", "step", "saved step", "step in place"]


def check(rows, V, dtype, K, how, pad, lead, grad_lead):
    print(f"gradients {rows} x {V} {dtype} K={K} {how} pad={pad} lead={lead}/{grad_lead}",
          flush=True)
    rng = np.random.default_rng(rows + V + K + HOWS.index(how))
    z = rng.normal(0, 3, (rows, V)).astype(np.float32)
    z[::6, :70] = -np.inf  # masked, listed tokens among them
    z[::6, 0] = 1.0
    if dtype == "bf16":
        z = bf16(z)
    ids, values = edge_lists(rng, rows, V, K)
    ids[::6][ids[::6] < 70] = 0
    g = rng.normal(0, 1, rows).astype(np.float32)
    g[min(4, rows - 1)] = 0.0
    loss, grad = grads_of(z, ids, values, 1.5, g, dtype, how, pad, lead, grad_lead)
    for r in range(rows):
        want_loss, want, loss_bound, bound = distill_plain(z[r], ids[r], values[r], 1.5, True)
        assert abs(loss[r] - want_loss) <= loss_bound + U * abs(want_loss), r
        want = want * float(g[r])
        bound = (bound + 4 * U * np.abs(want)) * abs(float(g[r])) + 1e-37
        over = excess(grad[r], want, bound + 4 * U * np.abs(want), dtype)
        assert np.all(over <= 1), (r, int(np.argmax(over)), over.max())


# f32: 6 rows are two vectors a thread, 14 four; bf16: 6 and 105.
@pytest.mark.parametrize("dtype,rows", [("f32", 6), ("f32", 14), ("bf16", 6), ("bf16", 105)])
@pytest.mark.parametrize("how", HOWS)
@pytest.mark.parametrize("V,pad,lead,grad_lead", [(81920, 0, 0, 0), (80003, 0, 0, 0),
                                                  (80003, 5, 1, 17), (79872, 1, 3, 63)])
def test_gradients_by_chunks(dtype, rows, how, V, pad, lead, grad_lead):
    check(rows, V, dtype, 20, how, pad, lead, grad_lead)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("how", ["backward in place", "step"])
@pytest.mark.parametrize("K", [1, 64, 65, 256])
def test_lists_of_any_length_by_chunks(dtype, how, K):
    check(14, 80003, dtype, K, how, 2, 7, 9)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_short_rows_go_backward_by_chunks_too(dtype):
    """The backward pass alone takes rows of any length by chunks: of less than a
    chunk, and of a line more or less than one."""
    for V in (1, 7, 300, 2047, 4095, 4096 - 31, 8192 + 33):
        K = min(V, 5)
        for how in ("backward", "backward in place"):
            rng = np.random.default_rng(V)
            z = rng.normal(0, 3, (9, V)).astype(np.float32)
            if dtype == "bf16":
                z = bf16(z)
            ids = np.stack([rng.choice(V, K, replace=False) for _ in range(9)]).astype(np.uint32)
            values, g = rng.normal(0, 1, (9, K)).astype(np.float32), np.ones(9, np.float32)
            _, grad = grads_of(z, ids, values, 1.0, g, dtype, how, V % 5, V % 7, V % 61)
            for r in range(9):
                _, want, _, bound = distill_plain(z[r], ids[r], values[r], 1.0, True)
                bound = bound + 4 * U * np.abs(want) + 1e-37
                assert np.all(excess(grad[r], want, bound, dtype) <= 1), (V, how, r)


@pytest.mark.parametrize("rows", [6, 200])
def test_rows_without_a_list_have_no_gradient_whatever_comes_in(rows):
    """NaN and infinite loss gradients of rows with empty lists: 6 rows by chunks,
    200 by whole rows."""
    V = 80003
    rng = np.random.default_rng(41)
    z = bf16(rng.normal(0, 2, (rows, V)).astype(np.float32))
    ids = np.tile(np.uint32([5, 6]), (rows, 1))
    ids[:3] = NO
    g = np.ones(rows, np.float32)
    g[0], g[1], g[4] = np.nan, np.inf, np.nan
    for how in HOWS:
        _, grad = grads_of(z, ids, np.zeros((rows, 2), np.float32), 1.0, g, "bf16", how, 0, 0, 0)
        assert not grad[:3].any() and np.isnan(grad[4]).all()
