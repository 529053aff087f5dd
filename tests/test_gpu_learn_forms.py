"""Forms of the losses of drawn tokens that few sizes reach: more long f32 rows than the
pairs' launch works out, also captured, and steps of 1024 threads a row of bf16 with an
entropy bonus."""
import numpy as np
import pytest

import jf_sampler as J
import test_gpu_clipped as clipped
import test_gpu_preference as preference
from learning_cases import ABSENT
from scoring_cases import device_rows, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,V", [("f32", 110001), ("bf16", 140001)])
def test_preference_losses_of_many_long_rows(dtype, V):
    """Forward and backward passes and a step, as calls and captured, replayed with other
    rows, tokens and lengths in the same buffers and the program's own calls between."""
    import torch
    rows, rng = 1100, np.random.default_rng(21)
    active = [0, 1, 7, 300, 301, 640, 641, 1030, 1090, 1099]
    spans = [[0, 8, 301, 641, 1097], [0, 1, 1, 301, 1100], [2, 300, 640, 1050, 1095]]
    cases = [preference.sparse_rows(rng, V, rows, active, dtype) for _ in spans]
    t, d_tokens, d_ref, at = (v.clone() for v in cases[0][:4])
    d_offsets = preference._ids(spans[0])
    s, gl = J.Scorer(V, rows), torch.tensor([0.5, -2.0], device="cuda")
    out = [dict(loss=torch.zeros(2, device="cuda"), scores=torch.zeros(4, device="cuda"),
                logprobs=torch.zeros(rows, device="cuda"),
                saved=torch.zeros((rows, 4), device="cuda"), grad=torch.zeros_like(t))
           for _ in range(2)]
    a, b = (s.preference_args(t, d_tokens, d_offsets, reference_logprobs=d_ref, grad_loss=gl, **o)
            for o in out)

    def calls():
        s.launch_preference(a)
        s.launch_preference_backward(a)
        s.launch_preference_step(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        calls()
    for n, (case, span) in enumerate(list(zip(cases, spans)) + [(cases[0], spans[0])]):
        for how in ("calls", "graph"):
            print(f"many long rows {dtype} {V} inputs {n} {how}", flush=True)
            for to, v in zip((t, d_tokens, d_ref), case):
                to.copy_(v)
            d_offsets.copy_(preference._ids(span))
            for o in out:
                for v in o.values():
                    v.fill_(7.0)
            (calls if how == "calls" else graph.replay)()
            torch.cuda.synchronize()
            x, tokens, ref = case[4:]
            # Rows without a token belong to sequences all the same.
            small = np.uint32([np.searchsorted(active, o) for o in span])
            args = (x, tokens, small, ref, 1.0, 0.1, 0.0, 0.0, "sigmoid", False, [0.5, -2.0], dtype)
            rest = torch.ones(rows, dtype=torch.bool, device="cuda")
            rest[at] = False
            for o in out:
                preference.check(*args, dict(loss=host(o["loss"]), scores=host(o["scores"]),
                                             logprobs=host(o["logprobs"][at]),
                                             grad=host(o["grad"][at])))
                assert not o["grad"][rest].any() and not o["logprobs"][rest].any()
    s.close()


@pytest.mark.parametrize("rows,place", [(6, "loss gradients"), (6, "tokens"), (180, "none"),
                                        (180, "logits")])
@pytest.mark.parametrize("entropy", [0.1, -0.2])
def test_bf16_steps_of_1024_threads_with_an_entropy_bonus(rows, place, entropy):
    """Few rows whose losses take the place of an input, and many."""
    import torch
    V, rng = 170001, np.random.default_rng(rows)
    x, tokens, A, old, ref = clipped.batch(rng, V, rows, 0.9, 0.2, 0.2, "bf16")
    tokens[4] = ABSENT[0]
    g = rng.normal(0, 1, rows).astype(np.float32)
    t, _ = device_rows(x, "bf16", pad=1, lead=3)
    gl, d_tokens = clipped._f32(g), clipped._ids(tokens)
    loss = {"loss gradients": gl, "tokens": d_tokens.view(torch.float32)}.get(
        place, torch.full((rows,), 7.0, device="cuda"))
    grad = t if place == "logits" else torch.full((rows, V), 7.0, device="cuda",
                                                  dtype=torch.bfloat16)
    out = dict(loss=loss, logprobs=torch.zeros(rows, device="cuda"),
               kl=torch.zeros(rows, device="cuda"), entropy=torch.zeros(rows, device="cuda"))
    s = J.Scorer(V, rows)
    s.launch_clipped_step(s.clipped_args(
        t, d_tokens, clipped._f32(A), old_logprobs=clipped._f32(old),
        reference_logprobs=clipped._f32(ref), kl_weight=0.1, entropy_weight=entropy,
        temperature=0.9, saved=torch.empty((rows, 4), device="cuda"), grad_loss=gl, grad=grad,
        **out))
    picked = np.r_[0:6, rows - 6:rows]
    full = (x, tokens, A, old, ref, 0.9, 0.2, 0.2, 0.1, entropy, g, "bf16")
    got = dict({k: host(v) for k, v in out.items()}, grad=host(grad))
    clipped.check(*(v[picked] if isinstance(v, np.ndarray) else v for v in full),
                  {k: v[picked] for k, v in got.items()})
    assert all(not got["grad"][r].any() for r in np.flatnonzero(tokens >= V))
    s.close()
