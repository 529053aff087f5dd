"""A clipped loss whose outputs take the place of its tokens: each wave of a row's block
has its token before any of the row's numbers is written, also in rows without one."""
import numpy as np
import pytest

import jf_sampler as J
from learning_cases import ABSENT
from scoring_cases import device_rows, host
from test_gpu_clipped import _f32, _ids, batch, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("output", ["loss", "logprobs", "kl", "entropy"])
@pytest.mark.parametrize("rows,V", [(5, 700), (600, 2001), (30, 90001), (110, 90001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("step", [False, True])
def test_outputs_in_place_of_the_tokens(output, rows, V, dtype, step):
    import torch
    print(f"outputs over tokens: {output} {rows} x {V} {dtype} step {step}", flush=True)
    rng = np.random.default_rng(rows)
    x, tokens, A, old, ref = batch(rng, V, rows, 1.0, 0.2, 0.2, dtype)
    none = rng.random(rows) < 0.5
    tokens[none] = rng.choice(ABSENT, int(none.sum()))
    g = rng.normal(0, 1, rows).astype(np.float32)
    t, _ = device_rows(x, dtype)
    d_tokens = _ids(tokens)
    out = {k: torch.full((rows,), 7.0, device="cuda") for k in ("loss", "logprobs", "kl", "entropy")}
    out[output] = d_tokens.view(torch.float32)
    saved, grad = torch.empty((rows, 4), device="cuda"), torch.full_like(t, 7.0)
    s = J.Scorer(V, rows)
    a = s.clipped_args(t, d_tokens, _f32(A), old_logprobs=_f32(old), reference_logprobs=_f32(ref),
                       kl_weight=0.1, entropy_weight=0.1, saved=saved, **out,
                       **(dict(grad_loss=_f32(g), grad=grad) if step else {}))
    if step:
        s.launch_clipped_step(a)
    else:
        s.launch_clipped(a)
        s.launch_clipped_backward(s.clipped_args(t, _ids(tokens), None, entropy_weight=0.1,
                                                 saved=saved, grad_loss=_f32(g), grad=grad))
    got = dict({k: host(v) for k, v in out.items()}, grad=host(grad))
    without = tokens >= V
    for name in got:
        assert not got[name][without].any(), name
    picked = np.r_[:5, rows - 5:rows]
    full = (x, tokens, A, old, ref, 1.0, 0.2, 0.2, 0.1, 0.1, g)
    check(*(v[picked] if isinstance(v, np.ndarray) else v for v in full), dtype,
          {k: v[picked] for k, v in got.items()})
    s.close()
