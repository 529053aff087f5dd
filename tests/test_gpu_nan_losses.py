"""A row whose log-probability is NaN has a NaN loss, also where its own stand in for the
old policy's and the ratio is 1; others keep theirs."""
import numpy as np
import pytest

from learning_cases import ABSENT
from test_gpu_clipped import check, run

pytestmark = pytest.mark.gpu


# Rows taken whole by blocks that share one and by a block each, by chunks with their losses
# in the gradient's blocks and before them, and 1024 threads a row.
@pytest.mark.parametrize("rows,V", [(8, 700), (80, 700), (8, 80001), (48, 80001), (104, 90001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mode", ["separate", "step", "in place"])
@pytest.mark.parametrize("entropy", [0.0, 0.1])
def test_nan_is_not_hidden(rows, V, dtype, mode, entropy):
    print(f"NaN losses {rows} x {V} {dtype} {mode} {entropy}", flush=True)
    x = np.random.default_rng(V).normal(0, 2, V).astype(np.float32) + \
        np.zeros((rows, 1), np.float32)
    x.view(np.uint32)[...] &= 0xffff0000  # values of both types
    kind, tokens, A = np.arange(rows) % 8, np.full(rows, 5, np.uint32), np.ones(rows, np.float32)
    bad = (kind == 1) | (kind == 2) | (kind == 3)
    x[kind == 1, V - 1] = np.nan
    x[kind == 2, 0] = np.inf
    x[kind == 3], A[kind == 3] = np.nan, 0.0
    x[kind == 4], tokens[kind == 4] = np.nan, ABSENT[0]
    x[kind == 5, 5] = -np.inf  # a token without probability: lp is -infinity, r is 1
    args = (tokens, A, None, None, 1.0, 0.2, 0.2, 0.0, entropy, np.ones(rows), dtype)
    got = run(x, *args, mode=mode)
    assert np.isnan(got["loss"][bad]).all() and np.isnan(got["logprobs"][bad]).all()
    assert not got["loss"][kind == 4].any()
    assert np.isneginf(got["logprobs"][kind == 5]).all() and np.isfinite(got["loss"][~bad]).all()
    if not entropy:
        assert (got["loss"][kind == 5] == -1).all()
    plain = np.flatnonzero(kind == 0)[:2]
    check(x[plain], tokens[plain], A[plain], *args[2:-2], np.ones(2), dtype,
          {k: v[plain] for k, v in got.items()})
