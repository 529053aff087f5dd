"""Gradients that are documented to be 0 whatever a row's logits, over rows that hold
NaN and +infinity: of losses whose gradient is 0, and of losses without a slope; in
every form that a backward pass and a step have."""
import numpy as np
import pytest

import test_gpu_clipped as clipped
import test_gpu_preference as preference
from scoring_cases import bf16

pytestmark = pytest.mark.gpu

# A row of each, by turns.
PLAIN, NAN_MASKED, INF_MASKED, NAN_FLAT, INF_FLAT, NAN_LEARNED = range(6)


def rows_of(rng, rows, V, dtype):
    x = rng.normal(0, 2, V).astype(np.float32) + np.zeros((rows, 1), np.float32)
    x = bf16(x) if dtype == "bf16" else x
    kind = np.arange(rows) % 6
    x[kind == NAN_MASKED, V // 2] = np.nan
    x[kind == INF_MASKED, V - 1] = np.inf
    x[kind == NAN_FLAT] = np.nan
    x[kind == INF_FLAT, 0] = np.inf
    x[kind == NAN_LEARNED, 3] = np.nan
    return x, kind


# Steps whose blocks share a row; a block a row of 512 threads; few long rows by chunks,
# each block with its row's loss; more of them, the losses before; 1024 threads a row, f32
# and both types.
SIZES = [(6, 700), (66, 700), (6, 80001), (42, 80001), (102, 90001), (180, 170001)]


@pytest.mark.parametrize("rows,V", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mode", ["separate", "step", "in place"])
def test_losses_of_rows(rows, V, dtype, mode):
    x, kind = rows_of(np.random.default_rng(rows), rows, V, dtype)
    tokens = np.full(rows, 5, np.uint32)
    A = np.where((kind == NAN_FLAT) | (kind == INF_FLAT), 0, 1).astype(np.float32)
    g = np.ones(rows, np.float32)
    g[(kind == NAN_MASKED) | (kind == INF_MASKED)] = 0
    g[kind == INF_FLAT] = np.nan  # a loss without a slope has no gradient whatever comes in
    # No entropy, one that is only asked for, one that is weighted.
    for entropy, asked in ((0.0, False), (0.0, True), (0.1, True)):
        print(f"zero gradients {rows} x {V} {dtype} {mode} {entropy} {asked}", flush=True)
        got = clipped.run(x, tokens, A, None, None, 1.0, 0.2, 0.2, 0.0, entropy, g, dtype, mode,
                          all_outputs=asked)["grad"]
        plain = got[kind == PLAIN]
        assert np.isfinite(plain).all() and plain.any(axis=1).all()
        assert not got[(kind == NAN_MASKED) | (kind == INF_MASKED)].any()
        flat = got[(kind == NAN_FLAT) | (kind == INF_FLAT)]
        assert np.isnan(flat).all() if entropy else not flat.any()
        assert np.isnan(got[kind == NAN_LEARNED]).all()


@pytest.mark.parametrize("rows,V", [(8, 700), (160, 700), (8, 80001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mode", ["separate", "step", "in place"])
def test_losses_of_pairs(rows, V, dtype, mode):
    x, _ = rows_of(np.random.default_rng(rows), rows, V, dtype)
    half, quarter = rows // 2, rows // 4
    x[half:] = x[0]  # a pair of bad rows and one without
    offsets = np.uint32([0, quarter, half, half + quarter, rows])
    tokens = np.full(rows, 5, np.uint32)
    for g in ([0.0, 1.0], [0.0, 0.0], [1.0, 0.0]):
        got = preference.run(x, tokens, offsets, None, 1.0, 0.1, 0.0, 0.0, "sigmoid", True, g,
                             dtype, mode)
        assert np.isnan(got["loss"][0]) and np.isfinite(got["loss"][1])
        assert np.isnan(got["grad"][:half]).all() if g[0] else not got["grad"][:half].any()
        rest = got["grad"][half:]
        assert np.isfinite(rest).all() and rest.any() == (g[1] != 0)
