"""Best alternatives of batches large enough for four vectors a thread (more than
2^20 f32 or 2^23 bf16 tokens a launch): ids exact against 64 bits, values within
their bounds, in rows of every order that the search for them meets, at any
alignment, over vocabularies around the chunk's and the group's sizes."""
import numpy as np
import pytest

from scoring_cases import bf16, rank_of, score_plain
from test_gpu_logprobs import NO, _ordered, near, run

pytestmark = pytest.mark.gpu

KINDS = ["normal", "constant", "falling", "rising", "few values", "one value at the top",
         "one lane", "one column", "two levels", "masked", "masked by the lowest value",
         "fewer than asked for", "nothing", "NaN", "infinity"]
FAR = float(np.finfo(np.float32).max)


def row_of_kind(kind, V, rng):
    if kind in ("normal", "NaN", "infinity"):
        x = rng.normal(0, 3, V)
        if kind != "normal":
            at = rng.choice(V, 5, replace=False)
            x[at[:3]] = np.nan if kind == "NaN" else np.inf
            x[at[3:]] = -np.inf
        return x
    if kind.startswith("masked"):
        away = -np.inf if kind == "masked" else -3.3895314e38
        return np.where(rng.random(V) < 0.01, rng.normal(0, 3, V), away)
    if kind in ("fewer than asked for", "nothing"):
        x = np.full(V, -np.inf)
        if kind != "nothing":
            x[rng.choice(V, 3, replace=False)] = -3e38, 1.0, 1.0
        return x
    return _ordered(kind, V, rng)


def best_of(x, k):
    """The k first ids by (logit down, id up), NaN and -infinity left out."""
    ids = np.flatnonzero(x > -np.inf)
    if len(ids) > k:
        v = x[ids]
        ids = ids[v >= np.partition(v, len(v) - k)[len(v) - k]]
    return ids[np.lexsort((ids, -x[ids].astype(np.float64)))][:k]


def batch(rows, V, dtype, rng):
    """Every kind in turn from a random one on, the last tokens of some rows their
    best."""
    first = int(rng.integers(len(KINDS)))
    x = np.stack([row_of_kind(KINDS[(first + r) % len(KINDS)], V, rng) for r in range(rows)])
    x = x.astype(np.float32)
    x[::7, V - 1] = 40.0
    x[3::7, 0] = 40.0
    return bf16(x) if dtype == "bf16" else x


def check(rows, V, dtype, top, rank, pad=0, lead=0, seed=0):
    print(f"alternatives {rows} x {V} {dtype} top={top} rank={rank} pad={pad} lead={lead}",
          flush=True)
    rng = np.random.default_rng(seed + V + top)
    x = batch(rows, V, dtype, rng)
    T = rng.choice([0.5, 1.0, 2.0, 0.0], rows)
    tokens = rng.integers(0, V, (rows, 2)).astype(np.uint32) if rank else None
    got = run(x, dtype, tokens=tokens, temperatures=T, top=top, pad=pad, lead=lead)
    for r in range(rows):
        _, lp, lse, lp_bound, lse_bound = score_plain(x[r], T[r] or 1.0)
        # Past the outputs' range: a token of a lowest value at a temperature below 1.
        lp = np.where(np.abs(lp) > FAR, np.copysign(np.inf, lp), lp)
        near(got["lse"][r], lse, lse_bound, ("lse", r))
        best = best_of(x[r], top)
        n, ids = len(best), got["top_ids"][r].view(np.uint32)
        np.testing.assert_array_equal(ids[:n], best, err_msg=str(r))
        assert np.all(ids[n:] == NO) and np.all(np.isneginf(got["top_logprobs"][r][n:]))
        near(got["top_logprobs"][r][:n], lp[best], lp_bound[best], ("top", r))
        if rank:
            near(got["logprobs"][r], lp[tokens[r]], lp_bound[tokens[r]], ("logprobs", r))
            assert got["ranks"][r] == rank_of(x[r], tokens[r, 0]), r


# Up to 4,096 groups a row, and more; V within a chunk of 4,096 or 8,192 tokens, a
# group and a lane of its end.
@pytest.mark.parametrize("top", [1, 5, 20, 32, 33, 64, 127, 128])
@pytest.mark.parametrize("V,rows", [(100003, 17), (98304, 16), (98305, 16), (70001, 31),
                                    (262144, 16), (262145, 16), (300001, 16)])
def test_f32_batches(top, V, rows):
    assert rows * V > 1 << 20
    check(rows, V, "f32", top, rank=top % 2 == 0, pad=V % 4, lead=V % 3)


@pytest.mark.parametrize("top", [5, 20, 64, 128])
@pytest.mark.parametrize("V,rows", [(100003, 84), (98304, 86), (262208, 33), (300001, 28),
                                    (524288, 17)])
def test_bf16_batches(top, V, rows):
    assert rows * V > 1 << 23
    check(rows, V, "bf16", top, rank=top % 20 == 0, pad=V % 4, lead=V % 3)


@pytest.mark.parametrize("dtype,V", [("f32", 8191), ("bf16", 16449)])
@pytest.mark.parametrize("top", [5, 128])
def test_batches_of_two_launches(dtype, V, top):
    """More rows than a launch with alternatives takes: the first launch's threads
    take four vectors, the last one's two."""
    check(540, V, dtype, top, rank=True, pad=1, lead=5)
