"""Log-probabilities (jf_logprobs) against a plain implementation in 64 bits:
values within the bound of their roundings, ids and ranks exact with ties to
the lowest id, over vocabularies around the group's and the chunk's sizes,
both types, strides and alignments."""
import numpy as np
import pytest

import jf_sampler as J
from scoring_cases import bf16, device_rows, host, order, rank_of, score_plain

pytestmark = pytest.mark.gpu

NO = 0xFFFFFFFF


def run(x, dtype="f32", tokens=None, temperatures=None, top=0, ranks=True, pad=0, lead=0,
        scorer=None):
    """Host results of one call: lse, logprobs, ranks, top_ids, top_logprobs."""
    import torch
    rows, V = x.shape
    t, _ = device_rows(x, dtype, pad, lead)
    out = dict(lse=torch.full((rows,), 7.0, device="cuda"))
    kw = {}
    if tokens is not None:
        kw["tokens"] = torch.from_numpy(np.ascontiguousarray(tokens, np.uint32).view(np.int32)).cuda()
        out["logprobs"] = torch.full(tokens.shape, 7.0, device="cuda")
        if ranks:
            out["ranks"] = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    if temperatures is not None:
        kw["temperatures"] = torch.tensor(temperatures, dtype=torch.float32, device="cuda")
    if top:
        out["top_ids"] = torch.full((rows, top), -7, dtype=torch.int32, device="cuda")
        out["top_logprobs"] = torch.full((rows, top), 7.0, device="cuda")
    s = scorer or J.Scorer(V, rows)
    s.logprobs(t, **out, **kw)
    torch.cuda.synchronize()
    got = {k: v.cpu().numpy() for k, v in out.items()}
    if scorer is None:
        s.close()
    return got


def near(got, want, bound, what):
    got, want, bound = np.broadcast_arrays(*(np.asarray(v, np.float64)
                                             for v in (got, want, bound)))
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite], err_msg=str(what))
    off = np.abs(got[finite] - want[finite])
    assert np.all(off <= bound[finite]), (what, off.max(), bound[finite].min())


def check(x, got, tokens=None, temperatures=None, top=0, ranks=True):
    rows, V = x.shape
    for r in range(rows):
        T = 1.0
        if temperatures is not None:
            t = float(np.float32(temperatures[r]))
            T = t if np.finfo(np.float32).tiny <= t < np.inf else 1.0
        _, lp, lse, lp_bound, lse_bound = score_plain(x[r], T)
        near(got["lse"][r], lse, lse_bound, ("lse", r))
        if tokens is not None:
            for i, token in enumerate(tokens[r].tolist()):
                known = token < V
                near(got["logprobs"][r, i], lp[token] if known else -np.inf,
                     lp_bound[token] if known else 0, ("logprob", r, i))
            if ranks:
                first = tokens[r, 0]
                assert got["ranks"][r] == (rank_of(x[r], first) if first < V else 0), r
        if top:
            best = order(x[r])[:top]
            n = len(best)
            np.testing.assert_array_equal(got["top_ids"][r].view(np.uint32)[:n], best)
            assert np.all(got["top_ids"][r].view(np.uint32)[n:] == NO)
            assert np.all(np.isneginf(got["top_logprobs"][r][n:]))
            near(got["top_logprobs"][r][:n], lp[best], lp_bound[best], ("top", r))


def both(x, dtype, **kw):
    if dtype == "bf16":
        x = bf16(x)
    place = {k: kw.pop(k) for k in ("pad", "lead") if k in kw}
    print(f"logprobs {x.shape} {dtype} {place} top={kw.get('top', 0)}", flush=True)
    got = run(x, dtype, **kw, **place)
    check(x, got, **kw)
    return got


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 8191, 8192, 8193, 16385, 20011])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top", [0, 1, 5, 33, 128])
def test_log_probabilities(V, dtype, top):
    rng = np.random.default_rng(V + top)
    rows = 5
    x = rng.normal(0, 5, (rows, V)).astype(np.float32)
    tokens = rng.integers(0, V, (rows, 3)).astype(np.uint32)
    tokens[0, 0], tokens[1, 0], tokens[2, 1], tokens[3, 0] = 0, V - 1, NO, V
    both(x, dtype, tokens=tokens, temperatures=[1.0, 0.0, 0.5, 3.0, np.inf], top=top,
         pad=V % 4, lead=V % 3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_output_alone(dtype):
    rng = np.random.default_rng(2)
    x = rng.normal(0, 3, (3, 9000)).astype(np.float32)
    tokens = rng.integers(0, 9000, (3, 1)).astype(np.uint32)
    both(x, dtype)
    both(x, dtype, tokens=tokens, ranks=False)
    both(x, dtype, top=128)
    both(x, dtype, tokens=tokens, ranks=False, top=7)


# Orders that crowd the best tokens into few groups, few threads or one value.
def _ordered(how, V, rng):
    i = np.arange(V)
    if how == "constant":
        return np.zeros(V)
    if how == "falling":
        return -0.01 * i
    if how == "rising":
        return 0.01 * i
    if how == "few values":
        return rng.integers(0, 3, V).astype(float)
    if how == "one value at the top":
        return np.where(rng.random(V) < 0.3, 5.0, rng.normal(0, 1, V))
    if how == "one lane":  # the best tokens 16,384 apart: one thread's groups
        return np.where(i % 16384 < 64, 9.0 - 1e-3 * (i % 97), rng.normal(0, 1, V))
    if how == "one column":  # one token a group, every group
        return np.where(i % 64 == 17, 3.0 + 1e-4 * i, -1.0)
    if how == "two levels":  # ties across the cut between whole groups
        return np.where(i // 64 % 2 == 1, 2.0, 1.0)
    raise ValueError(how)


@pytest.mark.parametrize("how", ["constant", "falling", "rising", "few values",
                                 "one value at the top", "one lane", "one column", "two levels"])
@pytest.mark.parametrize("top", [1, 2, 20, 64, 127, 128])
@pytest.mark.parametrize("V", [700, 40000])
def test_orders_that_crowd_the_best(how, top, V):
    rng = np.random.default_rng(top)
    x = np.stack([_ordered(how, V, rng), _ordered(how, V, rng)]).astype(np.float32)
    both(x, "f32", top=top)
    both(x, "bf16", top=top)


# Zeros of both signs are equal; subnormal logits keep their order.
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 20, 64, 128])
def test_zeros_and_subnormals(dtype, top):
    rng = np.random.default_rng(top)
    V = 9000
    x = np.stack([rng.normal(0, 1e-39, V), np.where(rng.random(V) < 0.5, 0.0, -0.0),
                  np.where(rng.random(V) < 0.99, -1e-39, -0.0),
                  np.where(rng.random(V) < 0.002, 1e-39, -3.0)]).astype(np.float32)
    tokens = rng.integers(0, V, (4, 1)).astype(np.uint32)
    both(x, dtype, tokens=tokens, top=top)


# Masks of the lowest value that leave fewer tokens than are listed, as many and more.
@pytest.mark.parametrize("V", [300, 30000, 151936])
@pytest.mark.parametrize("top", [20, 128])
def test_rows_masked_by_the_lowest_value(V, top):
    rng = np.random.default_rng(V)
    x = rng.normal(0, 3, (6, V)).astype(np.float32)
    for r, left in enumerate((0, 1, 5, top - 1, top, top + 1)):
        keep = rng.choice(V, left, replace=False)
        row = np.full(V, -3.3895314e38, np.float32)  # the lowest bf16
        row[keep] = x[r, keep]
        x[r] = row
    both(x, "f32", top=top)
    both(x, "bf16", top=top)


# Around the vocabularies at which a finishing thread takes 4, 8, 12 and 16 groups.
@pytest.mark.parametrize("V", [n * 16384 + d for n in (4, 8, 12, 16) for d in (0, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_groups_a_thread_takes(V, dtype):
    rng = np.random.default_rng(V)
    x = rng.normal(0, 3, (2, V)).astype(np.float32)
    x[0, V - 1], x[1, V - 70] = 40.0, 40.0
    for top in (3, 40, 128):
        both(x, dtype, top=top)


def test_the_largest_vocabulary():
    rng = np.random.default_rng(9)
    V = 524288
    x = np.stack([rng.normal(0, 2, V), _ordered("one lane", V, rng), np.zeros(V)]).astype(np.float32)
    tokens = np.uint32([[V - 1], [16384], [300000]])
    both(x, "bf16", tokens=tokens, top=128)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_rows(dtype):
    """-infinity and the type's lowest value as masks: whole rows, all but a
    few tokens, whole chunks."""
    rng = np.random.default_rng(4)
    V = 20000
    x = rng.normal(0, 3, (7, V)).astype(np.float32)
    lowest = np.float32(-3.3895314e38)
    x[0] = -np.inf
    x[1, :] = -np.inf
    x[1, [3, 19999, 8192]] = [1.0, 1.0, 2.0]
    x[2, 8192:16384] = -np.inf
    x[3] = lowest
    x[4, rng.random(V) < 0.99] = lowest
    x[5, :] = -np.inf
    x[5, 12345] = -80.0
    x[6, 1:] = lowest
    tokens = np.uint32([[5], [3], [9000], [7], [0], [12345], [0]])
    got = both(x, dtype, tokens=tokens, top=20)
    assert np.isneginf(got["lse"][0]) and got["ranks"][0] == 6
    assert np.all(got["top_ids"][0] == -1)


def test_rows_with_nan_and_infinity():
    """lse and log-probabilities become NaN; lists hold the other tokens."""
    rng = np.random.default_rng(6)
    V = 10000
    x = rng.normal(0, 3, (4, V)).astype(np.float32)
    x[0, 77] = np.nan
    x[1, [9, 9000]] = np.inf
    x[2] = np.nan
    x[3, ::2] = np.nan
    got = run(x, tokens=np.uint32([[5], [9000], [3], [2]]), top=6)
    assert np.all(np.isnan(got["lse"])) and np.all(np.isnan(got["logprobs"]))
    for r in range(4):
        best = order(x[r])[:6]
        np.testing.assert_array_equal(got["top_ids"][r].view(np.uint32)[:len(best)], best)
        assert np.all(got["top_ids"][r][len(best):] == -1)
        assert np.all(np.isnan(got["top_logprobs"][r][:len(best)]))
    assert got["ranks"][1] == 2 and got["ranks"][2] == 1 and got["ranks"][3] == 1
    assert got["ranks"][0] == rank_of(x[0], 5)


@pytest.mark.parametrize("rows", [1, 3, 300, 1100, 2500])
def test_many_rows_share_the_scratch(rows):
    """More rows than one launch with alternatives takes, and few enough that
    a row's blocks change in number; a smaller call follows a larger one."""
    rng = np.random.default_rng(rows)
    V = 8200
    x = bf16(rng.normal(0, 3, (rows, V)).astype(np.float32))
    tokens = rng.integers(0, V, (rows, 1)).astype(np.uint32)
    T = (0.5 + rng.random(rows)).astype(np.float32)
    s = J.Scorer(V, rows)
    for kw in (dict(top=3), dict(top=0)):
        check(x, run(x, "bf16", tokens=tokens, temperatures=T, scorer=s, **kw), tokens, T, **kw)
    half = (rows + 1) // 2
    check(x[:half], run(x[:half], "bf16", tokens=tokens[:half], scorer=s, top=128),
          tokens[:half], top=128)
    s.close()


def test_repeats_are_bit_identical_and_replay_under_a_graph():
    import torch
    rng = np.random.default_rng(12)
    V, rows = 30011, 6
    t, _ = device_rows(rng.normal(0, 3, (rows, V)).astype(np.float32), "f32", 1, 1)
    tokens = torch.from_numpy(rng.integers(0, V, (rows, 2)).astype(np.int32)).cuda()
    out = dict(lse=torch.zeros(rows, device="cuda"), logprobs=torch.zeros((rows, 2), device="cuda"),
               ranks=torch.zeros(rows, dtype=torch.int32, device="cuda"),
               top_ids=torch.zeros((rows, 20), dtype=torch.int32, device="cuda"),
               top_logprobs=torch.zeros((rows, 20), device="cuda"))
    s = J.Scorer(V, rows)
    a = s.logprobs_args(t, tokens=tokens, **out)

    def bits():
        torch.cuda.synchronize()
        return [v.cpu().numpy().view(np.int32).copy() for v in out.values()]
    s.launch_logprobs(a)
    want = bits()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.launch_logprobs(a)
    for turn in range(4):
        for v in out.values():
            v.zero_()
        if turn % 2:
            s.launch_logprobs(a)
            torch.cuda.synchronize()
        graph.replay()
        for w, g in zip(want, bits()):
            np.testing.assert_array_equal(g, w)
    del graph
    s.close()


def test_refusals():
    import torch
    V, rows = 100, 2
    t, _ = device_rows(np.zeros((rows, V), np.float32), "f32")
    s = J.Scorer(V, rows)
    lse = torch.zeros(rows, device="cuda")
    ids = torch.zeros((rows, 3), dtype=torch.int32, device="cuda")
    lps = torch.zeros((rows, 3), device="cuda")

    def refused(message, args=None, **change):
        a = s.logprobs_args(t, **(dict(lse=lse) if args is None else args))
        for k, v in change.items():
            setattr(a, k, v)
        with pytest.raises(J.JfError) as e:
            s.launch_logprobs(a)
        assert e.value.code == J.JF_ERR_INVALID_ARGUMENT and message in e.value.message, \
            e.value.message

    refused("batch width", rows=0)
    refused("batch width", rows=3)
    refused("dtype", dtype=2)
    refused("null logits", logits=None)
    refused("aligned", logits=t.data_ptr() + 3)
    refused("stride is below", logits_stride=V - 1)
    refused("nothing to score", args={})
    refused("more than 128", top=129)
    refused("alternatives need", top=3)
    refused("alternatives need", args=dict(top_ids=ids))
    refused("scored tokens need", args=dict(tokens=ids))
    refused("stride is below the token count", args=dict(tokens=ids, logprobs=lps), token_stride=2)
    refused("ranks need", out_ranks=ids.data_ptr())
    for bad in (dict(lse=lse[:1]), dict(lse=lse.double()), dict(tokens=ids.long(), logprobs=lps),
                dict(top_ids=ids[:, ::2], top_logprobs=lps), dict(temperatures=lse[:1], lse=lse)):
        with pytest.raises(ValueError):
            s.logprobs_args(t, **bad)
    assert not lse.any() and not lps.any()
    for vocabulary, max_rows, message in ((0, 1, "geometry"), (524289, 1, "524288"),
                                          (10, 0, "row count"), (10, (1 << 22) + 1, "row count")):
        with pytest.raises(J.JfError) as e:
            J.Scorer(vocabulary, max_rows)
        assert message in e.value.message
    s.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_signalling_nan_hides_no_other_token(dtype):
    """A NaN that signals, in the groups of the best tokens: the lists hold the
    other tokens all the same."""
    import torch
    rng = np.random.default_rng(40)
    V = 12000
    x = bf16(rng.normal(0, 3, (2, V)).astype(np.float32))
    best = order(x[0])[:30]
    t, _ = device_rows(x, dtype)
    at = torch.from_numpy((best[:3] // 64 * 64 + (best[:3] % 64 + 1) % 64).copy()).cuda()
    if dtype == "f32":
        t.view(torch.int32)[0, at] = 0x7F810000
    else:
        t.view(torch.int16)[0, at] = 0x7F81
    ids = torch.zeros((2, 20), dtype=torch.int32, device="cuda")
    lps = torch.zeros((2, 20), device="cuda")
    s = J.Scorer(V, 2)
    s.logprobs(t, top_ids=ids, top_logprobs=lps)
    seen = x.copy()
    seen[0, at.cpu().numpy()] = np.nan
    for r in range(2):
        np.testing.assert_array_equal(ids[r].cpu().numpy(), order(seen[r])[:20])
    assert torch.isnan(lps[0]).all() and not torch.isnan(lps[1]).any()
    s.close()
