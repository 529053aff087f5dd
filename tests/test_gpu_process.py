"""Processed logits (jf_process_logits) against a plain implementation in 64
bits: unedited tokens bit for bit, edited ones within the bound of their
roundings, over vocabularies around the chunk's and the mask word's sizes,
both types, strides and alignments; written out and in place."""
import numpy as np
import pytest

import jf_sampler as J
from scoring_cases import bf16, device_rows, excess, host, process_bound, process_plain

pytestmark = pytest.mark.gpu

NO = 0xFFFFFFFF


def _words(V, history, generated, mark):
    w = np.zeros(V, np.uint32)
    J.rebuild_penalty_words(w, history, generated, None, mark)
    return w


def _masks(rng, rows, V, share=0.3):
    admitted = rng.random((rows, V)) < share
    words = np.zeros((rows, (V + 31) // 32 * 32), bool)
    words[:, :V] = admitted
    bits = (words.reshape(rows, -1, 32) << np.arange(32, dtype=np.uint64)).sum(2)
    return admitted, bits.astype(np.uint32)


POLICIES = [dict(), dict(repetition=1.3), dict(presence=0.7, frequency=0.2),
            dict(repetition=0.8, presence=-0.5, frequency=1.5), dict(constrained=True),
            dict(repetition=1.2, frequency=0.1, constrained=True), dict(exclude_stop=True),
            dict(presence=2.0, constrained=True, exclude_stop=True)]


def _run(V, rows, dtype, out_dtype, pad=0, lead=0, out_pad=0, in_place=False, seed=0, x=None,
         biases=7, extras=True, history=900, kinds=POLICIES):
    """Every row its own policy; returns nothing, checks every element."""
    import torch
    print(f"process V={V} rows={rows} {dtype}->{out_dtype} pad={pad} lead={lead} "
          f"in_place={in_place}", flush=True)
    rng = np.random.default_rng(seed + V)
    if x is None:
        x = rng.normal(0, 4, (rows, V)).astype(np.float32)
    if dtype == "bf16":
        x = bf16(x)
    policies = [J.policy(**kinds[r % len(kinds)]) for r in range(rows)]
    stops = (V // 2, V - 1)
    n = max(2, min(2 * V, history))
    table = J.PenaltyTable(V, rows, n + 8)
    words, bias, extra = [], [], np.zeros((rows, 5), np.uint32)
    bias_table = J.BiasTable(V, rows, max(1, biases))
    for r in range(rows):
        h = rng.integers(0, V, n).astype(np.uint32)
        table.rebuild(r, h, n // 2, None, True)
        words.append(_words(V, h, n // 2, True))
        b = rng.choice(V, min(V, biases), replace=False)
        values = rng.uniform(-9, 9, len(b)).astype(np.float32)
        values[::4] = -np.inf
        bias.append(dict(zip(b.tolist(), values.tolist())))
        bias_table.set(r, b, values)
        # A token of the history, one twice, one that may be neither, one
        # past the vocabulary.
        extra[r] = [h[0], V // 3, V // 3, rng.integers(0, V), NO]
    admitted, masks = _masks(rng, rows, V)
    t, buf = device_rows(x, dtype, pad, lead)
    if in_place:
        out, out_buf = t, buf
    else:
        out, out_buf = device_rows(np.zeros_like(x), out_dtype, out_pad, lead)
    around = out_buf.clone()
    kw = {}
    if extras:
        ex = torch.from_numpy(extra.view(np.int32)).cuda()
        kw = dict(extra_tokens=ex, extra_counts=[5 if r % 3 else 0 for r in range(rows)],
                  extra_stride=5)
    s = J.Scorer(V, rows)
    s.process(t, policies, out, masks=torch.from_numpy(masks.view(np.int32)).cuda(),
              stop_tokens=stops, penalties=table, penalty_rows=list(range(rows)),
              biases=bias_table, bias_rows=[None if r % 4 == 3 else r for r in range(rows)], **kw)
    torch.cuda.synchronize()
    got = host(out)
    for r in range(rows):
        p = policies[r]
        penalized = p.repetition != 1 or p.presence != 0 or p.frequency != 0
        want, edited, size = process_plain(
            x[r], p, words[r] if penalized else None,
            extra[r] if extras and r % 3 else (), bias[r] if r % 4 != 3 else None,
            admitted[r] if p.flags & J.JF_POLICY_CONSTRAINED else None,
            stops if p.flags & J.JF_POLICY_EXCLUDE_STOP else ())
        plain = x[r] if out_dtype == "f32" else bf16(x[r])
        np.testing.assert_array_equal(got[r][~edited], plain[~edited])
        off = np.isinf(want) | np.isnan(want)
        np.testing.assert_array_equal(got[r][edited & off], want[edited & off])
        on = edited & ~off
        over = excess(got[r][on], want[on], process_bound(size[on]), out_dtype)
        assert np.all(over <= 1), (V, r, over.max())
    # Nothing around the rows is written.
    inside = torch.zeros_like(out_buf, dtype=torch.bool)
    inside[lead:lead + rows * out.stride(0)].view(rows, -1)[:, :V] = True
    assert torch.equal(out_buf[~inside], around[~inside])
    table.close()
    bias_table.close()
    s.close()


@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 8191, 8192, 8193, 20011])
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"),
                                       ("f32", "bf16")])
def test_processed_logits(V, dtype, out):
    _run(V, 9, dtype, out, pad=V % 3, lead=V % 5, out_pad=(V + 1) % 4)


@pytest.mark.parametrize("V", [1, 1000, 8192, 20011])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place(V, dtype):
    _run(V, 9, dtype, dtype, pad=3, lead=1, in_place=True)


# Outputs that go past the caches, from rows that start anywhere in a line.
@pytest.mark.parametrize("V,rows,dtype,out,in_place", [
    (50021, 130, "f32", "f32", False), (50021, 130, "bf16", "f32", False),
    (50021, 260, "bf16", "bf16", False), (50021, 260, "f32", "bf16", False),
    (50021, 130, "f32", "f32", True), (50021, 260, "bf16", "bf16", True),
    (8191, 800, "bf16", "f32", False), (65536, 200, "bf16", "bf16", False)])
def test_large_outputs_at_any_alignment(V, rows, dtype, out, in_place):
    _run(V, rows, dtype, out, pad=3, lead=V % 7, out_pad=V % 4, in_place=in_place)


@pytest.mark.parametrize("dtype,out,in_place", [
    ("f32", "f32", False), ("bf16", "f32", False), ("bf16", "bf16", False), ("bf16", "bf16", True)])
def test_large_masked_outputs_at_any_alignment(dtype, out, in_place):
    _run(50021, 340, dtype, out, pad=3, lead=5, out_pad=1, in_place=in_place,
         kinds=[k for k in POLICIES if k.get("constrained") or k.get("exclude_stop")])


@pytest.mark.parametrize("V,rows", [(2, 3300000), (3, 2200000), (7, 1000000), (40, 160000)])
def test_many_short_rows(V, rows):
    import torch
    buf = torch.full((rows * V + 64,), 5.0, device="cuda")
    out = buf[33:33 + rows * V].view(rows, V)
    t = torch.randn((rows, V), device="cuda")
    s = J.Scorer(V, rows)
    s.process(t, [J.policy(exclude_stop=True)] * rows, out, stop_tokens=(1, NO))
    want = t.clone()
    want[:, 1] = -float("inf")
    assert torch.equal(out, want)
    assert bool((buf[:33] == 5).all()) and bool((buf[33 + rows * V:] == 5).all())
    s.close()


@pytest.mark.parametrize("biases,history", [(700, 900), (3001, 900), (10, 12000), (2500, 12000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_long_lists_fill_a_chunk(biases, history, in_place):
    """More entries and biases than a block has threads, and than its LDS
    stages, in one chunk."""
    _run(9001 if history > 9000 else 3001, 8, "f32", "f32", biases=biases, history=history,
         in_place=in_place)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_special_values(dtype):
    """NaN, infinities and the lowest value, edited, masked and left alone."""
    rng = np.random.default_rng(3)
    x = rng.normal(0, 4, (8, 1000)).astype(np.float32)
    special = np.float32([np.nan, np.inf, -np.inf, -3.3895314e38, 0.0, -0.0, 1e-40])
    for r in range(8):
        at = rng.choice(1000, 400, replace=False)
        x[r, at] = special[rng.integers(0, len(special), 400)]
    _run(1000, 8, dtype, dtype, x=x)
    _run(1000, 8, dtype, dtype, x=x, in_place=True)


def test_masks_that_leave_nothing_and_rows_by_index():
    """Rows whose mask admits no token are -infinity throughout; mask_rows and
    extra_offsets address other rows' data."""
    import torch
    V, rows = 5000, 3
    rng = np.random.default_rng(1)
    x = rng.normal(0, 3, (rows, V)).astype(np.float32)
    admitted, masks = _masks(rng, 2, V)
    masks[1] = 0
    t, _ = device_rows(x, "f32")
    out = torch.zeros_like(t)
    table = J.PenaltyTable(V, 1, 8)
    table.rebuild(0, [5, 6], 1, None, False)
    ex = torch.tensor([0, 0, 0, 7, 6], dtype=torch.int32).cuda()
    s = J.Scorer(V, rows)
    s.process(t, [J.policy(constrained=True), J.policy(constrained=True),
                  J.policy(presence=1.0, frequency=0.5)], out,
              masks=torch.from_numpy(masks.view(np.int32)).cuda(), mask_rows=[1, 0, 0],
              penalties=table, penalty_rows=[0, 0, 0], extra_tokens=ex, extra_counts=[0, 0, 2],
              extra_offsets=[0, 0, 3])
    got = host(out)
    assert np.all(np.isneginf(got[0]))
    np.testing.assert_array_equal(np.isneginf(got[1]), ~admitted[0])
    want = x[2].copy()
    want[6] -= np.float32(1.0 + 0.5 * 2)  # once generated, once extra
    want[7] -= np.float32(1.5)
    np.testing.assert_array_equal(got[2], want)
    s.close()


def test_changed_tables_and_policies_reach_the_next_call():
    """A second call with other policies, biases and counts answers for them."""
    import torch
    V = 3000
    x = np.zeros((1, V), np.float32)
    t, _ = device_rows(x, "f32")
    out = torch.zeros_like(t)
    table, bias = J.PenaltyTable(V, 1, 8), J.BiasTable(V, 2, 4)
    table.rebuild(0, [1, 2], 1, None, False)
    bias.set(0, [9, 4], [2.0, -3.0])
    s = J.Scorer(V, 4)
    kw = dict(penalties=table, penalty_rows=[0], biases=bias)
    s.process(t, [J.policy(presence=1.0)], out, bias_rows=[0], **kw)
    first = host(out)[0]
    table.count(0, [2, 3])
    bias.set(0, [], [])
    bias.set(1, [7], [5.0])
    s.process(t, [J.policy(frequency=0.25)], out, bias_rows=[1], **kw)
    second = host(out)[0]
    s.process(t, [J.policy()], out, bias_rows=[0], **kw)
    third = host(out)[0]
    want = np.zeros((3, V))
    want[0, [2, 9, 4]] = [-1.0, 2.0, -3.0]
    want[1, [2, 3, 7]] = [-0.5, -0.25, 5.0]
    np.testing.assert_array_equal(np.stack([first, second, third]), want)
    s.close()


def test_a_sampler_draws_the_same_from_processed_logits():
    """The selection over processed logits with a neutral policy picks the
    tokens that the selection with the penalties and masks picks."""
    import torch
    V, rows = 30000, 12
    rng = np.random.default_rng(8)
    x = rng.normal(0, 3, (rows, V)).astype(np.float32)
    admitted, masks = _masks(rng, rows, V, 0.05)
    table = J.PenaltyTable(V, rows, 600)
    for r in range(rows):
        table.rebuild(r, rng.integers(0, V, 500).astype(np.uint32), 250, None, True)
    t, _ = device_rows(x, "f32")
    m = torch.from_numpy(masks.view(np.int32)).cuda()
    u = torch.from_numpy(rng.random(rows).astype(np.float32)).cuda()
    cut = [dict(), dict(temperature=0.8, top_k=40), dict(temperature=1.1, top_p=0.9)]
    edit = dict(repetition=1.2, presence=0.3, frequency=0.2, constrained=True)
    a = torch.zeros(rows, dtype=torch.int32).cuda()
    b = torch.zeros_like(a)
    sampler, s = J.Sampler(V, rows), J.Scorer(V, rows)
    kw = dict(penalties=table, penalty_rows=list(range(rows)), masks=m)
    full = [J.policy(**cut[r % 3], **edit) for r in range(rows)]
    sampler.sample(t, full, a, uniforms=u, **kw)
    s.process(t, full, t, **kw)
    sampler.sample(t, [J.policy(**cut[r % 3]) for r in range(rows)], b, uniforms=u)
    np.testing.assert_array_equal(a.cpu().numpy(), b.cpu().numpy())
    s.close()
    sampler.close()


def test_another_stream_and_graph_replays():
    """On a stream of its own, and captured once the records are uploaded;
    replays, with eager work between, equal the eager result."""
    import torch
    V, rows = 9000, 4
    rng = np.random.default_rng(5)
    x = rng.normal(0, 3, (rows, V)).astype(np.float32)
    t, _ = device_rows(x, "bf16")
    bias = J.BiasTable(V, rows, 50)
    for r in range(rows):
        bias.set(r, rng.choice(V, 50, replace=False), rng.normal(0, 3, 50))
    out, s = torch.zeros((rows, V), device="cuda"), J.Scorer(V, rows)
    a, keep = s.process_args(t, [J.policy()] * rows, out, biases=bias, bias_rows=range(rows))
    s.launch_process(a)
    want = host(out)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out.zero_()
        s.launch_process(a)
    side.synchronize()
    np.testing.assert_array_equal(host(out), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.launch_process(a)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        np.testing.assert_array_equal(host(out), want)
    del graph
    s.close()


def test_refusals():
    import torch
    V, rows = 100, 2
    t, _ = device_rows(np.zeros((rows, V), np.float32), "f32")
    out = torch.zeros_like(t)
    s, pol = J.Scorer(V, rows), [J.policy()] * rows

    def refused(message, code=J.JF_ERR_INVALID_ARGUMENT, **change):
        a, keep = s.process_args(t, change.pop("policies", pol), out, **change.pop("kw", {}))
        for k, v in change.items():
            setattr(a, k, v)
        with pytest.raises(J.JfError) as e:
            s.launch_process(a)
        assert e.value.code == code and message in e.value.message, e.value.message

    refused("batch width", rows=0)
    refused("batch width", rows=3)
    refused("logits dtype", dtype=7)
    refused("processed logits dtype", out_dtype=7)
    refused("null logits", logits=None)
    refused("null processed logits", out=None)
    refused("stride is below", logits_stride=V - 1)
    refused("stride is below", out_stride=V - 1)
    refused("aligned", logits=t.data_ptr() + 2)
    refused("aligned", out=out.data_ptr() + 1)
    refused("in place", out=t.data_ptr(), out_stride=V + 1)
    refused("top_p", policies=[J.policy(top_p=2.0)] * 2)
    refused("no penalty table row", policies=[J.policy(presence=1.0)] * 2)
    refused("mask buffer", policies=[J.policy(constrained=True)] * 2)
    bias, other = J.BiasTable(V, 1, 4), J.BiasTable(V + 1, 1, 4)
    refused("no bias table row", kw=dict(biases=bias, bias_rows=[0, 1]))
    refused("no bias table row", kw=dict(bias_rows=[0, 0]))
    refused("vocabulary differs", kw=dict(biases=other, bias_rows=[0, 0]))
    table = J.PenaltyTable(V, 1, 4)
    table.rebuild(0, [1], 0, None, False)
    kw = dict(penalties=table, penalty_rows=[0, 0])
    refused("more than 16", policies=[J.policy(presence=1.0)] * 2,
            kw=dict(kw, extra_tokens=out, extra_counts=[17, 0], extra_stride=17))
    ex = dict(kw, extra_tokens=out, extra_counts=[1, 0], extra_offsets=[1 << 32, 0])
    refused("exceeds 32 bits", policies=[J.policy(presence=1.0)] * 2, kw=ex)
    for args, message in ((([V], [1.0]), "outside the vocabulary"), (([1, 1], [1.0, 2.0]), "twice"),
                          (([1], [float("nan")]), "finite"), (([1], [float("inf")]), "finite"),
                          ((range(5), [0.0] * 5), "exceed")):
        with pytest.raises(J.JfError) as e:
            bias.set(0, *args)
        assert message in e.value.message
    with pytest.raises(J.JfError):
        bias.set(1, [1], [1.0])
    with pytest.raises(ValueError):
        s.process_args(t[:, :50], pol, out)
    with pytest.raises(ValueError):
        s.process_args(t.half(), pol, out)
    with pytest.raises(ValueError):
        s.process_args(t, pol, out, bias_rows=[0])
    for masks, mask_rows in ((torch.zeros((2, 3), dtype=torch.int32), None),
                             (torch.zeros((1, 4), dtype=torch.int32), None),
                             (torch.zeros((2, 4), dtype=torch.int32), [0, 2]),
                             (torch.zeros((2, 4), dtype=torch.int64), None)):
        with pytest.raises(ValueError):
            s.process_args(t, pol, out, masks=masks.cuda(), mask_rows=mask_rows)
    # Nothing above reached the output.
    assert not out.any()
    s.close()


@pytest.mark.parametrize("rows", [3, 70])
def test_a_graph_replays_its_own_rows_whatever_the_scorer_does_since(rows):
    """Captured without masks and tables and with them; calls of the other kind, of
    fewer and of more rows come between, and each replay equals the eager call."""
    import torch
    V, rng = 6000, np.random.default_rng(12)
    x = rng.normal(0, 3, (rows, V)).astype(np.float32)
    _, masks = _masks(rng, rows, V)
    t, _ = device_rows(x, "f32")
    table, bias = J.PenaltyTable(V, rows, 40), J.BiasTable(V, rows, 9)
    for r in range(rows):
        table.rebuild(r, rng.integers(0, V, 30), 15, None, True)
        bias.set(r, rng.choice(V, 9, replace=False), rng.normal(0, 3, 9))
    m = torch.from_numpy(masks.view(np.int32)).cuda()
    s = J.Scorer(V, rows)
    edited = dict(masks=m, penalties=table, penalty_rows=range(rows), biases=bias,
                  bias_rows=range(rows))
    kinds = [([J.policy()] * rows, {}),
             ([J.policy(constrained=True, presence=0.5)] * rows, edited),
             ([J.policy(repetition=1.2)] * rows, dict(edited, masks=None)),
             ([J.policy(constrained=True)] * rows, dict(masks=m))]
    outs = [torch.zeros((rows, V), device="cuda") for _ in kinds]
    records = [s.process_args(t, p, o, **kw) for (p, kw), o in zip(kinds, outs)]
    stream, wants, graphs = torch.cuda.Stream(), [], []
    for (a, _), out in zip(records, outs):
        s.launch_process(a)
        wants.append(host(out))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.launch_process(a)
        graphs.append(graph)
    few_out = torch.zeros((2, V), device="cuda")
    few = s.process_args(t[:2], [J.policy(exclude_stop=True), J.policy(constrained=True)], few_out,
                         masks=m)
    for turn in range(3):
        for n, (graph, out) in enumerate(zip(graphs, outs)):
            for i in (few[0], records[(n + 1 + turn) % 4][0]):
                s.launch_process(i)
            torch.cuda.synchronize()
            for o in outs:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            np.testing.assert_array_equal(host(out), wants[n])
            assert not any(bool(o.any()) for k, o in enumerate(outs) if k != n)
    # A call with records of its own is refused inside a capture, and the scorer
    # goes on.
    s.launch_process(records[1][0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(J.JfError) as e:
            s.launch_process(few[0])
        s.launch_process(records[1][0])
    assert e.value.code == J.JF_ERR_LOGIC
    s.launch_process(few[0])
    assert few_out.any()
    torch.cuda.synchronize()
    outs[1].zero_()
    graph.replay()
    np.testing.assert_array_equal(host(outs[1]), wants[1])
    del graph, graphs, few_out
    s.close()
