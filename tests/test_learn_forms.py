"""Which launches the calls of the GPU tests' sizes are made of, so that these tests reach
the forms that they are there for (over a recording device; no GPU)."""
import pytest

import jf_sampler as J
from test_learn_host import CLIPPED, FORWARD, PREFERENCE, STEP, Host, kinds

TYPES = {"f32": J.JF_DTYPE_F32, "bf16": J.JF_DTYPE_BF16}


def launches(loss, call, rows, V, dtype, **fields):
    with Host(vocabulary=V, max_rows=rows) as h:
        names, make = (CLIPPED, h.clipped) if loss == "clipped" else (PREFERENCE, h.preference)
        a = make(rows, dtype=TYPES[dtype], logits_stride=V, grad_stride=V, **fields)
        # Apart from one another, as the tests' tensors are.
        for n, name in enumerate(("tokens", "grad_loss", "offsets", "advantages", "out_loss")):
            if hasattr(a, name) and name not in fields:
                setattr(a, name, (8 << 30) + (n << 26))
        rc, log = h.call(names[call], h.scorer, a)
        assert rc == 0
        return log


@pytest.mark.parametrize("rows,V,dtype,want", [
    (6, 700, "f32", "step"), (66, 700, "f32", "step"), (6, 80001, "f32", "score grad"),
    (42, 80001, "f32", "score rows grad"), (42, 80001, "bf16", "score rows grad"),
    (102, 90001, "f32", "step"), (102, 90001, "bf16", "score rows grad"),
    (180, 170001, "f32", "step"), (180, 170001, "bf16", "step")])
def test_steps(rows, V, dtype, want):
    log = launches("clipped", STEP, rows, V, dtype)
    assert kinds(log) == want.split()
    if want == "step":
        size = 4 if dtype == "f32" else 2
        assert log[0]["blocks"] == (4 if rows == 6 else 1)
        assert log[0]["threads"] == (1024 if V * size > 320 << 10 else 512)


def test_preference_losses_of_many_long_rows():
    for call, behind in ((FORWARD, []), (STEP, ["grad"])):
        for dtype in TYPES:
            log = launches("preference", call, 1100, 110001 if dtype == "f32" else 140001, dtype)
            assert kinds(log) == ["score", "pair_rows", "pairs"] + behind
            assert not log[2]["with_rows"]


# The forms whose accuracy is tested, by their first launch.
@pytest.mark.parametrize("loss,call,rows,V,dtype,want,threads", [
    ("preference", FORWARD, 256, 32000, "f32", "whole pairs", 512),
    ("preference", STEP, 128, 32000, "f32", "score pairs grad", None),
    ("clipped", STEP, 16, 32000, "f32", "step", 512),
    ("preference", FORWARD, 2048, 32000, "bf16", "whole pairs", 256),
    ("clipped", FORWARD, 2048, 32000, "bf16", "whole", 256),
    ("clipped", STEP, 512, 32000, "bf16", "step", 512),
    ("clipped", FORWARD, 64, 100003, "f32", "score rows", None),
    ("clipped", FORWARD, 256, 100003, "f32", "whole", 512),
    ("clipped", STEP, 16, 100003, "f32", "score grad", None),
    ("clipped", FORWARD, 256, 100003, "bf16", "whole", 512),
    ("preference", FORWARD, 2048, 151936, "f32", "score pair_rows pairs", None),
    ("clipped", STEP, 256, 151936, "f32", "step", 1024),
    ("preference", STEP, 2048, 151936, "bf16", "score pair_rows pairs grad", None),
    ("clipped", STEP, 256, 151936, "bf16", "step", 512),
    ("clipped", STEP, 16, 151936, "bf16", "score grad", None)])
def test_forms_whose_accuracy_is_tested(loss, call, rows, V, dtype, want, threads):
    log = launches(loss, call, rows, V, dtype)
    assert kinds(log) == want.split()
    assert threads is None or log[0]["threads"] == threads
    # The vectors a thread takes of a chunk, by the chunks a row.
    vectors = {(128, 32000): 4, (64, 100003): 4, (16, 100003): 4, (2048, 151936): 8,
               (16, 151936): 2}.get((rows, V))
    if "score" in want:
        chunk = 256 * (4 if dtype == "f32" else 8) * (4 if dtype == "bf16" and vectors == 8
                                                      else vectors)
        assert log[0]["segments"] == -(-V // chunk)


@pytest.mark.parametrize("rows,fields", [(6, dict(out_loss=5 << 33, grad_loss=5 << 33)),
                                         (6, dict(out_loss=5 << 33, tokens=5 << 33)), (180, {}),
                                         (180, dict(grad=1 << 30))])
def test_bf16_steps_of_1024_threads(rows, fields):
    log = launches("clipped", STEP, rows, 170001, "bf16", entropy_weight=0.1, **fields)
    assert kinds(log) == ["step"] and (log[0]["threads"], log[0]["blocks"]) == (1024, 1)
