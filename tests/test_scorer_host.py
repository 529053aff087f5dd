"""The scorer's host code over a recording device (tests/cpp/scorer_host.cpp; no
GPU): what it uploads, allocates, launches and refuses."""
import ctypes
import json
import os

import pytest

import jf_sampler as J

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "cpp", "_build", "libscorer_host.so")
vp, u32 = ctypes.c_void_p, ctypes.c_uint32
LOGITS, OUT, MASKS = 1 << 30, 2 << 30, 3 << 30  # addresses that nothing reads
STREAM = vp(64)


class Host:
    """The library over the recording device, and one scorer."""

    def __init__(self, vocabulary=1000, max_rows=4):
        assert os.path.exists(LIB), "build first: python tests/cpp/build.py"
        self.lib = ctypes.CDLL(LIB)
        self.lib.fake_log.restype = ctypes.c_char_p
        self.lib.jf_last_error.restype = ctypes.c_char_p
        self.device(0)
        self.capturing(False)
        self.vocabulary = vocabulary
        self.scorer = vp()
        self.log()
        assert self.lib.jf_scorer_create(vocabulary, max_rows, ctypes.byref(self.scorer)) == 0
        self.created = self.log()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.device(0)
        self.capturing(False)
        self.lib.jf_scorer_destroy(self.scorer)

    def log(self):
        """What has happened since the last look."""
        return [json.loads(line) for line in self.lib.fake_log().decode().splitlines()]

    def device(self, device):
        self.lib.fake_device(device)

    def capturing(self, capturing):
        self.lib.fake_capturing(1 if capturing else 0)

    def process(self, policies, **fields):
        """(return code, what happened)."""
        rows = len(policies)
        a = J.JfProcessArgs()
        a.rows, a.logits, a.out = rows, LOGITS, OUT
        a.dtype = a.out_dtype = J.JF_DTYPE_F32
        a.logits_stride = a.out_stride = self.vocabulary
        a.masks, a.mask_stride = MASKS, (self.vocabulary + 31) // 32
        a.policies = (J.JfPolicy * rows)(*policies)
        a.stop_token_0 = a.stop_token_1 = J.JF_NO_TOKEN
        for name, value in fields.items():
            setattr(a, name, value)
        rc = self.lib.jf_process_logits(self.scorer, ctypes.byref(a), STREAM)
        return rc, self.log()

    def refused(self, rc, code, message):
        assert rc == code and message in self.lib.jf_last_error().decode(), \
            (rc, self.lib.jf_last_error())


def kinds(log):
    return [e["what"] for e in log]


PLAIN, MASKED = J.policy(), J.policy(constrained=True)


def test_a_captured_call_brings_no_new_row_records():
    """Its upload would be replayed from a pinned buffer that other calls have
    filled since, and a call after it would take the records for uploaded."""
    with Host() as h:
        assert kinds(h.process([PLAIN] * 2)[1]) == ["copy", "process"]
        h.capturing(True)
        rc, log = h.process([MASKED] * 2)
        h.refused(rc, J.JF_ERR_LOGIC, "captured")
        assert not log
        # The same records as before are no upload.
        rc, log = h.process([PLAIN] * 2)
        assert rc == 0 and kinds(log) == ["process"]
        h.capturing(False)
        rc, log = h.process([MASKED] * 2)
        assert rc == 0 and kinds(log)[-2:] == ["copy", "process"]


def test_captured_calls_keep_their_row_records():
    """A captured call has its masks and tables fixed, so its replays have to read
    the records that go with them, whatever the scorer is called with since."""
    with Host() as h:
        records = next(e["at"] for e in h.created if e["what"] == "malloc")

        def call(policies, capture=False):
            h.capturing(capture)
            rc, log = h.process(policies)
            h.capturing(False)
            assert rc == 0
            assert not capture or kinds(log) == ["process"]
            uploads = [e for e in log if e["what"] == "copy"]
            for e in uploads:
                held[e["to"]] = bytes.fromhex(e["held"])
            (used,) = [e["rows"] for e in log if e["what"] == "process"]
            return used, held[used][:48 * len(policies)]

        held, graphs = {}, []
        for policies in ([PLAIN] * 2, [MASKED, PLAIN], [MASKED] * 4, [PLAIN] * 2):
            eager = call(policies)
            graphs.append(call(policies, capture=True))
            assert graphs[-1] == eager
            # Calls with and without new records behind the captured one.
            for other in (policies, [PLAIN, MASKED, MASKED], [MASKED], policies):
                call(other)
                for used, then in graphs:
                    assert held[used][:len(then)] == then
        # Calls that nothing captured share one place.
        places = len(held)
        for policies in ([PLAIN], [MASKED], [PLAIN] * 4):
            call(policies)
        assert len(held) == places == 1 + len(graphs) and records in held
        # Counted, and freed with the scorer.
        h.lib.jf_scorer_workspace_bytes.restype = ctypes.c_uint64
        bytes_before = sum(e["bytes"] for e in h.created if e["what"] == "malloc")
        assert h.lib.jf_scorer_workspace_bytes(h.scorer) == bytes_before + 4 * 4 * 48
        h.lib.jf_scorer_destroy(h.scorer)
        h.scorer = vp()
        freed = {e["at"] for e in h.log() if e["what"] == "free"}
        assert set(held) <= freed


def test_biases_are_not_set_inside_a_capture():
    with Host() as h:
        table = vp()
        assert h.lib.jf_bias_table_create(1000, 2, 4, ctypes.byref(table)) == 0
        h.log()
        tokens, biases = (u32 * 2)(3, 9), (ctypes.c_float * 2)(1.0, 2.0)
        args = (table, 1, tokens, biases, ctypes.c_uint64(2), STREAM)
        h.capturing(True)
        h.refused(h.lib.jf_bias_table_set(*args), J.JF_ERR_LOGIC, "captured")
        assert not h.log()
        # The row is as it was, and may be used.
        rc, _ = h.process([PLAIN], biases=table, bias_rows=(u32 * 1)(1))
        assert rc == J.JF_ERR_LOGIC  # its records are new
        h.capturing(False)
        assert h.process([PLAIN], biases=table, bias_rows=(u32 * 1)(1))[0] == 0
        assert h.lib.jf_bias_table_set(*args) == 0
        assert kinds(h.log()) == ["copy", "copy"]
        h.lib.jf_bias_table_destroy(table)


def test_tables_of_another_device_are_refused():
    with Host() as h:
        biases = vp()
        h.device(1)
        assert h.lib.jf_bias_table_create(1000, 1, 4, ctypes.byref(biases)) == 0
        h.device(0)
        h.lib.fake_penalty_table.restype = vp
        penalties = [vp(h.lib.fake_penalty_table(1000, device)) for device in (0, 1)]
        row = (u32 * 1)(0)
        h.log()
        rc, log = h.process([PLAIN], biases=biases, bias_rows=row)
        h.refused(rc, J.JF_ERR_INVALID_ARGUMENT, "bias table is on another device")
        assert not log
        penalized = [J.policy(presence=1.0)]
        rc, log = h.process(penalized, penalties=penalties[1], penalty_rows=row)
        h.refused(rc, J.JF_ERR_INVALID_ARGUMENT, "penalty table is on another device")
        assert not log
        assert h.process(penalized, penalties=penalties[0], penalty_rows=row)[0] == 0
        for table in penalties:
            h.lib.fake_penalty_table_free(table)
        h.lib.jf_bias_table_destroy(biases)


@pytest.mark.parametrize("vocabulary", [524289, 2 ** 32 - 2048, 2 ** 32 - 2047, 2 ** 32 - 1])
def test_bias_tables_take_no_larger_vocabulary_than_scorers(vocabulary):
    """Near 2^32 the number of a row's buckets wrapped to none, and setting a row
    then counted past a vector of one."""
    with Host() as h:
        table = vp(1)
        rc = h.lib.jf_bias_table_create(vocabulary, 1, 1, ctypes.byref(table))
        h.refused(rc, J.JF_ERR_INVALID_ARGUMENT, "524288 tokens")
        assert not table.value and not h.log()
        assert h.lib.jf_bias_table_create(524288, 1, 1, ctypes.byref(table)) == 0
        h.lib.jf_bias_table_destroy(table)


def test_a_bias_table_whose_bytes_pass_64_bits_is_out_of_memory():
    """2^30 + 1 rows of 2^31 - 1 entries are 2^64 bytes and a few: a table of a few
    bytes was made."""
    with Host() as h:
        table = vp(1)
        rc = h.lib.jf_bias_table_create(1, (1 << 30) + 1, (1 << 31) - 1, ctypes.byref(table))
        h.refused(rc, J.JF_ERR_NO_MEMORY, "bias entries")
        assert not table.value and not h.log()


def scratch(h):
    """{address: bytes} of the scorer's device memory."""
    return {e["at"]: e["bytes"] for e in h.created if e["what"] == "malloc"}


def score(h, rows, dtype=0, top=0):
    a = J.JfLogprobsArgs()
    a.rows, a.dtype, a.logits, a.logits_stride = rows, dtype, LOGITS, h.vocabulary
    a.out_lse = OUT
    if top:
        a.top, a.out_top_ids, a.out_top_logprobs = top, OUT, OUT
    assert h.lib.jf_logprobs(h.scorer, ctypes.byref(a), STREAM) == 0
    return h.log()


def distill(h, rows, dtype=0, call="jf_distill_step", saved=None):
    a = J.JfDistillArgs()
    a.rows, a.dtype, a.logits, a.logits_stride = rows, dtype, LOGITS, h.vocabulary
    a.temperature, a.teacher_ids, a.teacher_values = 1.0, MASKS, MASKS
    a.teacher_stride = a.teacher_count = 256
    a.out_loss, a.grad_loss, a.grad, a.grad_stride = OUT, OUT, OUT, h.vocabulary
    a.saved = saved
    assert getattr(h.lib, call)(h.scorer, ctypes.byref(a), STREAM) == 0
    return h.log()


@pytest.mark.parametrize("vocabulary", [1, 3, 2048, 2049, 32000, 73728, 73729, 151936, 262144,
                                        524288])
def test_scratch_holds_what_every_launch_takes(vocabulary):
    for max_rows in (1, 5, 111, 112, 409, 513, 65536, 4194304):
        with Host(vocabulary, max_rows) as h:
            held = scratch(h)
            for rows in sorted({1, 2, 100, 111, 112, 148, 296, 408, 409, 512, 513, 20000, 55189,
                                max_rows}):
                if rows > max_rows:
                    continue
                for dtype in (0, 1):
                    for log in (score(h, rows, dtype), score(h, rows, dtype, top=128),
                                distill(h, rows, dtype), distill(h, rows, dtype, "jf_distill")):
                        for e in log:
                            if "segments" in e:
                                parts = e["row_count"] * e["segments"]
                                assert 8 * parts <= held[e["partials"]], (max_rows, rows, e)
                                assert 4 * parts <= held[e["aheads"]], (max_rows, rows, e)
                                if e["top"]:
                                    assert 4 * e["row_count"] * e["groups"] <= held[e["maxima"]]
                            if e["what"] in ("loss", "grad") and e["saved"]:
                                assert 4 * e["row_count"] * 258 <= held[e["saved"]], (max_rows, e)


def test_scratch_of_rows_is_that_of_one_launch():
    """Its launches follow one another on the same parts. One launch over 151,936
    tokens takes 55,188 rows at most, in chunks of at least 2,048 tokens."""
    with Host(151936, 4194304) as h:
        parts = 55188 * 75
        sizes = sorted(scratch(h).values())
        assert sizes.count(8 * parts) == 1 and sizes.count(4 * parts) == 1
        assert max(score(h, 4194304), key=lambda e: e["row_count"])["row_count"] == 55188
    with Host(1000, 8) as h:
        assert {8 * 8, 4 * 8} <= set(scratch(h).values())


def test_distillation_records_are_those_of_steps_by_chunks():
    """Only steps of fewer rows than are taken whole keep them in the scorer: none
    of short rows, fewer than 112 or a row's f32 bytes / 5120 of long ones."""
    for vocabulary, rows in ((1000, 0), (73728, 0), (73729, 111), (151936, 117), (524288, 408)):
        for max_rows in (5, 4194304):
            with Host(vocabulary, max_rows) as h:
                size = min(rows, max_rows) * 258 * 4
                held = scratch(h)
                saved = {e["saved"] for n in range(1, min(rows, max_rows) + 1)
                         for e in distill(h, n) if e["what"] == "grad"}
                assert [held[at] for at in saved] == [size] * bool(rows)
                # That is all: rows, parts and maxima beside it.
                used = {e[name] for log in (score(h, 1, top=1), h.process([PLAIN])[1]) for e in log
                        for name in ("rows", "partials", "aheads", "maxima") if name in e}
                assert set(held) == used | saved
                h.lib.jf_scorer_workspace_bytes.restype = ctypes.c_uint64
                assert h.lib.jf_scorer_workspace_bytes(h.scorer) == sum(held.values())


def test_steps_of_whole_rows_are_one_launch():
    with Host(1000, 200000) as h:
        assert [e["row_count"] for e in distill(h, 200000)] == [200000]
    with Host(151936, 200000) as h:
        assert [(e["what"], e["row_count"]) for e in distill(h, 55188 + 117)] == [
            ("step", 55188), ("score", 117), ("loss", 117), ("grad", 117)]
