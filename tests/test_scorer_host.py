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
        rc = self.lib.jf_process_logits(self.scorer, ctypes.byref(a), None)
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
