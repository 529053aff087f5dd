"""What the binding of the operators over rows of logits refuses before a record
goes to the library, with host tensors that say they are on a GPU (no GPU)."""
import pytest
import torch

import jf_sampler as J

V, ROWS = 100, 3


class OnGpu(torch.Tensor):
    """A host tensor that gives itself out for one of GPU `index`."""
    index = 0
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.index))

    def get_device(self):
        return self.index


def on(t, index=0):
    t = t.as_subclass(OnGpu)
    t.index = index
    return t


def scorer():
    """One without a library's handle: it builds records and launches none."""
    s = J.Scorer.__new__(J.Scorer)
    s.handle, s.vocabulary, s.max_rows, s.device = None, V, ROWS, 0
    return s


PENALIZED = [J.policy(presence=1.0)] * ROWS


def extras(tokens, policies=PENALIZED, **kw):
    x = on(torch.zeros((ROWS, V)))
    return scorer().process_args(x, policies, x, extra_tokens=tokens, **kw)


def test_extra_tokens_are_32_bit_ids():
    for dtype in (torch.int64, torch.float32, torch.int16, torch.uint8):
        with pytest.raises(ValueError, match="extra tokens"):
            extras(on(torch.zeros(8, dtype=dtype)), extra_counts=[1, 0, 2], extra_stride=2)
    for dtype in (torch.int32, torch.uint32):
        extras(on(torch.zeros(8, dtype=dtype)), extra_counts=[1, 0, 2], extra_stride=2)


@pytest.mark.parametrize("size,ok", [(0, False), (5, False), (6, True)])
@pytest.mark.parametrize("where", [dict(extra_stride=2), dict(extra_offsets=[5, 9, 4])])
def test_extra_tokens_hold_what_the_rows_take(size, ok, where):
    """Rows take [0, 1), nothing and [4, 6), or [5, 6) and [4, 6)."""
    tokens = on(torch.zeros(size, dtype=torch.int32))
    if ok:
        a, keep = extras(tokens, extra_counts=[1, 0, 2], **where)
        assert a.extra_tokens == tokens.data_ptr()
    else:
        with pytest.raises(ValueError, match="extra tokens"):
            extras(tokens, extra_counts=[1, 0, 2], **where)


def test_extra_tokens_of_a_wider_buffer():
    """Rows of a view are addressed by its own stride."""
    wide = on(torch.zeros((ROWS, 7), dtype=torch.int32)[:, 2:5])
    extras(wide, extra_counts=[3] * ROWS, extra_stride=7)
    with pytest.raises(ValueError, match="extra tokens"):
        extras(wide, extra_counts=[3, 3, 4], extra_stride=7)


def test_extra_tokens_that_no_row_reads():
    """Rows without penalties take none; counts and places that the library
    refuses are left to it."""
    none = on(torch.zeros(0, dtype=torch.int32))
    extras(none, policies=[J.policy()] * ROWS, extra_counts=[9] * ROWS, extra_stride=16)
    for counts, offsets in (([17, 0, 0], None), ([0, 0, 1], [0, 0, 1 << 32]), ([0, -1, 0], None)):
        extras(none, extra_counts=counts, extra_offsets=offsets, extra_stride=16)


def test_masks_are_32_bit_words():
    x = on(torch.zeros((ROWS, V)))
    for dtype in (torch.float32, torch.int64, torch.int16):
        with pytest.raises(ValueError, match="masks"):
            scorer().process_args(x, PENALIZED, x, masks=on(torch.zeros((ROWS, 8), dtype=dtype)))
    for dtype in (torch.int32, torch.uint32):
        scorer().process_args(x, PENALIZED, x, masks=on(torch.zeros((ROWS, 4), dtype=dtype)))


def test_tensors_are_on_the_scorers_gpu():
    """A tensor of another GPU: its address means nothing on the scorer's, and a
    trainer's current stream there is not the one that the tensor's work is on."""
    def t(*shape, dtype=torch.float32):
        return on(torch.zeros(shape, dtype=dtype))
    i32 = torch.int32
    x, ids, values = t(ROWS, V), t(ROWS, 2, dtype=i32), t(ROWS, 2)
    s = scorer()
    calls = ((s.process_args, dict(logits=x, policies=PENALIZED, out=x, masks=t(ROWS, 4, dtype=i32),
                                   extra_tokens=t(8, dtype=i32))),
             (s.logprobs_args, dict(logits=x, tokens=ids, temperatures=t(ROWS), lse=t(ROWS),
                                    logprobs=values, ranks=t(ROWS, dtype=i32), top_ids=ids,
                                    top_logprobs=values)),
             (s.distill_args, dict(logits=x, teacher_ids=ids, teacher_values=values, loss=t(ROWS),
                                   lse=t(ROWS), saved=t(ROWS, 4), grad_loss=t(ROWS), grad=x)))
    for build, kw in calls:
        build(**kw)
        for name, value in kw.items():
            if torch.is_tensor(value):
                with pytest.raises(ValueError, match="cuda:1, not on cuda:0"):
                    build(**dict(kw, **{name: on(value.clone(), 1)}))
                with pytest.raises(ValueError, match="not on the GPU"):
                    build(**dict(kw, **{name: torch.zeros(value.shape, dtype=value.dtype)}))


def test_numpy_counts_offsets_and_strides():
    import numpy as np
    tokens = on(torch.zeros(8, dtype=torch.int32))
    extras(tokens, extra_counts=np.array([1, 0, 2]), extra_stride=np.int64(2))
    extras(tokens, extra_counts=np.array([1, 0, 2]), extra_offsets=np.array([0, 0, 6]))
    with pytest.raises(ValueError, match="extra tokens"):
        extras(tokens, extra_counts=np.array([1, 0, 2]), extra_stride=np.int64(4))
