"""What the torch functions write through addresses counts as written for autograd, as
where torch's own functions write in place: a graph that has saved it refuses its backward
pass instead of taking the new values."""
import pytest

import jf_sampler as J

pytestmark = pytest.mark.gpu

ROWS, V = 4, 300


def inputs():
    import torch
    torch.manual_seed(1)
    leaf = torch.randn((ROWS, V), device="cuda", requires_grad=True)
    tokens = torch.tensor([3, -1, 5, 299], dtype=torch.int32, device="cuda")
    return leaf, tokens, torch.randn(ROWS, device="cuda"), torch.full((ROWS,), -5.0, device="cuda")


def taken(scorer, leaf, tokens, A, reference, **out):
    """A call of each loss with its optional outputs."""
    import torch
    from jf_sampler.train import clipped_loss, preference_loss
    if "scores" in out:
        offsets = torch.arange(ROWS + 1, dtype=torch.int32, device="cuda")
        return preference_loss(scorer, leaf, tokens, offsets, reference, **out)
    return clipped_loss(scorer, leaf, tokens, A, None, reference, **out)


OUTPUTS = [("logprobs", "kl", "entropy"), ("scores", "logprobs")]


def test_clipped_gradients():
    import torch
    from jf_sampler.train import clip_gradients
    clipper = J.GradientClipper(2)
    w = torch.randn(50, device="cuda", requires_grad=True)
    b = torch.nn.Parameter(torch.randn(7, device="cuda").bfloat16())
    w.grad, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    b.grad = torch.randn_like(b)
    penalty = (w.grad * w.grad).sum()
    versions = w.grad._version, b.grad._version
    clip_gradients(clipper, [w, b], 0.5)
    assert (w.grad._version, b.grad._version) == (versions[0] + 1, versions[1] + 1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        penalty.backward()
    clipper.close()


@pytest.mark.parametrize("names", OUTPUTS)
def test_outputs_for_a_trainer_s_records(names):
    import torch
    leaf, *rest = inputs()
    scorer = J.Scorer(V, ROWS)
    out = {k: torch.empty(ROWS, device="cuda") for k in names}
    other = torch.ones(ROWS, device="cuda", requires_grad=True)
    taken(scorer, leaf, *rest, **out).sum().backward()
    for name in names:
        product = (other * out[name]).sum()
        version = out[name]._version
        loss = taken(scorer, leaf, *rest, **out)
        assert out[name]._version == version + 1
        with pytest.raises(RuntimeError, match="inplace operation"):
            product.backward()
        loss.sum().backward()  # no part of it is saved by the losses themselves
    scorer.close()


@pytest.mark.parametrize("names", OUTPUTS)
def test_inference_tensors_have_no_versions(names):
    import torch
    from jf_sampler.train import clip_gradients
    leaf, *rest = inputs()
    scorer, clipper = J.Scorer(V, ROWS), J.GradientClipper(1)
    want = {k: torch.empty(ROWS, device="cuda") for k in names}
    taken(scorer, leaf, *rest, **want)
    with torch.inference_mode():
        out = {k: torch.empty(ROWS, device="cuda") for k in names}
        taken(scorer, leaf.detach(), *rest, **out)
        for k in names:
            assert torch.equal(out[k], want[k])
        leaf.grad = torch.full((ROWS, V), 2.0, device="cuda")
        assert abs(clip_gradients(clipper, leaf, 1.0).item() - 2 * (ROWS * V) ** 0.5) < 1e-4
    for handle in (scorer, clipper):
        handle.close()
