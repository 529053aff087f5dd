"""A norm alone may be written anywhere, also over an element of its gradients: these have
all been read by then. Where gradients are written it is refused."""
import pytest

import jf_sampler as J
from scoring_cases import U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tensors", [1, 3, 200])
@pytest.mark.parametrize("order", [2.0, float("inf")])
def test_a_norm_over_an_element_of_a_gradient(tensors, order):
    import torch
    torch.manual_seed(tensors)
    grads = [torch.randn(9000 + n, device="cuda") for n in range(tensors)]
    before = [g.clone() for g in grads]
    whole = torch.cat(before).double()
    want = float(whole.abs().max() if order != 2 else whole.square().sum().sqrt())
    clipper = J.GradientClipper(tensors)
    for at in (0, 8999):
        norm = grads[-1][at:at + 1]
        for g, b in zip(grads, before):
            g.copy_(b)
        for launch in (clipper.launch_scale, clipper.launch_clip):
            with pytest.raises(J.JfError, match="share"):
                launch(clipper.args(grads, norm=norm, max_norm=1.0, order=order))
        clipper.launch_norm(clipper.args(grads, norm=norm, order=order))
        assert abs(norm.item() - want) <= (U + 1e-12) * want
        # Nothing else.
        norm.copy_(before[-1][at:at + 1])
        assert all(torch.equal(g, b) for g, b in zip(grads, before))
    clipper.close()
