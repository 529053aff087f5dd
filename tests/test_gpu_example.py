"""The example that runs processed logits, the sampler, log-probabilities and
the distillation loss together: the loss falls, drawn tokens are possible and
the lists ordered."""
import os
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "examples"))


def test_the_draft_model_learns():
    import distill_draft
    losses, scores = distill_draft.run(steps=40, say=lambda line: print(line, flush=True))
    assert np.mean(losses[-5:]) < 0.8 * np.mean(losses[:5])
    assert np.isfinite(scores["logprobs"]).all() and (scores["ranks"] >= 1).all()
    assert np.all(np.diff(scores["top_logprobs"], axis=1) <= 0)
