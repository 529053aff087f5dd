"""Trains a small draft model on what a served model's decode steps hand out.

Each step, the teacher's logits of a batch are processed (penalties over each
request's history, a bias list, a grammar mask), a token is drawn from them,
and the row's log-probabilities are taken: the drawn token's with its rank, as
a server reports them, and the best tokens, which are the draft model's lesson
(jf_sampler.train.distill_loss). The models are linear maps of random states,
enough to show the calls and that the loss falls; the states are a few batches
that come again, as a trainer's epochs do.

Usage: python examples/distill_draft.py [--steps N]"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "justfit-llm_amd"))

import jf_sampler as J  # noqa: E402
from jf_sampler.train import distill_loss  # noqa: E402

VOCABULARY, WIDTH, ROWS, LISTED, TEMPERATURE = 32000, 128, 48, 32, 1.0


def run(steps=60, seed=0, say=print):
    """The mean losses of the steps, and the last step's scores."""
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    teacher = torch.randn((WIDTH, VOCABULARY), generator=g, device="cuda") * 0.35
    student = torch.zeros((WIDTH, VOCABULARY), device="cuda", requires_grad=True)
    optimizer = torch.optim.Adam([student], lr=0.01)

    # Requests: a third plain, a third with penalties, a third constrained.
    policies = [J.policy(temperature=0.8, top_p=0.95, **(
        dict(), dict(repetition=1.1, frequency=0.2), dict(constrained=True))[r % 3])
        for r in range(ROWS)]
    neutral = [J.policy(temperature=0.8, top_p=0.95)] * ROWS
    history = J.PenaltyTable(VOCABULARY, ROWS, 4096)
    biases = J.BiasTable(VOCABULARY, ROWS, 8)
    for r in range(ROWS):
        history.rebuild(r, rng.integers(0, VOCABULARY, 64), 32, None, True)
        biases.set(r, rng.choice(VOCABULARY, 8, replace=False), [-float("inf")] * 4 + [3.0] * 4)
    words = torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31, (ROWS, VOCABULARY // 32))
                             .astype(np.int32)).cuda()
    scorer, sampler = J.Scorer(VOCABULARY, ROWS), J.Sampler(VOCABULARY, ROWS)
    tokens = torch.zeros((ROWS, 1), dtype=torch.int32, device="cuda")
    scores = dict(logprobs=torch.empty((ROWS, 1), device="cuda"),
                  ranks=torch.empty(ROWS, dtype=torch.int32, device="cuda"),
                  top_ids=torch.empty((ROWS, LISTED), dtype=torch.int32, device="cuda"),
                  top_logprobs=torch.empty((ROWS, LISTED), device="cuda"))
    processed = torch.empty((ROWS, VOCABULARY), device="cuda")
    batches = torch.randn((4, ROWS, WIDTH), generator=g, device="cuda")
    losses = []
    for step in range(steps):
        states = batches[step % 4]
        scorer.process(states @ teacher, policies, processed, masks=words, penalties=history,
                       penalty_rows=range(ROWS), biases=biases, bias_rows=range(ROWS))
        # The edits are in the logits; the sampler only cuts and draws.
        sampler.sample(processed, neutral, tokens.view(-1),
                       uniforms=torch.rand(ROWS, generator=g, device="cuda"))
        scorer.logprobs(processed, tokens=tokens, **scores)
        logits = states @ student
        loss = distill_loss(scorer, logits, scores["top_ids"], scores["top_logprobs"],
                            temperature=TEMPERATURE, normalize=True).mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        history.count_rows(range(ROWS), tokens.view(-1).cpu().numpy().view(np.uint32))
        losses.append(loss.item())
        if step % 20 == 0 or step == steps - 1:
            say(f"step {step}: loss {losses[-1]:.4f}, drawn tokens' mean log-probability "
                f"{float(scores['logprobs'].mean()):.3f}, median rank "
                f"{int(scores['ranks'].median())}")
    out = {k: v.cpu().numpy() for k, v in scores.items()}
    for handle in (scorer, sampler, history, biases):
        handle.close()
    return losses, out


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=60)
    run(parser.parse_args().steps)
