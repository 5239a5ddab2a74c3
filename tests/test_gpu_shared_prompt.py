"""The shared-prompt example: prompt, drafts, commits and a decode step agree
with a prefill of every sequence's whole text.

States are float sums in two orders (1e-5 of the 2-norm, as the operators'
own tests hold them, on each side). Logits go through attention outputs and
linear inputs rounded to bf16 on both sides, which a float difference moves
across a midpoint now and then: 2^-7 of the largest logit."""
import os
import sys

import pytest

from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "project-k3x_b200", "examples"))


@pytest.mark.parametrize("prompt,sequences,drafts,rounds", [(300, 5, 3, 3), (1, 2, 1, 2), (131, 40, 2, 1)])
def test_example_agrees_with_whole_texts(prompt, sequences, drafts, rounds):
    torch_cuda()
    import shared_prompt
    got = shared_prompt.main(prompt, sequences, drafts, rounds)
    assert got["committed"] >= sequences * rounds
    assert got["state_error"] <= 2e-5 and got["logits_error"] <= 2.0 ** -7, got
