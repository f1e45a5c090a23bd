"""The example's decoder, served from pages, against recomputing every prefix without a cache.

Both sides run the same bf16 layers; the attention outputs differ by the rounding of the softmax weights
(2^-8, 2^-11 with an 8-bit cache) and of the sums, at most two bf16 units of their size, which two layers carry
to the logits: 2^-5 of their norm leaves them a factor of four. An 8-bit cache rounds keys and values by 2^-4 at
most, a third of that in the mean, and a key's share of a score's error falls with sqrt(head_dim): 0.15."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,budget,bound", [(torch.bfloat16, 0, 2.0 ** -5), (torch.bfloat16, 64, 2.0 ** -5),
                                                (torch.float8_e4m3fn, 0, 0.15)])
def test_decoder_from_pages(cuda, dtype, budget, bound):
    """With a budget of all pages the sparse path has to give the same as the dense one."""
    import paged_decode as example
    steps = 18
    model, prompts, forced, logits = example.generate([3, 47, 300], steps, dtype, budget)
    assert torch.isfinite(logits).all()
    for b, p in enumerate(prompts):
        for t in (0, 1, 2, steps // 2, steps):
            want = example.recompute(model, torch.cat([p, forced[:t, b]])).float()
            off = float((logits[t, b].float() - want).norm() / want.norm())
            assert off <= bound, (b, t, off)


def test_decoder_with_few_pages_a_step(cuda):
    """A budget below the context: finite, repeatable, and the steps that still fit it unchanged."""
    import paged_decode as example
    dense = example.generate([3, 200], 12)[-1]
    sparse, again = (example.generate([3, 200], 12, budget=6)[-1] for _ in "ab")
    assert torch.isfinite(sparse).all() and torch.equal(sparse, again)
    assert not torch.equal(sparse[:, 1], dense[:, 1])
    # sequence 0 never has more than one page
    assert float((sparse[:, 0].float() - dense[:, 0].float()).norm() / dense[:, 0].float().norm()) <= 2.0 ** -5
