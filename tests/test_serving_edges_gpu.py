"""The serving operators where they are easiest to get wrong: clusters whose CTAs start at different times,
batches and prefixes beyond one CTA's or one tile's share, indices outside their buffers, axes of one element."""

from __future__ import annotations

import math

import pytest
import torch

from test_serving_gpu import check_sample, clear_error_word, gen, params, sy  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# sample_tokens
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("vocab", [4097, 8200, 20001])
def test_sample_many_short_clusters_at_once(sy, vocab):
    """Clusters of 2, 4 and 8 CTAs with next to nothing to read, thousands of them from three streams at once, so that
    the CTAs of one start at different times. Every row repeats one of 16, and so does its token."""
    g = gen(vocab)
    x = 3 * torch.randn(16, vocab, generator=g, device="cuda")
    args = params(16, vocab)
    check_sample(sy, x, *args)
    want, logprob = sy.sample_tokens(x, *args, return_logprob=True)
    times = 64
    many, margs = x.repeat(times, 1), [a.repeat(times) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(sy.sample_tokens(many, *margs, return_logprob=True))
    torch.cuda.synchronize()
    for token, lp in got:
        assert torch.equal(token, want.repeat(times))
        assert torch.equal(lp.nan_to_num(1.0), logprob.repeat(times).nan_to_num(1.0))
