"""generate: samples that cannot go on, parameters as whole numbers, and its further refusals."""

from __future__ import annotations

import pytest
import torch

from switchyard.decoder import Decoder, DecoderConfig

pytestmark = pytest.mark.gpu


def small(dtype=torch.bfloat16, **kw):
    torch.manual_seed(0)
    cfg = DecoderConfig(vocab_size=97, d_model=128, n_layers=2, n_heads=2, d_ff=256, n_blocks=2, max_seq_len=128,
                        residual="switchyard", sources="arena", tie_embeddings=False, **kw)
    return Decoder(cfg).cuda().to(dtype)


def test_a_sample_with_nothing_to_draw_from_ends():
    """Tokens from 85 on have NaN embeddings: a sample that draws one has NaN logits at the next step. It ends with -1,
    and the other samples draw what they draw when it is healthy."""
    from switchyard.generate import generate

    model = small()
    prompt = torch.arange(20, device="cuda")
    u = torch.rand(6, 40, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    healthy, _ = generate(model, prompt, 40, 6, u=u)
    with torch.no_grad():
        model.embed.weight[85:] = float("nan")
    tokens, logprobs = generate(model, prompt, 40, 6, u=u)
    high = healthy >= 85
    after = high.cumsum(1) - high.int() > 0  # behind the first token from 85 on
    assert 0 < int(after[:, -1].sum()) < 40, "both kinds of samples are there"
    assert torch.equal(tokens, healthy.masked_fill(after, -1))
    assert torch.equal(logprobs.isnan(), after)


def test_a_prompt_with_nothing_to_draw_from():
    from switchyard.generate import generate

    model = small(torch.float16)
    with torch.no_grad():
        model.lm_head.weight.fill_(float("nan"))
    tokens, logprobs = generate(model, torch.arange(5, device="cuda"), 3, 4)
    assert (tokens == -1).all() and logprobs.isnan().all()


def test_whole_numbers_as_parameters():
    from switchyard.generate import generate

    model = small()
    prompt = torch.arange(7, device="cuda")
    u = torch.rand(3, 5, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    want = generate(model, prompt, 5, 3, u=u, temperature=1.0, top_p=1.0, min_p=0.0)
    got = generate(model, prompt, 5, 3, u=u, temperature=1, top_k=0, top_p=1, min_p=0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    greedy, _ = generate(model, prompt, 5, 3, u=u, temperature=0)
    assert torch.equal(greedy, generate(model, prompt, 5, 3, u=u, temperature=0.0)[0])


def test_the_default_dtype_does_not_matter():
    from switchyard.generate import generate

    model = small()
    prompt = torch.arange(7, device="cuda")

    def draw():
        g = torch.Generator("cuda").manual_seed(4)
        return generate(model, prompt, 5, 3, temperature=0.8, top_p=0.9, min_p=0.01, generator=g)

    want = draw()
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        got = draw()
    finally:
        torch.set_default_dtype(before)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[1].dtype == torch.float32


@pytest.mark.parametrize("page_size", [0, -8, 12])
def test_page_sizes_that_are_refused(page_size):
    from switchyard.generate import generate

    with pytest.raises(ValueError, match="page_size"):
        generate(small(), torch.arange(7, device="cuda"), 2, 3, page_size=page_size)
