"""generate: cached decoding against the decoder's own forward, and its refusals."""

from __future__ import annotations

import pytest
import torch

from switchyard.decoder import Decoder, DecoderConfig

pytestmark = pytest.mark.gpu


def small(residual, dtype=torch.bfloat16, sources="arena"):
    torch.manual_seed(0)
    cfg = DecoderConfig(vocab_size=331, d_model=256, n_layers=4, n_heads=4, d_ff=512, n_blocks=4,
                        max_seq_len=400, residual=residual, sources=sources)
    model = Decoder(cfg)
    with torch.no_grad():
        for p in model.parameters():  # logits with some spread, sites that do not mix uniformly
            if p.ndim == 2:
                p.mul_(4)
        for site in model.attn_res or []:
            site.w.normal_(std=0.05)
    return model.cuda().to(dtype)


@pytest.mark.parametrize("residual", ["switchyard", "attnres", "standard"])
@pytest.mark.parametrize("prompt_len", [1, 70])
def test_cached_steps_follow_the_forward(residual, prompt_len):
    """The log-probability of every drawn token agrees with the whole sequence's forward: both round the hidden
    state to bf16 (2^-8) once an operation, some hundred operations deep, in different orders."""
    from switchyard.generate import generate

    model = small(residual)
    prompt = torch.randint(0, 331, (prompt_len,), device="cuda")
    u = torch.rand(9, 5, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    tokens, logprobs = generate(model, prompt, 5, 9, u=u, page_size=16)
    assert tokens.shape == logprobs.shape == (5, 9) and int(tokens.min()) >= 0 and int(tokens.max()) < 331
    whole = torch.cat([prompt.expand(5, -1), tokens], 1)
    with torch.no_grad():
        logits = model(whole)[:, prompt_len - 1:-1].double()
    want = logits.log_softmax(-1).gather(-1, tokens[..., None])[..., 0]
    spread = logits.std()
    assert (logprobs.double() - want).abs().max() <= 0.05 * spread + 0.05, (logprobs - want).abs().max()
    again, _ = generate(model, prompt, 5, 9, u=u, page_size=16)
    assert torch.equal(again, tokens)


def test_greedy_samples_agree_and_filters_apply():
    from switchyard.generate import generate

    model = small("switchyard", torch.float16)
    prompt = torch.randint(0, 331, (33,), device="cuda")
    tokens, logprobs = generate(model, prompt, 3, 6, temperature=0.0)
    assert (tokens == tokens[0]).all() and not logprobs.any()
    one, _ = generate(model, prompt, 3, 6, top_k=1)
    assert torch.equal(one, tokens)
    some, lp = generate(model, prompt, 64, 2, top_k=5, top_p=0.9, min_p=0.01)
    assert int(torch.unique(some[:, 0]).numel()) <= 5 and (lp <= 0).all()


def test_refusals():
    from switchyard.generate import generate

    model = small("standard")
    prompt = torch.zeros(4, dtype=torch.long, device="cuda")
    for bad in (dict(prompt=prompt[None]), dict(prompt=prompt[:0]), dict(n_samples=0), dict(max_new=0),
                dict(max_new=397), dict(prompt=prompt.cpu()), dict(u=torch.zeros(2, 2, device="cuda"))):
        args = {**dict(prompt=prompt, n_samples=2, max_new=3), **bad}
        with pytest.raises(ValueError):
            generate(model, **args)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        generate(small("standard", torch.float32), prompt, 2, 3)
