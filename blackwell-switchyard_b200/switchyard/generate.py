"""Continuations of one prompt by the Block AttnRes decoder, many at once.

:func:`generate` reads a prompt once, keeps its keys and values in pages that all
samples share, and then decodes ``n_samples`` continuations together: each step
rotates and appends the new token's keys and values (:func:`~switchyard.append_kv`),
attends over the shared prompt and each sample's own pages
(:func:`~switchyard.attend_paged`) and draws the next tokens
(:func:`~switchyard.sample_tokens`). The residual stream between the sublayers is
the decoder's own: the Block AttnRes sites run the forward kernels over the arena.

The reference trains only; it has no counterpart. The model is used as it is
(:class:`~switchyard.decoder.Decoder`, bf16 or fp16 on a GPU), and its weights are
not touched.
"""

from __future__ import annotations

import torch

from .arena import stage_partial
from .decoder import CausalSelfAttention, Decoder, folded_form
from .serving import append_kv, attend_paged, sample_tokens
from .triton_op import block_attn_res_triton

__all__ = ["PagedCache", "generate"]


class PagedCache:
    """Keys and values of every layer, ``[layers, 2, pages, heads, page_size,
    head_dim]``: the pages of one shared prefix, then the pages of each of
    ``batch`` sequences. Page numbers are the same in all layers."""

    def __init__(self, layers: int, heads: int, head_dim: int, batch: int, prefix_len: int,
                 own_len: int, dtype: torch.dtype, device, page_size: int = 64) -> None:
        if batch < 1 or prefix_len < 0 or own_len < 0:
            raise ValueError("batch must be positive, prefix_len and own_len not negative")
        if page_size < 1 or page_size % 8:
            raise ValueError(f"page_size must be a positive multiple of 8, got {page_size}")
        ahead, own = -(-prefix_len // page_size), -(-own_len // page_size)
        self.page_size, self.prefix_len = page_size, prefix_len
        self.kv = torch.empty(layers, 2, ahead + batch * own, heads, page_size, head_dim,
                              dtype=dtype, device=device)
        self.prefix_pages = torch.arange(ahead, dtype=torch.int32, device=device)
        self.table = ahead + torch.arange(batch * own, dtype=torch.int32, device=device).view(batch, own)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)

    def own_slots(self, n: int) -> torch.Tensor:
        """Slots of the ``n`` tokens a sequence appends next, ``[batch * n]``."""
        at = self.lens.long()[:, None] + torch.arange(n, device=self.lens.device)
        pages = self.table.long().gather(1, at // self.page_size)
        return (pages * self.page_size + at % self.page_size).flatten()

    def prefix_slots(self) -> torch.Tensor:
        return torch.arange(self.prefix_len, device=self.lens.device)


def _attend(op: CausalSelfAttention, x, cache: PagedCache, layer: int, slots, positions, rope, own):
    """The attention sublayer of ``x [batch, n, d_model]`` over the cache."""
    b, n, d = x.shape
    h, hd = op.n_heads, op.head_dim
    k_cache, v_cache = cache.kv[layer]
    q, k, v = (p(x).view(b * n, h, hd) for p in (op.q_proj, op.k_proj, op.v_proj))
    q = append_kv(k, v, k_cache, v_cache, slots, q=q, positions=positions, cos=rope[0], sin=rope[1])
    y = attend_paged(q.view(b, n, h, hd), k_cache, v_cache, **own)
    return op.o_proj(y.reshape(b, n, d))


def _step(model: Decoder, ids, cache: PagedCache, slots, positions, own) -> torch.Tensor:
    """The hidden state of ``ids [batch, n]`` before the final norm."""
    cfg = model.cfg
    rope = (model.rope_cos.float(), model.rope_sin.float())  # a cast model keeps rounded tables

    def sublayer(i, x):
        sub = model.sublayers[i]
        x = sub.norm(x)
        if isinstance(sub.op, CausalSelfAttention):
            return _attend(sub.op, x, cache, i // 2, slots, positions, rope, own)
        return sub.op(x)

    x = model.embed(ids)
    if not cfg.uses_attnres:
        for i in range(cfg.n_sublayers):
            x = x + sublayer(i, x)
        return x

    arena = torch.empty(cfg.n_blocks + 1, *x.shape, device=x.device, dtype=x.dtype)
    arena[0].copy_(x)
    fused = cfg.residual == "switchyard"

    def site(i, sources):
        w = model.attn_res[i].w * model.attn_res[i].g
        mix = block_attn_res_triton if fused else folded_form
        return mix(arena[:sources], w, cfg.norm_eps)

    done, partial = 1, None  # completed blocks, the running block's sum
    for i in range(cfg.n_sublayers):
        if i and i % cfg.block_size == 0:
            done, partial = done + 1, None
        out = sublayer(i, site(i, done + (partial is not None)))
        if partial is None:
            partial = arena[done].copy_(out)
        else:
            # the slot itself holds the running sum: it is read before it is written
            partial = stage_partial(partial.clone(), out, arena[done]) if fused else arena[done].add_(out)
    return site(cfg.n_sublayers, done + 1)


@torch.no_grad()
def generate(
    model: Decoder,
    prompt: torch.Tensor,
    n_samples: int,
    max_new: int,
    u: torch.Tensor | None = None,
    temperature: float = 1.0,
    top_k: int | None = None,
    top_p: float | None = None,
    min_p: float | None = None,
    generator: torch.Generator | None = None,
    page_size: int = 64,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Draw ``n_samples`` continuations of ``prompt`` (int64 ``[tokens]``, on the
    model's GPU), ``max_new`` tokens each.

    ``u`` (fp32 ``[max_new, n_samples]`` in [0, 1)) are the random numbers; without
    it they come from ``generator``. The sampling parameters are
    :func:`~switchyard.sample_tokens`'s. Returns the tokens ``[n_samples, max_new]``
    and their log-probabilities under the distribution they were drawn from. A
    sample that meets logits with nothing to draw from (all NaN after an overflow)
    ends there: its tokens are -1 and its log-probabilities NaN from then on.
    One host synchronisation at most, when the caller reads the result.
    """
    cfg = model.cfg
    weight = model.embed.weight
    if prompt.ndim != 1 or prompt.numel() == 0:
        raise ValueError(f"prompt must be [tokens] and not empty, got {tuple(prompt.shape)}")
    if n_samples < 1 or max_new < 1:
        raise ValueError(f"n_samples and max_new must be positive, got {n_samples} and {max_new}")
    if not weight.is_cuda or prompt.device != weight.device:
        raise ValueError("the model and the prompt must be on one CUDA device")
    if weight.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"generate takes a bfloat16 or float16 model, got {weight.dtype}")
    length, dev = prompt.numel(), weight.device
    if length + max_new > cfg.max_seq_len:
        raise ValueError(f"{length} + {max_new} tokens exceed max_seq_len {cfg.max_seq_len}")
    if u is None:
        u = torch.rand(max_new, n_samples, generator=generator, device=dev, dtype=torch.float32)
    elif u.shape != (max_new, n_samples):
        raise ValueError(f"u must be [{max_new}, {n_samples}], got {tuple(u.shape)}")

    cache = PagedCache(cfg.n_layers, cfg.n_heads, cfg.head_dim, n_samples, length, max_new,
                       weight.dtype, dev, page_size)
    # the prompt, once: one sequence whose own pages are the shared ones
    alone = dict(page_table=cache.prefix_pages[None],
                 kv_lens=torch.full((1,), length, dtype=torch.int32, device=dev))
    at = torch.arange(length, dtype=torch.int32, device=dev)
    h = _step(model, prompt[None], cache, cache.prefix_slots(), at, alone)
    logits = model.lm_head(model.final_norm(h[:, -1])).expand(n_samples, -1)

    def per_sample(x, dtype=torch.float32):
        return None if x is None else torch.full((n_samples,), x, dtype=dtype, device=dev)

    draw = dict(temperature=per_sample(temperature), top_k=per_sample(top_k, torch.int32),
                top_p=per_sample(top_p), min_p=per_sample(min_p))
    tokens = torch.empty(max_new, n_samples, dtype=torch.int64, device=dev)
    logprobs = torch.empty(max_new, n_samples, dtype=torch.float32, device=dev)
    together = dict(page_table=cache.table, kv_lens=cache.lens, prefix_pages=cache.prefix_pages,
                    prefix_len=length)
    for t in range(max_new):
        tokens[t], logprobs[t] = sample_tokens(logits, u[t], return_logprob=True, **draw)
        if t + 1 == max_new:
            break
        slots, positions = cache.own_slots(1), cache.lens + length
        cache.lens += 1
        # a sample that has ended goes on with token 0 in the batch; what it draws is dropped below
        h = _step(model, tokens[t][:, None].clamp(min=0), cache, slots, positions, together)
        logits = model.lm_head(model.final_norm(h[:, -1]))
    ended = (tokens < 0).cumsum(0) > 0
    return tokens.masked_fill_(ended, -1).t(), logprobs.masked_fill_(ended, float("nan")).t()
