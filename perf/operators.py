"""What the serving operators are measured on.

Three operators serve a decoder that continues one prompt with many samples at once: ``append_kv`` (rotate
the new queries and keys, write the new keys and values into pages), ``attend_paged`` (attention over a prefix
that the whole batch shares and over each sequence's own pages) and ``sample_tokens`` (the next token of each
row from given random numbers). ``run`` computes them in elementary torch operations in 32 bits, or, where
``own`` is set, by the framework's calls. The default decoder of this repository has 16 heads of 128 and a
vocabulary of 32000; its sequences have 2048 to 4096 tokens. The other sizes are generic.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def _append(tokens, q_heads, kv_heads, head_dim, rot, page, pad, prefill, dtype):
    return {"op": "append", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "rot": rot, "page": page, "pad": pad, "prefill": prefill, "dtype": dtype}


def _attend(batch, q_len, prefix, own_max, q_heads, kv_heads, head_dim, page, dtype):
    return {"op": "attend", "batch": batch, "q_len": q_len, "prefix": prefix, "own_max": own_max,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype}


def _sample(batch, vocab, dtype, params, masked):
    return {"op": "sample", "batch": batch, "vocab": vocab, "dtype": dtype, "params": params, "masked": masked}


def listed():
    return [
        # one sequence decodes one token: nothing but latency
        {"name": "append_decode_1", **_append(1, 16, 16, 128, 128, 16, 0, False, "bf16")},
        # a batch padded to the size that a captured graph was made for, shared key heads, half of each head rotated
        {"name": "append_decode_64_padded", **_append(64, 32, 8, 64, 32, 32, 3, False, "f16")},
        # a long prompt enters the cache
        {"name": "append_prefill_8192", **_append(8192, 16, 16, 128, 128, 64, 0, True, "bf16")},
        # one sequence decodes at a moderate length, no shared prefix
        {"name": "attend_decode_1", **_attend(1, 1, 0, 517, 16, 16, 128, 16, "bf16")},
        # eight samples of one prompt, early in their own text
        {"name": "attend_samples_8", **_attend(8, 1, 2048, 200, 16, 16, 128, 16, "bf16")},
        # four long sequences with nothing in common
        {"name": "attend_long_4", **_attend(4, 1, 0, 65536, 32, 8, 128, 64, "bf16")},
        # drafts of five tokens are verified for 24 samples; group of three, odd lengths
        {"name": "attend_verify_24", **_attend(24, 5, 1999, 333, 24, 8, 64, 32, "f16")},
        # a prompt of the decoder's longest length is read
        {"name": "attend_prefill_4096", **_attend(1, 4096, 0, 4096, 16, 16, 128, 64, "bf16")},
        # many samples of one long document
        {"name": "attend_samples_128", **_attend(128, 1, 16384, 512, 32, 8, 128, 64, "bf16")},
        # the next token of one sequence
        {"name": "sample_1", **_sample(1, 32000, "f32", "nucleus", 0.0)},
        # a batch whose users set different things; 16-bit logits tie; most tokens barred by a grammar
        {"name": "sample_64_mixed", **_sample(64, 32000, "bf16", "mixed", 0.7)},
        # a large batch over a large, odd vocabulary
        {"name": "sample_256_mixed", **_sample(256, 131071, "f32", "mixed", 0.0)},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    q_heads, kv_heads = rng.choice([(16, 16), (32, 8), (24, 8), (8, 1), (12, 4), (10, 2)])
    head_dim, page = rng.choice([64, 80, 96, 128, 128]), rng.choice([8, 16, 24, 32, 64, 128])
    if op == "append":
        tokens = _log(rng, 1, 8192)
        rot = rng.choice([head_dim, head_dim, head_dim // 2])
        pad = rng.choice([0, 0, min(3, tokens - 1)])
        return _append(tokens, q_heads, kv_heads, head_dim, rot, page, pad, rng.random() < 0.5,
                       rng.choice(["bf16", "f16", "f32"]))
    if op == "sample":
        return _sample(_log(rng, 1, 256), _log(rng, 1000, 131071), rng.choice(["f32", "bf16", "f16"]),
                       rng.choice(["mixed", "nucleus", "temperature"]), rng.choice([0.0, 0.0, 0.7, 0.99]))
    kind = rng.choice(["samples", "samples", "alone", "verify", "prefill"])
    if kind == "prefill":
        n = _log(rng, 64, 4096)
        batch = max(1, min(4, 4096 // n))
        return _attend(batch, n, rng.choice([0, _log(rng, 1, 1024)]) if n <= 2048 else 0, n,
                       min(q_heads, 16), min(kv_heads, 4) if q_heads > 16 else kv_heads, head_dim, page, dtype)
    batch = _log(rng, 1, 128)
    q_len = rng.randint(2, 8) if kind == "verify" else 1
    prefix = 0 if kind == "alone" else _log(rng, 1, 16384)
    most = min(65536, 4 * 65536 * 8 // (batch * kv_heads)) if kind == "alone" else 1024
    own_max = _log(rng, q_len, most)
    if q_len > 1:
        prefix = min(prefix, 2048)
    return _attend(batch, q_len, prefix, own_max, q_heads, kv_heads, head_dim, page, dtype)


def _own_lens(case):
    """The sequences' own lengths: spread evenly from q_len to own_max, in a scattered order."""
    b, q, most = case["batch"], case["q_len"], case["own_max"]
    if b == 1:
        return [most]
    return [q + (most - q) * ((i * 37 + b - 1) % b) // (b - 1) for i in range(b)]


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        t, d = case["tokens"], case["head_dim"]
        live = t - case["pad"]
        rows = t * case["q_heads"] + live * 2 * case["kv_heads"]
        turned = t * case["q_heads"] + live * case["kv_heads"]
        return {"bytes": 2 * rows * d * size + live * case["rot"] * 4 + 12 * t, "flops": 3 * turned * case["rot"]}
    if case["op"] == "attend":
        lens, q, p = _own_lens(case), case["q_len"], case["prefix"]
        keys = p + sum(lens)
        rows = case["batch"] * q * case["q_heads"]
        pairs = case["batch"] * q * p + sum(sum(range(n - q + 1, n + 1)) for n in lens)
        return {"bytes": (2 * keys * case["kv_heads"] + 2 * rows) * case["head_dim"] * size + 4 * rows,
                "flops": 4 * pairs * case["q_heads"] * case["head_dim"]}
    n = case["batch"] * case["vocab"]
    return {"bytes": n * size + 32 * case["batch"], "flops": 4 * n}


# ---------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------


def _angles(length, rot, device):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    ang = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    def shuffled(n):
        return torch.randperm(n, generator=gen, device=dev)

    if case["op"] == "append":
        t, hq, hk, d, page = (case[x] for x in ("tokens", "q_heads", "kv_heads", "head_dim", "page"))
        qkv = normal(t, (hq + 2 * hk) * d)  # one projection's output: the three are strided views of it
        q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=1)
        length = 16384
        cos, sin = _angles(length, case["rot"], dev)
        if case["prefill"]:  # consecutive tokens fill page after page
            pages = (t + page - 1) // page
            table = shuffled(pages + pages // 4 + 1)
            at = torch.arange(t, device=dev)
            slots = table[at // page] * page + at % page
            positions = at + int(torch.randint(0, length - t, (1,), generator=gen, device=dev))
        else:  # every token is another sequence's: a page and an offset of its own
            table = shuffled(t + t // 4 + 1)
            slots = table[:t] * page + torch.randint(0, page, (t,), generator=gen, device=dev)
            positions = torch.randint(0, length, (t,), generator=gen, device=dev)
        slots[t - case["pad"]:] = -1
        cache = [torch.zeros(table.numel(), hk, page, d, device=dev, dtype=dtype) for _ in range(2)]
        return {"case": case, "q": q.view(t, hq, d), "k": k.view(t, hk, d), "v": v.view(t, hk, d),
                "k_cache": cache[0], "v_cache": cache[1], "slots": slots, "positions": positions.int(),
                "cos": cos, "sin": sin}

    if case["op"] == "attend":
        b, n, hq, hk, d, page = (case[x] for x in ("batch", "q_len", "q_heads", "kv_heads", "head_dim", "page"))
        lens = torch.tensor(_own_lens(case), device=dev)
        need, ahead = (lens + page - 1) // page, (case["prefix"] + page - 1) // page
        total = ahead + int(need.sum())
        pages = shuffled(total).int()
        width = int(need.max())
        first = need.cumsum(0) - need
        at = torch.arange(width, device=dev)
        table = torch.where(at < need[:, None], pages[(ahead + first[:, None] + at).clamp(max=total - 1)], -1)
        return {"case": case, "q": normal(b, n, hq, d) * 1.5, "k_cache": normal(total, hk, page, d),
                "v_cache": normal(total, hk, page, d), "page_table": table.int(), "kv_lens": lens.int(),
                "prefix_pages": pages[:ahead].contiguous(), "prefix_len": case["prefix"]}

    b, v = case["batch"], case["vocab"]
    # a few tokens stand out and the rest trail off, as a trained model's logits do
    x = torch.randn(b, v, generator=gen, device=dev)
    x = 2.2 * x + 5.0 * torch.relu(x - 3.0)
    if case["masked"]:
        barred = torch.rand(b, v, generator=gen, device=dev) < case["masked"]
        barred[:, v // 2] = False  # a grammar leaves something
        x = x.masked_fill(barred, -math.inf)

    def pick(values):
        values = torch.tensor(values, device=dev)
        return values[torch.randint(0, len(values), (b,), generator=gen, device=dev)]

    kinds = {
        "mixed": ([0.0, 0.6, 0.8, 1.0, 1.3], [0, 0, 20, 50, 400], [1.0, 0.8, 0.9, 0.95], [0.0, 0.0, 0.02, 0.1]),
        "nucleus": ([0.7, 0.8, 1.0], [0], [0.9, 0.95], [0.0]),
        "temperature": ([0.8, 1.0, 1.1], [0], [1.0], [0.0]),
    }[case["params"]]
    return {"case": case, "logits": x.to(dtype), "u": torch.rand(b, generator=gen, device=dev),
            "temperature": pick(kinds[0]), "top_k": pick(kinds[1]).int(), "top_p": pick(kinds[2]),
            "min_p": pick(kinds[3])}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _turn(x, cos, sin):
    """Rotate the two halves of the first 2 * cos.shape[-1] columns against each other, in 32 bits."""
    h = cos.shape[-1]
    x, c, s = x.float(), cos[:, None], sin[:, None]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], dim=-1)


def _plain_append(s):
    cos, sin = s["cos"][s["positions"].long()], s["sin"][s["positions"].long()]
    live = s["slots"] >= 0
    page = s["k_cache"].shape[2]
    at = s["slots"][live]
    s["k_cache"][at // page, :, at % page] = _turn(s["k"], cos, sin)[live].to(s["k_cache"].dtype)
    s["v_cache"][at // page, :, at % page] = s["v"][live]
    return {"q": _turn(s["q"], cos, sin).to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    q, table, p = s["q"].float(), s["page_table"], s["prefix_len"]
    b, n, hq, d = q.shape
    hk = s["k_cache"].shape[1]
    g = hq // hk
    q = q.view(b, n, hk, g, d) / math.sqrt(d)

    def ahead(cache):  # [hk, prefix, d]
        return cache[s["prefix_pages"].long()].float().transpose(0, 1).reshape(hk, -1, d)[:, :p]

    def mine(cache):  # [b, hk, keys, d]
        return cache[table.clamp(min=0).long()].float().transpose(1, 2).reshape(b, hk, -1, d)

    shared = q.permute(2, 0, 1, 3, 4).reshape(hk, b * n * g, d)
    alone = q.permute(0, 2, 1, 3, 4).reshape(b, hk, n * g, d)
    ls = (shared @ ahead(s["k_cache"]).transpose(1, 2)).view(hk, b, n * g, p).transpose(0, 1)
    la = alone @ mine(s["k_cache"]).transpose(2, 3)
    at = torch.arange(la.shape[-1], device=q.device)
    until = s["kv_lens"].long()[:, None] - n + 1 + torch.arange(n, device=q.device)
    seen = at < until.repeat_interleave(g, dim=1)[:, None, :, None]
    la = la.masked_fill(~seen, -math.inf)
    logits = torch.cat([ls, la], dim=-1)
    top = logits.amax(-1, keepdim=True).clamp(min=-1e30)
    e = (logits - top).exp()
    total = e.sum(-1, keepdim=True)
    out = e[..., p:] @ mine(s["v_cache"])
    out = out + (e[..., :p].transpose(0, 1).reshape(hk, b * n * g, p) @ ahead(s["v_cache"])).view(
        hk, b, n * g, d).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (top + total.log()).squeeze(-1)
    out = out.view(b, hk, n, g, d).transpose(1, 2).reshape(b, n, hq, d)
    return {"out": out.to(s["q"].dtype), "lse": lse.view(b, hk, n, g).transpose(1, 2).reshape(b, n, hq)}


def _plain_sample(s):
    # Weights are whole numbers, exp(x - max) in units of 2^-40, so sums have no rounding and no order.
    t = s["temperature"]
    greedy = (t <= 0)[:, None]
    x = s["logits"].float() * torch.where(t > 0, 1.0 / t, 1.0)[:, None]
    e = (x - x.amax(-1, keepdim=True)).exp()
    w = (e * 2.0**40).round().long()
    # the order of the filters: highest first, ties to the lowest index
    _, order = x.sort(dim=-1, descending=True, stable=True)
    ranked = w.gather(1, order)
    rank = torch.arange(x.shape[1], device=x.device)
    k = torch.where(s["top_k"] > 0, s["top_k"], x.shape[1])[:, None]
    k = torch.where(greedy, 1, k)
    ranked = ranked.masked_fill(rank >= k, 0)
    before = ranked.cumsum(-1) - ranked
    p = s["top_p"].double()[:, None]
    goal = (p * ranked.sum(-1, keepdim=True).double()).ceil().long()
    kept = (rank == 0) | (before < goal) | (p >= 1)
    kept &= e.gather(1, order) >= s["min_p"].clamp(max=1.0)[:, None]
    ranked = ranked * kept
    w = torch.zeros_like(w).scatter(1, order, ranked)
    total = w.sum(-1, keepdim=True)
    aim = (s["u"].double()[:, None] * total.double()).floor().long().minimum(total - 1)
    token = (w.cumsum(-1) <= aim).sum(-1)
    mass = w.gather(1, token[:, None]).float() / total.float()
    return {"token": token, "logprob": mass.log().squeeze(1)}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[op](state)
    package = str(Path(__file__).resolve().parent.parent / "blackwell-switchyard_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import switchyard

    s = state
    if op == "append":
        q = switchyard.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], q=s["q"],
                                 positions=s["positions"], cos=s["cos"], sin=s["sin"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "attend":
        out, lse = switchyard.attend_paged(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_lens"],
                                           prefix_pages=s["prefix_pages"], prefix_len=s["prefix_len"],
                                           return_lse=True)
        return {"out": out, "lse": lse}
    token, logprob = switchyard.sample_tokens(s["logits"], s["u"], temperature=s["temperature"],
                                              top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                              return_logprob=True)
    return {"token": token, "logprob": logprob}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    dev = s[{"append": "q", "attend": "q", "sample": "logits"}[case["op"]]].device
    if case["op"] == "append":
        h, page = case["rot"] // 2, case["page"]
        z = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]

        def turned(x):
            x = x.double()
            y = torch.complex(x[..., :h], x[..., h:2 * h]) * z
            return torch.cat([y.real, y.imag, x[..., 2 * h:]], dim=-1)

        n = case["tokens"] - case["pad"]
        flat = {}
        for name, new in (("k_cache", turned(s["k"])), ("v_cache", s["v"].double())):
            rows = s[name].double().transpose(1, 2).reshape(-1, case["kv_heads"], case["head_dim"])
            rows = rows.index_copy(0, s["slots"][:n], new[:n])
            flat[name] = rows.view(-1, page, case["kv_heads"], case["head_dim"]).transpose(1, 2).contiguous()
        return {"q": turned(s["q"]), **flat}

    if case["op"] == "attend":
        b, n, hq, hk, d, page = (case[x] for x in ("batch", "q_len", "q_heads", "kv_heads", "head_dim", "page"))
        out = torch.zeros(b, n, hq, d, dtype=torch.float64, device=dev)
        lse = torch.zeros(b, n, hq, dtype=torch.float64, device=dev)
        lens = _own_lens(case)

        def rows(cache, pages, count):
            got = cache[pages.long()].double()
            return torch.cat(list(got.unbind(0)), dim=1)[:, :count] if count else got.new_zeros(hk, 0, d)

        lead = [rows(s[c], s["prefix_pages"], case["prefix"]) for c in ("k_cache", "v_cache")]
        for i in range(b):
            mine = s["page_table"][i, : (lens[i] + page - 1) // page]
            k, v = (torch.cat([lead[j], rows(s[c], mine, lens[i])], dim=1)
                    for j, c in enumerate(("k_cache", "v_cache")))
            last = case["prefix"] + lens[i] - n + torch.arange(n, device=dev)
            bar = torch.arange(k.shape[1], device=dev)[None] > last[:, None]
            for j in range(hq):
                a = s["q"][i, :, j].double() @ k[j * hk // hq].T * d**-0.5
                a.masked_fill_(bar, -math.inf)
                lse[i, :, j] = a.logsumexp(1)
                out[i, :, j] = a.softmax(1) @ v[j * hk // hq]
        return {"out": out, "lse": lse}

    logprob = torch.zeros(case["batch"], dtype=torch.float64, device=dev)
    for i in range(case["batch"]):
        t = float(s["temperature"][i])
        # the scaled logits are rounded to 32 bits by definition: their order decides the filters
        x = (s["logits"][i].float() * (1.0 / s["temperature"][i] if t > 0 else 1.0)).double()
        order = x.sort(descending=True, stable=True).indices
        w = (x[order] - x.max()).exp()
        k = 1 if t <= 0 else int(s["top_k"][i]) or len(w)
        w[k:] = 0
        p = float(s["top_p"][i])
        if p < 1:
            cut = int((w.cumsum(0) < p * w.sum()).sum()) + 1
            w[cut:] = 0
        w[w < float(s["min_p"][i])] = 0
        w = torch.zeros_like(w).index_copy(0, order, w)
        token = int((w.cumsum(0) <= float(s["u"][i]) * w.sum()).sum())
        logprob[i] = (w[min(token, len(w) - 1)] / w.sum()).log()
    return {"token": None, "logprob": logprob}
