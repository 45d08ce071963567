"""append_kv, attend_paged and sample_tokens against plain implementations in 64 bits.

Tolerances follow from the arithmetic, u being the unit roundoff of the 16-bit type (2^-8 or 2^-11): an appended element is rounded once from fp32; an attention output is a sum of weights rounded to
16 bits times values, divided in fp32 and rounded once; tokens are whole numbers and have to be equal.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}  # fp16's subnormal half step
T16 = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def sy():
    import switchyard

    return switchyard


@pytest.fixture(autouse=True)
def clear_error_word():
    from switchyard import _native

    _native.device_error()
    yield
    assert _native.device_error() == 0, "a kernel left an error in the device error word"


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def angles(length, half):
    inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    a = torch.arange(length, dtype=torch.float64)[:, None] * inv
    return a.cos().float().cuda(), a.sin().float().cuda()


# ---------------------------------------------------------------------------
# append_kv
# ---------------------------------------------------------------------------


def turned64(x, cos, sin):
    h = cos.shape[-1]
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


def near_turned(got, x, cos, sin):
    """One rounding of an fp32 result whose three operations err by at most 3 * 2^-24 of |x1| + |x2|."""
    want = turned64(x, cos, sin)
    h = cos.shape[-1]
    a, b = x.double()[..., :h].abs(), x.double()[..., h:2 * h].abs()
    size = torch.cat([a + b, a + b, torch.zeros_like(x.double()[..., 2 * h:])], -1)
    bound = UNIT[x.dtype] * want.abs() + 3 * 2.0**-24 * size * (1 + UNIT[x.dtype]) + TINY[x.dtype]
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hk,d,half,page", [
    (1, 16, 16, 128, 64, 16), (5, 32, 8, 64, 32, 8), (3, 3, 1, 80, 20, 24), (2, 2, 2, 34, 5, 3),
    (7, 4, 2, 7, 3, 1), (130, 8, 8, 96, 48, 32), (2, 1, 1, 2, 1, 64), (3, 2, 1, 512, 256, 16),
    (2, 70, 3, 1024, 512, 2),
])
def test_append(sy, dtype, tokens, hq, hk, d, half, page):
    g = gen(tokens * 7 + d)
    qkv = torch.randn(tokens, (hq + 2 * hk) * d, generator=g, device="cuda").to(dtype)
    q, k, v = qkv.split([hq * d, hk * d, hk * d], 1)
    q, k, v = q.view(tokens, hq, d), k.view(tokens, hk, d), v.view(tokens, hk, d)
    pages = (tokens + page - 1) // page + 2
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    cos, sin = angles(300, half)
    pos = torch.randint(0, 300, (tokens,), generator=g, device="cuda").int()
    kc = torch.full((pages, hk, page, d), math.nan, device="cuda", dtype=dtype)
    vc = torch.full_like(kc, math.nan)
    qr = sy.append_kv(k, v, kc, vc, slots, q=q, positions=pos, cos=cos, sin=sin)
    c, s = cos[pos.long()], sin[pos.long()]
    near_turned(qr, q, c, s)
    near_turned(kc[slots // page, :, slots % page], k, c, s)
    assert torch.equal(vc[slots // page, :, slots % page], v)
    rest = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    rest[slots // page, slots % page] = False
    assert kc.transpose(1, 2)[rest].isnan().all() and vc.transpose(1, 2)[rest].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_padding_views_and_no_rotation(sy, dtype):
    g = gen(3)
    layers = torch.zeros(2, 2, 6, 3, 8, 40, device="cuda", dtype=dtype)  # [layer, k or v, page, head, row, d]
    k = torch.randn(5, 3, 40, generator=g, device="cuda").to(dtype)
    v = torch.randn(3, 5, 40, generator=g, device="cuda").to(dtype).transpose(0, 1)
    slots = torch.tensor([7, -1, 0, 47, -1], device="cuda")
    assert sy.append_kv(k, v, layers[1, 0], layers[1, 1], slots) is None
    want = torch.zeros_like(layers)
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            want[1, 0, s // 8, :, s % 8], want[1, 1, s // 8, :, s % 8] = k[t], v[t]
    assert torch.equal(layers, want)
    # a slab of a wider tensor whose rows start off any 16-byte boundary
    wide = torch.zeros(6, 3, 8, 43, device="cuda", dtype=dtype)
    sy.append_kv(k, v, wide[..., 3:], wide.clone()[..., 3:], slots)
    assert torch.equal(wide[..., 3:], want[1, 0]) and not wide[..., :3].any()


def test_append_empty_and_q_of_padding(sy):
    kc = torch.zeros(1, 2, 8, 16, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(0, 2, 16, device="cuda").bfloat16()
    none = torch.zeros(0, dtype=torch.long, device="cuda")
    assert sy.append_kv(x, x, kc, kc.clone(), none, q=x).shape == (0, 2, 16)
    cos, sin = angles(9, 8)
    x = torch.randn(1, 2, 16, device="cuda").bfloat16()
    pos = torch.tensor([8], device="cuda", dtype=torch.int32)
    got = sy.append_kv(x, x, kc, kc.clone(), torch.tensor([-5], device="cuda"), q=x, positions=pos, cos=cos, sin=sin)
    near_turned(got, x, cos[8:], sin[8:])
    assert not kc.any()


def test_append_indices_outside_are_not_followed(sy):
    from switchyard import _native

    kc, vc = (torch.zeros(2, 1, 8, 16, device="cuda") for _ in range(2))
    cos, sin = angles(4, 8)
    x = torch.randn(3, 1, 16, device="cuda")
    pos = torch.tensor([0, 4, -1], device="cuda", dtype=torch.int32)
    sy.append_kv(x, x, kc, vc, torch.tensor([16, 1, 2], device="cuda"), q=x, positions=pos, cos=cos, sin=sin)
    assert _native.device_error() == 4
    assert not kc.any() and not vc.any()


# ---------------------------------------------------------------------------
# attend_paged
# ---------------------------------------------------------------------------


def paged(seed, lens, n, hq, hk, d, page, prefix, dtype, junk=math.nan, q_scale=1.0):
    """Inputs, and the contiguous keys and values of the prefix and of every sequence; what no key uses is junk."""
    g = gen(seed)
    b = len(lens)
    need = [(x + page - 1) // page for x in lens]
    ahead = (prefix + page - 1) // page
    total = ahead + sum(need) + 1
    order = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.full((b, max(need + [0]) + 1), -7, device="cuda", dtype=torch.int32)
    caches, lead, own = [], [], []
    for _ in range(2):
        cache = torch.full((total, hk, page, d), junk, device="cuda", dtype=dtype)
        x = torch.randn(hk, prefix, d, generator=g, device="cuda").to(dtype)
        lead.append(x)
        for i in range(ahead):
            part = x[:, i * page:(i + 1) * page]
            cache[int(order[i]), :, : part.shape[1]] = part
        at, mine = ahead, []
        for s, m in enumerate(lens):
            x = torch.randn(hk, m, d, generator=g, device="cuda").to(dtype)
            mine.append(x)
            for i in range(need[s]):
                part = x[:, i * page:(i + 1) * page]
                cache[int(order[at + i]), :, : part.shape[1]] = part
                table[s, i] = order[at + i]
            at += need[s]
        caches.append(cache)
        own.append(mine)
    q = (q_scale * torch.randn(b, n, hq, d, generator=g, device="cuda")).to(dtype)
    kw = dict(prefix_pages=order[:ahead].contiguous(), prefix_len=prefix)
    args = (q, caches[0], caches[1], table, torch.tensor(lens, device="cuda", dtype=torch.int32))
    return args, kw, lead, own


def check_attend(out, lse, args, kw, lead, own, scale=None):
    q, dtype = args[0], args[0].dtype
    b, n, hq, d = q.shape
    g = hq // lead[0].shape[0]
    scale = d**-0.5 if scale is None else scale
    u = UNIT[dtype]
    for s in range(b):
        k = torch.cat([lead[0], own[0][s]], 1).double().repeat_interleave(g, 0)
        v = torch.cat([lead[1], own[1][s]], 1).double().repeat_interleave(g, 0)
        m = own[0][s].shape[1]
        a = torch.einsum("nhd,hkd->hnk", q[s].double(), k) * scale
        size = torch.einsum("nhd,hkd->hnk", q[s].double().abs(), k.abs()) * abs(scale)
        # the whole prefix, and of the sequence's own keys those up to the query's own place
        last = kw["prefix_len"] + (m - n + torch.arange(n, device="cuda")).clamp(min=-1)
        bar = torch.arange(k.shape[1], device="cuda") > last[:, None]
        a = a.masked_fill(bar, -math.inf)
        want_lse = a.logsumexp(-1) if k.shape[1] else torch.full((hq, n), -math.inf, device="cuda").double()
        p = (a - want_lse[..., None]).exp().nan_to_num(0.0)
        want = torch.einsum("hnk,hkd->nhd", p, v)
        size_v = torch.einsum("hnk,hkd->nhd", p, v.abs())
        # logits: fp32 sums of d exact products (2^-23 d of their sizes at most, far less as the sums go pairwise)
        # and the exponential's argument and value (2^-22 of the logit's size, 2^-21)
        ds = 2.0**-20 * (1 + size.masked_fill(bar, 0).amax(-1)) if k.shape[1] else torch.zeros(hq, n, device="cuda").double()
        # weights rounded to 16 bits, the result once more; fp16 weights below 2^-20 of the highest have fewer bits
        small = 2.0**-31 * k.shape[1] * float(v.abs().amax()) if dtype == torch.float16 and k.shape[1] else 0.0
        bound = (1.01 * u + 2 * ds.T[..., None]) * size_v + 1.01 * u * want.abs() + small + TINY[dtype]
        err = (out[s].double() - want).abs()
        assert (err <= bound).all(), f"sequence {s}: {float((err / bound.clamp(min=1e-30)).max())} of the bound"
        if lse is not None:
            dl = (lse[s].double() - want_lse.T).abs().nan_to_num(0.0)
            assert torch.equal(lse[s].isinf(), want_lse.T.isinf())
            assert (dl <= ds.T + 2.0**-23 * want_lse.T.abs().nan_to_num(0.0, 0.0, 0.0)).all(), float(dl.max())


SHAPES = [
    # lens, n, hq, hk, d, page, prefix
    ([1], 1, 1, 1, 64, 8, 0),
    ([517], 1, 16, 16, 128, 16, 0),
    ([128], 1, 4, 1, 128, 128, 0),
    ([129, 0, 1, 127, 128, 255, 256, 257], 1, 8, 2, 128, 24, 0),
    ([3, 1, 40, 17, 200], 1, 16, 16, 128, 16, 130),
    ([3, 1, 40, 17, 200], 1, 6, 2, 80, 8, 1),
    ([0, 0, 0], 1, 4, 4, 64, 16, 129),
    ([5, 9, 333], 5, 24, 8, 64, 32, 199),
    ([5, 9, 333], 5, 24, 8, 64, 32, 0),
    ([2, 0, 4], 3, 8, 1, 96, 8, 0),  # queries ahead of every key
    ([2, 0, 4], 3, 8, 1, 96, 8, 5),
    ([300], 300, 4, 4, 128, 64, 0),
    ([257], 257, 6, 2, 128, 32, 0),
    ([130], 129, 8, 1, 64, 8, 100),
    ([64, 64], 64, 8, 8, 8, 8, 33),
    ([7] * 70, 1, 8, 8, 128, 16, 300),
    ([11] * 33, 1, 32, 8, 128, 16, 257),
    ([140, 30], 20, 20, 1, 40, 40, 77),
    ([1000, 1], 1, 128, 1, 128, 64, 640),
    ([1000, 1], 1, 130, 1, 128, 64, 640),
    ([4097], 1, 8, 8, 128, 16, 4095),
]


@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attend(sy, dtype, case):
    lens, n, hq, hk, d, page, prefix = SHAPES[case]
    args, kw, lead, own = paged(case, lens, n, hq, hk, d, page, prefix, dtype)
    out, lse = sy.attend_paged(*args, **kw, return_lse=True)
    check_attend(out, lse, args, kw, lead, own)
    assert torch.equal(sy.attend_paged(*args, **kw), out), "the same call gives the same bits"


@pytest.mark.parametrize("dtype", T16)
def test_attend_sharp_and_growing_logits(sy, dtype):
    """Logits spread over hundreds, growing along the keys: the running maximum moves in most tiles."""
    args, kw, lead, own = paged(1, [700, 300], 1, 8, 2, 64, 16, 300, dtype)
    q, kc, vc, table, lens = args
    for x in (lead[0], *own[0]):
        ramp = torch.linspace(0.05, 4, x.shape[1], device="cuda")[None, :, None]
        x.copy_((x.float().abs() * ramp).to(dtype))
    for i, pg in enumerate(kw["prefix_pages"].tolist()):
        part = lead[0][:, i * 16:(i + 1) * 16]
        kc[pg, :, : part.shape[1]] = part
    for s in range(2):
        for i in range((int(lens[s]) + 15) // 16):
            part = own[0][s][:, i * 16:(i + 1) * 16]
            kc[int(table[s, i]), :, : part.shape[1]] = part
    q.copy_(q.abs())
    out, lse = sy.attend_paged(*args, **kw, scale=0.25, return_lse=True)
    check_attend(out, lse, args, kw, lead, own, scale=0.25)


def test_attend_equal_logits_and_large_negative(sy):
    """All logits equal (zero queries), and all of them at -1e4: the softmax is uniform in both."""
    for fill in (0.0, -100.0):
        args, kw, lead, own = paged(2, [129, 5], 1, 4, 4, 64, 8, 131, torch.bfloat16)
        args[0].fill_(1.0)
        args[1].fill_(fill)
        for x in (lead[0], *own[0]):
            x.fill_(fill)
        out, lse = sy.attend_paged(*args, **kw, scale=1.5625, return_lse=True)
        check_attend(out, lse, args, kw, lead, own, scale=1.5625)


def test_attend_views(sy):
    """q as a view of one projection, the caches as slices of one tensor over layers, the table as a column slice."""
    args, kw, lead, own = paged(4, [40, 77], 2, 4, 2, 64, 16, 50, torch.bfloat16)
    q, kc, vc, table, lens = args
    both = torch.full((3, 2, *kc.shape), math.nan, device="cuda", dtype=kc.dtype)
    both[1, 0], both[1, 1] = kc, vc
    wide = torch.full((2, 2, 4 * 64 + 72), math.nan, device="cuda", dtype=q.dtype)
    wide[..., 8:8 + 256] = q.view(2, 2, 256)
    qv = wide[..., 8:8 + 256].view(2, 2, 4, 64)
    tv = torch.cat([table, table], 1)[:, : table.shape[1]]
    want = sy.attend_paged(*args, **kw)
    assert torch.equal(sy.attend_paged(qv, both[1, 0], both[1, 1], tv, lens, **kw), want)
    # page-major rows ([pages, page_size, kv_heads, head_dim] seen through a transpose)
    rows = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc)]
    assert torch.equal(sy.attend_paged(q, *rows, table, lens, **kw), want)
    # a q whose rows are not 16-byte aligned is copied
    odd = torch.zeros(2, 2, 4, 67, device="cuda", dtype=q.dtype)
    odd[..., 1:65] = q
    assert torch.equal(sy.attend_paged(odd[..., 1:65], kc, vc, table, lens, **kw), want)


def test_attend_empty(sy):
    kc = torch.zeros(1, 2, 8, 16, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(0, 1, 2, 16, device="cuda", dtype=torch.bfloat16)
    z = torch.zeros(0, device="cuda", dtype=torch.int32)
    out, lse = sy.attend_paged(q, kc, kc, z.view(0, 1), z, return_lse=True)
    assert out.shape == (0, 1, 2, 16) and lse.shape == (0, 1, 2)
    # sequences without pages
    q = torch.zeros(2, 1, 2, 16, device="cuda", dtype=torch.bfloat16)
    z = torch.zeros(2, device="cuda", dtype=torch.int32)
    out, lse = sy.attend_paged(q, kc, kc, z.view(2, 1)[:, :0], z, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()


def test_attend_another_stream(sy):
    args, kw, lead, own = paged(5, [300, 20], 1, 8, 8, 128, 16, 200, torch.bfloat16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out, lse = sy.attend_paged(*args, **kw, return_lse=True)
    side.synchronize()
    check_attend(out, lse, args, kw, lead, own)


def test_attend_graph_replays_with_new_lengths(sy):
    args, kw, lead, own = paged(6, [90, 170], 1, 8, 8, 128, 16, 40, torch.bfloat16)
    q, kc, vc, table, lens = args
    sy.attend_paged(*args, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = sy.attend_paged(*args, **kw, return_lse=True)
    for new in ([90, 170], [1, 133], [64, 0]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        cut = [[x[:, :m] for x, m in zip(side, new)] for side in own]
        check_attend(out, lse, args, kw, lead, cut)


def test_attend_indices_outside_are_not_followed(sy):
    from switchyard import _native

    args, kw, lead, own = paged(7, [40, 20], 1, 4, 4, 64, 16, 0, torch.bfloat16, junk=0.0)
    q, kc, vc, table, lens = args
    table[0, 1] = kc.shape[0]
    out = sy.attend_paged(*args, **kw)
    assert _native.device_error() == 4 and out.isfinite().all()
    table[0, 1] = -1
    out = sy.attend_paged(*args, **kw)
    assert _native.device_error() == 4 and out.isfinite().all()
    table[0, 1] = 0
    lens[1] = 16 * table.shape[1] + 1
    table[1] = 0
    out = sy.attend_paged(*args, **kw)
    assert _native.device_error() == 4 and out.isfinite().all()


def test_refusals(sy):
    args, kw, _, _ = paged(8, [20, 9], 1, 4, 2, 64, 16, 30, torch.bfloat16, junk=0.0)
    q, kc, vc, table, lens = args

    def no(error, match, *a, **k):
        with pytest.raises(error, match=match):
            sy.attend_paged(*a, **{**kw, **k})

    no(ValueError, "dtype", q.half(), kc, vc, table, lens)
    no(ValueError, "bfloat16 or float16", q.float(), kc.float(), vc.float(), table, lens)
    no(ValueError, "head_dim", q[..., :60], kc, vc, table, lens)
    no(ValueError, "multiple of 8", q[..., :60], kc[..., :60], vc[..., :60], table, lens)
    no(ValueError, "page_size", q, kc[:, :, :12], vc[:, :, :12], table, lens)
    no(ValueError, "q_heads", q[:, :, :3], kc, vc, table, lens)
    no(ValueError, "page_table", q, kc, vc, table[:1], lens)
    no(ValueError, "page_table", q, kc, vc, table.long(), lens)
    no(ValueError, "kv_lens", q, kc, vc, table, lens.long())
    no(ValueError, "prefix_pages", *args, prefix_len=33)
    no(ValueError, "prefix_pages", *args, prefix_pages=None)
    no(ValueError, "prefix_len", *args, prefix_len=-1)
    no(ValueError, "last dimension", q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, table, lens)
    for scale in (0.0, -1.0, math.nan, math.inf):
        no(ValueError, "scale", *args, scale=scale)
    no(ValueError, "CUDA", q, kc, vc, table.cpu(), lens)
    no(RuntimeError, "no backward", q.clone().requires_grad_(), kc, vc, table, lens)

    x = torch.zeros(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    slots = torch.zeros(2, device="cuda", dtype=torch.int64)
    cos, sin = angles(4, 32)
    pos = slots.int()
    for bad in (dict(k=x[:, :1]), dict(v=x[:1]), dict(k=x.half()), dict(slots=slots.int()), dict(slots=slots[:1]),
                dict(q=x[:1]), dict(q=x.float()), dict(positions=pos), dict(positions=pos, cos=cos, sin=sin.half()),
                dict(positions=pos, cos=cos, sin=sin[:3]), dict(positions=slots, cos=cos, sin=sin),
                dict(positions=pos, cos=cos.repeat(1, 2), sin=sin.repeat(1, 2))):
        with pytest.raises(ValueError):
            sy.append_kv(**{**dict(k=x, v=x, k_cache=kc, v_cache=vc, slots=slots), **bad})
    with pytest.raises(RuntimeError, match="no backward"):
        sy.append_kv(x.clone().requires_grad_(), x, kc, vc, slots)

    logits, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    for bad in (dict(u=u[:1]), dict(u=u.double()), dict(top_k=u), dict(top_p=u[:1]), dict(min_p=u.half()),
                dict(logits=logits.double()), dict(logits=logits[0])):
        with pytest.raises(ValueError):
            sy.sample_tokens(**{**dict(logits=logits, u=u), **bad})
    with pytest.raises(RuntimeError, match="no backward"):
        sy.sample_tokens(logits.clone().requires_grad_(), u)


# ---------------------------------------------------------------------------
# sample_tokens
# ---------------------------------------------------------------------------


def sample64(logits, u, temperature, top_k, top_p, min_p):
    """The definition on one row in numpy: whole-number weights, Python integers."""
    f32 = np.float32
    x = logits.astype(f32) * (f32(1) / f32(temperature) if temperature > 0 else f32(1))
    x = np.where(np.isnan(x), f32(-np.inf), x)
    top = x.max()
    if top == -np.inf:
        return -1, math.nan
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.where(x == top, f32(1), torch.from_numpy(x - top).cuda().exp().cpu().numpy())
    w = np.rint(e.astype(np.float64) * 2.0**40).astype(np.int64)
    order = np.argsort(-x, kind="stable")
    k = 1 if temperature <= 0 else (top_k if top_k > 0 else len(x))
    order = order[:k]
    total = int(w[order].sum())
    if top_p < 1:
        goal = max(1, math.ceil(float(f32(top_p)) * float(total)))
        before = np.cumsum(w[order]) - w[order]
        order = order[before < goal]
    order = order[e[order] >= min(f32(min_p), f32(1))]
    kept = np.zeros_like(w)
    kept[order] = w[order]
    total = int(kept.sum())
    aim = min(math.floor(float(f32(u)) * float(total)), total - 1)
    token = int((np.cumsum(kept) <= aim).sum())
    return token, math.log(int(kept[token]) / total)


def check_sample(sy, logits, u, temperature, top_k, top_p, min_p):
    token, logprob = sy.sample_tokens(
        logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, return_logprob=True)
    rows = logits.float().cpu().numpy()
    for r in range(len(rows)):
        want, lp = sample64(rows[r], float(u[r]), float(temperature[r]), int(top_k[r]), float(top_p[r]),
                            float(min_p[r]))
        assert int(token[r]) == want, f"row {r}"
        got = float(logprob[r])
        # w and the total rounded to fp32, their quotient and logarithm: 4 * 2^-24 and 2 ulp of the result
        assert math.isnan(got) if math.isnan(lp) else abs(got - lp) <= 2.0**-21 + 2.0**-22 * abs(lp), f"row {r}"


def params(rows, seed):
    g = gen(seed)

    def pick(values):
        t = torch.tensor(values, device="cuda")
        return t[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]

    return (torch.rand(rows, generator=g, device="cuda"), pick([0.0, 0.3, 0.7, 1.0, 1.7, -1.0]),
            pick([0, -1, 1, 2, 5, 50, 10**6]).int(), pick([1.0, 0.0, 0.05, 0.5, 0.9, 0.99, 1.5]),
            pick([0.0, 0.0, 0.01, 0.3, 1.0, 2.0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 257, 1000, 1025, 4096, 32000, 50257, 131071, 262144])
def test_sample(sy, dtype, vocab):
    rows = 24
    g = gen(vocab)
    x = (3 * torch.randn(rows, vocab, generator=g, device="cuda")).to(dtype)
    check_sample(sy, x, *params(rows, vocab + 1))


@pytest.mark.parametrize("vocab", [7, 1024, 5000, 40000])
def test_sample_ties_masks_and_extremes(sy, vocab):
    g = gen(vocab)
    rows = []
    base = torch.randn(vocab, generator=g, device="cuda")
    rows.append(torch.zeros(vocab, device="cuda"))  # all equal
    rows.append(base.round())  # many ties
    rows.append(torch.where(base > 1, base, -math.inf))
    rows.append(torch.full((vocab,), -math.inf, device="cuda"))
    rows.append(torch.full((vocab,), torch.finfo(torch.float32).min, device="cuda"))
    rows.append(torch.where(base > 0, base, torch.finfo(torch.float32).min))
    rows.append(torch.where(base > 0.5, math.nan, base))
    rows.append(torch.full((vocab,), math.nan, device="cuda"))
    one = torch.full((vocab,), -math.inf, device="cuda")
    one[vocab - 1] = -3.0
    rows.append(one)
    inf = base.clone()
    inf[vocab // 2], inf[vocab - 1] = math.inf, math.inf
    rows.append(inf)
    rows.append(base * 1e30)
    rows.append(base * 1e-30)
    rows.append(torch.where(base > 0, 0.0, -0.0))
    rows.append(torch.arange(vocab, device="cuda") * -0.01)
    x = torch.stack(rows)
    for seed in range(4):
        check_sample(sy, x, *params(len(rows), seed))
    ones = torch.ones(len(rows), device="cuda")
    zero = torch.zeros_like(ones)
    for u in (0.0, 1.0 - 2.0**-24):
        check_sample(sy, x, u * ones, ones, zero.int(), ones, zero)
        check_sample(sy, x, u * ones, ones, 3 + zero.int(), 0.7 * ones, zero)


def test_sample_defaults_scalars_and_views(sy):
    g = gen(11)
    x = torch.randn(6, 700, generator=g, device="cuda")
    u = torch.rand(6, generator=g, device="cuda")
    one, zero = torch.ones(6, device="cuda"), torch.zeros(6, device="cuda")
    want = sy.sample_tokens(x, u, one, zero.int(), one, zero)
    assert want.dtype == torch.int64 and torch.equal(sy.sample_tokens(x, u), want)
    wide = torch.full((6, 711), math.nan, device="cuda")
    wide[:, 5:705] = x
    assert torch.equal(sy.sample_tokens(wide[:, 5:705], u), want)
    assert torch.equal(sy.sample_tokens(x.t().contiguous().t(), u), want)
    assert torch.equal(sy.sample_tokens(x[:1].expand(6, 700), u), sy.sample_tokens(x[:1].repeat(6, 1), u))
    assert torch.equal(sy.sample_tokens(x, u, temperature=0.0), x.argmax(1))
    assert torch.equal(sy.sample_tokens(x, u, 0.7, 40, 0.9, 0.05),
                       sy.sample_tokens(x, u, 0.7 * one, 40 + zero.int(), 0.9 * one, 0.05 * one))
    assert sy.sample_tokens(x[:0], u[:0]).shape == (0,)


def test_sample_follows_the_distribution(sy):
    """Frequencies of 200 000 draws lie within five standard deviations of the probabilities."""
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], device="cuda")
    n = 200_000
    u = torch.rand(n, generator=gen(1), device="cuda")
    got = sy.sample_tokens(x.expand(n, 5), u)
    p = x.double().softmax(0)
    freq = torch.bincount(got, minlength=5).double() / n
    assert ((freq - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()
