"""The serving operators where they are easiest to get wrong: clusters whose CTAs start at different times,
batches and prefixes beyond one CTA's or one tile's share, indices outside their buffers, axes of one element."""

from __future__ import annotations

import math

import pytest
import torch

from test_serving_gpu import (  # noqa: F401  (sy and clear_error_word are fixtures)
    angles,
    check_attend,
    check_sample,
    clear_error_word,
    gen,
    near_turned,
    paged,
    params,
    sy,
)

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


def test_sample_top_p_cut_between_two_doubles(sy):
    """Sums of weights beyond 2^53 and a cut right behind what the bins next to the maximum hold: S = 2^60 + W, a
    number that no double is, and a goal of S + 64, the double that S rounds to. One more token than those bins' is
    kept, the highest of the rest."""
    d = torch.arange(6.94, 7.1, 2.0**-21, dtype=torch.float64, device="cuda").float()
    w = ((-d).exp().double() * 2.0**40).round().long()
    near = int((w % 256 == 192).nonzero()[0])  # 2^60 + w is 64 below a multiple of 256
    s = 2**60 + int(w[near])
    goal = s + 64
    assert int(float(s)) == goal and goal % 256 == 0
    p = 1.0 - 2.0**-24
    # lower weights so that p of the total is the goal
    table = torch.linspace(7.2, 27.0, 200_000, dtype=torch.float64, device="cuda").float()
    weights = ((-table).exp().double() * 2.0**40).round().long().cpu().numpy()
    total, rest, at = math.ceil(goal / p), [], 0
    left = total - s
    table = table.cpu().numpy()
    while left > 0:
        at += int((weights[at:] <= left).argmax())
        if weights[at] > left:
            break
        rest.append(float(table[at]))
        left -= int(weights[at])
    total -= left
    assert math.ceil(p * float(total)) == goal, "the inputs are as described"
    x = torch.cat([-torch.tensor(rest[::-1], device="cuda"), torch.zeros(2**20, device="cuda"), -d[near:near + 1]])
    ones = torch.ones(2, device="cuda")
    u = torch.tensor([0.0, 1.0 - 2.0**-24], device="cuda")
    token = sy.sample_tokens(x.expand(2, -1), u, top_p=p * ones)
    assert int(token[0]) == rest[::-1].index(rest[0]), "of the rest only the highest, at its lowest index, is kept"
    check_sample(sy, x.expand(2, -1), u, ones, 0 * ones.int(), p * ones, 0 * ones)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [262145, 700_001, 1 << 22])
def test_sample_slices_beyond_shared_memory(sy, dtype, vocab):
    """Slices that do not fit in shared memory are read again from global memory: random rows, one of equal logits and
    one of few values (more ties in a bin than its list holds)."""
    x = 3 * torch.randn(5, vocab, generator=gen(vocab), device="cuda")
    x[0] = 1.0
    x[1] = x[1].round()
    x[2] = torch.where(x[2] > 2, x[2], -math.inf)
    x = x.to(dtype)
    u = torch.rand(5, generator=gen(1), device="cuda")
    one = torch.ones(5, device="cuda")
    zero = torch.zeros_like(one)
    check_sample(sy, x, u, 0.7 * one, 60 + zero.int(), 0.8 * one, zero)
    check_sample(sy, x, u, one, zero.int(), 0.9 * one, 0.01 * one)
    check_sample(sy, x, u, one, zero.int(), one, zero)
    check_sample(sy, x, u, zero, zero.int(), one, zero)


# ---------------------------------------------------------------------------
# attend_paged
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,n,hq,hk,d,page,prefix", [
    ([130] * 20, 130, 16, 16, 128, 16, 0),  # 320 units: most are finished in one run
    ([145] * 12, 145, 16, 16, 64, 8, 0),
    ([131] * 11, 131, 16, 16, 40, 8, 3),
    ([200, 61, 1], 33, 3, 1, 128, 8, 0),  # 99 rows of a unit; tiles of 72 keys, 61 keys, one key
    ([97, 98, 99, 100], 1, 21, 1, 128, 24, 131),  # 84 rows over the prefix, 21 over a sequence
    ([65, 2, 127], 2, 62, 2, 64, 16, 70),  # 62 rows a unit, 186 over the prefix: the second stream has 58
])
def test_attend_rows_and_keys_that_leave_lanes_idle(sy, dtype, lens, n, hq, hk, d, page, prefix):
    """Rows that end inside a warp (its lanes part where O is stored) and keys that end inside a tile (they part where
    V is cleared): the tensor memory loads that follow take whole warps."""
    args, kw, lead, own = paged(sum(lens) + n, lens, n, hq, hk, d, page, prefix, dtype)
    out, lse = sy.attend_paged(*args, **kw, return_lse=True)
    check_attend(out, lse, args, kw, lead, own)
    assert torch.equal(sy.attend_paged(*args, **kw), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,n,hq,hk,d,page,prefix", [
    ([7] * 75, 1, 32, 8, 128, 16, 300),  # 300 rows over the prefix: two row tiles, the second with 44
    ([1, 50, 9] * 43, 1, 32, 8, 64, 8, 129),  # 516 rows: a third tile of four rows
    ([30] * 5, 30, 8, 2, 128, 64, 200),  # 120 rows a sequence, 600 over the prefix
    ([3] * 400, 1, 4, 4, 64, 8, 20),  # two sequences a thread in the scan over the lengths
    ([0, 1, 0, 130, 5] * 160, 1, 8, 2, 128, 16, 0),  # 800 sequences, some of them empty
    ([5] * 389, 5, 6, 2, 80, 8, 0),
])
def test_attend_many_sequences(sy, dtype, lens, n, hq, hk, d, page, prefix):
    args, kw, lead, own = paged(len(lens), lens, n, hq, hk, d, page, prefix, dtype)
    out, lse = sy.attend_paged(*args, **kw, return_lse=True)
    check_attend(out, lse, args, kw, lead, own)
    assert torch.equal(sy.attend_paged(*args, **kw), out)


# ---------------------------------------------------------------------------
# append_kv
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_what_q_holds_for_indices_outside(sy, dtype):
    """Partial rotation: q is zero in all its columns where the position lies outside, and rotated as ever where only
    the slot does. The cache rows of both tokens stay as they were."""
    from switchyard import _native

    kc, vc = (torch.full((2, 1, 8, 40), 7.0, device="cuda", dtype=dtype) for _ in range(2))
    cos, sin = angles(4, 8)
    x = torch.randn(4, 1, 40, generator=gen(1), device="cuda").to(dtype)
    pos = torch.tensor([0, 4, -1, 3], device="cuda", dtype=torch.int32)
    q = sy.append_kv(x, x, kc, vc, torch.tensor([3, 1, 2, 16], device="cuda"), q=x, positions=pos, cos=cos, sin=sin)
    assert _native.device_error() == 4
    assert not q[1:3].any()
    for t in (0, 3):
        near_turned(q[t:t + 1], x[t:t + 1], cos[pos[t:t + 1].long()], sin[pos[t:t + 1].long()])
    kept = torch.ones(2, 8, dtype=torch.bool, device="cuda")
    kept[0, 3] = False
    assert (kc[:, 0][kept] == 7).all() and (vc[:, 0][kept] == 7).all()
    assert torch.equal(vc[0, :, 3], x[0])


def test_attend_axes_of_one_element_may_have_any_stride(sy):
    """A cache of one page, and one of one key head, whose strides along those axes are no multiples of 16 bytes."""
    for lens, hk in (([13], 2), ([40, 5], 1)):
        args, kw, lead, own = paged(9, lens, 1, 4, hk, 64, 64, 0, torch.bfloat16)
        q, kc, vc, table, n = args
        if hk == 2:  # one page alone
            page = int(table[0, 0])
            kc, vc, table = kc[page:page + 1], vc[page:page + 1], torch.zeros_like(table)
        want = sy.attend_paged(q, kc, vc, table, n)
        strides = [(s if m > 1 else 13) for s, m in zip(kc.stride(), kc.shape)]
        odd = [torch.as_strided(c, c.shape, strides, c.storage_offset()) for c in (kc, vc)]
        assert torch.equal(sy.attend_paged(q, *odd, table, n), want)
        thin = [torch.as_strided(x, x.shape, [3 if m == 1 else s for s, m in zip(x.stride(), x.shape)]) for x in (q,)]
        assert torch.equal(sy.attend_paged(*thin, kc, vc, table, n), want)


def test_attend_scale_that_overflows_is_refused(sy):
    args, kw, _, _ = paged(10, [20], 1, 2, 2, 64, 16, 0, torch.bfloat16)
    for scale in (2.4e38, 1e39, 1e-46):  # the last is zero in 32 bits
        with pytest.raises(ValueError, match="scale"):
            sy.attend_paged(*args, scale=scale)
    out = sy.attend_paged(args[0].zero_(), *args[1:], scale=2.3e38)
    assert out.isfinite().all()


def test_attend_what_stands_in_for_indices_outside(sy):
    """A page outside the cache reads as zero keys and values, which count; a length outside is cut to the table."""
    from switchyard import _native

    args, kw, lead, own = paged(7, [40, 48], 1, 4, 4, 64, 16, 37, torch.bfloat16)
    q, kc, vc, table, lens = args
    for page in (kc.shape[0], -1, 2**31 - 1):
        bad = table.clone()
        bad[0, 1] = page
        out, lse = sy.attend_paged(q, kc, vc, bad, lens, **kw, return_lse=True)
        assert _native.device_error() == 4
        zeroed = [[side[0].clone(), side[1]] for side in own]
        for side in zeroed:
            side[0][:, 16:32] = 0
        check_attend(out, lse, args, kw, lead, zeroed)
    # a table of exactly three pages: sequence 1 fills it
    whole = table[:, :3].contiguous()
    want = sy.attend_paged(q, kc, vc, whole, lens, **kw)
    far = torch.stack([lens[0], torch.full_like(lens[0], 2**31 - 1)])
    assert torch.equal(sy.attend_paged(q, kc, vc, whole, far, **kw), want)
    assert _native.device_error() == 4
    out, lse = sy.attend_paged(q, kc, vc, table, torch.stack([lens[0], -lens[1]]), **kw, return_lse=True)
    assert _native.device_error() == 4
    check_attend(out, lse, args, kw, lead, [[side[0], side[1][:, :0]] for side in own])


# ---------------------------------------------------------------------------
# what the header says of workspaces
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("batch,n,hq,hk,d,width,prefix", [
    (1, 1, 16, 16, 128, 33, 0), (128, 1, 32, 8, 128, 8, 16384), (24, 5, 24, 8, 64, 11, 1999), (1, 4096, 16, 16, 128, 64, 0),
    (1024, 8, 128, 8, 128, 16, 0), (3, 129, 4, 4, 80, 16, 50),
])
def test_attend_workspace_is_as_documented(batch, n, hq, hk, d, width, prefix):
    import ctypes

    from switchyard import _native
    from test_serving_cpu import Attend

    args = Attend(batch=batch, q_len=n, q_heads=hq, kv_heads=hk, head_dim=d, pages=99, page_size=64,
                  table_width=width, table_row=width, prefix_len=prefix, scale=1.0)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    rows, line = n * (hq // hk), 4 * (2 + (64 if d <= 64 else 128))
    wide = rows > 128
    shared = prefix > 0 and batch > 1 and not wide
    most = (4 * sms * 128 if wide else 2 * (batch * hk + sms) * rows) * line
    if shared:
        most += 2 * (hk * -(-batch * rows // 256) + sms) * min(128, batch * rows) * line
    most += 4 * (batch * -(-rows // 256) + 1)
    got = _native.lib.sy_attend_workspace(ctypes.byref(args))
    assert most <= got <= most + 5 * 16
