"""Refusals of the serving functions: wrong arguments raise before anything is launched (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def sy():
    import switchyard

    return switchyard


def test_cpu_tensors_are_refused(sy):
    x = torch.zeros(1, 1, 8)
    cache = torch.zeros(1, 1, 8, 8)
    i32, i64 = torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        sy.append_kv(x, x, cache, cache, i64)
    with pytest.raises(ValueError, match="CUDA"):
        sy.attend_paged(x[None], cache, cache, i32[None], i32)
    with pytest.raises(ValueError, match="CUDA"):
        sy.sample_tokens(torch.zeros(1, 4), torch.zeros(1))


def test_wrong_shapes_are_refused(sy):
    x, cache = torch.zeros(1, 1, 8), torch.zeros(1, 1, 8, 8)
    i32, i64 = torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="k_cache and v_cache"):
        sy.append_kv(x, x, cache, cache[0], i64)
    with pytest.raises(ValueError, match="k_cache and v_cache"):
        sy.attend_paged(x[None], cache[0], cache, i32[None], i32)
    with pytest.raises(ValueError, match="logits must be"):
        sy.sample_tokens(torch.zeros(4), torch.zeros(1))
    with pytest.raises(ValueError, match="logits must be"):
        sy.sample_tokens(torch.zeros(1, 0), torch.zeros(1))


class Append(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q k v q_out k_cache v_cache slots positions cos sin").split()]
                + [(n, ctypes.c_int64) for n in (
                    "tokens q_heads kv_heads head_dim rot_half rope_len rope_row pages page_size q_tok q_head k_tok "
                    "k_head v_tok v_head kc_page kc_head kc_row vc_page vc_head vc_row").split()]
                + [("dtype", ctypes.c_int32)])


class Attend(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in (
                    "q k_cache v_cache out lse page_table kv_lens prefix_pages workspace").split()]
                + [("workspace_bytes", ctypes.c_int64)]
                + [(n, ctypes.c_int64) for n in (
                    "batch q_len q_heads kv_heads head_dim pages page_size table_width table_row prefix_len q_b q_t "
                    "q_h kc_page kc_head kc_row vc_page vc_head vc_row").split()]
                + [("scale", ctypes.c_float), ("dtype", ctypes.c_int32)])


class Sample(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in (
                    "logits u temperature top_k top_p min_p token logprob workspace").split()]
                + [(n, ctypes.c_int64) for n in "workspace_bytes rows vocab logits_row".split()]
                + [("dtype", ctypes.c_int32)])


def test_abi_checks_arguments():
    from switchyard import _native as N

    L = N.lib
    good = dict(k=16, v=16, k_cache=16, v_cache=16, slots=16, tokens=2, kv_heads=1, head_dim=8, pages=1, page_size=8)

    def append(**kw):
        return L.sy_append_kv(ctypes.byref(Append(**{**good, **kw})), None)

    assert L.sy_append_kv(None, None) == N.SY_ERR_ARG
    assert append(tokens=0) == N.SY_OK
    assert append(dtype=7) == N.SY_ERR_DTYPE
    for bad in (dict(tokens=-1), dict(kv_heads=0), dict(head_dim=0), dict(page_size=0), dict(k=None), dict(slots=None),
                dict(q_heads=2), dict(positions=16), dict(positions=16, cos=16, sin=16, rot_half=5, rope_len=4, rope_row=5),
                dict(positions=16, cos=16, sin=16, rot_half=4, rope_len=0, rope_row=4)):
        assert append(**bad) == N.SY_ERR_ARG, bad

    good_a = dict(q=16, k_cache=16, v_cache=16, out=16, page_table=16, kv_lens=16, batch=1, q_len=1, q_heads=2,
                  kv_heads=1, head_dim=64, pages=4, page_size=16, table_width=2, table_row=2, scale=0.125)

    def attend(**kw):
        return L.sy_attend(ctypes.byref(Attend(**{**good_a, **kw})), None)

    assert attend(batch=0) == N.SY_OK and attend(q_len=0) == N.SY_OK
    assert attend(dtype=9) == N.SY_ERR_DTYPE
    for bad in (dict(dtype=N.SY_F32), dict(head_dim=12), dict(head_dim=136), dict(page_size=12)):
        assert attend(**bad) == N.SY_ERR_UNSUPPORTED, bad
    # query rows further apart than 32 bits of 16 bytes
    assert attend(q_h=1 << 36) == N.SY_ERR_UNSUPPORTED
    assert attend(batch=3, q_b=1 << 34) == N.SY_ERR_UNSUPPORTED
    for bad in (dict(q=None), dict(q=8), dict(out=None), dict(kv_lens=None), dict(q_heads=3, kv_heads=2),
                dict(prefix_len=5), dict(prefix_len=-1), dict(kc_row=4), dict(q_h=3), dict(kc_page=-8),
                dict(table_width=1 << 28), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(page_table=None), dict(k_cache=None)):
        assert attend(**bad) == N.SY_ERR_ARG, bad
    assert L.sy_attend_workspace(None) == -N.SY_ERR_ARG

    good_s = dict(logits=16, u=16, token=16, rows=1, vocab=8, logits_row=8)

    def sample(**kw):
        return L.sy_sample(ctypes.byref(Sample(**{**good_s, **kw})), None)

    assert sample(rows=0) == N.SY_OK
    assert sample(dtype=-1) == N.SY_ERR_DTYPE
    for bad in (dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(rows=-1), dict(rows=2, logits_row=7), dict(u=None),
                dict(logits=None), dict(token=None)):
        assert sample(**bad) == N.SY_ERR_ARG, bad
