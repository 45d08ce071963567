"""Argument checks of the serving entry points at the edges of what they take (no GPU needed)."""

from __future__ import annotations

import ctypes

from test_serving_cpu import Attend, Sample


def test_strides_of_the_abi():
    """Strides that are no multiples of 16 bytes are refused along every axis that has two elements. (Calls that would
    pass every check are not made here: their pointers are made up.)"""
    from switchyard import _native as N

    good = dict(q=16, k_cache=16, v_cache=16, out=16, page_table=16, kv_lens=16, batch=2, q_len=2, q_heads=2,
                kv_heads=2, head_dim=64, pages=2, page_size=16, table_width=2, table_row=2, scale=0.125)
    for axis in "q_b q_t q_h kc_page kc_head kc_row vc_page vc_head vc_row".split():
        for stride in (4, -8, (1 << 38) + 8):
            args = Attend(**{**good, axis: stride})
            assert N.lib.sy_attend(ctypes.byref(args), None) == N.SY_ERR_ARG, (axis, stride)


def test_scale_times_log2_e_must_be_finite():
    """The kernels take their exponentials to base 2: a scale that overflows there gave NaN."""
    from switchyard import _native as N

    nothing = dict(q_len=1, q_heads=2, kv_heads=1, head_dim=64, pages=4, page_size=16)
    for scale, want in ((2.3e38, N.SY_OK), (2.4e38, N.SY_ERR_ARG), (2.9e38, N.SY_ERR_ARG)):
        assert N.lib.sy_attend(ctypes.byref(Attend(batch=0, scale=scale, **nothing)), None) == want, scale


def test_sampling_needs_no_workspace():
    from switchyard import _native as N

    def need(**kw):
        return N.lib.sy_sample_workspace(ctypes.byref(Sample(**{**dict(rows=64, vocab=32000, logits_row=32000), **kw})))

    assert need() == 0 and need(rows=0) == 0
    assert need(vocab=0) == -N.SY_ERR_ARG and need(dtype=9) == -N.SY_ERR_DTYPE
