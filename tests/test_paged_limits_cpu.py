"""Refusals of the paged-cache operators at the ends of what they accept (none
of these calls reaches a launch)."""
import pytest
import torch

from test_paged_cpu import BF16, _attn_args, _plan_args, _rc

# Arrays of 16 requests at addresses of their own, 4096 bytes apart.
APART = dict(requests=16, token_cap=32, q_start=4096, kv_len=2 * 4096, positions=3 * 4096, slots=4 * 4096, ring_out=5 * 4096,
             table=6 * 4096, ring=7 * 4096, lens=8 * 4096, new=9 * 4096, ring_state=10 * 4096)


@pytest.mark.parametrize("kw", [dict(kv_len=8 * 4096 + 8), dict(kv_len=8 * 4096 - 8), dict(kv_len=8 * 4096 + 15 * 8),
                                dict(q_start=9 * 4096 - 16 * 8), dict(positions=8 * 4096 + 8), dict(slots=9 * 4096 - 31 * 8),
                                dict(ring_out=10 * 4096 - 8), dict(ring_out=8 * 4096 + 15 * 8), dict(slots=10 * 4096 + 8)])
def test_plan_refuses_outputs_that_begin_or_end_inside_an_input(xn, kw):
    """One output shifted against an input by a few entries: other blocks would read what one has written."""
    assert _rc(xn, "xn_paged_plan", *_plan_args(**dict(APART, **kw))) == xn.XN_E_INVALID
    assert "input array" in xn.last_error()


@pytest.mark.parametrize("scale", [2.0 ** 127 * (1 + 2.0 ** -23), 2.5e38, 3.4e38])
def test_attention_refuses_scales_past_f32_in_base_2(xn, scale):
    assert _rc(xn, "xn_paged_attention", *_attn_args(scale=scale)) == xn.XN_E_INVALID
    assert "scale" in xn.last_error()


def test_attention_takes_the_largest_scale(xn):
    assert _rc(xn, "xn_paged_attention", *_attn_args(scale=2.0 ** 127, n=0)) == xn.XN_OK


def test_norm_of_no_columns_still_has_scales(xn):
    """Rows of no columns have a scale each: the call needs a place for them, and nothing else."""
    norm = lambda scales, group: _rc(xn, "xn_rms_norm_q8", None, scales, None, None, None, None, 5, 0, group, 1e-5, BF16, None)  # noqa: E731
    assert norm(None, 0) == xn.XN_E_INVALID and "null" in xn.last_error()
    assert norm(None, 32) == xn.XN_OK


class NoTruth:
    def __bool__(self):
        raise ValueError("no truth value")


def test_what_an_argument_raises_comes_through(xn):
    """An argument whose truth value raises stops the call with that, before anything else is looked at."""
    pool = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int64)
    table = torch.zeros(9, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no truth value"):
        xn.paged_append_rope(torch.zeros(4, 12 * 64, dtype=torch.bfloat16), 8, 2, table, table, pool, pool, i, i,
                             interleaved=NoTruth())
