"""Refusals of the paged-cache operators and of the 8-bit RMSNorm at the C ABI
and in the Python binding (none of these calls reaches a launch), and the
plain restatements themselves."""
import ctypes

import pytest
import torch

import paged_ref

P = 16  # a non-null, 16-byte-aligned address that no refused call touches
BF16 = 1


def _rc(xn, name, *args):
    return getattr(xn.lib(), name)(*args)


def _plan_args(**kw):
    a = dict(q_start=P, kv_len=P, positions=P, slots=P, ring_out=P, table=P, ring=P, lens=2 * P, new=3 * P, ring_state=2 * P,
             requests=2, max_blocks=4, n_pages=8, page_size=16, token_cap=4, err=None, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(requests=-1), "negative"), (dict(requests=8193), "exceed"), (dict(page_size=24), "page size"),
    (dict(page_size=4), "page size"), (dict(page_size=512), "page size"), (dict(n_pages=0), "out of range"),
    (dict(token_cap=-1), "negative"), (dict(kv_len=2 * P), "input array"), (dict(ring_out=2 * P), "input array"),
    (dict(q_start=3 * P), "input array"), (dict(slots=2 * P), "input array"), (dict(positions=3 * P), "input array"),
    (dict(table=None), "null"), (dict(slots=None), "null"), (dict(ring=None), "null"), (dict(max_blocks=1 << 32), "out of range")])
def test_plan_refusals(xn, kw, text):
    assert _rc(xn, "xn_paged_plan", *_plan_args(**kw)) == xn.XN_E_INVALID
    assert text in xn.last_error()


def _append_args(**kw):
    a = dict(q_out=P, k=P, v=P, qkv=P, cos=P, sin=P, positions=P, slots=P, n=4, h=8, hk=2, d=64, max_pos=100, n_pages=4,
             page_size=16, ps=2 * 16 * 64, hs=16 * 64, ss=64, interleaved=1, dtype=BF16, err=None, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(n=-1), "negative"), (dict(d=48), "head dim"), (dict(page_size=12), "page size"), (dict(ss=60), "16 bytes"),
    (dict(ss=32), "out of range"), (dict(hs=-64), "out of range"), (dict(k=8), "aligned"), (dict(q_out=None), "null"),
    (dict(slots=None), "null"), (dict(h=0), "empty"), (dict(n_pages=0), "out of range")])
def test_append_refusals(xn, kw, text):
    assert _rc(xn, "xn_paged_append_rope", *_append_args(**kw)) == xn.XN_E_INVALID
    assert text in xn.last_error()
    assert _rc(xn, "xn_paged_append_rope", *_append_args(dtype=3)) == xn.XN_E_DTYPE


def _attn_args(**kw):
    a = dict(out=P, q=P, k=P, v=P, table=P, q_start=P, kv_len=P, n=4, requests=2, h=8, hk=2, d=64, n_pages=4, page_size=16,
             max_blocks=4, q_stride=8 * 64, ps=2 * 16 * 64, hs=16 * 64, ss=64, max_new=2, window=0, scale=0.125, dtype=BF16,
             ws=P, ws_bytes=1 << 40, err=None, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(h=9), "times h_kv"), (dict(h=130, hk=2, q_stride=130 * 64), "times h_kv"), (dict(d=96), "head dim"),
    (dict(window=-1), "window"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=-1.0), "scale"), (dict(q_stride=8 * 64 - 8), "stride"),
    (dict(q_stride=8 * 64 + 4), "stride"), (dict(ws_bytes=64), "workspace"), (dict(ws=None), "null"), (dict(q=24), "aligned"),
    (dict(requests=8193), "exceed"), (dict(max_blocks=1 << 40), "out of range"), (dict(page_size=7), "page size"),
    (dict(ps=2 * 16 * 64 + 4), "16 bytes"), (dict(n=-4), "negative")])
def test_attention_refusals(xn, kw, text):
    assert _rc(xn, "xn_paged_attention", *_attn_args(**kw)) == xn.XN_E_INVALID
    assert text in xn.last_error()


def test_attention_workspace(xn):
    n = ctypes.c_int64()
    size = lambda *a: (_rc(xn, "xn_paged_attention_workspace", ctypes.byref(n), *a), n.value)  # noqa: E731
    assert size(16, 16, 16, 16, 64, 1, BF16)[0] == xn.XN_OK
    assert size(16, 16, 16, 5, 64, 1, BF16)[0] == xn.XN_E_INVALID
    assert size(16, 16, 16, 16, 64, 1, 4)[0] == xn.XN_E_DTYPE
    assert _rc(xn, "xn_paged_attention_workspace", None, 16, 16, 16, 16, 64, 1, BF16) == xn.XN_E_INVALID
    w = xn.paged_attention_workspace(16, 16, 16, 16, 64, 1, torch.bfloat16, "cpu")
    assert w.numel() == size(16, 16, 16, 16, 64, 1, BF16)[1]


def test_empty_calls_launch_nothing(xn):
    assert _rc(xn, "xn_paged_attention", *_attn_args(n=0, out=None, q=None, ws=None)) == xn.XN_OK
    assert _rc(xn, "xn_paged_append_rope", *_append_args(n=0, q_out=None)) == xn.XN_OK
    assert _rc(xn, "xn_rms_norm_q8", None, None, None, None, None, None, 0, 64, 0, 1e-5, BF16, None) == xn.XN_OK


@pytest.mark.parametrize("kw,code", [(dict(eps=0.0), "XN_E_INVALID"), (dict(group=48), "XN_E_INVALID"),
                                     (dict(group=128, cols=192), "XN_E_INVALID"), (dict(dtype=4), "XN_E_DTYPE"),
                                     (dict(scales=None), "XN_E_INVALID"), (dict(rows=-1), "XN_E_INVALID"),
                                     (dict(eps=float("nan")), "XN_E_INVALID")])
def test_norm_refusals(xn, kw, code):
    a = dict(dst=P, scales=P, res=None, src=P, alpha=P, branch=None, rows=2, cols=128, group=0, eps=1e-5, dtype=BF16, stream=None)
    a.update(kw)
    assert _rc(xn, "xn_rms_norm_q8", *a.values()) == getattr(xn, code)


def test_python_checks(xn):
    pool = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    table = torch.zeros(2, 4, dtype=torch.int32)
    i64 = lambda *v: torch.tensor(v, dtype=torch.int64)  # noqa: E731
    q = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(xn.XnError, match="no CPU path"):
        xn.paged_attention(q, pool, pool, table, i64(0, 1, 4), i64(3, 9), 0.125, max_new=3)
    with pytest.raises(xn.XnError, match="multiple of"):
        xn.paged_attention(q[:, :7], pool, pool, table, i64(0, 1, 4), i64(3, 9), 0.125, max_new=3)
    with pytest.raises(xn.XnError, match="share their strides"):
        xn.paged_attention(q, pool, pool.transpose(1, 2).contiguous().transpose(1, 2), table, i64(0, 1, 4), i64(3, 9), 0.125,
                           max_new=3)
    with pytest.raises(xn.XnError, match="shape mismatch"):
        xn.paged_attention(q, pool, pool, table, i64(0, 1), i64(3, 9), 0.125, max_new=3)
    with pytest.raises(xn.XnError, match="no CPU path"):
        xn.paged_plan(i64(1, 2), i64(1, 1), table, torch.zeros(8, dtype=torch.int32), i64(0, 8), 16, 4)
    with pytest.raises(xn.XnError, match="shape mismatch"):
        xn.paged_plan(i64(1, 2), i64(1), table, torch.zeros(8, dtype=torch.int32), i64(0, 8), 16, 4)
    with pytest.raises(xn.XnError, match="expected qkv"):
        xn.paged_append_rope(torch.zeros(4, 11 * 64), 8, 2, torch.zeros(9, 32), torch.zeros(9, 32), pool, pool, i64(0, 1, 2, 3),
                             i64(0, 1, 2, 3))
    x = torch.zeros(2, 96)
    with pytest.raises(xn.XnError, match="divisor"):
        xn.rms_norm_q8(x, torch.ones(96), 1e-5, group=64)
    with pytest.raises(xn.XnError, match="eps must be positive"):
        xn.rms_norm_q8(x, torch.ones(96), 0.0)
    with pytest.raises(xn.XnError, match="no CPU path"):
        xn.rms_norm_q8(x, torch.ones(96), 1e-5)


def test_plan_restatement_keeps_every_page_once():
    """Pages are neither lost nor shared over steps that grow, end and wrap the ring."""
    import random

    rng = random.Random(3)
    page, n_pages, n = 8, 40, 6
    table, ring, state, lens = [[-1] * 10 for _ in range(n)], list(range(n_pages)), [0, n_pages], [0] * n
    done = 0
    for _ in range(200):
        new = [rng.choice([-1, 0, 1, 1, 7, 19]) for _ in range(n)]
        got = paged_ref.plan(lens, new, table, ring, state, page, 64)
        if got is None:
            new = [-1] * n
            got = paged_ref.plan(lens, new, table, ring, state, page, 64)
        _, lens, _, slots, table, ring, state = got
        held = [p for i in range(n) for p in table[i][:-(-lens[i] // page)]]
        free = [ring[(state[0] + k) % n_pages] for k in range(state[1])]
        assert sorted(held + free) == list(range(n_pages))
        live = [s for s in slots if s >= 0]
        assert len(set(live)) == len(live)
        done += sum(k > 0 for k in new)
    assert done > 100
