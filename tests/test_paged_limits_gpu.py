"""The paged-cache operators and the 8-bit RMSNorm at the ends of what they
accept: request counts around a shared-memory limit, scores and scales at the
ends of f32's range, wide query groups, empty rows."""
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import paged_ref
from helpers import U32
from paged_ref import HALF_STEP
from test_paged_gpu import DT, Batch, _plan_state, _run_plan, i64

pytestmark = pytest.mark.gpu

REPO = Path(__file__).resolve().parents[1]


def _child(code, *args, **env):
    """Runs code in a process of its own (nothing launched before it); what it prints last, as JSON."""
    out = subprocess.run([sys.executable, "-c", code, str(REPO), *map(str, args)], env=dict(os.environ, **env),
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    return json.loads(out.stdout.strip().splitlines()[-1])


# -- plan ------------------------------------------------------------------------

PLAN_CHILD = r"""
import json, sys
sys.path[:0] = [sys.argv[1] + "/random-things_b200"]
import torch
import xn_fused as xn
n, dev = int(sys.argv[2]), "cuda:0"
new = torch.ones(n, dtype=torch.int64, device=dev)
table = torch.full((n, 1), -1, dtype=torch.int32, device=dev)
ring = torch.arange(n, dtype=torch.int32, device=dev)
p = xn.paged_plan(torch.zeros_like(new), new, table, ring, torch.tensor([0, n], device=dev), 8, n)
ids = torch.arange(n, device=dev)
print(json.dumps([torch.equal(p.slots, ids * 8), torch.equal(table[:, 0].long(), ids), torch.equal(p.q_start[1:], ids + 1)]))
"""


@pytest.mark.parametrize("n", [4061, 4062, 4095, 4096])
def test_plan_request_counts_at_the_default_shared_memory(n):
    """12 bytes a request meet the 48 KB that a block has without asking, of which a few hundred bytes are taken."""
    assert _child(PLAN_CHILD, n) == [True] * 3


def test_plan_request_counts_after_one_another(xn, cuda):
    for n in (4062, 8192, 4095, 4096, 4061):
        lens, table, ring, state = _plan_state(n, n, 8, 30, 6, n + 3)
        new = [i % 3 for i in range(n)]
        want = paged_ref.plan(lens, new, table, ring, state, 8, sum(new))
        assert list(want) == list(_run_plan(xn, cuda, lens, new, table, ring, state, 8, sum(new)))


@pytest.mark.parametrize("state,lens", [([0, (1 << 63) - 1], [5, 16]), ([0, (1 << 63) - 3], [5, 16]), ([(1 << 63) - 1, 2], [5, 16]),
                                        ([-(1 << 63), 2], [5, 16]), ([0, -(1 << 63)], [5, 16]), ([0, 2], [(1 << 63) - 1, 16]),
                                        ([0, 2], [-(1 << 63), 16])])
@pytest.mark.parametrize("new", [[-1, -1], [-1, 1], [3, -(1 << 63)]])
def test_plan_state_at_the_ends_of_64_bits(xn, cuda, state, lens, new):
    """A ring or lengths that cannot be, however large, change nothing."""
    table, ring = [[0, -1, -1], [1, 2, -1]], [9, 8, 7, 6, 5, 4, 3]
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = _run_plan(xn, cuda, lens, new, table, ring, state, 8, 6, err)
    assert int(err) & xn.XN_DEVERR_RANGE
    assert list(got) == [[0] * 3, lens, [-1] * 6, [-1] * 6, table, ring, state]


def test_plan_outputs_next_to_inputs(xn, cuda):
    """Arrays of one buffer, one behind the other, do not overlap; shifted by an entry they do."""
    n, cap = 40, 64
    lens, table, ring, state = _plan_state(1, n, 8, 30, 6, n + 3)
    new = [i % 3 for i in range(n)]
    want = paged_ref.plan(lens, new, table, ring, state, 8, cap)
    sizes = [n, n, n, n + 1, cap, 2, 2, cap]  # kv_len, lens, new, q_start, positions, ring state out, in, slots
    kv, le, ne, qs, po, ro, ri, sl = torch.full((sum(sizes),), 5, dtype=torch.int64, device=cuda).split(sizes)
    le.copy_(i64(lens)), ne.copy_(i64(new)), ri.copy_(i64(state))
    t, r = torch.tensor(table, dtype=torch.int32, device=cuda), torch.tensor(ring, dtype=torch.int32, device=cuda)
    p = xn.paged_plan(le, ne, t, r, ri, 8, cap, out=xn.PagedPlan(qs, kv, po, sl, ro))
    assert list(want) == [x.tolist() for x in (p.q_start, p.kv_len, p.positions, p.slots, t, r, p.ring_state)]
    both = torch.zeros(n + 1, dtype=torch.int64, device=cuda)
    with pytest.raises(xn.XnError, match="input array"):
        xn.paged_plan(both[1:], ne, t, r, ri, 8, cap, out=xn.PagedPlan(qs, both[:-1], po, sl, ro))


# -- attention: windows ----------------------------------------------------------

@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("new", [[5, 4, 3], [70, 40, 30]])
@pytest.mark.parametrize("window", [(1 << 31) - 1, 1 << 31, (1 << 63) - 1])
def test_attention_windows_longer_than_any_request(xn, cuda, dtype, new, window):
    """The longest windows hide nothing, tokens at negative positions (kv_len below the new tokens) among them."""
    b = Batch(cuda, dtype, 4, 2, 64, 16, [0, 0, 50], new, kv=[3, 0, 50 + new[2]])
    want = b.run(xn)
    assert torch.equal(b.run(xn, window=window), want)
    b.check(xn, window=window)


# -- attention: rows that no token sees ------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("window", [0, 1, 9])
def test_attention_single_tokens_over_stale_rows(xn, cuda, dtype, d, window):
    """Every count of unseen NaN rows in a key tile, at its end and before a window, in 64 requests at once, again and
    again: the lanes that read the zeroed rows are others than those that zero them."""
    b = Batch(cuda, dtype, 4, 2, d, 64, list(range(64)), [1] * 64, stale=float("nan"))
    b.check(xn, window=window)
    want = b.run(xn, window=window)
    for _ in range(50):
        assert torch.equal(b.run(xn, window=window), want)


# -- attention: large scores -----------------------------------------------------

def _one_key(dtype, value, h, hk, d, new, dev):
    """Requests of one cached key each that every row sees alone or with copies of it: all of q and k is `value`."""
    b = Batch(dev, dtype, h, hk, d, 16, [0] * 3, [1, new, 1])
    b.q[:], b.k[:] = value, torch.where(torch.isnan(b.k), b.k, value)
    return b


# Scores of up to 128 x 60000^2 x scale (f16) and of 2^96 x scale (bf16, f32): finite in f32.
HUGE = [("f16", 8000.0), ("f16", 60000.0), ("bf16", 8000.0), ("bf16", 60000.0), ("bf16", 2.0 ** 44), ("f32", 60000.0),
        ("f32", 2.0 ** 44)]


@pytest.mark.parametrize("dtype,value", HUGE)
@pytest.mark.parametrize("h,hk,d", [(4, 2, 64), (8, 1, 128), (2, 2, 32)])
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("scale", [None, 1.0, 1e6, 2.0 ** 127])
def test_attention_equal_scores_of_any_size(xn, cuda, dtype, value, h, hk, d, new, scale):
    """Keys of one and the same score weigh alike, however large it is: rows of one key give its value, others the mean.

    The scores of a row are sums of equal terms in equal order, so they are equal to the last bit and every weight is 1;
    a chunk's bound is that of the weights' and the output's sums and rounding alone."""
    b = _one_key(dtype, value, h, hk, d, new, cuda)
    if scale is not None:
        b.scale = scale
    got = b.run(xn).view(-1, h, d).double().cpu()
    for i, (lo, hi) in enumerate(zip(b.start, b.start[1:])):
        v = b.v[b.table[i, :-(-b.kv[i] // 16)].long()].transpose(1, 2).reshape(-1, hk, d)[:b.kv[i]].double()
        ref = torch.stack([v[:t + 1].mean(0) for t in range(hi - lo)]).repeat_interleave(h // hk, 1)
        mag = torch.stack([v[:t + 1].abs().mean(0) for t in range(hi - lo)]).repeat_interleave(h // hk, 1)
        # Up to 90 terms of weight 1 (exact in every type): 90 roundings of the sum, one of the quotient, one of the output.
        tol = 92 * 2 * U32 * mag + HALF_STEP[DT[dtype]] * 1.01 * ref.abs()
        assert ((got[lo:hi] - ref).abs() <= tol).all()
        assert torch.equal(got[lo], v[0].repeat_interleave(h // hk, 0))  # one key: its value, exactly


@pytest.mark.parametrize("dtype,value", HUGE)
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_attention_the_largest_of_huge_scores_takes_all(xn, cuda, dtype, value, new, order):
    """Keys whose scores lie far apart: each row gives the value of its largest, whether the maximum moves with every
    tile or stands from the first."""
    h, hk, d, n = 4, 2, 64, 400
    b = Batch(cuda, dtype, h, hk, d, 16, [n], [new])
    kv = b.kv[0]
    step = torch.linspace(0.25, 1.0, kv, dtype=torch.float64)
    step = step if order == "rising" else step.flip(0)
    at = b.table[0, :-(-kv // 16)].long()
    rows = (value * step).to(DT[dtype])
    keys = torch.zeros(at.numel() * 16, dtype=DT[dtype])
    keys[:kv] = rows
    b.k[at] = keys.view(-1, 1, 16, 1).expand(-1, hk, -1, d)
    b.q[:] = value
    got = b.run(xn).view(-1, h, d).double().cpu()
    v = b.v[at].transpose(1, 2).reshape(-1, hk, d)[:kv].double()
    exact = rows.double()
    for t in range(new):
        # Keys of the largest (rounded) size share the weight; the next smaller one is 2^-8 or more below, which is
        # more than 2^20 in the exponent.
        top = exact[:n + t + 1] == exact[:n + t + 1].max()
        ref, mag = v[:n + t + 1][top].mean(0), v[:n + t + 1][top].abs().mean(0)
        tol = (int(top.sum()) + 2) * 2 * U32 * mag + HALF_STEP[DT[dtype]] * 1.01 * ref.abs()
        assert ((got[t] - ref.repeat_interleave(h // hk, 0)).abs() <= tol.repeat_interleave(h // hk, 0)).all(), t


# -- attention: groups and hints -------------------------------------------------

@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("h,hk,d", [(21, 1, 64), (33, 1, 32), (64, 1, 128), (48, 2, 64), (128, 2, 32)])
def test_attention_wide_groups(xn, cuda, dtype, h, hk, d):
    Batch(cuda, dtype, h, hk, d, 16, [300, 5, 0], [1, 1, 1]).check(xn)
    Batch(cuda, dtype, h, hk, d, 32, [200, 0, 70], [30, 17, 1], packed=True).check(xn, window=40)


@pytest.mark.parametrize("hint", [0, 1, 4, 100])
def test_attention_hint_f16(xn, cuda, hint):
    Batch(cuda, "f16", 8, 2, 128, 16, [100, 1000, 5], [1, 1, 1]).check(xn, max_new=hint)
    Batch(cuda, "f16", 8, 2, 64, 16, [100, 1000, 5], [50, 7, 30]).check(xn, max_new=hint)



# -- attention: the largest sizes --------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hint", [1, 64])
def test_attention_as_many_requests_as_there_may_be(xn, cuda, dtype, hint):
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 12, (xn.XN_PAGED_MAX_REQUESTS,), generator=g).tolist()
    Batch(cuda, dtype, 2, 1, 32, 8, lens, [1] * len(lens)).check(xn, max_new=hint)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("window", [1, 100, 1000])
def test_attention_positions_up_to_the_last(xn, cuda, dtype, new, window):
    """A window at the end of the longest request there may be, its pages three that repeat."""
    page, h, hk, d, dt = 256, 4, 2, 64, DT[dtype]
    blocks = (2 ** 31 - 1024) // page
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, hk, page, d, generator=g).to(dt) for _ in range(2))
    q = torch.randn(new, h, d, generator=g).to(dt)
    table = (torch.arange(blocks, dtype=torch.int32) % 3).view(1, -1)
    kv, start, scale = blocks * page, i64([0, new]), d ** -0.5
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = xn.paged_attention(q.to(cuda), k.to(cuda), v.to(cuda), table.to(cuda), start.to(cuda), i64([kv], cuda), scale,
                             max_new=new, window=window, err_flag=err)
    # The same request without the blocks that no token sees.
    first = (kv - new - window) // page
    ref, tol = paged_ref.attention(q, k, v, table[:, first:], start, i64([kv - first * page]), scale, window)
    paged_ref.check_attention(got, ref, tol)
    assert int(err) == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("new", [1, 20])
def test_attention_long_history(xn, cuda, dtype, new):
    """A third of a million keys of one head: every part of the work list a piece of the same few rows."""
    Batch(cuda, dtype, 4, 1, 64, 256, [333333], [new]).check(xn)


# -- 8-bit norm ------------------------------------------------------------------

def test_norm_q8_scale_is_the_quotient_by_448(xn, cuda):
    """Rows of ones under an eps that vanishes have y = alpha exactly: each group's scale is alpha / 448, rounded once,
    from the smallest magnitude to the largest and infinity."""
    g = torch.Generator().manual_seed(1)
    bits = torch.randint(1, 0x7f800000, (1 << 16,), generator=g)
    small = torch.randint(1, 0x05000000, (1 << 14,), generator=g)  # subnormal quotients, and the first normal ones
    edges = [1, 2, 223, 224, 225, 448, 0x7fffff, 0x800000, 0x800001, 0x7f7fffff, 0x7f800000]
    edges += [(e << 23) + m for e in range(1, 255) for m in (0, 1, 0x600000, 0x5fffff, 0x600001, 0x7fffff)]
    mag = torch.cat([bits, small, torch.tensor(edges)]).int().view(torch.float32)
    # A quotient of 24 bits by 7 is never as near to half way between two normal floats as the double's rounding.
    want = (mag.double() / 448.0).float()
    normal = want >= 2.0 ** -126
    assert normal.sum() > 60000 and (~normal).sum() > 10000
    alpha = mag.repeat_interleave(32).to(cuda)
    x = torch.ones(1, alpha.numel(), device=cuda)
    for lo, n in ((0, 8192), (1 << 21, 8192), (0, alpha.numel())):  # rows in registers, a row too wide for them
        _, s, _ = xn.rms_norm_q8(x[:, lo:lo + n], alpha[lo:lo + n], 1e-30, group=32)
        s, part = s[0].cpu(), slice(lo // 32, (lo + n) // 32)
        assert torch.equal(torch.where(normal[part], s, 0.0), torch.where(normal[part], want[part], 0.0))
        # Subnormal: half a step of 2^-149, either way of a half, and the step's own 2^-24 of a step.
        off = (s.double() - mag[part].double() / 448.0).abs()[~normal[part]]
        assert (off <= 2.0 ** -150 * (1 + 2.0 ** -23)).all()


def test_norm_q8_rows_of_no_columns(xn, cuda):
    """The largest of no values is 0, and so is the scale."""
    s = torch.full((5,), 7.0, device=cuda)
    q, got, _ = xn.rms_norm_q8(torch.empty(5, 0, device=cuda), torch.empty(0, device=cuda), 1e-5, scales=s)
    assert got is s and s.eq(0).all() and q.shape == (5, 0)


# -- binding ---------------------------------------------------------------------

def test_out_of_memory_is_torchs_exception(xn, cuda):
    """An output that cannot be allocated raises what torch's own operators raise, and nothing is lost."""
    ring = torch.arange(8, dtype=torch.int32, device=cuda)
    args = i64([0], cuda), i64([1], cuda), torch.full((1, 1), -1, dtype=torch.int32, device=cuda), ring, i64([0, 8], cuda), 8
    torch.cuda.set_per_process_memory_fraction(0.05)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            xn.paged_plan(*args, (1 << 31) - 1)  # 34 GB
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert xn.paged_plan(*args, 1).slots.tolist() == [0]
