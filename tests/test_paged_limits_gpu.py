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
