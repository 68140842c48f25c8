"""The bounded waits of the paged attention's TMA kernels report their give-up
as a device status and return, instead of hanging.

The waits cannot run out with valid arguments, so the tests lower their limit
through XN_PAGED_WAIT_CLOCKS (read once per process) in a child process, on
valid inputs: with 0 the warps of the softmax give up before their first wait,
while copies and score products are under way, and the others find nobody to
wait for; with 1 waits give up whose data is not there when they look. The kernels must still let their copies and products in
flight end (that keeps the full limit), write NaN to the rows they had not
finished, set XN_DEVERR_WAIT and return with the CUDA context usable. No GPU
fault is involved: every copy and product completes normally."""
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

REPO = Path(__file__).resolve().parents[1]

CHILD = r"""
import itertools, json, math, sys
sys.path[:0] = [sys.argv[1] + "/random-things_b200"]
import torch
import xn_fused as xn
dev, page, h, hk, d = torch.device("cuda:0"), 16, 4, 2, int(sys.argv[2])
g = torch.Generator(device=dev).manual_seed(0)
res = []
for dtype in (torch.bfloat16, torch.float16):
    # Single tokens and chunks: requests shorter than the ring of tiles, longer ones, ones cut into pieces.
    for lens, new in (([0, 40, 3000, 9000], [1] * 4), ([0, 40, 3000, 9000], [20, 130, 64, 200])):
        kv = [a + b for a, b in zip(lens, new)]
        held = [-(-n // page) for n in kv]
        table = torch.zeros(len(kv), max(held), dtype=torch.int32)
        at = 0
        for i, c in enumerate(held):
            table[i, :c] = torch.arange(at, at + c)
            at += c
        k, v = (torch.randn(at, hk, page, d, device=dev, generator=g).to(dtype) for _ in range(2))
        start = [0] + list(itertools.accumulate(new))
        q = torch.randn(start[-1], h, d, device=dev, generator=g).to(dtype)
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        i64 = lambda x: torch.tensor(x, device=dev)
        for _ in range(3):
            out = xn.paged_attention(q, k, v, table.to(dev), i64(start), i64(kv), 1 / math.sqrt(d), max_new=max(new), err_flag=err)
        ref = []
        for i, (n, t) in enumerate(zip(lens, new)):
            kk, vv = (x[table[i, :held[i]].long().to(dev)].transpose(1, 2).reshape(-1, hk, d)[:n + t].float() for x in (k, v))
            s = torch.einsum("thgd,khd->hgtk", q[start[i]:start[i + 1]].float().view(t, hk, h // hk, d), kk) / math.sqrt(d)
            seen = torch.arange(n + t, device=dev) <= torch.arange(n, n + t, device=dev)[:, None]
            w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            ref.append(torch.einsum("hgtk,khd->thgd", w, vv).reshape(t, h * d))
        ref, got = torch.cat(ref), out.float()
        nan = torch.isnan(got)
        res.append(dict(err=int(err), nan=float(nan.float().mean()), off=float(torch.where(nan, 0.0, (got - ref).abs()).max())))
torch.cuda.synchronize()
ok = torch.ones(1000, device=dev).sum().item() == 1000.0
print(json.dumps([ok, res]))
"""


def _child(d, clocks=None):
    env = dict(os.environ)
    env.pop("XN_PAGED_WAIT_CLOCKS", None)
    if clocks is not None:
        env["XN_PAGED_WAIT_CLOCKS"] = str(clocks)
    out = subprocess.run([sys.executable, "-c", CHILD, str(REPO), str(d)], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    ok, res = json.loads(out.stdout.strip().splitlines()[-1])
    assert ok
    return res


@pytest.mark.parametrize("d", [32, 64, 128])
def test_waits_that_give_up_at_once(d):
    for r in _child(d, 0):
        assert r["err"] == 2 and r["nan"] == 1.0, r  # XN_DEVERR_WAIT


# Values are means of up to 9000 normal ones: below 6, so a rounding of the weights, of the output and of the
# reference's f32 sums together is below 3 half steps of 6 in bf16.
TOL = 3 * 6 * 2.0 ** -8


@pytest.mark.parametrize("d", [32, 64, 128])
def test_waits_that_give_up_soon(d):
    """Each row is right or NaN, and NaN come with the status."""
    for r in _child(d, 1):
        assert r["off"] <= TOL and (r["err"] == 2 if r["nan"] > 0 else r["err"] in (0, 2)), r


@pytest.mark.parametrize("d", [32, 64, 128])
def test_waits_at_their_own_limit(d):
    for r in _child(d):
        assert r["err"] == 0 and r["nan"] == 0.0 and r["off"] <= TOL, r
