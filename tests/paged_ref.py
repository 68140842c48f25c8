"""Plain 64-bit restatements of the paged-cache operators and of the 8-bit
RMSNorm, with the error bounds that the tests allow the kernels."""
from __future__ import annotations

import math

import torch

from helpers import U32, sum_error_bound

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def plan(lens, new, table, ring, state, page, cap):
    """The documented step on Python lists; None where it does not fit. Returns
    (q_start, kv_len, positions, slots, table, ring, state)."""
    n_pages, blocks = len(ring), len(table[0]) if table else 0
    table, ring = [list(r) for r in table], list(ring)
    head, count = state
    held = [-(-n // page) for n in lens]
    need = [0 if k < 0 else -(-(n + k) // page) - h for n, k, h in zip(lens, new, held)]
    if sum(need) > count or sum(max(k, 0) for k in new) > cap or any(h + k > blocks for h, k in zip(held, need)):
        return None
    taken = 0
    for i, k in enumerate(need):
        for j in range(k):
            table[i][held[i] + j] = ring[(head + taken) % n_pages]
            taken += 1
    back = 0
    for i, k in enumerate(new):
        if k < 0:
            for j in range(held[i]):
                ring[(head + count + back) % n_pages] = table[i][j]
                back += 1
    q_start, positions, slots = [0], [], []
    for i, k in enumerate(new):
        for p in range(lens[i], lens[i] + max(k, 0)):
            positions.append(p)
            slots.append(table[i][p // page] * page + p % page)
        q_start.append(len(positions))
    pad = [-1] * (cap - len(positions))
    kv = [0 if k < 0 else n + k for n, k in zip(lens, new)]
    return q_start, kv, positions + pad, slots + pad, table, ring, [(head + taken) % n_pages, count - taken + back]


def rope(x, cos, sin, interleaved):
    """x [N, h, d] rotated with cos / sin rows [N, d/2], in 64 bits; and the sum of the products' magnitudes."""
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
    else:
        a, b = x.chunk(2, -1)
    y1, y2 = a * c - b * s, a * s + b * c
    m1, m2 = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat([u, v], -1))
    return join(y1, y2), join(m1, m2)


def attention(q, k_pages, v_pages, table, q_start, kv_len, scale, window=0):
    """(ref, tol) [N, H, D] in 64 bits (NaN: rows outside all requests) on CPU tensors.

    The bound. A score is a dot product of D terms and a multiplication, so it
    is off by at most ds = 2 (D + 2) u scale sum |q_d k_d| (u = 2^-24; twice
    that for accumulators that truncate), exp2's argument by 2 u |s - m| log2 e
    more, exp2 itself by 2^-22 relative, or 2^-16 where 16-bit weights make more
    pointless. A weight is then off by a factor exp(e), e = the sum of those,
    so a quotient of sums by 2 e. 16-bit weights are rounded: half a step w, and
    half the smallest f16 (2^-25) where they are subnormal. The sums of n terms
    are off by sum_error_bound. Last, the output's rounding."""
    n, h, d = q.shape
    hk, page = k_pages.shape[1], k_pages.shape[2]
    g, n_pages = h // hk, k_pages.shape[0]
    u16 = 0.0 if q.dtype == torch.float32 else HALF_STEP[q.dtype]
    ref = torch.full((n, h, d), math.nan, dtype=torch.float64)
    tol = torch.zeros((n, h, d), dtype=torch.float64)
    for i in range(len(kv_len)):
        lo, hi, kv = int(q_start[i]), int(q_start[i + 1]), int(kv_len[i])
        if hi == lo:
            continue
        blocks = table[i, :-(-kv // page)].long()
        ok = (blocks >= 0) & (blocks < n_pages)
        at = torch.where(ok, blocks, 0)
        k, v = (torch.where(ok[:, None, None, None], x[at], 0).transpose(1, 2).reshape(-1, hk, d)[:kv].double()
                for x in (k_pages, v_pages))
        for t in range(lo, hi):
            p = kv - (hi - lo) + (t - lo)
            first = max(0, p - window + 1) if window else 0
            if p < 0:
                ref[t] = 0.0
                continue
            kk, vv = k[first:p + 1], v[first:p + 1]
            qq = q[t].double().view(hk, g, d)
            s = torch.einsum("hgd,khd->hgk", qq, kk) * scale
            w = torch.softmax(s, -1)
            ref[t] = torch.einsum("hgk,khd->hgd", w, vv).reshape(h, d)
            mag = torch.einsum("hgd,khd->hgk", qq.abs(), kk.abs()) * scale
            e = 2 * (d + 2) * U32 * mag + 2 * U32 * 1.5 * (s - s.amax(-1, keepdim=True)).abs() + (2.0 ** -22 if u16 == 0 else 2.0 ** -16)
            e = e.nan_to_num(0.0, 0.0, 0.0).amax(-1)[..., None]
            a = torch.einsum("hgk,khd->hgd", w, vv.abs())
            small = vv.abs().sum(0)[:, None] * (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
            tol[t] = (a * (2 * e + u16) + small + torch.as_tensor(sum_error_bound(kk.shape[0], 2 * a.numpy()))).reshape(h, d)
    tol += ref.abs().nan_to_num(0.0) * HALF_STEP[q.dtype] * 1.01 + 1e-30
    return ref, tol


def check_attention(got, ref, tol, what=""):
    """got [N, H * D]: every row of a request within the bound; infinities and NaN where the formula has them."""
    got = got.double().cpu().view(ref.shape)
    live = torch.ones(ref.shape[0], dtype=torch.bool)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN pattern differs"
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities differ"
    err = torch.where(fin, (got - ref).abs(), 0.0)
    bad = (err > tol) & fin
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {int(live.sum()) * ref.shape[1] * ref.shape[2]} off, worst "
                           f"{float((err / tol).max()):.2f} times the bound at {bad.nonzero()[0].tolist()}")
    return float((err / tol).max())


def rms_norm_q8(x, alpha, eps, branch, group):
    """(h, y, scales) in 64 bits, y and scales of the rounded h."""
    h = x if branch is None else (x.float() + branch.float()).to(x.dtype)
    f = h.double()
    y = f / torch.sqrt((f * f).mean(-1, keepdim=True) + eps) * alpha.double()
    scales = y.view(*y.shape[:-1], -1, group or y.shape[-1]).abs().amax(-1) / 448.0
    return h, y, scales if group else scales[..., 0]
