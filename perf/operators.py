"""The paged-cache serving operators, measured: their cases, their plain forms in elementary torch operations and
the calls a program makes of them.

Four operators that serve requests of different lengths from one pool of cache pages:
  plan    request lengths -> pages taken from / returned to a free ring, block tables, positions, slots;
  append  packed QKV projection -> RoPE on q and k, k and v rows into their pages;
  attend  a chunk of new tokens per request (one for decoding) over the pages, causal, with a sliding window;
  norm    RMSNorm with the residual's addition, output in 8 bits (e4m3) with one scale per row or column group.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESZ = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # One decoding step's bookkeeping for a small batch of streams: latency alone counts.
        dict(name="plan-decode-16", op="plan", requests=16, page=16, max_len=256, chunk=1, chunks=0, ending=0.0, mix=1),
        # A large server's step: thousands of requests, some ending, some with whole prompt chunks.
        dict(name="plan-mixed-4096", op="plan", requests=4096, page=16, max_len=4096, chunk=512, chunks=96, ending=0.05, mix=2),
        # The streaming speech decoder's step (16 streams, 16 heads of 64): the smallest append.
        dict(name="append-decode-16x16x64", op="append", dtype="bf16", tokens=16, heads=16, kv_heads=16, dim=64, page=16,
             interleaved=True, mix=3),
        # A prefill's worth of tokens of the 32 / 8 heads of 128 layer, half-split rotation.
        dict(name="append-prefill-32768x32x128", op="append", dtype="bf16", tokens=32768, heads=32, kv_heads=8, dim=128,
             page=64, interleaved=False, mix=4),
        # The speech decoder's attention step: 16 streams of up to 256 frames, one new frame each.
        dict(name="attend-decode-16x16x64", op="attend", dtype="bf16", requests=16, heads=16, kv_heads=16, dim=64, page=16,
             min_new=1, max_new=1, min_len=64, max_len=256, window=0, mix=5),
        # Decoding 64 requests of very different long histories, grouped heads: bound by the cache's bytes.
        dict(name="attend-decode-64x32x128-long", op="attend", dtype="bf16", requests=64, heads=32, kv_heads=8, dim=128, page=64,
             min_new=1, max_new=1, min_len=500, max_len=16000, window=0, mix=6),
        # One whole prompt of 8192 tokens into an empty cache: bound by the matrix products.
        dict(name="attend-prefill-1x8192x32x128", op="attend", dtype="bf16", requests=1, heads=32, kv_heads=8, dim=128, page=64,
             min_new=8192, max_new=8192, min_len=0, max_len=0, window=0, mix=7),
        # A continuous batch: ragged chunks, single tokens among them, over ragged histories; half precision.
        dict(name="attend-chunk-12x24x128-ragged", op="attend", dtype="f16", requests=12, heads=24, kv_heads=8, dim=128, page=32,
             min_new=1, max_new=777, min_len=0, max_len=5000, window=0, mix=8),
        # The codec's transformer on 4 streams: 8 heads of 64, context 250 as a sliding window, 32-bit values.
        dict(name="attend-window-4x8x64-f32", op="attend", dtype="f32", requests=4, heads=8, kv_heads=8, dim=64, page=16,
             min_new=100, max_new=250, min_len=0, max_len=1000, window=250, mix=9),
        # The norm in front of a decoding step's 8-bit products.
        dict(name="norm-decode-16x4096", op="norm", dtype="bf16", rows=16, cols=4096, group=0, residual=True, mix=10),
        # The same of a prefill, scales by groups of 128 columns.
        dict(name="norm-prefill-32768x4096", op="norm", dtype="bf16", rows=32768, cols=4096, group=128, residual=True, mix=11),
        # Rows of a ragged width, 32-bit values, no residual.
        dict(name="norm-4111x1333-f32", op="norm", dtype="f32", rows=4111, cols=1333, group=0, residual=False, mix=12),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "norm", "norm"])
    mix = rng.randrange(1 << 30)
    dtype = rng.choice(["bf16", "f16", "bf16", "f16", "f32"])
    page = rng.choice([8, 16, 32, 64, 128, 256])
    if op == "plan":
        requests = _log(rng, 1, 4096)
        return dict(op=op, requests=requests, page=page, max_len=_log(rng, 1, 4096), chunk=_log(rng, 1, 512),
                    chunks=rng.randint(0, min(requests, 96)), ending=rng.choice([0.0, 0.05, 0.5]), mix=mix)
    if op == "append":
        dim, kv_heads, group = rng.choice([32, 64, 128]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
        top = 32768 * 48 * 128 // ((group + 2) * kv_heads * dim * (2 if dtype == "f32" else 1))
        return dict(op=op, dtype=dtype, tokens=_log(rng, 1, min(top, 32768)), heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    page=page, interleaved=rng.random() < 0.5, mix=mix)
    if op == "norm":
        cols = rng.choice([_log(rng, 16, 16384), 64 * _log(rng, 1, 256), 128 * _log(rng, 1, 128)])
        group = rng.choice([0, 32, 64, 128])
        group = group if group and cols % group == 0 else 0
        top = 32768 * 4096 // (cols * (2 if dtype == "f32" else 1))
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, max(1, min(top, 65536))), cols=cols, group=group,
                    residual=rng.random() < 0.7, mix=mix)
    dim, kv_heads, group = rng.choice([32, 64, 128]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8])
    window = rng.choice([0, 0, _log(rng, 1, 4096)])
    if rng.random() < 0.5:  # decoding: one new token, or a few
        new, requests = rng.choice([1, 1, 1, rng.randint(2, 6)]), _log(rng, 1, 128)
        most = 64 * 16000 * 8 * 128 // (requests * kv_heads * dim * (2 if dtype == "f32" else 1))
        length = _log(rng, 1, max(2, min(most, 32000)))
        return dict(op=op, dtype=dtype, requests=requests, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page,
                    min_new=1, max_new=new, min_len=rng.choice([0, length // 3, length]), max_len=length, window=window, mix=mix)
    requests, new, length = _log(rng, 1, 24), _log(rng, 2, 4096), _log(rng, 1, 16000)
    # Scores of the padded plain form, and the gathered keys, within those of the largest listed cases.
    while (requests * kv_heads * group * new * (new + length) > 32 * 8192 * 8192 or
           requests * kv_heads * dim * (new + length) * (2 if dtype == "f32" else 1) > 64 * 16000 * 8 * 128):
        new, length = (new + 1) // 2, (length + 1) // 2
    return dict(op=op, dtype=dtype, requests=requests, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page,
                min_new=rng.choice([0, 1, new]), max_new=new, min_len=0, max_len=length, window=window, mix=mix)


# -- what a case's lengths are (by the case alone) ---------------------------------------------------------------

def _plan_lengths(case):
    """(lens, new) of the requests: most decode one token, `chunks` of them bring up to `chunk`, some end (-1)."""
    rng, n = random.Random(case["mix"]), case["requests"]
    lens = [rng.randint(0, case["max_len"]) for _ in range(n)]
    new = [1] * n
    for i in rng.sample(range(n), min(case["chunks"], n)):
        new[i] = rng.randint(0, case["chunk"])
    for i in range(n):
        if rng.random() < case["ending"]:
            new[i] = -1
    return lens, new


def _attend_lengths(case):
    """(tokens cached before, new tokens) of the requests; the largest of both occur."""
    rng, n = random.Random(case["mix"]), case["requests"]
    lens = [rng.randint(case["min_len"], case["max_len"]) for _ in range(n)]
    new = [rng.randint(case["min_new"], case["max_new"]) for _ in range(n)]
    lens[rng.randrange(n)] = case["max_len"]
    new[rng.randrange(n)] = case["max_new"]
    return lens, new


def _ceil(a, b):
    return -(-a // b)


# -- inputs ------------------------------------------------------------------------------------------------------

def _xn():
    pkg = str(Path(__file__).resolve().parents[1] / "random-things_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import xn_fused

    return xn_fused


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case, "xn": _xn() if own else None}
    dev = torch.device("cuda")
    dtype = DTYPES.get(case.get("dtype"))

    def randn(*shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=dev, dtype=torch.float32) * std + mean).to(dtype)

    def pool(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    if case["op"] == "plan":
        lens, new = _plan_lengths(case)
        page = case["page"]
        held = [_ceil(n, page) for n in lens]
        need = [max(0, _ceil(n + max(k, 0), page) - h) for n, k, h in zip(lens, new, held)]
        blocks = max(h + k for h, k in zip(held, need)) + 1
        n_pages = sum(held) + 2 * sum(need) + 8
        ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
        table = torch.full((len(lens), blocks), -1, dtype=torch.int32, device=dev)
        cols = torch.arange(blocks, device=dev)
        taken = torch.tensor(held, device=dev)
        table[cols[None, :] < taken[:, None]] = ids[:sum(held)]
        head = int(torch.randint(0, n_pages, (1,), generator=g, device=dev))
        ring = torch.full((n_pages,), -1, dtype=torch.int32, device=dev)
        free = ids[sum(held):]
        ring[(head + torch.arange(free.numel(), device=dev)) % n_pages] = free
        total = sum(max(k, 0) for k in new)
        s.update(lens=torch.tensor(lens, dtype=torch.int64, device=dev), new=torch.tensor(new, dtype=torch.int64, device=dev),
                 table=table, ring=ring, state=torch.tensor([head, free.numel()], dtype=torch.int64, device=dev),
                 cap=total + 7)
    elif case["op"] == "append":
        n, h, hk, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        n_pages = _ceil(n, page) + 4
        max_pos = 8192
        half = d // 2
        inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        ang = torch.arange(max_pos, dtype=torch.float64, device=dev)[:, None] * inv[None, :]
        s.update(qkv=randn(n, (h + 2 * hk) * d), cos=ang.cos().to(dtype), sin=ang.sin().to(dtype),
                 k=torch.zeros((n_pages, hk, page, d), dtype=dtype, device=dev),
                 v=torch.zeros((n_pages, hk, page, d), dtype=dtype, device=dev),
                 positions=torch.randint(0, max_pos, (n,), generator=g, device=dev),
                 slots=torch.randperm(n_pages * page, generator=g, device=dev)[:n])
    elif case["op"] == "attend":
        lens, new = _attend_lengths(case)
        page, h, hk, d = case["page"], case["heads"], case["kv_heads"], case["dim"]
        total = [a + b for a, b in zip(lens, new)]
        held = [_ceil(n, page) for n in total]
        n_pages, blocks = sum(held) + 2, max(max(held), 1)
        ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
        table = torch.full((len(lens), blocks), -1, dtype=torch.int32, device=dev)
        table[torch.arange(blocks, device=dev)[None, :] < torch.tensor(held, device=dev)[:, None]] = ids[:sum(held)]
        start = torch.zeros(len(lens) + 1, dtype=torch.int64, device=dev)
        start[1:] = torch.cumsum(torch.tensor(new, device=dev), 0)
        s.update(q=randn(sum(new), h, d), k=pool(n_pages, hk, page, d), v=pool(n_pages, hk, page, d), table=table, start=start,
                 kv=torch.tensor(total, dtype=torch.int64, device=dev), scale=1.0 / math.sqrt(d), max_new=max(new),
                 max_kv=max(total))
        if own:  # a program keeps it from step to step
            s["workspace"] = s["xn"].paged_attention_workspace(sum(new), len(lens), h, hk, d, max(new), dtype, dev)
    else:
        rows, cols = case["rows"], case["cols"]
        s.update(x=randn(rows, cols), alpha=randn(cols, std=0.02, mean=1.0),
                 branch=randn(rows, cols, std=0.5) if case["residual"] else None, eps=1e-5)
    return s


# -- one pass ----------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        xn = s["xn"]
        if case["op"] == "plan":
            p = xn.paged_plan(s["lens"], s["new"], s["table"], s["ring"], s["state"], case["page"], s["cap"])
            return {"q_start": p.q_start, "kv_len": p.kv_len, "positions": p.positions, "slots": p.slots,
                    "ring_state": p.ring_state, "table": s["table"], "ring": s["ring"]}
        if case["op"] == "append":
            q = xn.paged_append_rope(s["qkv"], case["heads"], case["kv_heads"], s["cos"], s["sin"], s["k"], s["v"],
                                     s["positions"], s["slots"], interleaved=case["interleaved"])
            return {"q": q, "k": s["k"], "v": s["v"]}
        if case["op"] == "attend":
            return xn.paged_attention(s["q"], s["k"], s["v"], s["table"], s["start"], s["kv"], s["scale"],
                                      max_new=s["max_new"], window=case["window"], workspace=s["workspace"])
        q, scales, h = xn.rms_norm_q8(s["x"], s["alpha"], s["eps"], branch=s["branch"], group=case["group"])
        return {"q": q, "scales": scales, "h": h} if case["residual"] else {"q": q, "scales": scales}
    if case["op"] == "plan":
        return _plan(s)
    if case["op"] == "append":
        return _append(s)
    if case["op"] == "attend":
        return _attend(s)
    return _norm(s)


def _plan(s):
    page, cap, lens, table, ring = s["case"]["page"], s["cap"], s["lens"], s["table"].clone(), s["ring"].clone()
    n_pages, blocks = ring.numel(), table.shape[1]
    ends = s["new"] < 0
    new = s["new"].clamp(min=0)
    kv_len = torch.where(ends, 0, lens + new)
    held = (lens + page - 1) // page
    need = torch.where(ends, 0, (kv_len + page - 1) // page - held)
    back = torch.where(ends, held, 0)
    zero = torch.zeros(1, dtype=torch.int64, device=lens.device)
    q_start = torch.cat([zero, torch.cumsum(new, 0)])
    need_to, back_to = torch.cumsum(need, 0), torch.cumsum(back, 0)
    head, count = s["state"][0], s["state"][1]
    col = torch.arange(blocks, device=lens.device)[None, :]
    # Pages taken: a request's new blocks, in the order of requests, from the ring's head.
    at = head + (need_to - need - held)[:, None] + col
    taken = (col >= held[:, None]) & (col < (held + need)[:, None])
    out = torch.where(taken, ring[at % n_pages], table)
    # Pages returned: an ending request's blocks, behind the ring's last entry.
    to = head + count + (back_to - back)[:, None] + col
    given = col < back[:, None]
    spare = torch.cat([ring, ring[:1]])  # one entry more takes what is not given
    spare.scatter_(0, torch.where(given, to % n_pages, n_pages).reshape(-1), table.reshape(-1))
    # Tokens.
    tok = torch.arange(cap, device=lens.device)
    live = tok < q_start[-1]
    req = torch.searchsorted(q_start[1:], tok, right=True).clamp(max=lens.numel() - 1)
    pos = lens[req] + tok - q_start[req]
    blk = out[req, (pos // page).clamp(max=blocks - 1)].to(torch.int64)
    return {"q_start": q_start, "kv_len": kv_len, "positions": torch.where(live, pos, -1),
            "slots": torch.where(live, blk * page + pos % page, -1),
            "ring_state": torch.stack([(head + need_to[-1]) % n_pages, count - need_to[-1] + back_to[-1]]),
            "table": out, "ring": spare[:n_pages]}


def _append(s):
    case = s["case"]
    n, h, hk, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    dtype = s["qkv"].dtype
    x = s["qkv"].float().view(n, h + 2 * hk, d)
    c, sn = s["cos"].float()[s["positions"]][:, None, :], s["sin"].float()[s["positions"]][:, None, :]
    qk = x[:, :h + hk]
    if case["interleaved"]:
        a, b = qk[..., 0::2], qk[..., 1::2]
        y = torch.stack([a * c - b * sn, a * sn + b * c], -1).reshape(n, h + hk, d)
    else:
        a, b = qk[..., :d // 2], qk[..., d // 2:]
        y = torch.cat([a * c - b * sn, a * sn + b * c], -1)
    at, off = s["slots"] // page, s["slots"] % page
    s["k"][at, :, off] = y[:, h:].to(dtype)
    s["v"][at, :, off] = x[:, h + hk:].to(dtype)
    return {"q": y[:, :h].to(dtype), "k": s["k"], "v": s["v"]}


def _attend(s):
    """Scores of the padded batch [requests, kv heads, new * group, keys], softmax, weighted sum."""
    case, q, table, start, kv = s["case"], s["q"], s["table"], s["start"], s["kv"]
    page, h, hk, d = case["page"], case["heads"], case["kv_heads"], case["dim"]
    r, t, g, n = kv.numel(), s["max_new"], h // hk, q.shape[0]
    dev = q.device
    if n == 0:
        return q.reshape(0, h * d)
    length = table.shape[1] * page
    pages = table.clamp(min=0).to(torch.int64)
    k = s["k"][pages].permute(0, 2, 1, 3, 4).reshape(r, hk, length, d).float()
    new = start[1:] - start[:-1]
    tok = torch.arange(t, device=dev)[None, :]
    rows = (start[:-1, None] + tok).clamp(max=n - 1)
    x = q[rows].float().view(r, t, hk, g, d).permute(0, 2, 1, 3, 4).reshape(r, hk, t * g, d)
    x = torch.matmul(x, k.transpose(2, 3)).mul_(s["scale"])
    del k
    pos = (kv - new)[:, None] + tok
    key = torch.arange(length, device=dev)
    seen = key <= pos[:, :, None]
    if case["window"]:
        seen &= key > pos[:, :, None] - case["window"]
    x = x.view(r, hk, t, g, length).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    x = x.div_(x.sum(-1, keepdim=True)).view(r, hk, t * g, length)
    held = key[None, :] < kv[:, None]
    v = s["v"][pages].permute(0, 2, 1, 3, 4).reshape(r, hk, length, d).float()
    v = torch.where(held[:, None, :, None], v, 0.0)
    o = torch.matmul(x, v).view(r, hk, t, g, d).permute(0, 2, 1, 3, 4)
    at = torch.arange(n, device=dev)
    req = torch.searchsorted(start[1:], at, right=True)
    return o[req, at - start[req]].reshape(n, h * d).to(q.dtype)


def _norm(s):
    case, dtype = s["case"], s["x"].dtype
    h = s["x"] if s["branch"] is None else (s["x"].float() + s["branch"].float()).to(dtype)
    f = h.float()
    y = f / torch.sqrt((f * f).mean(-1, keepdim=True) + s["eps"]) * s["alpha"].float()
    group = case["group"] or case["cols"]
    y = y.view(case["rows"], -1, group)
    scales = y.abs().amax(-1) / 448.0
    q = torch.where(scales[..., None] > 0, y / scales[..., None], 0.0).to(torch.float8_e4m3fn)
    out = {"q": q.view(case["rows"], case["cols"]), "scales": scales if case["group"] else scales.view(-1)}
    return out if s["branch"] is None else {**out, "h": h}


# -- the definition in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    rows, cols = case["rows"], case["cols"]
    h = s["x"].double() if s["branch"] is None else s["x"].double() + s["branch"].double()
    hr = h.to(s["x"].dtype).double()
    y = s["alpha"].double() * hr * torch.rsqrt(hr.pow(2).sum(-1, keepdim=True) / cols + s["eps"])
    scales = y.view(rows, -1, case["group"] or cols).abs().max(-1).values / 448.0
    q = (y.view(rows, scales.shape[1], -1) / scales.unsqueeze(-1).clamp(min=1e-300)).view(rows, cols)
    out = {"q": q, "scales": scales if case["group"] else scales.view(-1)}
    return out if s["branch"] is None else {**out, "h": h}


def _exact_append(s):
    case = s["case"]
    h, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    x = s["qkv"].double().view(-1, h + 2 * hk, d)
    rot = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]].unsqueeze(1)
    qk = x[:, :h + hk]
    if case["interleaved"]:
        z = torch.view_as_complex(qk.reshape(*qk.shape[:2], d // 2, 2).contiguous()) * rot
        y = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(qk[..., :d // 2].contiguous(), qk[..., d // 2:].contiguous()) * rot
        y = torch.cat([z.real, z.imag], -1)

    def cache(rows):
        flat = torch.zeros((s["k"].shape[0] * page, hk, d), dtype=torch.float64, device=x.device)
        flat[s["slots"]] = rows
        return flat.view(-1, page, hk, d).transpose(1, 2).contiguous()

    return {"q": y[:, :h].contiguous(), "k": cache(y[:, h:]), "v": cache(x[:, h + hk:])}


def _exact_attend(s):
    case = s["case"]
    h, hk, d, page, w = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    lens, new = _attend_lengths(case)
    if work(case)["flops"] > 2e13:
        return None
    out = torch.zeros((s["q"].shape[0], h, d), dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, t) in enumerate(zip(lens, new)):
        if t == 0:
            continue
        pages = s["table"][i, :_ceil(n + t, page)].long()
        first = max(0, n - w + 1) if w else 0
        k = s["k"][pages].transpose(1, 2).reshape(-1, hk, d)[first:n + t].double()
        v = s["v"][pages].transpose(1, 2).reshape(-1, hk, d)[first:n + t].double()
        step = max(1, (1 << 27) // (k.shape[0] * h))
        for lo in range(0, t, step):
            hi = min(t, lo + step)
            q = s["q"][at + lo:at + hi].double().view(hi - lo, hk, h // hk, d)
            x = torch.einsum("thgd,khd->hgtk", q, k) * s["scale"]
            behind = torch.arange(n + lo, n + hi, device="cuda")[:, None] - torch.arange(first, n + t, device="cuda")[None, :]
            x[..., (behind < 0) | (behind >= (w or 1 << 60))] = -math.inf
            out[at + lo:at + hi] = torch.einsum("hgtk,khd->thgd", torch.softmax(x, -1), v).reshape(hi - lo, h, d)
        at += t
    return out.view(-1, h * d)


# -- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    if case["op"] == "plan":
        lens, new = _plan_lengths(case)
        page = case["page"]
        tokens = sum(max(k, 0) for k in new)
        moved = sum(_ceil(n, page) if k < 0 else _ceil(n + k, page) - _ceil(n, page) for n, k in zip(lens, new))
        first = sum(1 for n, k in zip(lens, new) if k > 0 and n % page)  # the page a request's tokens begin in
        return {"bytes": 8 * (4 * len(lens) + 1) + 16 * (tokens + 7) + 8 * moved + 4 * first + 32, "flops": 0}
    if case["op"] == "append":
        n, h, hk, d, e = case["tokens"], case["heads"], case["kv_heads"], case["dim"], ESZ[case["dtype"]]
        return {"bytes": n * (2 * (h + 2 * hk) * d * e + 16) + min(n, 8192) * d * e, "flops": 3 * n * (h + hk) * d}
    if case["op"] == "norm":
        n, e = case["rows"] * case["cols"], ESZ[case["dtype"]]
        scales = case["rows"] * (case["cols"] // case["group"] if case["group"] else 1)
        return {"bytes": n * (e * (3 if case["residual"] else 1) + 1) + 4 * scales + case["cols"] * e, "flops": 6 * n}
    lens, new = _attend_lengths(case)
    h, hk, d, e, w = case["heads"], case["kv_heads"], case["dim"], ESZ[case["dtype"]], case["window"]
    pairs = keys = 0
    for n, t in zip(lens, new):
        if not t:
            continue
        keys += n + t - (max(0, n - w + 1) if w else 0)
        if w:
            short = min(t, max(0, w - n))  # rows that see less than the window: n + 1 .. n + short keys
            pairs += short * n + short * (short + 1) // 2 + (t - short) * w
        else:
            pairs += t * n + t * (t + 1) // 2
    return {"bytes": 2 * keys * hk * d * e + 2 * sum(new) * h * d * e + 4 * _ceil(keys, case["page"]) + 16 * len(lens),
            "flops": 4 * pairs * h * d}
