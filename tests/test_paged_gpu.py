"""The paged-cache operators on the GPU against their 64-bit restatements:
plans exactly, the append and the attention within the derived bounds, over
ragged batches, every page size and layout, windows, empty rows, stale and
non-finite cache rows, bad tables, streams and captured graphs."""
import itertools
import math

import pytest
import torch

import paged_ref
from paged_ref import HALF_STEP, check_attention

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def i64(v, dev="cpu"):
    return torch.tensor(v, dtype=torch.int64, device=dev)


# -- plan ------------------------------------------------------------------------

def _plan_state(seed, n, page, max_len, blocks, spare):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, max_len + 1, (n,), generator=g).tolist()
    held = [-(-k // page) for k in lens]
    n_pages = sum(held) + spare
    ids = torch.randperm(n_pages, generator=g).tolist()
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-7] * (blocks - h))
        at += h
    head = int(torch.randint(0, n_pages, (1,), generator=g))
    ring = [-9] * n_pages
    for j, p in enumerate(ids[at:]):
        ring[(head + j) % n_pages] = p
    return lens, table, ring, [head, spare]


def _run_plan(xn, dev, lens, new, table, ring, state, page, cap, err=None):
    t, r = torch.tensor(table, dtype=torch.int32, device=dev), torch.tensor(ring, dtype=torch.int32, device=dev)
    p = xn.paged_plan(i64(lens, dev), i64(new, dev), t, r, i64(state, dev), page, cap, err_flag=err)
    return (p.q_start.tolist(), p.kv_len.tolist(), p.positions.tolist(), p.slots.tolist(), t.tolist(), r.tolist(),
            p.ring_state.tolist())


@pytest.mark.parametrize("n,page,max_len,chunk", [(1, 8, 0, 1), (1, 16, 40, 1), (7, 16, 100, 33), (33, 64, 500, 1),
                                                  (513, 8, 90, 5), (1500, 32, 64, 3), (8192, 16, 30, 2)])
def test_plan(xn, cuda, n, page, max_len, chunk):
    g = torch.Generator().manual_seed(n)
    new = torch.randint(-1, chunk + 1, (n,), generator=g).tolist()
    blocks = -(-(max_len + chunk) // page) + 1
    lens, table, ring, state = _plan_state(n, n, page, max_len, blocks, n * (chunk // page + 1) + 3)
    total = sum(max(k, 0) for k in new)
    for cap in (total, total + 9):
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        want = paged_ref.plan(lens, new, table, ring, state, page, cap)
        assert want is not None
        assert list(want) == list(_run_plan(xn, cuda, lens, new, table, ring, state, page, cap, err))
        assert int(err) == 0


def test_plan_no_requests(xn, cuda):
    none, ring = i64([], cuda), torch.tensor([5, 6], dtype=torch.int32, device=cuda)
    p = xn.paged_plan(none, none, torch.empty(0, 3, dtype=torch.int32, device=cuda), ring, i64([1, 1], cuda), 8, 4)
    assert p.q_start.tolist() == [0] and p.slots.tolist() == [-1] * 4 and p.ring_state.tolist() == [1, 1]


@pytest.mark.parametrize("what", ["pages", "tokens", "width", "negative", "long", "ring", "head"])
def test_plan_that_does_not_fit_changes_nothing(xn, cuda, what):
    lens, new, page, cap = [5, 16, 0], [4, 9, 20], 8, 33
    table, ring, state = [[0, -1, -1], [1, 2, -1], [-1, -1, -1]][:3], [9, 8, 7, 6, 5, 4, 3, 2, 1, 0], [8, 6]
    table = [r + [-1] for r in table]
    full = xn.XN_DEVERR_FULL
    bit = {"pages": full, "tokens": full, "width": full}.get(what, xn.XN_DEVERR_RANGE)
    ok = _run_plan(xn, cuda, lens, new, table, ring, state, page, cap)
    assert list(ok) == list(paged_ref.plan(lens, new, table, ring, state, page, cap))
    if what == "pages":
        state = [8, 4]
    elif what == "tokens":
        cap = 32
    elif what == "width":
        new = [4, 9 + 16, 4]
    elif what == "negative":
        lens = [5, -16, 0]
    elif what == "long":
        lens = [5, 33, 0]
    elif what == "ring":
        state = [8, 11]
    else:
        state = [10, 6]
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = _run_plan(xn, cuda, lens, new, table, ring, state, page, cap, err)
    assert int(err) == bit
    assert list(got) == [[0] * 4, lens, [-1] * cap, [-1] * cap, table, ring, state]


def test_plan_bad_page_loses_its_tokens_only(xn, cuda):
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = _run_plan(xn, cuda, [3, 8], [2, 2], [[99, -1], [1, -1]], [4, 5, 2, 3], [2, 2], 8, 4, err)
    assert int(err) == xn.XN_DEVERR_RANGE
    assert got[2] == [3, 4, 8, 9] and got[3] == [-1, -1, 16, 17]


# -- pools -----------------------------------------------------------------------

LAYOUTS = ["head-major", "slot-major", "k and v in one", "padded"]


def make_pools(n_pages, hk, page, d, dtype, dev, layout, fill):
    """Two pools [n_pages, hk, page, d] as views of differently laid out memory."""
    if layout == "head-major":
        k, v = (torch.full((n_pages, hk, page, d), fill, dtype=dtype, device=dev) for _ in range(2))
    elif layout == "slot-major":
        k, v = (torch.full((n_pages, page, hk, d), fill, dtype=dtype, device=dev).transpose(1, 2) for _ in range(2))
    elif layout == "k and v in one":
        both = torch.full((n_pages, 2, hk, page, d), fill, dtype=dtype, device=dev)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (torch.full((n_pages, hk, page, d + 24), fill, dtype=dtype, device=dev)[..., :d] for _ in range(2))
    return k, v


# -- append ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d,h,hk", [(32, 3, 3), (64, 16, 16), (128, 8, 2), (128, 5, 1)])
@pytest.mark.parametrize("interleaved", [True, False])
def test_append(xn, cuda, dtype, d, h, hk, interleaved):
    dt, page = DT[dtype], 16
    for n, layout in ((1, "head-major"), (37, "slot-major"), (131, "k and v in one"), (5, "padded")):
        g = torch.Generator().manual_seed(n + d)
        n_pages = -(-n // page) + 2
        qkv = torch.randn(n, (h + 2 * hk) * d, generator=g).to(dt)
        ang = torch.rand(50, d // 2, generator=g) * 6
        cos, sin = ang.cos().to(dt), ang.sin().to(dt)
        pos = torch.randint(0, 50, (n,), generator=g)
        slots = torch.randperm(n_pages * page, generator=g)[:n]
        if n > 2:
            slots[n // 2] = -1
        k, v = make_pools(n_pages, hk, page, d, dt, cuda, layout, 7.0)
        q = torch.full((n, h, d), 5.0, dtype=dt, device=cuda)
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        xn.paged_append_rope(qkv.to(cuda), h, hk, cos.to(cuda), sin.to(cuda), k, v, pos.to(cuda), slots.to(cuda),
                             interleaved=interleaved, q_out=q, err_flag=err)
        assert int(err) == 0
        x = qkv.view(n, h + 2 * hk, d)
        y, mag = paged_ref.rope(x[:, :h + hk], cos[pos], sin[pos], interleaved)
        # Two f32 operations on exact or once-rounded products, then the output's half step.
        tol = 3 * 2.0 ** -24 * mag + HALF_STEP[dt] * 1.01 * y.abs() + (2.0 ** -25 if dtype == "f16" else 1e-40)
        want_k, want_v = (torch.full((n_pages * page, hk, d), 7.0, dtype=torch.float64) for _ in range(2))
        tol_k = torch.zeros_like(want_k)
        live = slots >= 0
        want_k[slots[live]], tol_k[slots[live]] = y[live, h:], tol[live, h:]
        want_v[slots[live]] = x[live, h + hk:].double()
        flat = lambda t: t.double().cpu().transpose(1, 2).reshape(n_pages * page, hk, d)  # noqa: E731
        assert ((flat(k) - want_k).abs() <= tol_k).all()
        assert torch.equal(flat(v), want_v)
        want_q = torch.where(live[:, None, None], y[:, :h], 5.0)
        assert ((q.double().cpu() - want_q).abs() <= torch.where(live[:, None, None], tol[:, :h], 0.0)).all()


def test_append_matches_the_ring_append(xn, cuda):
    """f32: the same rotation as kv_append_rope up to the rounding of its products; v bit for bit."""
    b, h, d, t = 2, 4, 64, 3
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(b, t, 3 * h * d, generator=g).to(cuda)
    ang = torch.rand(20, d // 2, generator=g) * 6
    cos, sin = ang.cos().to(cuda), ang.sin().to(cuda)
    rk, rv = torch.zeros(b, h, 8, d, device=cuda), torch.zeros(b, h, 8, d, device=cuda)
    rq = xn.kv_append_rope(qkv, h, cos, sin, rk, rv, 4)
    k, v = torch.zeros(b, h, 8, d, device=cuda), torch.zeros(b, h, 8, d, device=cuda)
    pos = i64([4, 5, 6] * b, cuda)
    q = xn.paged_append_rope(qkv.view(b * t, -1), h, h, cos, sin, k, v, pos, pos + i64([0] * t + [8] * t, cuda))
    assert torch.equal(v, rv)
    assert torch.allclose(k, rk, rtol=0, atol=1e-6)
    assert torch.allclose(q.view(b, t, h, d).transpose(1, 2), rq, rtol=0, atol=1e-6)


def test_append_bad_slots_and_positions(xn, cuda):
    h, hk, d, page = 2, 1, 32, 8
    qkv = torch.ones(5, (h + 2 * hk) * d, device=cuda)
    cos, sin = torch.ones(10, d // 2, device=cuda), torch.zeros(10, d // 2, device=cuda)
    k, v = (torch.zeros(2, hk, page, d, device=cuda) for _ in range(2))
    q = torch.zeros(5, h, d, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    xn.paged_append_rope(qkv, h, hk, cos, sin, k, v, i64([0, 10, 3, -1, 4], cuda), i64([16, 0, -5, 1, 2], cuda), q_out=q,
                         err_flag=err)
    assert int(err) == xn.XN_DEVERR_RANGE
    assert q[4].eq(1).all() and q[:4].eq(0).all()
    assert k[0, 0, 2].eq(1).all() and k.sum() == d and v.sum() == d


# -- attention -------------------------------------------------------------------

class Batch:
    """A ragged batch on pages, every row of the pool that no request holds filled with `stale`."""

    def __init__(self, dev, dtype, h, hk, d, page, lens, new, seed=0, layout="head-major", stale=math.nan, packed=False, kv=None):
        g = torch.Generator().manual_seed(seed)
        dt = DT[dtype]
        self.kv = kv or [a + b for a, b in zip(lens, new)]
        held = [-(-n // page) for n in self.kv]
        self.n_pages = sum(held) + 2
        ids = torch.randperm(self.n_pages, generator=g).int()
        table = torch.full((len(lens), max(held) + 1), 2 ** 31 - 1, dtype=torch.int32)  # not to be read
        k = torch.full((self.n_pages, hk, page, d), stale, dtype=torch.float32)
        v = k.clone()
        at = 0
        for i, c in enumerate(held):
            table[i, :c] = ids[at:at + c]
            for j in range(c):
                rows = min(page, self.kv[i] - j * page)
                k[ids[at + j], :, :rows] = torch.randn(hk, rows, d, generator=g)
                v[ids[at + j], :, :rows] = torch.randn(hk, rows, d, generator=g)
            at += c
        self.k, self.v, self.table = k.to(dt), v.to(dt), table
        self.start = [0] + list(itertools.accumulate(new))
        n = self.start[-1]
        self.q = torch.randn(n, h, d, generator=g).to(dt)
        self.scale, self.max_new = 1.0 / math.sqrt(d), max(new)
        self.dk, self.dv = make_pools(self.n_pages, hk, page, d, dt, dev, layout, stale)
        self.dev, self.packed, self.h, self.hk, self.d = dev, packed, h, hk, d

    def run(self, xn, window=0, extra=0, max_new=None, **kw):
        self.dk.copy_(self.k)
        self.dv.copy_(self.v)
        n, h, d, dev = self.q.shape[0], self.h, self.d, self.dev
        q = self.q.to(dev)
        if self.packed:  # q as the first heads of a packed projection
            wide = torch.full((n, h + 2 * self.hk, d), math.nan, dtype=q.dtype, device=dev)
            wide[:, :h] = q
            q = wide[:, :h]
        if extra:
            q = torch.cat([q, torch.full((extra, h, d), math.nan, dtype=q.dtype, device=dev)])
        out = torch.full((n + extra, h * d), 3.0, dtype=q.dtype, device=dev)
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        got = xn.paged_attention(q, self.dk, self.dv, self.table.to(dev), i64(self.start, dev), i64(self.kv, dev), self.scale,
                                 max_new=self.max_new if max_new is None else max_new, window=window, err_flag=err, out=out, **kw)
        assert got is out and int(err) == 0
        if extra:
            assert out[n:].eq(3.0).all()
        return out[:n]

    def check(self, xn, window=0, **kw):
        ref, tol = paged_ref.attention(self.q, self.k, self.v, self.table, self.start, self.kv, self.scale, window)
        return check_attention(self.run(xn, window, **kw), ref, tol)


DECODE = [([0], [1]), ([15], [1]), ([16, 300, 64, 63, 127, 1], [1] * 6), ([700], [1]), ([5000, 3, 260], [1, 1, 1]),
          ([40, 100, 0], [2, 0, 3])]
CHUNK = [([0], [17]), ([0], [130]), ([100, 0, 7, 511, 64], [33, 64, 0, 1, 129]), ([3000], [65]), ([2, 900], [257, 100])]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("h,hk,d", [(4, 4, 64), (8, 2, 128), (3, 1, 32), (7, 1, 128), (16, 1, 64), (10, 2, 32)])
def test_attention_decode(xn, cuda, dtype, h, hk, d):
    for i, (lens, new) in enumerate(DECODE):
        b = Batch(cuda, dtype, h, hk, d, (8, 16, 32, 64, 128, 256)[i], lens, new, seed=i, layout=LAYOUTS[i % 4], packed=i % 2 == 1)
        b.check(xn, window=(0, 0, 0, 250, 0, 5)[i], extra=i % 3)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("h,hk,d", [(4, 4, 64), (8, 2, 128), (3, 1, 32), (5, 1, 128), (8, 1, 64), (20, 1, 32)])
def test_attention_chunk(xn, cuda, dtype, h, hk, d):
    for i, (lens, new) in enumerate(CHUNK):
        b = Batch(cuda, dtype, h, hk, d, (16, 8, 32, 256, 128)[i], lens, new, seed=i, layout=LAYOUTS[i % 4], packed=i % 2 == 0)
        b.check(xn, window=(0, 50, 0, 0, 300)[i], extra=i % 3)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 128, 1 << 40])
def test_attention_windows(xn, cuda, dtype, window):
    Batch(cuda, dtype, 4, 2, 64, 16, [0, 200, 64], [70, 3, 130]).check(xn, window=window)
    Batch(cuda, dtype, 4, 2, 128, 32, [0, 200, 64], [1, 1, 2]).check(xn, window=window)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("new", [[5, 9, 4], [40, 200, 70]])
def test_attention_rows_without_keys(xn, cuda, dtype, new):
    """kv_len below the number of new tokens: the first tokens sit at negative positions and give zeros."""
    b = Batch(cuda, dtype, 4, 2, 64, 16, [0, 0, 0], new, kv=[3, 0, new[2]])
    b.check(xn)
    out = b.run(xn).view(-1, 4, 64)
    assert out[:new[0] - 3].eq(0).all() and out[new[0]:new[0] + new[1]].eq(0).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lens,new", [([100], [1]), ([90, 30], [3, 4]), ([60, 150], [100, 40])])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_non_finite_keys_and_values_reach_their_readers_only(xn, cuda, dtype, lens, new, bad):
    """A NaN or infinity in a key or value row changes the tokens that see the row, as the formula says, and no others."""
    for where, window, last_only in itertools.product(("k", "v"), (0, 20), (False, True)):
        b = Batch(cuda, dtype, 4, 2, 64, 16, lens, new)
        for i, kv in enumerate(b.kv):
            # Rows of each request: its last token's, and one before its new tokens.
            for p in {kv - 1} if last_only else {kv - 1, max(0, kv - new[i] - 15)}:
                getattr(b, where)[b.table[i, p // 16], :, p % 16, 5:9] = bad
        ref, tol = paged_ref.attention(b.q, b.k, b.v, b.table, b.start, b.kv, b.scale, window)
        got = b.run(xn, window)
        check_attention(got, ref, tol, f"{where} window {window}")
        assert not torch.isfinite(ref).all()
        if last_only:  # tokens before the last one see nothing of it
            assert all(torch.isfinite(ref[lo:hi - 1]).all() for lo, hi in zip(b.start, b.start[1:]))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("new", [1, 90])
def test_attention_extreme_scores(xn, cuda, dtype, new):
    """Large scores (one key takes all the weight), equal ones, and all -inf (NaN by the formula)."""
    b = Batch(cuda, dtype, 4, 2, 64, 16, [300], [new])
    b.q *= 60
    b.check(xn)
    b.q *= 0
    b.check(xn)
    b = Batch(cuda, dtype, 4, 2, 64, 16, [100], [new])
    b.q = b.q.abs() + 0.1
    b.k[:] = torch.where(torch.isnan(b.k), b.k, -math.inf)
    out = b.run(xn)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_hint_does_not_decide_the_result(xn, cuda, dtype):
    """max_new chooses the kernel only: a batch of single tokens run as chunks, chunks run as single tokens."""
    Batch(cuda, dtype, 8, 2, 128, 16, [100, 1000, 5], [1, 1, 1]).check(xn, max_new=100)
    Batch(cuda, dtype, 8, 2, 128, 16, [100, 1000, 5], [50, 7, 30]).check(xn, max_new=1)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lens,new", [([100, 20], [1, 1]), ([100, 20], [40, 30])])
def test_attention_bad_pages(xn, cuda, dtype, lens, new):
    """Pages outside the pool read as zeros and are reported."""
    for page_id in (-1, 10 ** 6):
        b = Batch(cuda, dtype, 4, 2, 64, 16, lens, new)
        b.table[0, 2] = page_id
        ref, tol = paged_ref.attention(b.q, b.k, b.v, b.table, b.start, b.kv, b.scale)
        b.dk.copy_(b.k)
        b.dv.copy_(b.v)
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        got = xn.paged_attention(b.q.to(cuda), b.dk, b.dv, b.table.to(cuda), i64(b.start, cuda), i64(b.kv, cuda), b.scale,
                                 max_new=max(new), err_flag=err)
        assert int(err) == xn.XN_DEVERR_RANGE
        check_attention(got, ref, tol)


@pytest.mark.parametrize("new", [[1, 1, 1], [30, 40, 50]])
def test_attention_bad_lengths_skip_the_request(xn, cuda, new):
    b = Batch(cuda, "bf16", 4, 2, 64, 16, [50, 60, 70], new)
    ref, tol = paged_ref.attention(b.q, b.k, b.v, b.table, b.start, b.kv, b.scale)
    for kv1 in (-1, 16 * b.table.shape[1] + 1):
        kv = list(b.kv)
        kv[1] = kv1
        b.dk.copy_(b.k)
        b.dv.copy_(b.v)
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = torch.full((b.start[-1], 4 * 64), 3.0, dtype=torch.bfloat16, device=cuda)
        xn.paged_attention(b.q.to(cuda), b.dk, b.dv, b.table.to(cuda), i64(b.start, cuda), i64(kv, cuda), b.scale,
                           max_new=max(new), err_flag=err, out=out)
        assert int(err) == xn.XN_DEVERR_RANGE
        lo, hi = b.start[1], b.start[2]
        assert out[lo:hi].eq(3.0).all()
        keep = [t for t in range(b.start[-1]) if not lo <= t < hi]
        check_attention(out[keep], ref[keep], tol[keep])
    # Tokens beyond q, and q_start that descends.
    for start in ([0, new[0], b.start[2], b.start[-1] + 5], [0, b.start[2], new[0], b.start[-1]]):
        err.zero_()
        xn.paged_attention(b.q.to(cuda), b.dk, b.dv, b.table.to(cuda), i64(start, cuda), i64(b.kv, cuda), b.scale,
                           max_new=max(new), err_flag=err, out=out)
        assert int(err) == xn.XN_DEVERR_RANGE


def test_attention_shared_pages(xn, cuda):
    """Two requests with a common first page: the same row twice is fine."""
    b = Batch(cuda, "bf16", 8, 2, 64, 16, [40, 50], [1, 1])
    b.table[1, 0] = b.table[0, 0]
    b.check(xn)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_many_requests(xn, cuda, dtype):
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 40, (1300,), generator=g).tolist()
    Batch(cuda, dtype, 2, 1, 64, 8, lens, [1] * 1300).check(xn)
    lens = torch.randint(0, 40, (1100,), generator=g).tolist()
    new = torch.randint(0, 5, (1100,), generator=g).tolist()
    Batch(cuda, dtype, 2, 1, 32, 8, lens, new).check(xn, max_new=64)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_is_deterministic(xn, cuda, dtype):
    for lens, new in (([4000, 100], [1, 1]), ([3000], [100])):
        b = Batch(cuda, dtype, 8, 2, 128, 16, lens, new, stale=0.0)
        first = b.run(xn)
        for _ in range(3):
            assert torch.equal(first, b.run(xn))


def test_attention_pool_past_32_bit_offsets(xn, cuda):
    """Rows whose element offsets pass 2^31 and 2^32."""
    hk, page, d = 8, 256, 128
    n_pages = (1 << 32) // (hk * page * d) + 3  # 2^32 elements and a little more: 8.6 GB a pool
    k, v = (torch.empty(n_pages, hk, page, d, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    b = Batch(cuda, "bf16", 16, hk, d, page, [600, 500], [1, 1])
    c = Batch(cuda, "bf16", 16, hk, d, page, [600, 500], [60, 50])
    for x in (b, c):
        ref, tol = paged_ref.attention(x.q, x.k, x.v, x.table, x.start, x.kv, x.scale)
        ids = [n_pages - 1 - (n_pages // 9) * i for i in range(x.n_pages)]
        for i, to in enumerate(ids):
            k[to], v[to] = x.k[i].to(cuda), x.v[i].to(cuda)
        table = x.table.clone()
        for r, n in enumerate(x.kv):
            for j in range(-(-n // page)):
                table[r, j] = ids[int(x.table[r, j])]
        got = xn.paged_attention(x.q.to(cuda), k, v, table.to(cuda), i64(x.start, cuda), i64(x.kv, cuda), x.scale,
                                 max_new=x.max_new)
        check_attention(got, ref, tol)
    # The append reaches them too.
    slot = (n_pages - 1) * page + 3
    qkv = torch.randn(1, (2 + 2 * hk) * d, device=cuda).bfloat16()
    xn.paged_append_rope(qkv, 2, hk, torch.ones(1, d // 2, device=cuda).bfloat16(),
                         torch.zeros(1, d // 2, device=cuda).bfloat16(), k, v, i64([0], cuda), i64([slot], cuda))
    assert torch.equal(v[n_pages - 1, :, 3], qkv.view(-1, d)[2 + hk:])
    assert torch.equal(k[n_pages - 1, :, 3], qkv.view(-1, d)[2:2 + hk])


# -- together --------------------------------------------------------------------

class Server:
    """Requests on pages, stepped by plan, append and attention on random projections; a CPU mirror keeps every
    request's rows to compare with."""

    def __init__(self, dev, dt, h, hk, d, n, page, n_pages, blocks, cap, max_new):
        self.dev, self.dt, self.h, self.hk, self.d, self.page, self.cap, self.max_new = dev, dt, h, hk, d, page, cap, max_new
        self.k, self.v = (torch.full((n_pages, hk, page, d), math.nan, dtype=dt, device=dev) for _ in range(2))
        self.table = torch.full((n, blocks), -1, dtype=torch.int32, device=dev)
        self.ring = torch.arange(n_pages, dtype=torch.int32, device=dev)
        self.state, self.lens = i64([0, n_pages], dev), torch.zeros(n, dtype=torch.int64, device=dev)
        self.new = torch.zeros(n, dtype=torch.int64, device=dev)
        self.qkv = torch.zeros(cap, (h + 2 * hk) * d, dtype=dt, device=dev)
        ang = torch.rand(512, d // 2, generator=torch.Generator().manual_seed(9)) * 6
        self.cos, self.sin = ang.cos().to(dt).to(dev), ang.sin().to(dt).to(dev)
        self.out = torch.zeros(cap, h * d, dtype=dt, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        self.rows = [[] for _ in range(n)]

    def step(self, xn):
        self.plan = xn.paged_plan(self.lens, self.new, self.table, self.ring, self.state, self.page, self.cap, err_flag=self.err)
        q = xn.paged_append_rope(self.qkv, self.h, self.hk, self.cos, self.sin, self.k, self.v, self.plan.positions,
                                 self.plan.slots, err_flag=self.err)
        xn.paged_attention(q, self.k, self.v, self.table, self.plan.q_start, self.plan.kv_len, 1 / math.sqrt(self.d),
                           max_new=self.max_new, out=self.out, err_flag=self.err)
        self.lens.copy_(self.plan.kv_len)
        self.state.copy_(self.plan.ring_state)

    def feed(self, new, g):
        self.new.copy_(i64(new))
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=g).to(self.dt))
        x = self.qkv.cpu().view(self.cap, self.h + 2 * self.hk, self.d)
        at, self.queries = 0, []
        for i, k in enumerate(new):
            if k < 0:
                self.rows[i] = []
            for j in range(max(k, 0)):
                p = len(self.rows[i])
                c, s = self.cos[p:p + 1].cpu(), self.sin[p:p + 1].cpu()
                y = paged_ref.rope(x[at:at + 1, :self.h + self.hk], c, s, True)[0].to(self.dt)
                self.rows[i].append((y[0, self.h:], x[at, self.h + self.hk:]))
                self.queries.append((i, p, y[0, :self.h]))
                at += 1

    def check(self):
        assert int(self.err) == 0
        for at, (i, p, q) in enumerate(self.queries):
            k = torch.stack([r[0] for r in self.rows[i][:p + 1]]).double()
            v = torch.stack([r[1] for r in self.rows[i][:p + 1]]).double()
            qq = q.double().view(self.hk, -1, self.d)
            w = torch.softmax(torch.einsum("hgd,khd->hgk", qq, k) / math.sqrt(self.d), -1)
            ref = torch.einsum("hgk,khd->hgd", w, v).reshape(-1)
            # The mirror rounds q and k as the append does, but not always alike: a last bit of q and k moves a
            # score by at most u sqrt(d) |q| |k| scale ~ 2^-8 * 8 at these sizes, a weight by as much.
            u = HALF_STEP[self.dt]
            tol = (2 * u * 8 + 3 * u) * torch.einsum("hgk,khd->hgd", w, v.abs()).reshape(-1) + 2 * u * ref.abs() + 1e-5
            assert ((self.out[at].double().cpu() - ref).abs() <= tol).all(), (i, p)


@pytest.mark.parametrize("dtype,h,hk,d", [("bf16", 8, 2, 128), ("f32", 4, 4, 64)])
@pytest.mark.parametrize("graph", [False, True])
def test_serving_steps(xn, cuda, dtype, h, hk, d, graph):
    """Requests come with prompts, decode, end and make room for others; one captured graph serves every step."""
    s = Server(cuda, DT[dtype], h, hk, d, 5, 8, 60, 12, 96, 60)
    g = torch.Generator().manual_seed(4)
    steps = [[20, 0, 33, 1, 40], [1, 60, 1, 1, 1], [1, 1, 0, 5, 1], [-1, 1, 1, 1, -1], [17, 1, -1, 1, 2], [1, 1, 50, 1, 1]]
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.step(xn)  # no new tokens: nothing changes
        torch.cuda.current_stream().wait_stream(side)
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            s.step(xn)
    for new in steps:
        s.feed(new, g)
        cg.replay() if graph else s.step(xn)
        s.check()
        assert s.plan.kv_len.tolist() == [len(r) for r in s.rows]


def test_serving_on_another_stream_and_two_graphs(xn, cuda):
    """Work follows the stream that is current; two graphs with workspaces of their own may run at once."""
    side = torch.cuda.Stream()
    b = Batch(cuda, "bf16", 8, 2, 128, 16, [500, 90], [1, 1], stale=0.0)
    c = Batch(cuda, "bf16", 8, 2, 128, 16, [700, 30], [90, 40], stale=0.0, seed=5)
    want = [b.run(xn), c.run(xn)]
    torch.cuda.synchronize()
    graphs = []
    for x in (b, c):
        q, table, start, kv = x.q.to(cuda), x.table.to(cuda), i64(x.start, cuda), i64(x.kv, cuda)
        ws = xn.paged_attention_workspace(q.shape[0], 2, 8, 2, 128, x.max_new, q.dtype, cuda)
        out = torch.zeros(q.shape[0], 8 * 128, dtype=q.dtype, device=cuda)
        torch.cuda.synchronize()
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            xn.paged_attention(q, x.dk, x.dv, table, start, kv, x.scale, max_new=x.max_new, workspace=ws, out=out)
        graphs.append((cg, out, (q, table, start, kv, ws)))
    for _ in range(20):
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
    torch.cuda.synchronize()
    for (_, out, _), w in zip(graphs, want):
        assert torch.equal(out, w)
    with torch.cuda.stream(side):
        got = b.run(xn)
    side.synchronize()
    assert torch.equal(got, want[0])
