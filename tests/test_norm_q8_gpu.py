"""The 8-bit RMSNorm on the GPU against 64 bits: h bit for bit, scales within
their rounding, values within half an e4m3 step of what they stand for."""
import math

import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _check(xn, cuda, dtype, rows, cols, group, residual, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * scale).to(dtype)
    branch = (torch.randn(rows, cols, generator=g) * scale).to(dtype) if residual else None
    alpha = (1 + 0.1 * torch.randn(cols, generator=g)).to(dtype)
    h, y, s = paged_ref.rms_norm_q8(x, alpha, 1e-5, branch, group)
    q, scales, got_h = xn.rms_norm_q8(x.to(cuda), alpha.to(cuda), 1e-5, branch=None if branch is None else branch.to(cuda),
                                      group=group)
    assert torch.equal(got_h.cpu(), h)
    # y: the sum of squares (all positive: off by 4 sqrt(n) u relative, half that in the root) and six roundings.
    rel = (2 * math.sqrt(cols) + 6) * 2.0 ** -24
    assert ((scales.cpu().double() - s).abs() <= (rel + 2 * 2.0 ** -24) * s).all()
    # Half an e4m3 step: 2^-4 of the value, 2^-10 below the normal range (2^-6); plus what y and the scale are off by.
    unit = y / s.unsqueeze(-1).repeat_interleave(group or cols, -1).view(rows, cols).clamp(min=1e-300)
    tol = torch.maximum(unit.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64)) + unit.abs() * 4 * rel
    assert ((q.cpu().double() - unit).abs() <= tol).all()
    assert q.cpu().double().abs().amax(-1).eq(448).all() or scale == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,cols,group", [(1, 1, 0), (3, 7, 0), (5, 32, 32), (17, 64, 0), (9, 250, 0), (4, 192, 64), (33, 1024, 128),
                                             (2, 1333, 0), (6, 4096, 0), (6, 4096, 128), (3, 8200, 0), (2, 16384, 32),
                                             (2, 20001, 0), (2, 40000, 0), (2, 40064, 64), (2, 40960, 128), (3, 36896, 32)])
def test_norm_q8(xn, cuda, dtype, residual, rows, cols, group):
    _check(xn, cuda, DT[dtype], rows, cols, group, residual)


@pytest.mark.parametrize("dtype", DT)
def test_norm_q8_many_rows(xn, cuda, dtype):
    _check(xn, cuda, DT[dtype], 5001, 96, 32, True)
    _check(xn, cuda, DT[dtype], 4099, 16, 0, False)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("cols", [64, 250, 40000])
def test_norm_q8_special_rows(xn, cuda, dtype, cols):
    """Zeros give scale 0 and zeros; a NaN or an infinity reaches its row only; tiny rows keep their values."""
    dt = DT[dtype]
    x = torch.randn(5, cols, generator=torch.Generator().manual_seed(1)).to(dt)
    x[0] = 0
    x[1, 3] = math.nan
    x[2, 5] = math.inf
    x[3] *= 1e-4
    q, s, _ = xn.rms_norm_q8(x.to(cuda), torch.ones(cols, dtype=dt, device=cuda), 1e-5)
    q, s = q.float().cpu(), s.cpu()
    assert s[0] == 0 and q[0].eq(0).all()
    assert torch.isnan(s[1]) and torch.isnan(q[1]).all()
    # An infinity makes the sum infinite: inf * 0 is NaN there, the rest 0; NaN is the largest of the row.
    assert torch.isnan(s[2])
    assert torch.isfinite(q[3:]).all() and q[3:].abs().amax(-1).eq(448).all()
    # Weights of zero: scale 0.
    q, s, _ = xn.rms_norm_q8(x[4:].to(cuda), torch.zeros(cols, dtype=dt, device=cuda), 1e-5)
    assert s.eq(0).all() and q.float().eq(0).all()


def test_norm_q8_tiny_scales(xn, cuda):
    """Magnitudes whose scale has no f32 reciprocal."""
    x = torch.randn(2, 64, generator=torch.Generator().manual_seed(1)).to(cuda)
    a = torch.full((64,), 1e-36, device=cuda)
    q, s, _ = xn.rms_norm_q8(x, a, 1e-5)
    assert q.float().abs().amax(-1).eq(448).all()
    w, t, _ = xn.rms_norm_q8(x, torch.ones(64, device=cuda), 1e-5)
    assert (q.float() - w.float()).abs().le(w.float().abs() * 2.0 ** -3).all()


@pytest.mark.parametrize("cols", [256, 250, 40000])
def test_norm_q8_in_place_and_misaligned(xn, cuda, cols):
    """residual_out may be x or branch; rows that begin off a 16-byte boundary."""
    g = torch.Generator().manual_seed(2)
    x, b = (torch.randn(3, cols, generator=g).bfloat16().to(cuda) for _ in range(2))
    a = torch.ones(cols, dtype=torch.bfloat16, device=cuda)
    want = xn.rms_norm_q8(x, a, 1e-5, branch=b)
    for target in ("x", "b"):
        x2, b2 = x.clone(), b.clone()
        got = xn.rms_norm_q8(x2, a, 1e-5, branch=b2, residual_out=x2 if target == "x" else b2)
        for u, v in zip(got, want):
            assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))
    odd = torch.empty(3 * cols + 1, dtype=torch.bfloat16, device=cuda)[1:].view(3, cols)
    odd.copy_(x)
    got = xn.rms_norm_q8(odd, a, 1e-5, branch=b)
    assert torch.equal(got[2], want[2])
    assert torch.allclose(got[1], want[1], rtol=1e-5)
    if cols == 256:
        got, want = xn.rms_norm_q8(odd, a, 1e-5, branch=b, group=64), xn.rms_norm_q8(x, a, 1e-5, branch=b, group=64)
        assert torch.allclose(got[1], want[1], rtol=1e-5)


def test_norm_q8_feeds_an_8_bit_product(xn, cuda):
    """The values times their scales stand for the norm: a product with them is the norm's product to 8-bit accuracy."""
    g = torch.Generator().manual_seed(3)
    x, b = (torch.randn(64, 512, generator=g).bfloat16().to(cuda) for _ in range(2))
    a = (1 + 0.02 * torch.randn(512, generator=g)).bfloat16().to(cuda)
    w = torch.randn(512, 96, generator=g).to(cuda) / math.sqrt(512)
    y, h = xn.rms_norm_residual(x, b, a, 1e-5)
    q, s, h8 = xn.rms_norm_q8(x, a, 1e-5, branch=b)
    assert torch.equal(h, h8)
    got, want = (q.float() * s[:, None]) @ w, y.float() @ w
    # Each of 512 terms is off by at most 2^-4 of itself, with independent signs: 2^-4 / sqrt(3) of the norm.
    assert float((got - want).norm() / want.norm()) < 2.0 ** -4 / math.sqrt(3) + 2.0 ** -8
