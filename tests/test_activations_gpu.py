"""K9's activations by themselves: x = (1, 0, ..., 0) makes the sums of a column its weight's
first element, so every bf16 value, the infinities and NaN among them, runs through the
epilogue of each kernel (few rows, tiles, CTA pairs).

SiLU v / (1 + exp(-v)): exp is good to 2 + 1.173 |v| units of 2^-23 and the division to 2
(CUDA's bounds of __expf and __fdividef), 1.3e-5 at |v| = 88, so 2^-15 covers it; where the
denominator passes 2^126 (v < -87.3) the division gives 0 for |y| below 88.8 * 2^-126 < 2^-119.
GELU v Phi(v): 2.1e-6 down to v = -6; beyond, the exponent -v^2 log2(e) / 2, at most 149 in
size, is off by two roundings of 2^-24: 1.3e-5 of the value, again below 2^-15; results near
the smallest normal lose bits, 2^-126 at most. Then one rounding to bf16, 2^-8."""
import pytest
import torch

import a11spec

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ROWS = [1, 40, 2048]


def _exact(v, activation):
    v = v.double()
    return v / (1 + torch.exp(-v)) if activation == "silu" else v * 0.5 * torch.special.erfc(-v * 0.5 ** 0.5)


def _first(values):
    """[n, 8] with the values in the first column."""
    w = torch.zeros(values.numel(), 8, dtype=BF, device="cuda")
    w[:, 0] = values
    return w


def _x(rows):
    return _first(torch.ones(rows, device="cuda"))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_every_bf16_value(dev, rows, gated, activation):
    v = torch.arange(65536, device=dev, dtype=torch.int32).to(torch.int16).view(BF)
    ref = _exact(v, activation)
    for lo in range(0, 65536, 2048 if rows == 40 else 65536):
        part = slice(lo, lo + (2048 if rows == 40 else 65536))
        w = _first(v[part])
        if gated:
            y = a11spec.linear(_x(rows), _first(torch.ones_like(v[part])), gate=w, activation=activation)
        else:
            y = a11spec.linear(_x(rows), w, activation=activation)
        assert torch.equal(y[:1].expand_as(y).view(torch.int16), y.view(torch.int16))  # all rows alike
        got, want = y[0].double(), ref[part]
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[want.isinf()], want[want.isinf()])
        ok = want.isfinite()
        tol = want.abs() * (2.0 ** -8 + 2.0 ** -15) * (1 + 2.0 ** -8) + 2.0 ** (-119 if activation == "silu" else -126)
        bad = ok & ~((got - want).abs() <= tol)
        assert not bool(bad.any()), (v[part][bad][:5], got[bad][:5], want[bad][:5])


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("activation,lo,error", [("silu", -4.0, 2.0 ** -19), ("gelu", -4.0, 1.0e-6), ("gelu", -6.0, 2.1e-6)])
def test_error_in_fp32(dev, rows, activation, lo, error):
    """The activation's own error, seen past the output's rounding: act(u) v + r with r the
    rounded -act(u) v and, of 128 v, the one that leaves the least. Taken are the u (nearly
    all) where that is below 2^-14 of act(u) v, so that its rounding is below 2^-22; the
    product and the sum add 2^-24 each."""
    u = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF).double()
    u = u[u.isfinite() & (u >= lo) & (u <= 8.0) & (u.abs() >= 2.0 ** -8)]
    act = _exact(u, activation)
    m = torch.arange(128, 256, dtype=torch.float64) / 128
    product = act[:, None] * m
    left = (product - product.to(BF).double()).abs() / product.abs()
    least, best = left.min(1)
    fine = least < 2.0 ** -14
    assert float(fine.double().mean()) > 0.9
    u, act, v = u[fine], act[fine], m[best[fine]]
    r = -(act * v).to(BF).double()
    want = act * v + r
    y = a11spec.linear(_x(rows), _first(v.to(dev)), gate=_first(u.to(dev)), activation=activation,
                       residual=r.to(dev, BF).expand(rows, -1).contiguous())
    off = (y.double().cpu() - want).abs() / (act * v).abs()
    assert float(off.max()) <= error + 2.0 ** -22 + 2.0 ** -23, (float(off.max()), float(u[off.amax(0).argmax()]))
