"""K8, K9 and K10 where a rounding, a schedule or an error path can go wrong."""
import pytest
import torch

import a11spec

pytestmark = pytest.mark.gpu
BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


# --------------------------------------------------------------------------- K8
@pytest.mark.parametrize("dtype,factors", [(F32, (7, 41, 61, 63, 119)), (BF, (7,))])
@pytest.mark.parametrize("dim", [256, 235])
def test_norm_e4m3_is_the_rounded_quotient(dev, dtype, factors, dim):
    """out = y / scale rounded to nearest even, at quotients that are exact ties.

    Row m holds m * t * 2^-40 with t every midpoint of two e4m3 neighbours and
    +-448; eps = 1 swamps the squares, so the reciprocal root is 1 and the scale
    m * 2^-40 exactly. A product with a rounded 1 / m would miss the ties."""
    ties = torch.tensor([s * k * 2.0 ** j for s in (1, -1) for k in range(17, 32, 2) for j in range(-10, 4)])
    ties = torch.cat([torch.tensor([448.0, -448.0]), ties])
    t = torch.zeros(dim)
    t[:len(ties)] = ties
    want = t.to(E4).to(dev)
    scale = torch.tensor(factors, dtype=F32) * 2.0 ** -40
    x = (scale[:, None] * t[None]).to(dev, dtype)
    assert torch.equal(x.double().cpu(), scale.double()[:, None] * t.double()[None])  # nothing is rounded so far
    y, s, _ = a11spec.add_rms_norm(x, torch.ones(dim, device=dev, dtype=dtype), eps=1.0, out_dtype=E4)
    assert torch.equal(s.cpu(), scale)
    for i in range(len(factors)):
        assert torch.equal(y[i].float(), want.float()), factors[i]


@pytest.mark.parametrize("rows,dim", [(300, 200), (64, 5003), (40, 16384)])
@pytest.mark.parametrize("magnitude", [-65, -30, 0, 55])
def test_norm_e4m3_follows_its_own_fp32_output(dev, rows, dim, magnitude):
    """The same call with fp32 output gives y; out and scales are its quotients, bit for
    bit, for rows from 2^-65 to 2^55 (eps = 1 keeps the small ones small). The quotients
    are taken of tensors: torch divides a CUDA tensor by a number as a product."""
    g = torch.Generator(device="cuda").manual_seed(rows + dim)
    x = torch.randn(rows, dim, generator=g, device="cuda") * 2.0 ** magnitude
    w = 2.0 ** torch.randint(-6, 7, (dim,), generator=g, device="cuda") * torch.randn(dim, generator=g, device="cuda")
    y, _, _ = a11spec.add_rms_norm(x, w, eps=1.0)
    q, s, _ = a11spec.add_rms_norm(x, w, eps=1.0, out_dtype=E4)
    top = y.abs().amax(1)
    assert torch.equal(s, top / torch.full_like(top, 448.0))
    assert torch.equal(q.float(), (y / s[:, None].expand_as(y)).to(E4).float())
