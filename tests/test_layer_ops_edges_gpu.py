"""K8, K9 and K10 where a rounding, a schedule or an error path can go wrong."""
import pytest
import torch

import a11spec
from test_layer_ops_gpu import _cache, _check_attn

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


# --------------------------------------------------------------------------- K10
def _pieces(ws, B, Hkv):
    """Pieces that each (sequence, KV head) was cut into: the merge counters behind the status word (256 bytes)."""
    return ws[256:256 + 4 * B * Hkv].view(torch.int32).view(B, Hkv)


@pytest.mark.parametrize("slots,long_at,ctx,short,Hq,Hkv,D", [(64, 5, 15000, 0, 32, 4, 128), (256, 255, 60000, 0, 8, 1, 64),
                                                              (200, 0, 12000, 20, 4, 2, 64)])
def test_one_long_sequence_among_empty_slots_is_cut(dev, slots, long_at, ctx, short, Hq, Hkv, D):
    """A padded batch of single tokens: many slots are empty or short, one sequence is long.
    The average over the slots is below 16 pages; the long sequence's pages are still
    shared by many CTAs."""
    lens = [short + b % 3 if short else 0 for b in range(slots)]
    new = [1 if short else 0] * slots
    lens[long_at], new[long_at] = ctx, 1
    assert sum((c + n + 15) // 16 for c, n in zip(lens, new)) <= 16 * slots
    args = _cache(17, lens, new, 1, Hq, Hkv, D)
    a, la, ws = _check_attn(args)
    assert int(_pieces(ws, slots, Hkv)[long_at].min()) >= 16
    b, lb, _ = _check_attn(args)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_short_sequences_stay_whole(dev):
    lens = [(37 * b) % 250 for b in range(60)]
    args = _cache(18, lens, [1] * 60, 1, 8, 2, 128)
    _, _, ws = _check_attn(args)
    assert int(_pieces(ws, 60, 2).max()) == 0


# --------------------------------------------------------------------------- errors
def test_failed_allocation_is_torchs_error(dev):
    """An output that does not fit raises torch.OutOfMemoryError, as callers that shrink
    their batch expect, and the next call works. The limit is this process's own."""
    x, w = torch.ones(200000, 8, dtype=BF, device=dev), torch.ones(4096, 8, dtype=BF, device=dev)  # 1.6 GB of output
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (64 << 20)) / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            a11spec.linear(x, w)
        y = a11spec.linear(x[:1000], w)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert bool((y == 8).all())
    assert a11spec.linear(x, w).shape == (200000, 4096)
