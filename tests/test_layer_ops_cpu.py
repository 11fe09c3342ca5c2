"""What K8, K9 and K10 refuse, without a GPU: the C entry points check their
arguments before they touch the device, and the torch wrappers want CUDA tensors."""
import math

import pytest
import torch

import a11spec
from a11spec import _lib
from a11spec._lib import lib

P, ODD = 0x10000, 0x10001  # addresses that are never read: every call below is refused


def _refused(rc, code, words):
    assert rc == code, (rc, lib.a11s_last_error())
    assert words in lib.a11s_last_error().decode(), lib.a11s_last_error()


def _norm(**kw):
    a = dict(dtype=_lib.BF16, x=P, xs=64, res=None, rs=0, w=P, rows=4, dim=64, eps=1e-6, sum=None, ss=0,
             odt=_lib.BF16, out=P, os=64, sc=None, st=None)
    a.update(kw)
    return lib.a11s_add_rms_norm(*a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(dtype=_lib.E4M3), _lib.EINVAL, "dtype"), (dict(odt=_lib.F32), _lib.EINVAL, "out_dtype"),
    (dict(rows=-1), _lib.EINVAL, "sizes"), (dict(dim=0), _lib.EINVAL, "sizes"),
    (dict(dim=16385, xs=16385, os=16385), _lib.EUNSUPPORTED, "16384"),
    (dict(xs=63), _lib.EINVAL, "stride"), (dict(os=0), _lib.EINVAL, "stride"), (dict(res=P, rs=8), _lib.EINVAL, "stride"),
    (dict(res=P, rs=64, sum=P, ss=2), _lib.EINVAL, "stride"), (dict(eps=-1.0), _lib.EINVAL, "eps"),
    (dict(eps=math.nan), _lib.EINVAL, "eps"), (dict(x=None), _lib.EINVAL, "null"), (dict(w=None), _lib.EINVAL, "null"),
    (dict(out=None), _lib.EINVAL, "null"), (dict(sc=P), _lib.EINVAL, "scales"), (dict(odt=_lib.E4M3), _lib.EINVAL, "scales"),
    (dict(x=ODD), _lib.EINVAL, "aligned"), (dict(out=ODD), _lib.EINVAL, "aligned"),
])
def test_norm_refusals(kw, code, words):
    _refused(_norm(**kw), code, words)


def test_norm_without_rows_is_fine():
    assert _norm(rows=0, x=None) == _lib.OK


def _linear(**kw):
    a = dict(dtype=_lib.BF16, x=P, xs=64, sx=None, w=P, sw=None, g=None, sg=None, b=None, gb=None, rows=4, K=64, N=40,
             act=0, res=None, rs=0, out=P, os=40, ws=None, wsb=0, st=None)
    a.update(kw)
    return lib.a11s_linear(*a.values())


E4 = dict(dtype=_lib.E4M3, sx=P, sw=P)


@pytest.mark.parametrize("kw,code,words", [
    (dict(dtype=_lib.F32), _lib.EINVAL, "dtype"), (dict(rows=-1), _lib.EINVAL, "sizes"), (dict(N=0), _lib.EINVAL, "sizes"),
    (dict(K=60), _lib.EINVAL, "multiples of 8"), (dict(xs=65), _lib.EINVAL, "multiples of 8"),
    (dict(K=72, xs=72, **E4), _lib.EINVAL, "multiples of 16"), (dict(xs=56), _lib.EINVAL, "stride"),
    (dict(os=39), _lib.EINVAL, "stride"), (dict(res=P, rs=1), _lib.EINVAL, "stride"), (dict(act=3), _lib.EINVAL, "activation"),
    (dict(act=-1), _lib.EINVAL, "activation"), (dict(gb=P), _lib.EINVAL, "gate_bias"), (dict(x=None), _lib.EINVAL, "null"),
    (dict(w=None), _lib.EINVAL, "null"), (dict(out=None), _lib.EINVAL, "null"), (dict(sx=P), _lib.EINVAL, "scales"),
    (dict(dtype=_lib.E4M3), _lib.EINVAL, "scales"), (dict(g=P, **E4), _lib.EINVAL, "scales"),
    (dict(sg=P, **E4), _lib.EINVAL, "scales"), (dict(x=P + 8), _lib.EINVAL, "16-byte"), (dict(w=P + 2), _lib.EINVAL, "16-byte"),
    (dict(g=P + 2), _lib.EINVAL, "16-byte"), (dict(out=ODD), _lib.EINVAL, "aligned"), (dict(ws=P, wsb=8), _lib.ENOSPACE, "256"),
])
def test_linear_refusals(kw, code, words):
    _refused(_linear(**kw), code, words)


def _attn(**kw):
    a = dict(q=P, qs=1024, k=P, v=P, pages=8, table=P, maxp=4, ctx=P, nn=None, B=2, N=3, Hq=8, Hkv=2, D=128, kv=64, scale=0.1,
             out=P, lse=None, ws=P, wsb=256, st=None)
    a.update(kw)
    return lib.a11s_chunk_attention(*a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(D=96), _lib.EUNSUPPORTED, "head_dim"), (dict(Hq=7), _lib.EUNSUPPORTED, "multiple"),
    (dict(Hq=258), _lib.EUNSUPPORTED, "128"), (dict(N=0), _lib.EINVAL, "size"), (dict(B=-1), _lib.EINVAL, "size"),
    (dict(pages=0), _lib.EINVAL, "size"), (dict(kv=0), _lib.EINVAL, "size"), (dict(kv=65), _lib.EINVAL, "page table"),
    (dict(qs=1016), _lib.EINVAL, "q_stride"), (dict(qs=1028), _lib.EINVAL, "q_stride"), (dict(scale=0.0), _lib.EINVAL, "scale"), (dict(scale=math.inf), _lib.EINVAL, "scale"), (dict(q=None), _lib.EINVAL, "null"),
    (dict(ctx=None), _lib.EINVAL, "null"), (dict(ws=None), _lib.EINVAL, "null"), (dict(out=P + 2), _lib.EINVAL, "16-byte"),
    (dict(wsb=128), _lib.ENOSPACE, "workspace"), (dict(B=1, N=1, kv=32768, maxp=2048), _lib.ENOSPACE, "workspace"),
])
def test_chunk_attention_refusals(kw, code, words):
    _refused(_attn(**kw), code, words)


def test_wrappers_want_cuda_tensors():
    t = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(a11spec.A11Error, match="CUDA"):
        a11spec.add_rms_norm(t, t[0])
    with pytest.raises(a11spec.A11Error, match="CUDA"):
        a11spec.linear(t, t)
    with pytest.raises(a11spec.A11Error, match="CUDA"):
        a11spec.chunk_attention(t.view(1, 1, 4, 64), t, t, t, t)


def test_row_strides():
    """The wrappers' row strides: views whose rows are evenly spaced, and nothing else."""
    f = _lib.fast.row_stride
    t = torch.zeros(4, 6, 3, 136, dtype=torch.bfloat16)
    assert f(t, 136) == 136 and f(t[:, :, 1, :128], 128) == 408 and f(t[:, :1, 1, :128], 128) == 6 * 408
    assert f(t[:1, :1, :1, :128], 128) == 128 and f(t[0, 0, 0, :8], 8) == 8 and f(t[:0], 136) == 136
    for v in (t[:, 1:3, 1], t.transpose(0, 1)[..., :128], t[..., ::2], t[0, 0, 0, ::2], t[0, 0]):
        with pytest.raises(a11spec.A11Error):
            f(v, v.shape[-1] if v.dim() > 2 or v.stride(-1) > 1 else 8)


def test_wrappers_refuse_other_objects():
    t = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: a11spec.add_rms_norm([1.0], t), lambda: a11spec.linear(None, t), lambda: a11spec.linear(3, t),
                 lambda: a11spec.chunk_attention("q", t, t, t, t)):
        with pytest.raises(a11spec.A11Error, match="tensor"):
            call()
    with pytest.raises(a11spec.A11Error, match="activation"):
        a11spec.linear(t, t, activation="relu")


def test_chunk_attention_split_plan():
    """Splits as seen through the workspace size, on the 148 SMs assumed without a device:
    a long cache with one row per KV head is split, a long chunk is not."""
    f = a11spec.ops.chunk_attention_workspace_bytes
    assert f(1, 4096, 32, 4, 128, 16384) == 256
    assert f(1, 1, 32, 4, 128, 32768) > 256
    assert f(0, 1, 32, 4, 128, 64) == 256 and f(1, 0, 32, 4, 128, 64) == 0


@pytest.mark.parametrize("kw", [dict(rows=2 ** 30 + 1), dict(N=2 ** 30 + 8, os=2 ** 30 + 8), dict(K=2 ** 29 + 8, xs=2 ** 29 + 8),
                                dict(K=2 ** 30, xs=2 ** 30, N=1, os=1, **E4)])
def test_linear_refuses_sizes_beyond_32_bit_offsets(kw):
    _refused(_linear(**kw), _lib.EUNSUPPORTED, "beyond")
