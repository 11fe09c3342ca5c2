"""K8 (add_rms_norm), K9 (linear) and K10 (chunk_attention) against their fp64
forms (layer_reference.py has the forms and derives every tolerance)."""
import math

import pytest
import torch

import a11spec
import layer_reference as R
from a11spec import _lib, ops

pytestmark = pytest.mark.gpu
BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rnd(g, *shape, std=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


# --------------------------------------------------------------------------- K8
def _check_norm(x, w, res, eps, y, scales, h):
    ref, href = R.norm(x, w, res, eps)
    if res is not None:
        u = R.U[x.dtype]
        assert R.worst(h, href, href.abs() * (u * (1 + 2.0 ** -20) + 2.0 ** -24) + 2.0 ** -134) <= 1
    if scales is None:
        assert R.worst(y, ref, ref.abs() * (2.0 ** -19 + R.U[y.dtype]) * (1 + 2.0 ** -7) + 2.0 ** -134) <= 1
    else:
        s = (ref.abs().amax(-1) / 448).clamp_min(2.0 ** -100)
        assert R.worst(scales, s, s * 2.0 ** -18) <= 1
        v = ref / s[..., None]
        assert R.worst(y.float(), v, v.abs() * (2.0 ** -17 + 2.0 ** -4) + 2.0 ** -10) <= 1


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("rows,dim", [(1, 2048), (3, 1), (5, 7), (9, 64), (2, 256), (17, 264), (33, 257), (4, 1025),
                                      (6, 4999), (3, 5000), (2, 8192), (2, 8200), (2, 16384), (1, 16383), (300, 128)])
def test_norm(dev, dtype, e4m3, rows, dim):
    g = _gen(rows * 100003 + dim)
    x, res = _rnd(g, rows, dim, dtype=dtype), _rnd(g, rows, dim, std=2.0, dtype=dtype)
    w = (1 + _rnd(g, dim, std=0.1)).to(dtype)
    for r in (res, None):
        y, s, h = a11spec.add_rms_norm(x, w, residual=r, eps=1e-5, out_dtype=E4 if e4m3 else None)
        assert (s is None) == (not e4m3) and (h is None) == (r is None)
        _check_norm(x, w, r, 1e-5, y, s, h)


def test_norm_views_and_in_place(dev):
    g = _gen(5)
    wide = _rnd(g, 4, 6, 3, 136, dtype=BF)
    x = wide[:, :, 1, 3:3 + 128]          # rows 408 elements apart, 2-byte aligned only
    w, res = _rnd(g, 128, dtype=BF), _rnd(g, 4, 6, 128, dtype=BF)
    keep = wide.clone()
    old = res.clone()
    y, _, h = a11spec.add_rms_norm(x, w, residual=res, sum_out=res)
    assert h.data_ptr() == res.data_ptr() and torch.equal(wide, keep)
    _check_norm(x, w, old, 1e-6, y, None, h)
    out = torch.full((24, 200), 7.0, dtype=BF, device="cuda")  # rows 200 apart: what lies between stays
    y2, _, _ = a11spec.add_rms_norm(x.reshape(24, 128), w, out=out[:, 8:136])
    _check_norm(x.reshape(24, 128), w, None, 1e-6, y2, None, None)
    assert bool((out[:, :8] == 7).all()) and bool((out[:, 136:] == 7).all())


def test_norm_zero_tiny_and_nonfinite_rows(dev):
    x = torch.ones(5, 512, device="cuda")
    x[0] = 0
    x[1] = 1e-30                          # below eps: y is tiny, the scale stays usable
    x[2, 7] = math.nan
    x[3, 9] = math.inf
    w = torch.ones(512, device="cuda")
    y, s, _ = a11spec.add_rms_norm(x, w, out_dtype=E4)
    yf = y.float()
    assert bool((yf[0] == 0).all()) and float(s[0]) == 2.0 ** -100
    want = 1e-30 / math.sqrt(1e-6) / 448
    assert abs(float(s[1]) / want - 1) < 1e-5 and bool((yf[1] == 448).all())
    assert bool(yf[2].isnan().all()) and bool(yf[3].isnan().all())
    assert bool((yf[4] == 448).all())
    y, _, _ = a11spec.add_rms_norm(x, w)
    assert bool(y[2].isnan().all())
    assert bool(y[3, 9].isnan()) and bool((y[3, :9] == 0).all())  # inf * 0, and finite * 0


def test_norm_empty(dev):
    y, s, h = a11spec.add_rms_norm(torch.empty(0, 64, dtype=BF, device="cuda"), torch.ones(64, dtype=BF, device="cuda"),
                                   residual=torch.empty(0, 64, dtype=BF, device="cuda"), out_dtype=E4)
    assert y.shape == (0, 64) and s.shape == (0,) and h.shape == (0, 64)


# --------------------------------------------------------------------------- K9
def _e4m3(t):
    s = t.abs().amax(1) / 448
    return (t / s[:, None]).to(E4), s


def _linear_case(seed, rows, K, N, e4m3, gated, bias, residual):
    g = _gen(seed)
    x, w, gate = _rnd(g, rows, K), _rnd(g, N, K, std=K ** -0.5), _rnd(g, N, K, std=K ** -0.5)
    kw = {}
    if e4m3:
        (x, kw["x_scale"]), (w, kw["weight_scale"]), (gate, gs) = _e4m3(x), _e4m3(w), _e4m3(gate)
        if gated:
            kw["gate_scale"] = gs
    else:
        x, w, gate = x.to(BF), w.to(BF), gate.to(BF)
    if gated:
        kw["gate"] = gate
    if bias:
        kw["bias"] = _rnd(g, N, std=0.5, dtype=BF)
        if gated:
            kw["gate_bias"] = _rnd(g, N, std=0.5, dtype=BF)
    if residual:
        kw["residual"] = _rnd(g, rows, N, std=2.0, dtype=BF)
    return x, w, kw


def _linear_ref(x, w, kw, activation):
    return R.linear(x, w, bias=kw.get("bias"), activation=activation, gate=kw.get("gate"), gate_bias=kw.get("gate_bias"),
                    residual=kw.get("residual"), sx=kw.get("x_scale"), sw=kw.get("weight_scale"), sg=kw.get("gate_scale"))


SIZES = [  # rows, K, N: the streaming kernel, the split tile, the CTA pair; whole and ragged in every direction
    (1, 16, 1), (1, 2048, 48), (7, 48, 17), (8, 208, 100), (13, 4096, 33), (24, 1040, 520), (32, 8192, 16), (32, 272, 1531),
    (5, 8, 40), (40, 8, 40), (33, 64, 8), (33, 16, 24), (64, 4096, 256), (100, 2064, 200), (128, 1008, 1531), (197, 1008, 515), (300, 512, 2048),
    (2048, 512, 2048), (2049, 144, 4104), (2300, 272, 2055), (4096, 64, 2056), (8200, 32, 1000),
]


@pytest.mark.parametrize("rows,K,N", SIZES)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("gated,activation,bias,residual", [(False, None, False, False), (False, "gelu", True, True),
                                                            (True, "silu", False, True), (True, "gelu", True, False)])
def test_linear(dev, rows, K, N, e4m3, gated, activation, bias, residual):
    if e4m3 and K % 16:
        K += 8  # rows of 16-byte multiples
    x, w, kw = _linear_case(rows + 7 * K + 31 * N, rows, K, N, e4m3, gated, bias, residual)
    ref, tol = _linear_ref(x, w, kw, activation)
    out = torch.full((rows, N), math.nan, dtype=BF, device="cuda")
    y = a11spec.linear(x, w, activation=activation, out=out, check_status=True, **kw)
    assert y.data_ptr() == out.data_ptr()
    r = R.worst(y, ref, tol)
    assert r <= 1, r
    assert torch.equal(y, a11spec.linear(x, w, activation=activation, **kw))  # equal calls, equal bits


@pytest.mark.parametrize("rows", [5, 150, 3000])
def test_linear_views_and_in_place_residual(dev, rows):
    K, N = 256, 264
    x, w, kw = _linear_case(rows, rows, K, N, False, False, True, True)
    wide = torch.full((rows, 2 * K + 8), math.nan, dtype=BF, device="cuda")
    wide[:, 8:8 + K] = x
    ref, tol = _linear_ref(x, w, kw, "silu")
    # in place: out is the residual, rows 512 elements apart; what lies between stays
    buf = torch.full((rows, 512), 3.0, dtype=BF, device="cuda")
    buf[:, 16:16 + N] = kw.pop("residual")
    y = a11spec.linear(wide[:, 8:8 + K], w, activation="silu", residual=buf[:, 16:16 + N], out=buf[:, 16:16 + N],
                       check_status=True, **kw)
    assert R.worst(y, ref, tol) <= 1
    assert bool((buf[:, :16] == 3).all()) and bool((buf[:, 16 + N:] == 3).all())
    # an odd pitch and an odd start: nothing but 2-byte alignment
    odd = torch.full((rows, N + 3), 5.0, dtype=BF, device="cuda")
    x2, w2, kw2 = _linear_case(rows, rows, K, N, False, False, True, True)
    y = a11spec.linear(x2, w2, activation="silu", out=odd[:, 1:1 + N], **kw2)
    assert R.worst(y, ref, tol) <= 1
    assert bool((odd[:, :1] == 5).all()) and bool((odd[:, 1 + N:] == 5).all())
    odd[:, 1:1 + N] = kw2.pop("residual")  # and in place there
    y = a11spec.linear(x2, w2, activation="silu", residual=odd[:, 1:1 + N], out=odd[:, 1:1 + N], **kw2)
    assert R.worst(y, ref, tol) <= 1
    assert bool((odd[:, :1] == 5).all()) and bool((odd[:, 1 + N:] == 5).all())


@pytest.mark.parametrize("rows", [3, 70, 2100])
def test_linear_nonfinite_rows_stay_in_their_rows(dev, rows):
    x, w, kw = _linear_case(1, rows, 512, 640, False, True, False, False)
    ref, tol = _linear_ref(x, w, kw, "silu")
    x[1, 100] = math.nan
    y = a11spec.linear(x, w, activation="silu", **kw)
    assert bool(y[1].isnan().all())
    keep = torch.arange(rows, device="cuda") != 1
    assert R.worst(y[keep], ref[keep], tol[keep]) <= 1


def test_linear_empty_and_leading_axes(dev):
    w = torch.randn(40, 64, device="cuda").to(BF)
    assert a11spec.linear(torch.empty(0, 64, dtype=BF, device="cuda"), w).shape == (0, 40)
    x = torch.randn(2, 3, 64, device="cuda").to(BF)
    y = a11spec.linear(x, w)
    assert y.shape == (2, 3, 40) and torch.equal(y.view(6, 40), a11spec.linear(x.view(6, 64), w))


def test_linear_outputs_past_32_bits(dev):
    """More than 2^31 output elements, on even and on odd rows: the last rows are right."""
    rows, K, N = 66000, 16, 32800
    g = _gen(77)
    x, w = _rnd(g, rows, K, dtype=BF), _rnd(g, N, K, dtype=BF)
    for n in (N, N - 1):
        y = a11spec.linear(x, w[:n], check_status=True)
        for lo in (0, 65400, rows - 100):
            ref, tol = R.linear(x[lo:lo + 100], w[:n])
            assert R.worst(y[lo:lo + 100], ref, tol) <= 1, (n, lo)
        del y


# --------------------------------------------------------------------------- K10
def _cache(seed, ctx, n_new, N, Hq, Hkv, D, extra_pages=3):
    """Pools whose unused places (free pages, slots past a sequence's end) hold NaN."""
    g = _gen(seed)
    B = len(ctx)
    need = [(c + n + 15) // 16 for c, n in zip(ctx, n_new)]
    P = sum(need) + extra_pages
    perm = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, max(max(need), 1) + 2), -1, dtype=torch.int32, device="cuda")
    k = torch.full((P, 16, Hkv, D), math.nan, dtype=BF, device="cuda")
    v = k.clone()
    at = 0
    for b in range(B):
        S = ctx[b] + n_new[b]
        table[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
        pos = torch.arange(S, device="cuda")
        page = table[b].long()[pos // 16]
        k[page, pos % 16] = _rnd(g, S, Hkv, D, dtype=BF)
        v[page, pos % 16] = _rnd(g, S, Hkv, D, dtype=BF)
    q = _rnd(g, B, N, Hq, D, std=1.5, dtype=BF)
    i32 = dict(dtype=torch.int32, device="cuda")
    return q, k, v, table, torch.tensor(ctx, **i32), torch.tensor(n_new, **i32)


def _check_attn(args, scale=None, **kw):
    q, k, v, table, ctx, nn = args
    ref, tol, lref, ltol = R.attention(q, k, v, table, ctx, nn if nn is not None else [q.shape[1]] * q.shape[0], scale)
    out = torch.full_like(q, math.nan)
    got, lse, ws = a11spec.chunk_attention(q, k, v, table, ctx, nn, scale=scale, want_lse=True, out=out,
                                           check_status=True, **kw)
    r, rl = R.worst(got, ref, tol), R.worst(lse, lref, ltol)
    assert r <= 1 and rl <= 1, (r, rl)
    return got, lse, ws


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (4, 4), (6, 2), (10, 2), (32, 4), (24, 8)])
@pytest.mark.parametrize("ctx,n_new,N", [
    ([0], [1], 1), ([15], [1], 1), ([16], [1], 1), ([127, 128, 129], [1, 1, 1], 1), ([0, 5, 300], [3, 0, 9], 9),
    ([0], [128], 128), ([1], [129], 130), ([77, 1000], [200, 65], 200), ([0, 0], [0, 0], 4), ([33], [513], 513),
])
def test_chunk_attention(dev, D, Hq, Hkv, ctx, n_new, N):
    _check_attn(_cache(sum(ctx) + N + Hq + D, ctx, n_new, N, Hq, Hkv, D))


@pytest.mark.parametrize("ctx,n_new,N,Hq,Hkv,D", [
    ([20000], [1], 1, 8, 1, 128), ([5000, 1, 130], [1, 1, 0], 2, 32, 4, 128), ([9000, 40, 3000], [7, 7, 1], 7, 6, 2, 64),
    ([4000, 2500], [40, 17], 40, 16, 2, 128), ([3000], [1], 1, 128, 1, 64), ([3000], [1], 1, 100, 1, 128),
])
def test_chunk_attention_split_caches(dev, ctx, n_new, N, Hq, Hkv, D):
    """Long caches and few rows: the KV range is split; short sequences have fewer splits than long ones."""
    args = _cache(3 + sum(ctx), ctx, n_new, N, Hq, Hkv, D)
    top = max(c + n for c, n in zip(ctx, n_new))
    assert ops.chunk_attention_workspace_bytes(len(ctx), N, Hq, Hkv, D, top) > 256
    a, la, _ = _check_attn(args, max_kv_len=top)
    b, lb, _ = _check_attn(args, max_kv_len=top)
    assert torch.equal(a, b) and torch.equal(la, lb)  # merged in a fixed order
    _check_attn(args, max_kv_len=128)                 # a bound that is too small costs speed only


@pytest.mark.parametrize("N", [1, 40])
def test_chunk_attention_pool_past_32_bits(dev, N):
    """Pages whose elements lie past 2^31 in the pool."""
    q, k, v, table, ctx, nn = _cache(14, [700, 90], [N, N], N, 16, 8, 128)
    big = 140000  # pages of 16 x 8 x 128 elements: 2.29e9
    kb, vb = (torch.empty(big, 16, 8, 128, dtype=BF, device="cuda") for _ in range(2))
    shift = big - k.shape[0]
    kb[shift:], vb[shift:] = k, v
    moved = torch.where(table >= 0, table + shift, table)
    want, wl, _ = _check_attn((q, k, v, table, ctx, nn))
    got, gl, _ = a11spec.chunk_attention(q, kb, vb, moved, ctx, nn, want_lse=True, check_status=True)
    assert torch.equal(got, want) and torch.equal(gl, wl)


def test_chunk_attention_many_sequences(dev):
    """More sequences than threads of a CTA, most of them short or empty; and more than
    the few-row kernel's page sums hold."""
    for B in (700, 2100):
        ctx = [(b * 37) % 90 if b % 5 else 0 for b in range(B)]
        nn = [1 if b % 3 else 0 for b in range(B)]
        args = _cache(15, ctx, nn, 1, 4, 2, 64)
        a, la, _ = _check_attn(args)
        b, lb, _ = _check_attn(args)
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_chunk_attention_one_long_among_short(dev):
    """Shares cut the long sequence many times and hold many short ones whole."""
    ctx = [30000] + [20 + 3 * b for b in range(60)]
    _check_attn(_cache(16, ctx, [1] * 61, 1, 8, 2, 128))


def test_chunk_attention_default_lengths_and_scale(dev):
    q, k, v, table, ctx, _ = _cache(9, [40, 41], [6, 6], 6, 16, 2, 128)
    _check_attn((q, k, v, table, ctx, None), scale=0.3)


def test_chunk_attention_matches_chain_trees(dev):
    """A chain tree of up to 64 nodes is a chunk: tree_attention on the same cache agrees."""
    q, k, v, table, ctx, nn = _cache(10, [100, 333], [64, 50], 64, 16, 2, 128)
    k, v = k.nan_to_num(0), v.nan_to_num(0)
    par = (torch.arange(64, device="cuda", dtype=torch.int32) - 1).expand(2, 64).contiguous()
    t, _, _ = a11spec.tree_attention(q, k, v, table, ctx, par, nn, max_kv_len=400, check_status=True)
    c, _, _ = _check_attn((q, k, v, table, ctx, nn), max_kv_len=400)
    _, tol, _, _ = R.attention(q, k, v, table, ctx, nn)
    assert R.worst(t, c, 2 * tol) <= 1


def test_chunk_attention_bad_pages_and_lengths(dev):
    q, k, v, table, ctx, nn = _cache(11, [40, 20, 30], [4, 4, 4], 4, 8, 1, 128)
    good, _, _ = _check_attn((q, k, v, table, ctx, nn))
    bad = table.clone()
    bad[1, 0] = k.shape[0]                                 # past the pool
    got, _, ws = a11spec.chunk_attention(q, k, v, bad, ctx, nn)
    assert ops.read_status(ws) == (_lib.EBOUNDS, 1)
    assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2]) and bool(got[1].isfinite().all())
    for b, (c, n) in enumerate(((-1, 4), (40, 5), (10 ** 6, 4))):  # negative, more than N, beyond the page table
        ctx2, nn2 = ctx.clone(), nn.clone()
        ctx2[b], nn2[b] = c, n
        got, _, ws = a11spec.chunk_attention(q, k, v, table, ctx2, nn2)
        assert ops.read_status(ws) == (_lib.EBOUNDS, b)
        assert bool((got[b] == 0).all())
        others = [i for i in range(3) if i != b]
        assert torch.equal(got[others], good[others])
    got, _, ws = a11spec.chunk_attention(q, k, v, table, ctx, nn)  # the next call clears the word
    assert ops.read_status(ws)[0] == _lib.OK and torch.equal(got, good)


def test_chunk_attention_nonfinite_scores(dev):
    """A NaN key reaches exactly the rows that see it."""
    q, k, v, table, ctx, nn = _cache(12, [10], [8], 8, 8, 1, 128)
    good, _, _ = _check_attn((q, k, v, table, ctx, nn))
    k[table[0].long()[14 // 16], 14 % 16] = math.nan  # token 4 of the chunk
    got, lse, _ = a11spec.chunk_attention(q, k, v, table, ctx, nn, want_lse=True)
    assert torch.equal(got[0, :4], good[0, :4]) and bool(got[0, 4:].isnan().all()) and bool(lse[0, 4:].isnan().all())


# --------------------------------------------------------------------------- together
def _layer(s):
    """A decoder layer's statements on the operators."""
    y, sc, _ = a11spec.add_rms_norm(s["h"], s["w_norm"], out_dtype=E4)
    qkv = a11spec.linear(y, s["w_qkv"], x_scale=sc, weight_scale=s["w_qkv_scale"])
    B, N = s["h"].shape[:2]
    q = qkv[..., :16 * 128].reshape(B, N, 16, 128)
    attn, _, _ = a11spec.chunk_attention(q, s["k"], s["v"], s["table"], s["ctx"], s["nn"], max_kv_len=190)
    o = a11spec.linear(attn.view(B, N, -1), s["w_o"])
    y, _, h = a11spec.add_rms_norm(o, s["w_norm"], residual=s["h"])
    return a11spec.linear(a11spec.linear(y, s["w_up"], gate=s["w_gate"], activation="silu"), s["w_down"], residual=h)


def _layer_state(seed, B, N):
    q, k, v, table, ctx, nn = _cache(seed, [150, 90][:B], [N] * B, N, 16, 2, 128)
    g = _gen(seed)
    s = dict(k=k, v=v, table=table, ctx=ctx, nn=nn, h=_rnd(g, B, N, 256, dtype=BF), w_norm=_rnd(g, 256, dtype=BF))
    s["w_qkv"], s["w_qkv_scale"] = _e4m3(_rnd(g, 16 * 128 + 512, 256, std=1 / 16))
    s["w_o"] = _rnd(g, 256, 2048, std=2048 ** -0.5, dtype=BF)
    s["w_up"], s["w_gate"] = _rnd(g, 512, 256, std=1 / 16, dtype=BF), _rnd(g, 512, 256, std=1 / 16, dtype=BF)
    s["w_down"] = _rnd(g, 256, 512, std=512 ** -0.5, dtype=BF)
    return s


@pytest.mark.parametrize("N", [1, 40])
def test_layer_captured_and_replayed(dev, N):
    """The operators in one graph; replays follow the inputs' new contents."""
    s = _layer_state(20, 2, N)
    want = _layer(s).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _layer(s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _layer(s)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    other = _layer_state(21, 2, N)
    for k in ("h", "w_o", "v"):
        if s[k].shape == other[k].shape:
            s[k].copy_(other[k].nan_to_num(0))
    want = _layer(s).clone()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_layers_on_two_streams(dev):
    """Two layers at once on streams of their own give what each gives alone."""
    a, b = _layer_state(22, 2, 40), _layer_state(23, 1, 33)
    wa, wb = _layer(a), _layer(b)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(sa):
            ga = [_layer(a) for _ in range(3)]
        with torch.cuda.stream(sb):
            gb = [_layer(b) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, wa) for x in ga) and all(torch.equal(x, wb) for x in gb)


def _chain(s, steps, each=lambda: None):
    """Norm, gated product, product, each writing what the next and the one after the next read."""
    for _ in range(steps):
        a11spec.add_rms_norm(s["h"], s["w"], residual=s["d"], sum_out=s["h"], out=s["y"])
        each()
        a11spec.linear(s["y"], s["up"], gate=s["gate"], activation="silu", out=s["a"])
        each()
        a11spec.linear(s["a"], s["down"], bias=s["bias"], out=s["d"])
        each()
        s["bias"].copy_(s["d"][0])  # a parameter that another library's kernel writes between calls
        each()


@pytest.mark.parametrize("rows,dim", [(1, 512), (20, 512), (70, 264), (300, 2048)])
def test_calls_in_a_row_see_each_others_results(dev, rows, dim):
    """Kernels that start over the tail of the one before read what it wrote:
    run together or captured, a chain in the same buffers gives the bits that it gives
    with a synchronisation after each call."""
    g = _gen(rows)
    s = dict(w=_rnd(g, dim, std=0.5, dtype=BF), up=_rnd(g, 2 * dim, dim, std=dim ** -0.5, dtype=BF), bias=_rnd(g, dim, dtype=BF),
             gate=_rnd(g, 2 * dim, dim, std=dim ** -0.5, dtype=BF), down=_rnd(g, dim, 2 * dim, std=dim ** -0.5, dtype=BF),
             h=_rnd(g, rows, dim, dtype=BF), d=_rnd(g, rows, dim, dtype=BF))
    s["y"], s["a"] = torch.empty_like(s["h"]), torch.empty(rows, 2 * dim, device="cuda", dtype=BF)
    start = {k: s[k].clone() for k in ("h", "d", "bias")}

    def run(f):
        for k, v in start.items():
            s[k].copy_(v)
        f()
        torch.cuda.synchronize()
        return torch.cat([s["h"], s["d"]]).clone()

    want = run(lambda: _chain(s, 40, torch.cuda.synchronize))
    assert bool(want.isfinite().all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _chain(s, 40)
    for _ in range(4):
        assert torch.equal(run(lambda: _chain(s, 40)), want)
        assert torch.equal(run(graph.replay), want)


@pytest.mark.parametrize("N", [1, 40])
def test_graph_with_a_fork_and_a_join(dev, N):
    """Two layers on forked streams in one graph, their results added after the join."""
    a, b = _layer_state(24, 2, N), _layer_state(25, 2, N)
    h0 = b["h"].clone()

    def both(side):
        x = _layer(a)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = _layer(b)
        z = _layer(dict(a, h=x))
        torch.cuda.current_stream().wait_stream(side)
        return _layer(dict(a, h=a11spec.add_rms_norm(z, a["w_norm"], residual=y)[0])), y

    b["h"] = h0 * 2
    want = [t.clone() for t in both(torch.cuda.Stream())]
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = both(side)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
