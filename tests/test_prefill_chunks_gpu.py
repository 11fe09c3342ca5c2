"""TreeDecoder.prefill in chunks: what it computes, and that the cache and the
logits do not depend on how the prompt is cut (beyond the roundings)."""
import pytest
import torch

from a11spec import ops
from a11spec.decoder import SpeculativeDecoder
from a11spec.generate import speculative_stream
from a11spec.ops import KVPagePool
from a11spec.tree_model import TreeDecoder, synthetic_tensors
from test_tree_decoder_gpu import CFG, GOLD, PAGES, TOL_REL

pytestmark = pytest.mark.gpu
B, T = 2, 300


def _prefill(dev, fused, chunk):
    """(model, pages of the prompts [B, ...], logits of the last chunk, calls of the LM head)."""
    model = TreeDecoder(synthetic_tensors(CFG, int(GOLD["weight_seed"])), CFG, PAGES, dev, fused=fused)
    heads = []
    head = model._head
    model._head = lambda hn: heads.append(hn.shape[1]) or head(hn)
    pool = KVPagePool(PAGES, dev)
    table = torch.full((B, 32), -1, dtype=torch.int32, device=dev)
    ctx = torch.zeros(B, dtype=torch.int32, device=dev)
    pool.reserve(table, ctx, torch.full((B,), T, dtype=torch.int32, device=dev), check_status=True)
    tokens = torch.randint(0, CFG.vocab, (B, T), generator=torch.Generator().manual_seed(5)).to(dev, torch.int32)
    logits = model.prefill(tokens, table, chunk=chunk)
    return model, table, logits, heads


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("chunk", [64, 100, 512])
def test_head_runs_on_the_last_chunk_only(dev, fused, chunk):
    model, _, logits, heads = _prefill(dev, fused, chunk)
    last = T - (T - 1) // chunk * chunk
    assert heads == [last] and logits.shape == (B, last, CFG.vocab)
    assert model.forwards == -(-T // chunk)


def _cached(pool, table, layer):
    """K or V of the prompts' positions [B, T, Hkv, D]."""
    pos = torch.arange(T, device=table.device)
    return pool[layer, table[:, pos // 16].long(), pos % 16].double()


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("chunk", [100, 512])
def test_cache_and_logits_do_not_depend_on_the_chunks(dev, fused, chunk):
    """Chunks of 64 (chain trees) against longer ones (chunk attention), all positions of
    both sequences.

    Layer 0 has no attention before its K and V: only the order of the projections' sums
    differs (256 products of magnitude sum below 2^4.5: 2^-23 * 256 * 2^4.5 each, below
    2^-10 together), so a projection may round to the neighbouring bf16 value (2^-7
    relative at most). V is that. K's pair (k1, k2) then turns by the same angle, which
    moves a component by up to 2^-7 (|k1| + |k2|) <= 2^-7 sqrt(2) of the pair's length, and
    is rounded again (a neighbour: 2^-7). Layer 1 and the logits come out of two bf16
    pipelines that are each within TOL_REL of exact arithmetic, row by row."""
    a, ta, la, _ = _prefill(dev, fused, 64)
    b, tb, lb, _ = _prefill(dev, fused, chunk)
    va, vb = _cached(a.v_pool, ta, 0), _cached(b.v_pool, tb, 0)
    assert bool(((va - vb).abs() <= 2.0 ** -7 * va.abs() + 2.0 ** -9).all())
    ka, kb = _cached(a.k_pool, ta, 0), _cached(b.k_pool, tb, 0)
    half = CFG.head_dim // 2
    length = torch.sqrt(ka[..., :half] ** 2 + ka[..., half:] ** 2).repeat(1, 1, 1, 2)
    assert bool(((ka - kb).abs() <= 2.0 ** -7 * (1.4143 * length + ka.abs()) + 2.0 ** -8).all())
    for pa, pb in ((a.k_pool, b.k_pool), (a.v_pool, b.v_pool)):
        x, y = _cached(pa, ta, 1).flatten(2), _cached(pb, tb, 1).flatten(2)
        assert float(x.abs().amax(2).min()) > 0  # every position was written
        assert float(((x - y).abs().amax(2) / x.abs().amax(2)).max()) <= 2 * TOL_REL
    n = min(la.shape[1], lb.shape[1])
    x, y = la[:, -n:].double(), lb[:, -n:].double()
    assert float(((x - y).abs().amax(2) / x.abs().amax(2)).max()) <= 2 * TOL_REL


@pytest.mark.parametrize("fused", [False, True])
def test_stream_prefills_in_long_chunks(dev, fused, monkeypatch):
    """speculative_stream(prefill_chunk=...) takes the prompt through chunk attention and
    commits the tokens that the default commits, up to the first step where the reference's
    own top two logits are closer than a rounding."""
    calls = []
    attend = ops.chunk_attention
    monkeypatch.setattr(ops, "chunk_attention", lambda q, *a, **k: calls.append(q.shape[1]) or attend(q, *a, **k))
    model = TreeDecoder(synthetic_tensors(CFG, int(GOLD["weight_seed"])), CFG, PAGES, dev, fused=fused)
    dec = SpeculativeDecoder(table=torch.zeros((1 << 10, 4, 2), dtype=torch.int32), log2_buckets=10, width_root=2, width_inner=1,
                             max_depth=5, max_nodes=16, temperature=None, device=dev)
    prompt = torch.from_numpy(GOLD["prompt"]).to(dev).view(1, -1).contiguous()
    out = []
    for new in speculative_stream(model, prompt, 24, dec, KVPagePool(PAGES, dev), max_pages=16, learn=True, prefill_chunk=512):
        out += new[0]
    assert calls == [prompt.shape[1] - 1] * CFG.n_layers
    first_close = int((GOLD["gaps"] < 0.1).argmax()) if (GOLD["gaps"] < 0.1).any() else 24
    n = min(first_close, 20)
    assert out[:n] == GOLD["tokens"].tolist()[:n]
