"""TreeDecoder on the library's own layer operators (fused=True, fused="e4m3")
and prompts in chunks longer than a tree.

bf16: the golden decode of the reference (test_tree_decoder_gpu.py) within the
same bound as the unfused stack: both round to bf16 where the reference does,
the fused one less often.
e4m3: rounding to e4m3 is off by a relative 0.026 (rms: half a step is 2^-4 at
most, uniform in between), so a product of two rounded operands by 0.037. Per
layer three such products reach the residual stream (q/k/v, gate, up); were
they all to add up, two layers would move the logits by 2 * 3 * 0.037 = 0.22 of
their norm."""
import numpy as np
import pytest
import torch

from a11spec.decoder import SpeculativeDecoder
from a11spec.generate import speculative_stream
from a11spec.ops import KVPagePool
from a11spec.tree_model import DecoderConfig, TreeDecoder, synthetic_tensors
from test_tree_decoder_gpu import CFG, GOLD, PAGES, TOL_REL

pytestmark = pytest.mark.gpu


def _model(dev, fused, cfg=CFG, extra=None):
    t = synthetic_tensors(cfg, int(GOLD["weight_seed"]))
    t.update(extra or {})
    return TreeDecoder(t, cfg, PAGES, dev, fused=fused)


def _pool(dev, T):
    pool = KVPagePool(PAGES, dev)
    table = torch.full((1, 32), -1, dtype=torch.int32, device=dev)
    ctx = torch.zeros(1, dtype=torch.int32, device=dev)
    pool.reserve(table, ctx, torch.full((1,), T, dtype=torch.int32, device=dev), check_status=True)
    return pool, table, ctx


def _decode(model, dev, steps=None):
    """Teacher-forced one-token logits over the golden sequence."""
    prompt = torch.from_numpy(GOLD["prompt"]).to(dev).view(1, -1)
    T = prompt.shape[1]
    pool, table, ctx = _pool(dev, T - 1)
    model.prefill(prompt[:, :T - 1], table)
    one = torch.ones(1, dtype=torch.int32, device=dev)
    par = torch.full((1, 1), -1, dtype=torch.int32, device=dev)
    tok, out = int(GOLD["prompt"][-1]), []
    for k in range(steps or len(GOLD["tokens"])):
        grown = ctx.clone()
        pool.reserve(table, grown, one, check_status=True)
        out.append(model.forward_tree(torch.tensor([[tok]], dtype=torch.int32, device=dev), par, one, table, ctx)[0, 0].float())
        ctx.copy_(grown)
        tok = int(GOLD["tokens"][k])
    return torch.stack(out)


def test_fused_decode_matches_reference(dev):
    got = _decode(_model(dev, True), dev).cpu().numpy()
    want = np.asarray(GOLD["logits"][:len(got)])
    err = np.abs(got - want).max(1) / np.abs(want).max(1)
    assert err.max() <= TOL_REL, err.max()


def test_e4m3_decode_stays_near(dev):
    a, b = _decode(_model(dev, False), dev, 16), _decode(_model(dev, "e4m3"), dev, 16)
    assert float((a - b).norm() / a.norm()) <= 0.22


def test_fused_with_biases_and_head_norms(dev):
    """The optional tensors: biases of every projection, norms of the q and k heads."""
    g = torch.Generator().manual_seed(5)
    extra = {}
    for l in range(CFG.n_layers):
        for name, n in (("attn_q", 1024), ("attn_v", 128), ("attn_output", 256), ("ffn_gate", 512), ("ffn_up", 512), ("ffn_down", 256)):
            extra[f"blk.{l}.{name}.bias"] = 0.3 * torch.randn(n, generator=g)
        for name in ("attn_q_norm", "attn_k_norm"):
            extra[f"blk.{l}.{name}.weight"] = 1 + 0.1 * torch.randn(128, generator=g)
    a, b = (_decode(_model(dev, f, extra=extra), dev, 8) for f in (False, True))
    # both are within TOL_REL of exact arithmetic, row by row
    assert float(((a - b).abs().amax(1) / a.abs().amax(1)).max()) <= 2 * TOL_REL


@pytest.mark.parametrize("fused", [False, True, "e4m3"])
@pytest.mark.parametrize("chunk", [100, 512])
def test_long_chunks_prefill_as_chain_trees(dev, fused, chunk):
    """The prompt's last logits and K/V, in chunks of 64 (chain trees) and longer
    (chunk attention): the attention's roundings differ, by less than the bound
    between two bf16 pipelines."""
    T = 300
    tokens = torch.randint(0, CFG.vocab, (1, T), generator=torch.Generator().manual_seed(3)).to(dev, torch.int32)
    logits = []
    for c in (64, chunk):
        model = _model(dev, fused)
        pool, table, ctx = _pool(dev, T)
        logits.append(model.prefill(tokens, table, chunk=c)[0, -1].float())
    rel = 0.22 if fused == "e4m3" else 2 * TOL_REL  # e4m3: a flipped rounding upstream counts as any other
    assert float((logits[0] - logits[1]).abs().max() / logits[0].abs().max()) <= rel


def test_fused_speculative_stream(dev):
    """Speculative generation on the fused stack commits its own greedy tokens."""
    def stream(table):
        dec = SpeculativeDecoder(table=table, log2_buckets=10, width_root=2, width_inner=1, max_depth=5, max_nodes=16,
                                 temperature=None, device=dev)
        prompt = torch.from_numpy(GOLD["prompt"]).to(dev).view(1, -1).contiguous()
        out, forwards = [], 0
        for new in speculative_stream(_model(dev, True), prompt, 24, dec, KVPagePool(PAGES, dev), max_pages=16, learn=True):
            out += new[0]
            forwards += 1
        return out, forwards
    out, _ = stream(torch.zeros((1 << 10, 4, 2), dtype=torch.int32))
    first_close = int(np.argmax(GOLD["gaps"] < 0.1)) if (GOLD["gaps"] < 0.1).any() else 24
    n = min(first_close, 20)
    assert out[:n] == GOLD["tokens"].tolist()[:n]


def test_fused_refusals(dev):
    t = synthetic_tensors(CFG, 1)
    with pytest.raises(ValueError, match="fused"):
        TreeDecoder(t, CFG, 4, dev, fused="fp4")
    with pytest.raises(ValueError, match="bfloat16"):
        TreeDecoder(t, CFG, 4, dev, compute_dtype=torch.float32, fused=True)
    odd = DecoderConfig(n_layers=1, n_embd=264, n_head=8, n_head_kv=1, head_dim=128, n_ff=512, vocab=512)
    with pytest.raises(ValueError, match="multiple of 16"):
        TreeDecoder(synthetic_tensors(odd, 1), odd, 4, dev, fused="e4m3")
