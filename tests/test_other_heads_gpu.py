"""TreeDecoder with heads that tree attention does not take (64 wide, or groups other than
8): prefill and token-by-token decoding run through chunk attention; trees of several
nodes are refused as before."""
import dataclasses

import pytest
import torch

import a11spec
from a11spec.ops import KVPagePool
from a11spec.tree_model import TreeDecoder, rms_norm, rotary, synthetic_tensors
from test_tree_decoder_gpu import CFG, PAGES, TOL_REL

pytestmark = pytest.mark.gpu
T, STEPS = 90, 4


def _exact(t, cfg, tokens):
    """Logits [B, T, V] of the whole sequence in fp64 from the weights as the model holds them (bf16)."""
    w = {k: v.to(torch.bfloat16).double().cuda() for k, v in t.items()}
    B, n = tokens.shape
    pos = torch.arange(n, device="cuda").expand(B, n)
    seen = torch.ones(n, n, device="cuda", dtype=torch.bool).tril()
    h = w["token_embd.weight"][tokens.long()]
    for l in range(cfg.n_layers):
        b = f"blk.{l}."
        x = rms_norm(h, w[b + "attn_norm.weight"], cfg.rms_eps)
        q, k, v = (torch.matmul(x, w[b + f"attn_{c}.weight"].T).view(B, n, -1, cfg.head_dim) for c in "qkv")
        q, k = rotary(q, k, pos, cfg.rope_base)
        k, v = (z.repeat_interleave(cfg.n_head // cfg.n_head_kv, dim=2) for z in (k, v))
        s = torch.einsum("bihd,bjhd->bhij", q, k) / cfg.head_dim ** 0.5
        p = torch.softmax(s.masked_fill(~seen, -torch.inf), dim=-1)
        o = torch.einsum("bhij,bjhd->bihd", p, v).reshape(B, n, -1)
        h = h + torch.matmul(o, w[b + "attn_output.weight"].T)
        x = rms_norm(h, w[b + "ffn_norm.weight"], cfg.rms_eps)
        g = torch.matmul(x, w[b + "ffn_gate.weight"].T)
        h = h + torch.matmul(g * torch.sigmoid(g) * torch.matmul(x, w[b + "ffn_up.weight"].T), w[b + "ffn_down.weight"].T)
    return torch.matmul(rms_norm(h, w["output_norm.weight"], cfg.rms_eps), w["output.weight"].T)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("head_dim,n_head,n_head_kv", [(64, 6, 2), (128, 4, 4)])
@pytest.mark.parametrize("chunk", [64, 512])
def test_prefill_and_decode(dev, fused, head_dim, n_head, n_head_kv, chunk):
    cfg = dataclasses.replace(CFG, head_dim=head_dim, n_head=n_head, n_head_kv=n_head_kv)
    t = synthetic_tensors(cfg, 4)
    model = TreeDecoder(t, cfg, PAGES, dev, fused=fused)
    B = 2
    tokens = torch.randint(0, cfg.vocab, (B, T + STEPS), generator=torch.Generator().manual_seed(8)).to(dev, torch.int32)
    ref = _exact(t, cfg, tokens)
    pool = KVPagePool(PAGES, dev)
    table = torch.full((B, 16), -1, dtype=torch.int32, device=dev)
    ctx = torch.zeros(B, dtype=torch.int32, device=dev)
    pool.reserve(table, ctx, torch.full((B,), T, dtype=torch.int32, device=dev), check_status=True)
    got = [model.prefill(tokens[:, :T].contiguous(), table, chunk=chunk)]
    one, par = torch.ones(B, dtype=torch.int32, device=dev), torch.full((B, 1), -1, dtype=torch.int32, device=dev)
    for i in range(STEPS):
        grown = ctx.clone()
        pool.reserve(table, grown, one, check_status=True)
        got.append(model.forward_tree(tokens[:, T + i:T + i + 1].contiguous(), par, one, table, ctx))
        ctx.copy_(grown)
    got = torch.cat(got, dim=1).double()
    want = ref[:, -got.shape[1]:]
    # one bf16 pipeline against exact arithmetic: half of what two may differ by
    assert float(((got - want).abs().amax(2) / want.abs().amax(2)).max()) <= TOL_REL
    two = torch.tensor([[-1, 0]] * B, dtype=torch.int32, device=dev)
    with pytest.raises(a11spec.A11Error, match="a11s_tree_attention"):
        model.forward_tree(tokens[:, :2].contiguous(), two, 2 * one, table, ctx)
