"""Calls of the decoding operators that their documentation allows and ordinary use does not make, on
the GPU against the plain evaluations in 64 bits (tests/decode_ref.py)."""
import math

import pytest
import torch

from tests import decode_ref as ref

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope='module')
def nlp():
    import gluonnlp_amd
    return gluonnlp_amd


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_select_from_views_with_axes_of_one(nlp, dtype):
    """One beam an item, logits as a view of a time-major output; one row as a view of a column."""
    N, V = 4, 1000
    g = _gen(1)
    rows = (3 * torch.randn(N, V, generator=g)).to(dtype).cuda()
    s = -torch.rand(N, 1, generator=g).cuda()
    want = ref.select(rows, s, None)
    for x in (rows[None].transpose(0, 1), rows.unsqueeze(1), rows):
        got = nlp.sequence_sampler.beam_search_select(x, s)
        assert torch.equal(got[1].cpu().long(), want[1])
        assert torch.equal(got[2].cpu().long(), want[2])
        # a logsumexp off by a few half steps of the largest term, the score rounded once
        assert ((got[0].cpu().double() - want[0]).abs()
                <= (want[0].abs() + 20) * 2.0 ** -24 * 8).all()
    for x in (rows[0].reshape(V, 1).t(), rows[0].reshape(V, 1, 1).transpose(0, 2)):
        got = nlp.sequence_sampler.beam_search_select(x, s[:1])
        assert got[2].cpu().long().tolist() == want[2][:1].tolist()


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_attention_with_a_bias_or_mask_over_no_keys(nlp, dtype):
    """Keys from Lm on are not seen; with Lm = 0 nothing is, and the result is zeros."""
    B, H, Lq, d, T = 2, 3, 2, 64, 700
    g = _gen(2)
    c = nlp.kv_cache.QuantKVCache(B, H, d, T, ctx='cuda')
    c.set_length(T)
    x = torch.randn(B, T, H, d, generator=g).to(dtype).cuda()
    c.write(x, x)
    q = torch.randn(B, Lq, H, d, generator=g).to(dtype).cuda()
    e, m = torch.zeros(B, H, Lq, T).cuda(), torch.ones(B, Lq, T, dtype=torch.bool).cuda()
    table = torch.zeros(H, 5).to(dtype).cuda()
    for kw in (dict(edge_scores=e[..., :0]), dict(mask=m[..., :0]), dict(mask=m[:1, :1, :0]),
               dict(edge_scores=e[..., :0], mask=m[..., :1]),
               dict(edge_scores=e[..., :0], mask=m[..., :0]),
               dict(edge_table=table, mask=m[..., :0])):
        for causal in (True, False):
            for bound in (1, T):                   # one and several workgroups a sequence
                c._bound = bound
                got = nlp.attention_cell.multi_head_dot_attn_cached(q, c, causal=causal, **kw)
                assert got.shape == (B, Lq, H * d) and (got == 0).all()


def test_memory_lengths_beyond_the_memory(nlp):
    """A decoder's step on 4-bit states: lengths beyond the memory are all of it."""
    torch.manual_seed(3)
    m = nlp.models.T5Decoder(d_model=64, d_kv=16, d_ff=96, num_layers=1, num_heads=4).cuda()
    for p in m.parameters():
        with torch.no_grad():
            p.copy_(0.2 * torch.randn(p.shape))
    g = _gen(4)
    mem, x = torch.randn(3, 11, 64, generator=g).cuda(), torch.randn(3, 1, 64, generator=g).cuda()
    outs = []
    with torch.no_grad():
        for vl in ([11, 11, 4], [12, 500, 4]):
            states = m.init_quant_states(mem, torch.tensor(vl).cuda(), 4)
            outs.append(m.incremental_decode(x, None, states, None, None)[0])
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1])
