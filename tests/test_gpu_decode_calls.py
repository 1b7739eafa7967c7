"""Calls of the decoding operators that their documentation allows and ordinary use does not make, on
the GPU against the plain evaluations in 64 bits (tests/decode_ref.py)."""
import math

import pytest
import torch

from tests import decode_ref as ref
from tests.test_gpu_decode import _check, _filled

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


# ------------------------------------------------------------------ attention, past a wave's first tile
def _rising(nlp, g, B, Hc, d, T, lengths, dtype):
    """_filled with keys that grow five-fold towards the end: the largest score comes late, and what is
    summed up until then is scaled down."""
    c, _, _, _ = _filled(nlp, g, B, Hc, d, T, T, lengths, dtype)
    grow = 1 + 4 * torch.arange(T)[None, :, None, None] / T
    k = (torch.randn(B, T, Hc, d, generator=g) * grow).to(dtype)
    v = (torch.randn(B, T, Hc, d, generator=g) + 0.5).to(dtype)
    c.set_length(T)
    kk, vv = k.clone(), v.clone()
    for b in range(B):
        kk[b, int(lengths[b]):] = math.nan
        vv[b, int(lengths[b]):] = math.nan
    c.write(kk.cuda(), vv.cuda())
    c.set_length(torch.as_tensor(lengths).int().cuda())
    (qk, ks, km), (qv, _, _) = ref.quantise(k), ref.quantise(v)
    return c, qk, qv, (ks.max().item(), km.abs().max().item(), qv.abs().max().item())


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('d', [64, 128, 72])
@pytest.mark.parametrize('Lq,share', [(1, 1), (2, 1), (1, 4), (3, 3), (10, 2)])
def test_attention_over_many_tiles(nlp, dtype, d, Lq, share):
    """One workgroup a sequence, and several with a few rounds of tiles each: rows of 1, 2, 4 and 16,
    with and without bias and mask; lengths that end inside a round."""
    B, Hc = 3, 1
    for T, lengths in ((2100, [2100, 1337, 513]), (1025, [1025, 1024, 1])):
        g = _gen(T + d + Lq)
        c, k, v, size = _rising(nlp, g, B, Hc, d, T, lengths, dtype)
        q = torch.randn(B, Lq, share, d, generator=g).to(dtype)
        e = torch.randn(1, share, Lq, T, generator=g).to(dtype)
        table = torch.randn(share, 300, generator=g).to(dtype)
        m = torch.rand(B, Lq, T, generator=g) < 0.8
        m[1, 0, 300:] = False                               # nothing left after the first tiles
        m[0, Lq - 1, :1000] = False                         # nothing in them
        t = math.sqrt(d)
        tol = ref.attention_tolerance(q, *size, T, t, dtype)
        for kw in ({}, dict(edge=e, mask=m), dict(table=table)):
            want = ref.attention(q, k, v, lengths, share, temperature=t, **kw)
            names = {'edge': 'edge_scores', 'table': 'edge_table', 'mask': 'mask'}
            dev = {names[n]: x.cuda() for n, x in kw.items()}
            for bound in (1, 700, T):
                c._bound = bound
                got = nlp.attention_cell.multi_head_dot_attn_cached(q.cuda(), c, **dev)
                _check(got.reshape(B, Lq, share, d), want, tol)


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('d,B,Hc,T', [(64, 65, 8, 520), (128, 33, 8, 270)])
def test_attention_of_many_sequences(nlp, dtype, d, B, Hc, T):
    """More sequences and heads than are split: the first tiles are requested before the lengths are
    known.  Lengths of 0 and 1 among them; NaN behind all of them."""
    g = _gen(d)
    lengths = torch.randint(2, T + 1, (B,), generator=g)
    lengths[:6] = torch.tensor([0, 1, T, 0, T - 1, 65])
    c, k, v, size = _filled(nlp, g, B, Hc, d, T, T, lengths, dtype)
    c._bound = T
    t = math.sqrt(d)
    for Lq in (1, 2, 3, 5):
        q = torch.randn(B, Lq, Hc, d, generator=g).to(dtype)
        got = nlp.attention_cell.multi_head_dot_attn_cached(q.cuda(), c)
        want = ref.attention(q, k, v, lengths, temperature=t)
        _check(got.reshape(B, Lq, Hc, d), want,
               ref.attention_tolerance(q, *size, T, t, dtype))
        assert (got[0] == 0).all() and (got[3] == 0).all()
        m = torch.rand(B, Lq, T, generator=g) < 0.7
        got = nlp.attention_cell.multi_head_dot_attn_cached(q.cuda(), c, mask=m.cuda())
        want = ref.attention(q, k, v, lengths, mask=m, temperature=t)
        _check(got.reshape(B, Lq, Hc, d), want,
               ref.attention_tolerance(q, *size, T, t, dtype))


def test_reordering_with_a_cache_that_does_not_fit(nlp):
    """Refused with everything as it was."""
    g = _gen(7)
    x = torch.randn(6, 33, generator=g).cuda()
    before = x.clone()
    c = nlp.kv_cache.QuantKVCache(5, 2, 64, 8, ctx='cuda')
    p = torch.tensor([[2, 0, 1], [1, 1, 0]]).cuda()
    states = [x, c]
    with pytest.raises(ValueError):
        nlp.sequence_sampler.reorder_states(states, p, out=states)
    assert torch.equal(x, before)


def test_states_and_their_cache_move_once(nlp):
    g = _gen(8)
    rows = nlp.kv_cache.QuantKVCache(6, 2, 64, 20, ctx='cuda')
    lengths = torch.tensor([3, 20, 7, 0, 12, 1])
    k = torch.randn(6, 20, 2, 64, generator=g).cuda()
    rows.set_length(20)
    rows.write(k, -k)
    rows.set_length(lengths.cuda())
    memory = nlp.kv_cache.QuantKVCache(2, 2, 64, 5, ctx='cuda')
    before = rows.read()
    p = torch.tensor([[2, 0, 1], [1, 2, 0]])
    nlp.sequence_sampler.reorder_states(
        [nlp.kv_cache.QuantDecoderStates(rows, memory), rows], p.cuda())
    at = (torch.arange(2)[:, None] * 3 + p).reshape(-1)
    assert torch.equal(rows.length.cpu().long(), lengths[at])
    for a, b in zip(rows.read(), before):
        assert torch.equal(a.cpu(), b.cpu()[at])


@pytest.mark.parametrize('Lq', [1, 2, 4, 9])
def test_attention_averages_that_cancel(nlp, Lq):
    """bfloat16, 16 tokens of one weight whose values cancel, beside a token of zeros: what the two
    bfloat16 parts of a weight lose must not come in times 16 + n (the form in which codes are
    multiplied), but cancel as the values do."""
    H, d, T = 2, 64, 17
    b = -torch.arange(20, 200).float() / 64                     # (bfloat16 numbers, to 8 bits)
    b = b[b == b.bfloat16().float()]
    pv = torch.exp(b) * 0.125
    part = pv.bfloat16().float()
    lost = (pv - part - (pv - part).bfloat16().float()).abs() / pv
    b = b[lost.argmax()].item()
    assert lost.max() > 0.8 * 2.0 ** -18
    v = torch.empty(1, T, H, d)
    v[:, 0::2], v[:, 1::2] = -0.0625, 0.0625                    # codes 7 and 8
    v[..., 0], v[..., 1] = -0.9375, 0.9375                      # scale 1/8, minimum -0.9375, exactly
    v[:, 16] = 0
    assert torch.equal(ref.quantise(v)[0], v.double())
    c = nlp.kv_cache.QuantKVCache(1, H, d, T, ctx='cuda')
    c.extend(T)
    c.write(torch.zeros_like(v).cuda(), v.cuda())
    e = torch.full((1, 1, 1, T), b)
    e[..., 16] = 0
    q = torch.zeros(1, Lq, H, d, dtype=BF16)
    got = nlp.attention_cell.multi_head_dot_attn_cached(q.cuda(), c, causal=False, scaled=False,
                                                        edge_scores=e.cuda())
    want = ref.attention(q, torch.zeros_like(v).double(), v.double(), [T], causal=False, edge=e)
    # 32-bit sums over 17 tokens of products of at most 23.5 scales (half a step each, and 8 more to
    # join lanes and waves), the output's half step and that of exp(b) in the two large channels
    tol = 25 * 2.0 ** -24 * 23.5 * 0.125 + want.abs() * (2.0 ** -8 + 2.0 ** -20)
    err = (got.reshape(1, Lq, H, d).cpu().double() - want).abs()
    assert (err <= tol).all(), (err - tol).max()


def test_a_memory_reordered_in_place_is_projected_again(nlp):
    """Float states, the memory among them: after a reordering in place a step gives what it gives
    after one into new tensors."""
    torch.manual_seed(5)
    m = nlp.models.T5Decoder(d_model=64, d_kv=16, d_ff=96, num_layers=1, num_heads=4).cuda()
    for p in m.parameters():
        with torch.no_grad():
            p.copy_(0.2 * torch.randn(p.shape))
    g = _gen(9)
    mem = torch.randn(4, 7, 64, generator=g).cuda()
    x = torch.randn(4, 1, 64, generator=g).cuda()
    vl = torch.tensor([7, 5, 6, 7]).cuda()
    parents = torch.tensor([[1, 0], [1, 1]]).cuda()
    outs = []
    with torch.no_grad():
        for in_place in (False, True):
            mine = mem.clone()
            out, caches = m.incremental_decode(x, None, m._init_key_values(4, 'cuda'), mine, vl)
            states = (mine, caches)
            states = nlp.sequence_sampler.reorder_states(states, parents,
                                                         out=states if in_place else None)
            assert (states[0] is mine) == in_place
            out, _ = m.incremental_decode(x, None, states[1], states[0], vl)
            outs.append(out)
    assert torch.equal(*outs)
