"""The decoders on states held in 4 bits, and beam search over them: the operators run together, as
they are used."""
import itertools
import math

import pytest
import torch

from tests import decode_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def nlp():
    import gluonnlp_amd
    from gluonnlp_amd import _lib
    _lib.load()
    return gluonnlp_amd


class _FloatCache:
    """QuantKVCache's interface on float tensors: what the 4-bit cache approximates."""

    def __init__(self, batch_size, num_heads, head_units, max_length, num_layers=1, ctx=None,
                 layout='NTK'):
        self.batch_size, self.num_heads, self.head_units = batch_size, num_heads, head_units
        self.layout, self.max_length = layout, max_length
        self.kv = torch.zeros(2, num_layers, batch_size, max_length, num_heads, head_units,
                              device=ctx)
        self.length = torch.zeros(batch_size, dtype=torch.int32, device=ctx)

    def _ntk(self, x):
        return x.float().transpose(0, 1) if self.layout == 'TNK' else x.float()

    def set_length(self, n):
        self.length.copy_(n if isinstance(n, torch.Tensor) else torch.full_like(self.length, n))

    def extend(self, n):
        self.length += n

    def write(self, key, value, layer=0):
        for which, x in enumerate((key, value)):
            x = self._ntk(x)
            for b in range(self.batch_size):
                end = int(self.length[b])
                self.kv[which, layer, b, end - x.shape[1]:end] = x[b]

    def reorder(self, parents):
        K = parents.shape[1]
        at = (torch.arange(parents.shape[0], device=parents.device)[:, None] * K +
              parents).reshape(-1)
        self.kv = self.kv[:, :, at]
        self.length = self.length[at]


def _float_attention(query, cache, layer=0, causal=True, edge_table=None, scaled=True, layout=None):
    layout = layout or cache.layout
    q = query.transpose(0, 1) if layout == 'TNK' else query
    out = ref.attention(q, cache.kv[0, layer].cpu().double(), cache.kv[1, layer].cpu().double(),
                        cache.length.tolist(), causal=causal, table=edge_table,
                        temperature=math.sqrt(q.shape[-1]) if scaled else 1.0)
    out = out.to(query.device, query.dtype)
    out = out.transpose(0, 1) if layout == 'TNK' else out
    return out.reshape(out.shape[0], out.shape[1], -1).contiguous()


def _decoder(nlp, kind, layout, dtype='float32'):
    torch.manual_seed(3)
    if kind == 't5':
        m = nlp.models.T5Decoder(d_model=64, d_kv=16, d_ff=96, num_layers=2, num_heads=4,
                                 activation='gated-gelu', layout=layout, dtype=dtype)
    else:
        m = nlp.models.TransformerDecoder(num_layers=2, units=64, mem_units=64, hidden_size=96,
                                          num_heads=4, layout=layout, dtype=dtype,
                                          pre_norm=kind == 'pre', recurrent=kind == 'pre')
    for n, p in m.named_parameters():
        with torch.no_grad():
            p.copy_(0.2 * torch.randn(p.shape) + (1.0 if n.endswith('gamma') else 0.0))
    return m.cuda()


def _step(m, kind, layout, x, states, mem, vl):
    if kind == 't5':
        step = x.unsqueeze(1 if layout == 'NT' else 0)
        out, states = m.incremental_decode(step, None, states, mem, vl)
        return out.squeeze(1 if layout == 'NT' else 0), states
    return m.incremental_decode(x, states, mem, vl)


@pytest.mark.parametrize('layout', ['NT', 'TN'])
@pytest.mark.parametrize('kind', ['t5', 'post', 'pre'])
def test_quant_states_follow_the_float_states(nlp, monkeypatch, kind, layout):
    """With a cache and an attention in floats in the 4-bit ones' place, the path through
    init_quant_states and incremental_decode is the decoders' own: the same biases, scalings,
    memory lengths and orders."""
    m = _decoder(nlp, kind, layout)
    B, Lm, C, steps = 3, 11, 64, 6
    g = torch.Generator().manual_seed(1)
    mem = torch.randn(B, Lm, C, generator=g).cuda()
    mem = mem if layout == 'NT' else mem.transpose(0, 1).contiguous()
    vl = torch.tensor([11, 4, 7], dtype=torch.int32).cuda()
    xs = [torch.randn(B, C, generator=g).cuda() for _ in range(steps)]
    with torch.no_grad():
        states = m._init_key_values(B, 'cuda') if kind == 't5' else m.init_states(B, 'cuda')
        want = []
        for x in xs:
            out, states = _step(m, kind, layout, x, states, mem, vl)
            want.append(out)
        monkeypatch.setattr(nlp.kv_cache, 'QuantKVCache', _FloatCache)
        for mod in (nlp.models.t5, nlp.models.transformer):
            monkeypatch.setattr(mod, 'multi_head_dot_attn_cached', _float_attention)
        states = m.init_quant_states(mem, vl, max_length=steps)
        for x, w in zip(xs, want):
            out, states = _step(m, kind, layout, x, states, None, None)
            # two float32 evaluations of the same layers, sums of up to 96 terms
            assert (out - w).abs().max() <= 2e-5 * w.abs().max()


@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
@pytest.mark.parametrize('kind,layout', [('t5', 'NT'), ('t5', 'TN'), ('post', 'NT')])
def test_quant_states_with_beams(nlp, monkeypatch, kind, layout, dtype):
    """Decoding steps with reordering in between: every attention call against a plain evaluation
    on the values that its cache reads back."""
    m = _decoder(nlp, kind, layout, dtype)
    items, K, Lm, C, steps = 2, 3, 9, 64, 5
    g = torch.Generator().manual_seed(2)
    dt = getattr(torch, dtype)
    mem = torch.randn(items, Lm, C, generator=g).to(dt).cuda()
    mem = mem if layout == 'NT' else mem.transpose(0, 1).contiguous()
    vl = torch.tensor([9, 5]).cuda()
    real = nlp.attention_cell.multi_head_dot_attn_cached
    calls = []

    def checked(query, cache, layer=0, causal=True, edge_table=None, scaled=True, layout=None):
        got = real(query, cache, layer, causal=causal, edge_table=edge_table, scaled=scaled,
                   layout=layout)
        lay = layout or cache.layout
        k, v = cache.read(layer=layer)
        if cache.layout == 'TNK':
            k, v = k.transpose(0, 1), v.transpose(0, 1)
        q = query.transpose(0, 1) if lay == 'TNK' else query
        out = got.transpose(0, 1) if lay == 'TNK' else got
        t = math.sqrt(q.shape[-1]) if scaled else 1.0
        want = ref.attention(q, k.cpu().double(), v.cpu().double(), cache.length.tolist(),
                             causal=causal, table=edge_table, temperature=t)
        span = k.abs().max().item()
        tol = ref.attention_tolerance(q, 2 * span / 15, span, v.abs().max().item(), k.shape[1], t,
                                      dt)
        err = (out.reshape(want.shape).cpu().double() - want).abs().max().item()
        assert err <= tol
        calls.append(causal)
        return got
    for mod in (nlp.models.t5, nlp.models.transformer):
        monkeypatch.setattr(mod, 'multi_head_dot_attn_cached', checked)
    with torch.no_grad():
        states = m.init_quant_states(mem, vl, max_length=steps, beam_size=K)
        for step in range(steps):
            x = torch.randn(items * K, C, generator=g).to(dt).cuda()
            out, states = _step(m, kind, layout, x, states, None, None)
            assert out.shape == (items * K, C) and torch.isfinite(out).all()
            parents = torch.randint(0, K, (items, K), generator=g).int().cuda()
            before = states.self_cache.read(layer=1)[0]
            nlp.sequence_sampler.reorder_states(states, parents)
            at = (torch.arange(items).cuda()[:, None] * K + parents).reshape(-1)
            axis = 0 if layout == 'NT' else 1
            assert torch.equal(states.self_cache.read(layer=1)[0], before.index_select(axis, at))
    assert states.length.tolist() == [steps] * (items * K)
    assert len(calls) == steps * 4


def test_a_step_with_quant_states_is_captured(nlp):
    """One T5 decoding step as a graph, replayed: the lengths move on the device."""
    m = _decoder(nlp, 't5', 'NT', 'bfloat16')
    B, steps = 2, 6
    g = torch.Generator().manual_seed(5)
    mem = torch.randn(B, 7, 64, generator=g).bfloat16().cuda()
    xs = [torch.randn(B, 1, 64, generator=g).bfloat16().cuda() for _ in range(steps)]
    with torch.no_grad():
        states = m.init_quant_states(mem, None, steps)
        want = [m.incremental_decode(x, None, states, None, None)[0] for x in xs]
        states = m.init_quant_states(mem, None, steps)
        x = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        m.incremental_decode(x, None, states, None, None)          # (warm: library state)
        states.self_cache.reset()
        with torch.cuda.graph(graph):
            out, _ = m.incremental_decode(x, None, states, None, None)
        states.self_cache.reset()
        for i in range(steps):
            x.copy_(xs[i])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[i])


def test_gradients_are_refused(nlp):
    m = _decoder(nlp, 't5', 'NT')
    mem = torch.randn(1, 4, 64).cuda()
    states = m.init_quant_states(mem, None, 4)
    m.requires_grad_(True)             # (the framework's parameters ask for none by themselves)
    with pytest.raises(NotImplementedError, match='no_grad'):
        m.incremental_decode(torch.randn(1, 1, 64).cuda(), None, states, None, None)


def test_bias_table_reaches_all_distances(nlp):
    """The states keep T5's bias up to max_distance; what lies further has the last entry's."""
    m = _decoder(nlp, 't5', 'NT')
    far = 400
    full = m.relative_position_encoder.self_attn_bias_table(far)[:, :far]
    table = m.init_quant_states(torch.randn(1, 4, 64).cuda(), None, far).bias_table
    R = table.shape[1]
    assert R < far and torch.equal(table, full[:, far - R:])
    assert torch.equal(full[:, :far - R], table[:, :1].expand(-1, far - R))


def test_a_refused_step_counts_no_token(nlp):
    """Gradients and steps of another shape are refused before the lengths move."""
    for kind, shape in (('t5', (2, 1, 64)), ('post', (2, 64))):
        m = _decoder(nlp, kind, 'NT')
        states = m.init_quant_states(torch.randn(2, 4, 64).cuda(), None, 4)
        assert states.bias_table is None or not states.bias_table.requires_grad

        def step(x):
            return m.incremental_decode(x, None, states, None, None) if kind == 't5' else \
                m.incremental_decode(x, states, None, None)
        with torch.no_grad():
            step(torch.randn(*shape).cuda())
            with pytest.raises(ValueError, match='rows'):
                step(torch.randn(*((3,) + shape[1:])).cuda())
        with pytest.raises(NotImplementedError, match='no_grad'):
            step(torch.randn(*shape).cuda().requires_grad_(True))
        m.requires_grad_(True)
        with pytest.raises(NotImplementedError, match='no_grad'):
            step(torch.randn(*shape).cuda())
        assert states.length.tolist() == [1, 1]


# ------------------------------------------------------------------------------------ beam search
def _bigram(V, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(V, V, generator=g) * 2


@pytest.mark.parametrize('alpha', [0.0, 0.8])
def test_beam_search_finds_the_best(nlp, alpha):
    """A bigram model, a beam as wide as needed: the sampler's sequences are the best of all."""
    V, T, eos, N = 4, 3, 0, 2
    table = _bigram(V, 1)
    logp = torch.log_softmax(table.double(), -1)
    dev = table.cuda()
    seen = torch.zeros(N * 16, 1).cuda()

    def decoder(tokens, states):
        return dev[tokens.long()], [states[0] + 1]
    sampler = nlp.sequence_sampler.BeamSearchSampler(16, decoder, eos, alpha=alpha, length_base=5,
                                                     max_length=T, early_return=False)
    first = torch.tensor([1, 3]).cuda()
    samples, scores, vl = sampler(first, [seen])
    for n in range(N):
        every = {}
        for seq in itertools.product(range(V), repeat=T):
            cut = seq[:seq.index(eos) + 1] if eos in seq else seq
            s, prev = 0.0, int(first[n])
            for t in cut:
                s += logp[prev, t].item()
                prev = t
            every[cut] = s / (((5 + len(cut)) / 6.0) ** alpha)
        best = sorted(every.items(), key=lambda kv: -kv[1])
        got = [tuple(samples[n, k, 1:int(vl[n, k])].tolist()) for k in range(16)]
        assert len(set(got)) == 16 and set(got) <= set(every)
        # (scores are kept in float32 between the steps: T half steps, and the selection's own)
        for k in range(16):
            assert abs(scores[n, k].item() - every[got[k]]) <= 2e-5
        if alpha == 0.0:           # a prefix scores no less than what follows it: nothing is lost
            assert got[0] == best[0][0]


def test_beam_search_on_quant_states(nlp):
    """T5 decoder, tied output weights, 4-bit states: the sequences' scores are what teacher forcing
    of the same sequences gives on the same kind of states."""
    m = _decoder(nlp, 't5', 'NT')
    V, N, K, T = 40, 2, 4, 5
    g = torch.Generator().manual_seed(7)
    emb = torch.randn(V, 64, generator=g).cuda()
    mem = torch.randn(N, 6, 64, generator=g).cuda()
    vl = torch.tensor([6, 3]).cuda()
    first = torch.tensor([1, 2]).cuda()

    def decoder(tokens, states):
        h, states = m.incremental_decode(emb[tokens.long()].unsqueeze(1), None, states, None, None)
        return torch.matmul(h.squeeze(1), emb.t().contiguous()) * 0.2, states
    with torch.no_grad():
        sampler = nlp.sequence_sampler.BeamSearchSampler(K, decoder, 0, alpha=0.0, max_length=T)
        samples, scores, valid = sampler(first, m.init_quant_states(mem, vl, T, K))
        assert (scores[:, :-1] >= scores[:, 1:]).all()
        states = m.init_quant_states(mem, vl, T, K)
        total = torch.zeros(N * K, dtype=torch.float64).cuda()
        rows = samples.reshape(N * K, -1)
        for t in range(rows.shape[1] - 1):
            logits, states = decoder(rows[:, t].clamp(min=0), states)
            logp = torch.log_softmax(logits.double(), -1)
            nxt = rows[:, t + 1]
            got = logp.gather(1, nxt.clamp(min=0).long()[:, None])[:, 0]
            total += torch.where(nxt >= 0, got, torch.zeros_like(got))
        # scores in float32 between the steps; the caches of both runs hold the same codes
        assert (total.reshape(N, K) - scores.double()).abs().max().item() <= 1e-4
