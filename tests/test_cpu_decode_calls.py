"""What the wrappers of the decoding operators hand to the C entries, seen with the launch taken out:
strides, what is refused, and what has run when it is.  No GPU."""
import ctypes
import warnings

import numpy as np
import pytest
import torch


@pytest.fixture(scope='module')
def nlp():
    import gluonnlp_amd
    return gluonnlp_amd


@pytest.fixture
def calls(nlp, monkeypatch):
    """The arguments of the launches that a call would make; CPU tensors count as device 0's."""
    got = []
    monkeypatch.setattr(nlp._tensor, 'device_index', lambda first, *rest: 0)
    monkeypatch.setattr(nlp._tensor, 'require_device', lambda *tensors: torch.device('cpu'))
    monkeypatch.setattr(nlp._tensor, 'launch', lambda index, fn, *args: got.append(args))
    return got


# logits (N, K, V) or (N K, V) as views -> (view, beams); element (r, v) of all rows is 1000 r + v
def _views():
    N, V = 4, 50
    rows = torch.arange(N)[:, None] * 1000.0 + torch.arange(V)
    return {
        'time-major, one beam': (rows[None].transpose(0, 1), 1),
        'unsqueezed': (rows.unsqueeze(1), 1),
        'one beam, wide rows': (torch.cat([rows, rows], 1)[:, :V].unsqueeze(1), 1),
        'one row, 3-d': (rows[:1, None], 1),
        'one row of many columns': (rows.t().contiguous()[:, :1].t(), 1),
        'a column as a row': (rows[0].reshape(V, 1).t(), 1),
        'a column as a row, 3-d': (rows[0].reshape(V, 1, 1).transpose(0, 2), 1),
        'one item': (rows[None], N),
        'one item, last of a wider tensor': (torch.stack([rows, rows])[1:], N),
        'one item, wide rows': (torch.cat([rows, rows], 1)[None, :, :V], N),
        'two items': (rows.reshape(2, 2, V), 2),
        'two items, beams first': (rows.reshape(2, 2, V).transpose(0, 1).contiguous()
                                   .transpose(0, 1), 2),
        'two items, wide': (torch.cat([rows, rows], 1).reshape(2, 2, 2 * V)[..., :V], 2),
        'every other beam': (rows.reshape(2, 2, V).repeat_interleave(2, 1)[:, ::2], 2),
        'beams of longer items': (torch.cat([rows.reshape(2, 2, V)] * 2, 1)[:, :2], 2),
        'expanded': (rows[:1].expand(4, V), 2),
        'one token': (rows[:, :1], 2),
        'one token, expanded': (rows[:1, :1].expand(4, 1), 2),
        'one token, 3-d, one beam': (rows[:, :1, None].transpose(1, 2), 1),
    }


@pytest.mark.parametrize('name', sorted(_views()))
def test_rows_of_the_logits(nlp, monkeypatch, calls, name):
    """Row r is V neighbouring elements, r row strides from the pointer, whatever the view's strides
    of axes of one element are; none of it lies outside the tensor."""
    x, K = _views()[name]
    V = x.shape[-1]
    N = x.numel() // V // K
    first = x.untyped_storage().data_ptr()
    end = first + x.untyped_storage().nbytes()
    seen = []

    def read(index, fn, *args):             # (at the call: a copy made for it lives that long)
        d, at = nlp._lib.BeamDesc.from_buffer_copy(args[8]), args[4]
        assert (d.N, d.K, d.V) == (N, K, V) and d.row_stride >= V
        if first <= at < end:
            assert at + 4 * ((N * K - 1) * d.row_stride + V) <= end
        else:
            assert d.row_stride == V
        seen.append(torch.stack([torch.tensor((ctypes.c_float * V).from_address(
            at + 4 * r * d.row_stride)[:]) for r in range(N * K)]))
    monkeypatch.setattr(nlp._tensor, 'launch', read)
    nlp.sequence_sampler.beam_search_select(x, torch.zeros(N, K))
    assert len(seen) == 1 and torch.equal(seen[0], x.reshape(N * K, V))


@pytest.mark.parametrize('given', ['edge_scores', 'mask', 'both'])
def test_a_bias_or_mask_over_no_keys_is_given(nlp, calls, given):
    """Its address is not NULL, which would let every key through, and it reaches 0 keys."""
    B, H, Lq, d = 2, 3, 2, 64
    c = nlp.kv_cache.QuantKVCache(B, H, d, 40, ctx='cpu')
    c.set_length(40)
    e, m = torch.zeros(B, H, Lq, 40), torch.ones(B, Lq, 40, dtype=torch.bool)
    kw = {'edge_scores': dict(edge_scores=e[..., :0]), 'mask': dict(mask=m[..., :0]),
          'both': dict(edge_scores=e[:1, ..., :0], mask=m[..., :1])}[given]
    nlp.attention_cell.multi_head_dot_attn_cached(torch.zeros(B, Lq, H, d), c, **kw)
    a = nlp._lib.Kv4AttnDesc.from_buffer_copy(calls[0][3])
    assert a.Lm == 0
    assert bool(a.edge_scores) == ('edge_scores' in kw) and bool(a.mask) == ('mask' in kw)


@pytest.mark.parametrize('dtype', [torch.int32, torch.int64, torch.int16, torch.float32])
@pytest.mark.parametrize('layout', ['NT', 'TN'])
def test_memory_lengths_end_at_the_memory(nlp, calls, layout, dtype):
    """Lengths beyond the memory mean all of it, as in gen_mem_attn_mask: not the rest of the buffer,
    which is rounded up to 32 slots."""
    items, Lm, H, d = 4, 11, 2, 8
    mem = torch.zeros((items, Lm, H * d) if layout == 'NT' else (Lm, items, H * d))
    states = nlp.kv_cache.quant_decoder_states(mem, torch.tensor([11, 40, 3, 0]).to(dtype),
                                               [(lambda m: m, lambda m: m)], H, d, 5, 2, layout)
    assert states.memory_cache.length.tolist() == [11, 11, 3, 0]
    assert states.length.tolist() == [0] * 8


def _cache(nlp, B, **kw):
    return nlp.kv_cache.QuantKVCache(B, 1, 8, 4, ctx='cpu', **kw)


def test_a_reordering_is_refused_before_anything_moves(nlp, calls):
    """Tensors stay as they are when a cache that comes with them does not fit."""
    Q = nlp.kv_cache.QuantDecoderStates
    x = torch.zeros(6, 4)
    p = torch.zeros(2, 3, dtype=torch.int32)
    big = torch.zeros(1, 40, dtype=torch.int32)
    for parents, t, cache in ((p, x, _cache(nlp, 5)), (p, x, Q(_cache(nlp, 9), _cache(nlp, 3))),
                              (p, x, Q(_cache(nlp, 8), _cache(nlp, 2))),
                              (big, torch.zeros(40, 4), _cache(nlp, 40))):
        for states, out in (([t, cache], None), ([cache, t], None), ([[t], (cache,)], None)):
            with pytest.raises(ValueError):
                nlp.sequence_sampler.reorder_states(states, parents, out=out)
            with pytest.raises(ValueError):
                nlp.sequence_sampler.reorder_states(states, parents, out=states)
        with pytest.raises(ValueError):
            cache.reorder(parents)
    assert not calls


def test_a_cache_moves_once(nlp, calls):
    """Also when it is listed beside the states that hold it, or twice."""
    Q = nlp.kv_cache.QuantDecoderStates
    rows, memory = _cache(nlp, 6), _cache(nlp, 6)
    p = torch.zeros(2, 3, dtype=torch.int32)
    s = Q(rows, memory)
    for states, moved in (([rows, rows], [rows]), ([s, rows], [rows, memory]),
                          ([rows, s, memory], [rows, memory]), ([s, s], [rows, memory]),
                          ([Q(rows, _cache(nlp, 2)), rows], [rows])):
        del calls[:]
        nlp.sequence_sampler.reorder_states(states, p)
        assert len(calls) == 2 * len(moved)                  # tokens, then lengths
        at = [(ctypes.c_int64 * 1).from_address(c.length.data_ptr()) for c in moved]
        assert sorted(args[6] for args in calls if args[6]) == sorted(map(ctypes.addressof, at))


@pytest.mark.parametrize('early_return', [True, False])
@pytest.mark.parametrize('K', [1, 3])
def test_beam_search_of_no_items(nlp, calls, K, early_return):
    def decoder(tokens, states):
        assert tokens.shape == (0,) and tokens.dtype == torch.int32
        return torch.zeros(0, 7), states
    sampler = nlp.sequence_sampler.BeamSearchSampler(K, decoder, 1, max_length=4,
                                                     early_return=early_return)
    samples, scores, valid = sampler(torch.zeros(0, dtype=torch.int64), [torch.zeros(0, 5)])
    assert samples.shape == (0, K, 2 if early_return else 5) and samples.dtype == torch.int32
    assert scores.shape == (0, K) and valid.shape == (0, K)


def _normalizes(nlp, calls, *args, **kw):
    """What BeamSearchSampler(*args, **kw) asks the selection for."""
    del calls[:]
    sampler = nlp.sequence_sampler.BeamSearchSampler(
        2, lambda tokens, states: (torch.zeros(2, 7), states), 1, 1.0, 5, 1, *args, **kw)
    sampler(torch.zeros(1, dtype=torch.int64), [])
    return nlp._lib.BeamDesc.from_buffer_copy(calls[0][8]).normalize


def test_beam_search_of_log_probabilities(nlp, calls):
    """``normalize`` as in the selection; its earlier name, which elsewhere says the opposite, works
    on and warns."""
    with warnings.catch_warnings():
        warnings.simplefilter('error')
        assert _normalizes(nlp, calls) == 1
        assert _normalizes(nlp, calls, normalize=False) == 0
        assert _normalizes(nlp, calls, 1.0, False) == 0       # (the place that from_logits had)
    for given in (True, False):
        with pytest.warns(FutureWarning, match='normalize'):
            assert _normalizes(nlp, calls, from_logits=given) == given


@pytest.mark.parametrize('eos', [1, np.int64(1), torch.tensor(1), None])
def test_beam_search_feeds_the_end_to_finished_beams(nlp, monkeypatch, eos):
    """Whole numbers of any kind as the end of sentence; tokens stay int32."""
    fed = []

    def decoder(tokens, states):
        fed.append(tokens.clone())
        return torch.zeros(tokens.shape[0], 7), states

    def select(outputs, scores, finished, **kw):
        return (scores, torch.zeros(2, 3, dtype=torch.int32),
                torch.tensor([[-1, 4, 5], [6, -1, -1]], dtype=torch.int32),
                torch.zeros(2, 3, dtype=torch.bool))
    monkeypatch.setattr(nlp._tensor, 'require_device', lambda *tensors: torch.device('cpu'))
    monkeypatch.setattr(nlp.sequence_sampler, 'beam_search_select', select)
    monkeypatch.setattr(nlp.sequence_sampler, 'reorder_states', lambda states, *a, **kw: states)
    nlp.sequence_sampler.BeamSearchSampler(3, decoder, eos, max_length=2)(torch.tensor([2, 3]), [])
    pad = 0 if eos is None else 1
    assert [t.tolist() for t in fed] == [[2, 2, 2, 3, 3, 3], [pad, 4, 5, 6, pad, pad]]
    assert all(t.dtype == torch.int32 for t in fed)


def test_tensors_that_a_reordering_writes_count_it(nlp, monkeypatch, calls):
    """Their version moves, as in any change in place: a memory's projections, which the decoders
    keep with the states, are those of its values at the time."""
    monkeypatch.setattr(nlp._tensor, 'device_index', lambda *tensors: -1)    # (a CPU tensor's own)
    p = torch.zeros(2, 3, dtype=torch.int32)
    states = [torch.zeros(6, 4), (torch.zeros(6, 4), torch.zeros(5, 6, 2)), None]
    axes = [0, (0, 1), 0]
    flat = [states[0], *states[1]]

    def versions(x):
        return [t._version for t in x]
    before = versions(flat)
    nlp.sequence_sampler.reorder_states(states, p, axes)
    assert versions(flat) == before
    nlp.sequence_sampler.reorder_states(states, p, axes, out=states)
    assert all(a > b for a, b in zip(versions(flat), before))
    before, out = versions(flat), [torch.empty(6, 4), (torch.empty(6, 4), torch.empty(5, 6, 2)), None]
    nlp.sequence_sampler.reorder_states(states, p, axes, out=out)
    assert versions(flat) == before and all(versions([out[0], *out[1]]))
