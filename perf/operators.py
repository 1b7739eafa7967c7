"""The operators of incremental decoding, with their plain forms: a key / value cache held in 4 bits
(written, read back, attended over), the selection step of a beam search, and the reordering of the
decoding states that follows it.

The 4-bit format: every group of 64 consecutive channels of one token and head (the last group may
be shorter) holds a scale and a minimum in bfloat16 and a code 0..15 per channel,

    scale = bf16((max - min) * fl32(1 / 15)),  minimum = bf16(min)
    code  = clamp(rint((x - minimum) / scale), 0, 15),  value = code * scale + minimum

evaluated in 32 bits, so that a code is a definite whole number; a group without spread (a scale
below 2^-126) has scale and codes 0.

Each operator runs in its plain form (torch operations in 32 or 64 bits) or, where ``own`` is true,
as the calls that a user of ``gluonnlp_amd`` makes.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = 'cuda'
GROUP = 64
BF16, F32 = 'bfloat16', 'float32'


def _package():
    path = os.path.join(_ROOT, 'gluon-nlp_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    import gluonnlp_amd
    return gluonnlp_amd


def listed():
    return [
        # one decoding step of 16 sequences: the new token of every row goes into the cache
        dict(name='cache step', op='cache', rows=16, heads=12, units=64, new=1, past=200, ragged=False,
             dtype=BF16),
        # prompts of unequal length are cached at once, as after an encoder or a prompt pass
        dict(name='cache prompts', op='cache', rows=32, heads=16, units=64, new=512, past=0,
             ragged=True, dtype=BF16),
        # the smallest useful call: greedy decoding of one sentence with a T5 position bias
        dict(name='attention one sentence', op='attention', rows=1, heads=8, share=1, units=64,
             queries=1, keys=40, causal=True, bias='table', dtype=BF16),
        # a batch of sequences mid-way through their answers, ragged lengths
        dict(name='attention batch step', op='attention', rows=64, heads=16, share=1, units=64,
             queries=1, keys=1000, causal=True, bias='none', dtype=BF16),
        # beams that share their sentence's encoder memory: the beams are the queries
        dict(name='attention beams on memory', op='attention', rows=32, heads=12, share=1, units=64,
             queries=8, keys=512, causal=False, bias='none', dtype=BF16),
        # several tokens at once (a draft to verify) in float32, odd sizes, a dense bias
        dict(name='attention draft float32', op='attention', rows=7, heads=5, share=1, units=80,
             queries=5, keys=777, causal=True, bias='dense', dtype=F32),
        # the longest contexts, several query heads to one cached head
        dict(name='attention long context', op='attention', rows=8, heads=8, share=4, units=128,
             queries=1, keys=32768, causal=True, bias='none', dtype=BF16),
        # beam search on one sentence
        dict(name='select one sentence', op='select', items=1, beams=4, vocab=32128, finished=0.0,
             alpha=1.0, temperature=1.0, dtype=F32),
        # a large batch, some beams finished
        dict(name='select batch', op='select', items=64, beams=8, vocab=32128, finished=0.2,
             alpha=0.6, temperature=1.0, dtype=F32),
        # a multilingual vocabulary, bfloat16 logits, many beams
        dict(name='select large vocabulary', op='select', items=8, beams=16, vocab=250112,
             finished=0.1, alpha=1.0, temperature=0.8, dtype=BF16),
        # the states of a small decoder on one sentence
        dict(name='reorder one sentence', op='reorder', items=1, beams=4, tensors=12, length=60,
             heads=8, units=64, dtype=BF16, time_major=False),
        # the states of a deep decoder, a batch of sentences
        dict(name='reorder batch', op='reorder', items=16, beams=5, tensors=24, length=128,
             heads=12, units=64, dtype=BF16, time_major=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(['cache', 'attention', 'attention', 'select', 'reorder'])
    dtype = rng.choice([BF16, BF16, F32])
    if op == 'cache':
        units = rng.choice([64, 64, 128, rng.randint(1, 128)])
        heads = rng.randint(1, 20)
        new = rng.choice([1, _log(rng, 1, 2000)])
        rows = _log(rng, 1, max(1, min(256, 32 * 16 * 64 * 500 // (units * heads * new))))
        return dict(op=op, rows=rows, heads=heads, units=units, new=new, past=rng.randint(0, 300),
                    ragged=rng.random() < 0.5, dtype=dtype)
    if op == 'attention':
        units = rng.choice([64, 64, 128, rng.randint(8, 128)])
        heads, share = rng.randint(1, 16), rng.choice([1, 1, 1, 2, 4, 6])
        queries = rng.choice([1, 1, 1, _log(rng, 2, 40)])
        keys = _log(rng, queries, 30000)
        most = 8 * 8 * 4 * 128 * 32768 // (units * heads * share * queries * keys)
        return dict(op=op, rows=_log(rng, 1, max(1, min(128, most))), heads=heads, share=share,
                    units=units, queries=queries, keys=keys, causal=rng.random() < 0.7,
                    bias=rng.choice(['none', 'none', 'table', 'dense']), dtype=dtype)
    if op == 'select':
        vocab, beams = _log(rng, 40, 250000), _log(rng, 1, 24)
        items = _log(rng, 1, max(1, min(96, 16000000 // (vocab * beams))))
        return dict(op=op, items=items, beams=beams, vocab=vocab,
                    finished=rng.choice([0.0, 0.25, 0.7]), alpha=rng.choice([0.0, 0.6, 1.0]),
                    temperature=rng.choice([1.0, 1.0, 0.7, 1.3]), dtype=dtype)
    heads, units, beams, tensors = rng.randint(1, 16), rng.choice([64, 64, 48, 33]), _log(rng, 1, 20), \
        rng.randint(1, 30)
    length = _log(rng, 1, 512)
    most = 16 * 5 * 24 * 128 * 12 * 64 // (heads * units * beams * tensors * length)
    return dict(op=op, items=_log(rng, 1, max(1, min(64, most // 2))), beams=beams, tensors=tensors,
                length=length, heads=heads, units=units, dtype=dtype, time_major=rng.random() < 0.4)


# ---- inputs --------------------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _inputs(case, seed):
    """What the caller holds, apart from a cache: a dict of tensors, from the seed alone."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = getattr(torch, case['dtype'])
    op = case['op']
    if op == 'cache':
        B, H, d, n = case['rows'], case['heads'], case['units'], case['new']
        # projections: channels of unequal size and offset
        size = 0.3 + _randn(g, 2, 1, 1, H, d).abs()
        offset = 0.7 * _randn(g, 2, 1, 1, H, d)
        kv = (_randn(g, 2, B, n, H, d) * size + offset).to(dt)
        new = torch.full((B,), n, dtype=torch.int32, device=DEV)
        if case['ragged']:
            new = torch.randint((n + 1) // 2, n + 1, (B,), generator=g, device=DEV).int()
        past = torch.randint(case['past'] // 2, case['past'] + 1, (B,), generator=g, device=DEV).int()
        return dict(key=kv[0], value=kv[1], new_length=new, past=past)
    if op == 'attention':
        B, H, r, d = case['rows'], case['heads'], case['share'], case['units']
        n, L = case['queries'], case['keys']
        key = (_randn(g, B, L, H, d) * (0.3 + _randn(g, 1, 1, H, d).abs())
               + 0.5 * _randn(g, 1, 1, H, d)).to(dt)
        value = _randn(g, B, L, H, d).to(dt)
        query = (1.3 * _randn(g, B, n, H * r, d)).to(dt)
        length = torch.randint(max(n, (3 * L) // 4), L + 1, (B,), generator=g, device=DEV).int()
        bias = None
        if case['bias'] == 'table':      # by distance: the last entry is the query's own position
            bias = _randn(g, H * r, min(L, 160)).to(dt)
        elif case['bias'] == 'dense':
            bias = _randn(g, 1, H * r, n, L).to(dt)
        return dict(key=key, value=value, query=query, length=length, bias=bias)
    if op == 'select':
        N, K, V = case['items'], case['beams'], case['vocab']
        logits = (2.5 * _randn(g, N, K, V)).to(dt)
        scores = torch.sort(-6.0 * torch.rand(N, K, generator=g, device=DEV) - 1, dim=1,
                            descending=True)[0].float()
        finished = torch.rand(N, K, generator=g, device=DEV) < case['finished']
        return dict(logits=logits, scores=scores, finished=finished)
    N, K, L, H, d = case['items'], case['beams'], case['length'], case['heads'], case['units']
    shape = (L, N * K, H, d) if case['time_major'] else (N * K, L, H, d)
    states = [_randn(g, *shape).to(dt) for _ in range(case['tensors'])]
    parents = torch.randint(0, K, (N, K), generator=g, device=DEV).int()
    return dict(states=states, parents=parents, out=[torch.empty_like(s) for s in states])


def prepare(case, seed):
    x = dict(_inputs(case, seed), case=case)
    op = case['op']
    if op == 'cache':
        B, H, d, n = case['rows'], case['heads'], case['units'], case['new']
        room = case['past'] + n
        if own:
            x['cache'] = _package().kv_cache.QuantKVCache(B, H, d, room, ctx=DEV)
            x['cache'].set_length(x['past'] + x['new_length'])
        else:
            # (one slot more than the rows have: what is not to be stored goes there)
            x['codes'] = torch.zeros(2, B, room + 1, H, d, dtype=torch.uint8, device=DEV)
            x['steps'] = torch.zeros(2, 2, B, room + 1, H, -(-d // GROUP), device=DEV)
    elif op == 'attention':
        if own:
            B, L, H, d = x['key'].shape
            cache = x['cache'] = _package().kv_cache.QuantKVCache(B, H, d, L, ctx=DEV)
            cache.set_length(torch.full_like(x['length'], L))
            cache.write(x['key'], x['value'])
            cache.set_length(x['length'])
        else:
            x['quantised'] = [_quantise(x[t].float()) for t in ('key', 'value')]
        del x['key'], x['value']
    return x


# ---- plain forms ---------------------------------------------------------------------------------
def _spread(steps, d):
    """One value per group -> one per channel."""
    return steps.repeat_interleave(GROUP, dim=-1)[..., :d]


def _quantise(x):
    """x (..., d) in 32 bits -> codes (uint8), scale and minimum of each group."""
    d = x.shape[-1]
    pad = -d % GROUP
    shape = x.shape[:-1] + ((d + pad) // GROUP, GROUP)
    lo = torch.nn.functional.pad(x, (0, pad), value=math.inf).reshape(shape).amin(-1)
    hi = torch.nn.functional.pad(x, (0, pad), value=-math.inf).reshape(shape).amax(-1)
    scale = ((hi - lo) * (1.0 / 15)).bfloat16().float()
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    minimum = lo.bfloat16().float()
    s = _spread(scale, d)
    codes = torch.where(s > 0, torch.round((x - _spread(minimum, d)) / s), torch.zeros_like(x))
    return codes.clamp(0, 15).to(torch.uint8), scale, minimum


def _values(codes, scale, minimum):
    d = codes.shape[-1]
    return codes.float() * _spread(scale, d) + _spread(minimum, d)


def _cache_plain(x):
    n = x['case']['new']
    B = x['past'].shape[0]
    codes, scale, minimum = _quantise(torch.stack([x['key'], x['value']]).float())
    row = torch.arange(B, device=DEV)[:, None]
    token = torch.arange(n, device=DEV)
    keep = token < x['new_length'][:, None]
    slot = torch.where(keep, x['past'][:, None] + token, x['codes'].shape[2] - 1).long()
    x['codes'][:, row, slot] = codes
    x['steps'][0][:, row, slot] = scale
    x['steps'][1][:, row, slot] = minimum
    out = _values(x['codes'][:, row, slot], x['steps'][0][:, row, slot],
                  x['steps'][1][:, row, slot])
    out = torch.where(keep[None, :, :, None, None], out, torch.zeros_like(out)).to(x['key'].dtype)
    return out[0], out[1]


def _attention_plain(x):
    case, q = x['case'], x['query'].float()
    B, n, HQ, d = q.shape
    H, r, dev = case['heads'], case['share'], q.device
    key, value = (_values(*t).permute(0, 2, 1, 3) for t in x['quantised'])     # (B, H, L, d)
    L = key.shape[2]
    rows = q.reshape(B, n, H, r, d).permute(0, 2, 3, 1, 4).reshape(B, H, r * n, d)
    scores = torch.matmul(rows, key.transpose(2, 3).contiguous()).reshape(B, HQ, n, L)
    at = x['length'].long()[:, None] - n + torch.arange(n, device=dev)              # (B, n)
    j = torch.arange(L, device=dev)
    if case['bias'] == 'table':
        R = x['bias'].shape[1]
        entry = (R - 1 - (at[:, :, None] - j)).clamp(0, R - 1)                       # (B, n, L)
        scores = scores + x['bias'].float()[:, entry].permute(1, 0, 2, 3)
    elif case['bias'] == 'dense':
        scores = scores + x['bias'].float()
    scores = scores / math.sqrt(d)
    end = at + 1 if case['causal'] else x['length'].long()[:, None].expand(B, n)
    seen = (j < end[:, :, None])[:, None]                                          # (B, 1, n, L)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    weights = weights / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(weights.reshape(B, H, r * n, L), value.contiguous())
    out = out.reshape(B, H, r, n, d).permute(0, 3, 1, 2, 4).reshape(B, n, HQ * d)
    return out.to(x['query'].dtype)


_STEP, _EOS = 7, 1


def _select_plain(x):
    """In 64 bits: candidates of different beams come near each other."""
    case, K = x['case'], x['case']['beams']
    z = x['logits'].double() / case['temperature']
    N, _, V = z.shape
    top = z.amax(-1, keepdim=True)
    logp = z - top - torch.log(torch.exp(z - top).sum(-1, keepdim=True))
    before, after = (((K + s) / (K + 1.0)) ** case['alpha'] for s in (_STEP - 1, _STEP))
    prev = x['scores'].double()
    grown = (prev[:, :, None] * before + logp) / after
    grown = grown.masked_fill(x['finished'][:, :, None], -math.inf).reshape(N, K * V)
    kept = prev.masked_fill(~x['finished'], -math.inf)
    scores, at = torch.sort(torch.cat([grown, kept], 1), dim=1, descending=True, stable=True)
    scores, at = scores[:, :K], at[:, :K]
    was = at >= K * V
    parents = torch.where(was, at - K * V, at // V)
    tokens = torch.where(was, torch.full_like(at, -1), at % V)
    return scores.float(), parents.int(), tokens.int(), was | (tokens == _EOS)


def _reorder_plain(x):
    N, K = x['parents'].shape
    at = (torch.arange(N, device=DEV)[:, None] * K + x['parents']).reshape(-1)
    axis = 1 if x['case']['time_major'] else 0
    return [s.index_select(axis, at) for s in x['states']]


def run(x):
    op = x['case']['op']
    if not own:
        return {'cache': _cache_plain, 'attention': _attention_plain, 'select': _select_plain,
                'reorder': _reorder_plain}[op](x)
    nlp, case = _package(), x['case']
    if op == 'cache':
        cache, n = x['cache'], case['new']
        cache.write(x['key'], x['value'], new_length=x['new_length'])
        return cache.read(n, start=x['past'], dtype=case['dtype'])
    if op == 'attention':
        kw = {'table': dict(edge_table=x['bias']), 'dense': dict(edge_scores=x['bias'])}
        return nlp.attention_cell.multi_head_dot_attn_cached(
            x['query'], x['cache'], causal=case['causal'], query_head_units=case['units'],
            layout='NTK', **kw.get(case['bias'], {}))
    if op == 'select':
        return nlp.sequence_sampler.beam_search_select(
            x['logits'], x['scores'], x['finished'], eos_id=_EOS, step=_STEP, alpha=case['alpha'],
            length_base=case['beams'], temperature=case['temperature'])
    return nlp.sequence_sampler.reorder_states(
        x['states'], x['parents'], batch_axis=1 if case['time_major'] else 0, out=x['out'])


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    size = 2 if case['dtype'] == BF16 else 4
    op = case['op']
    if op == 'cache':
        tokens = case['rows'] * case['new'] * (0.75 if case['ragged'] else 1.0)
        held = case['units'] / 2 + 4 * -(-case['units'] // GROUP)
        moved = tokens * case['heads'] * 2 * (case['units'] * size + 2 * held)
        back = case['rows'] * case['new'] * case['heads'] * 2 * case['units'] * size
        return {'bytes': moved + back, 'flops': tokens * case['heads'] * 2 * case['units'] * 8}
    if op == 'attention':
        tokens = case['rows'] * case['heads'] * case['keys'] * 0.875
        held = case['units'] / 2 + 4 * -(-case['units'] // GROUP)
        rows = case['share'] * case['queries']
        ends = 2 * case['rows'] * case['heads'] * rows * case['units'] * size
        return {'bytes': 2 * tokens * held + ends, 'flops': 4 * tokens * rows * case['units']}
    if op == 'select':
        values = case['items'] * case['beams'] * case['vocab'] * (1 - case['finished'])
        return {'bytes': values * size + case['items'] * case['beams'] * 18, 'flops': 4 * values}
    n = case['tensors'] * case['items'] * case['beams'] * case['length'] * case['heads'] * case['units']
    chosen = 1 - (1 - 1 / case['beams']) ** case['beams']       # of the rows, some beam's parent
    return {'bytes': (1 + chosen) * n * size, 'flops': 0}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def _exact_values(x):
    """The numbers that the 4-bit format stands for; the choice of a code is defined in 32 bits."""
    x = x.float()
    parts = []
    for c in range(0, x.shape[-1], GROUP):
        part = x[..., c:c + GROUP]
        lo, hi = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        scale = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)).bfloat16()
        scale, lo = scale.float(), lo.bfloat16().float()
        flat = scale < 2.0 ** -126
        code = ((part - lo) / torch.where(flat, 1.0, scale)).round().clamp(0, 15)
        code = torch.where(flat, 0.0, code)
        parts.append(code.double() * torch.where(flat, 0.0, scale).double() + lo.double())
    return torch.cat(parts, -1)


def exact(case, seed):
    x = _inputs(case, seed)
    op = case['op']
    if op == 'cache':
        live = (torch.arange(case['new'], device=DEV) < x['new_length'][:, None])[..., None, None]
        return tuple(torch.where(live, _exact_values(x[t]), 0.0) for t in ('key', 'value'))
    if op == 'attention':
        B, n, HQ, d = x['query'].shape
        out = torch.zeros(B, n, HQ, d, dtype=torch.float64, device=DEV)
        key, value = _exact_values(x['key']), _exact_values(x['value'])
        lengths = x['length'].tolist()
        for b in range(B):
            T = lengths[b]
            at = torch.arange(T - n, T, device=DEV)
            j = torch.arange(T, device=DEV)
            for h in range(HQ):
                c = h // case['share']
                s = x['query'][b, :, h].double() @ key[b, :T, c].T
                if case['bias'] == 'table':
                    R = x['bias'].shape[1]
                    far = (at[:, None] - j).clamp(0, R - 1)
                    s = s + x['bias'][h].double().flip(0)[far]
                elif case['bias'] == 'dense':
                    s = s + x['bias'][0, h, :, :T].double()
                s = s / d ** 0.5
                if case['causal']:
                    s = torch.where(j <= at[:, None], s, -math.inf)
                out[b, :, h] = torch.softmax(s, -1) @ value[b, :T, c]
        return out.reshape(B, n, HQ * d)
    if op == 'select':
        K, V = case['beams'], case['vocab']
        logp = torch.log_softmax(x['logits'].double() / case['temperature'], -1)
        length = [((K + s) / (K + 1)) ** case['alpha'] for s in (_STEP - 1, _STEP)]
        prev = x['scores'].double()
        rows = torch.where(x['finished'][..., None], -math.inf,
                           (prev[..., None] * length[0] + logp) / length[1])
        kept = torch.where(x['finished'], prev, -math.inf)
        every = torch.cat([rows.flatten(1), kept], 1)
        at = torch.argsort(every, dim=1, descending=True, stable=True)[:, :K]
        was = at >= K * V
        tokens = torch.where(was, -1, at % V)
        return (every.gather(1, at), torch.where(was, at - K * V, at // V), tokens,
                was | (tokens == _EOS))
    N, K = x['parents'].shape
    axis = 1 if case['time_major'] else 0
    return [torch.cat([s.narrow(axis, i * K, K).index_select(axis, x['parents'][i])
                       for i in range(N)], axis) for s in x['states']]
