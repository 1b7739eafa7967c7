"""The decoding operators on the GPU against plain evaluations in 64 bits (tests/decode_ref.py):
the 4-bit key / value cache, attention over it, beam search selection, reordering of states."""
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


def _tokens(g, B, T, H, d, dtype):
    x = torch.randn(B, T, H, d, generator=g) * (0.3 + torch.randn(H, d, generator=g).abs()) + \
        0.7 * torch.randn(H, d, generator=g)
    return x.to(dtype)


def _to_layout(x, layout):       # (B, T, H, d) -> the layout's axes (a view)
    return {'NTK': x, 'NKT': x.permute(0, 2, 1, 3), 'TNK': x.permute(1, 0, 2, 3)}[layout]


def _from_layout(x, layout):
    return {'NTK': x, 'NKT': x.permute(0, 2, 1, 3), 'TNK': x.permute(1, 0, 2, 3)}[layout]


def _raw(c):
    return [c._k_codes.clone(), c._v_codes.clone(), c._k_par.clone(), c._v_par.clone()]


# ------------------------------------------------------------------------------------ the cache
@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('layout,B,H,d,T', [
    ('NTK', 2, 3, 64, 37), ('NTK', 1, 1, 1, 1), ('NKT', 3, 2, 7, 9), ('TNK', 2, 5, 80, 41),
    ('NTK', 2, 2, 128, 64), ('TNK', 1, 12, 64, 8), ('NKT', 2, 4, 33, 100), ('NTK', 3, 1, 96, 5)])
def test_write_read(nlp, dtype, layout, B, H, d, T):
    g = _gen(B * 1000 + d + T)
    k, v = _tokens(g, B, T, H, d, dtype), _tokens(g, B, T, H, d, dtype)
    c = nlp.kv_cache.QuantKVCache(B, H, d, T + 3, ctx='cuda', layout=layout)
    c.extend(T)
    c.write(_to_layout(k.cuda(), layout), _to_layout(v.cuda(), layout))
    gk, gv = c.read(T + 2, dtype='float32')
    for got, want in ((gk, k), (gv, v)):
        got = _from_layout(got.cpu(), layout).double()
        exact = ref.quantise(want)[0]
        # a value is code * scale + minimum rounded once: half a step of float32
        assert ((got[:, :T] - exact).abs() <= exact.abs() * 2.0 ** -24).all()
        assert (got[:, T:] == 0).all()
    bk, _ = c.read(T, dtype='bfloat16')
    exact = ref.quantise(k)[0]
    # rounded twice: to float32 and to bfloat16
    assert ((_from_layout(bk.cpu(), layout).double() - exact).abs()
            <= exact.abs() * (2.0 ** -8 + 2.0 ** -23)).all()


@pytest.mark.parametrize('d', [64, 100])
def test_token_by_token_is_the_prompt(nlp, d):
    B, H, T = 2, 3, 21
    g = _gen(5)
    k, v = _tokens(g, B, T, H, d, BF16).cuda(), _tokens(g, B, T, H, d, BF16).cuda()
    one = nlp.kv_cache.QuantKVCache(B, H, d, T, ctx='cuda')
    one.extend(T)
    one.write(k, v)
    steps = nlp.kv_cache.QuantKVCache(B, H, d, T, ctx='cuda')
    at = 0
    for n in (1, 1, 5, 8, 1, 3, 2):
        steps.extend(n)
        steps.write(k[:, at:at + n], v[:, at:at + n])
        at += n
    assert at == T
    for a, b in zip(_raw(one), _raw(steps)):
        assert torch.equal(a, b)


@pytest.mark.parametrize('idtype', [torch.int32, torch.int64])
def test_ragged_write_leaves_the_rest(nlp, idtype):
    B, H, d, T, room = 5, 2, 64, 12, 40
    g = _gen(9)
    old = _tokens(g, B, room, H, d, F32)
    new = _tokens(g, B, T, H, d, F32)
    c = nlp.kv_cache.QuantKVCache(B, H, d, room, num_layers=2, ctx='cuda')
    c.set_length(room)
    for layer in range(2):
        c.write(old.cuda(), old.cuda(), layer)
    past = torch.tensor([0, 3, 17, 28, 35])
    count = torch.tensor([12, 0, 5, 12, 7], dtype=idtype)     # row 3 fills the cache, row 4 runs over
    c.set_length((past + count).to(idtype).cuda())
    padded = new.clone()
    for b in range(B):
        padded[b, int(count[b]):] = math.nan                 # padding is not read
    c.write(padded.cuda(), padded.cuda(), layer=1, new_length=count.cuda())
    c.set_length(room)
    exact_old, exact_new = ref.quantise(old)[0], ref.quantise(new)[0]
    want = exact_old.clone()
    for b in range(B):
        for i in range(int(count[b])):
            if past[b] + i < room:
                want[b, past[b] + i] = exact_new[b, i]
    for layer, expect in ((0, exact_old), (1, want)):
        for got in c.read(layer=layer):
            assert ((got.cpu().double() - expect).abs() <= expect.abs() * 2.0 ** -24).all()
    # from a start of its own, below 0 and past the end too
    start = torch.tensor([0, -2, 30, 39, 45], dtype=idtype)
    c.set_length(38)
    got, _ = c.read(10, start=start.cuda(), layer=1)
    for b in range(B):
        for i in range(10):
            slot = int(start[b]) + i
            expect = want[b, slot] if 0 <= slot < 38 else torch.zeros(H, d, dtype=torch.float64)
            assert ((got[b, i].cpu().double() - expect).abs() <= expect.abs() * 2.0 ** -24).all()


def test_groups_out_of_the_ordinary(nlp):
    d, T = 64, 12
    x = torch.randn(1, T, 1, d, generator=_gen(1))
    x[0, 0] = 3.25                                   # no spread
    x[0, 1, 0, 5] = math.nan
    x[0, 2, 0, 0] = math.inf
    x[0, 3, 0, 63] = -math.inf
    x[0, 4, 0, :2] = torch.tensor([3e38, -3e38])     # range beyond float32
    x[0, 5] = torch.linspace(0, 1, d) * 1e-38        # scale below the smallest normal number
    x[0, 6] = torch.linspace(-1, 1, d) * 1e-30
    x[0, 7] = 1000 + torch.linspace(0, 1e-3, d)      # spread below the minimum's rounding
    x[0, 8] = 0
    x[0, 9] = torch.linspace(-1, 1, d) * 1e37
    x[0, 10, 0, :] = 3.4e38                          # the minimum rounds to infinity
    c = nlp.kv_cache.QuantKVCache(1, 1, d, T, ctx='cuda')
    c.extend(T)
    c.write(x.cuda(), x.cuda())
    exact = ref.quantise(x)[0]
    for got in c.read():
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(exact))
        ok = ~torch.isnan(exact)
        assert ((got[ok] - exact[ok]).abs() <= exact[ok].abs() * 2.0 ** -24 + 2.0 ** -149).all()
        assert [bool(torch.isnan(got[0, t]).all()) for t in range(T)] == \
            [t in (1, 2, 3, 4, 10) for t in range(T)]


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_strided_and_misaligned_tokens(nlp, dtype):
    B, T, H, d = 2, 11, 3, 64
    packed = torch.randn(B, T, 3 * H * d + 1, generator=_gen(2)).to(dtype).cuda()
    for off in (0, 1):                                # 16-byte aligned and not
        k = packed[..., off:off + H * d].unflatten(-1, (H, d))
        v = packed[..., off + 2 * H * d:off + 3 * H * d].unflatten(-1, (H, d))
        c = nlp.kv_cache.QuantKVCache(B, H, d, T, ctx='cuda')
        c.extend(T)
        c.write(k, v)
        for got, x in zip(c.read(), (k, v)):
            exact = ref.quantise(x)[0]
            assert ((got.cpu().double() - exact).abs() <= exact.abs() * 2.0 ** -24).all()
    # an inner stride other than 1
    k = torch.randn(B, T, d, H, generator=_gen(3)).to(dtype).cuda().transpose(2, 3)
    c = nlp.kv_cache.QuantKVCache(B, H, d, T, ctx='cuda')
    c.extend(T)
    c.write(k, k)
    exact = ref.quantise(k)[0]
    assert ((c.read()[0].cpu().double() - exact).abs() <= exact.abs() * 2.0 ** -24).all()


# ------------------------------------------------------------------------------------ attention
def _filled(nlp, g, B, Hc, d, T, room, lengths, dtype, poison=True, layout='NTK'):
    """A cache holding T tokens, the rows' own lengths set; slots behind them hold NaN groups."""
    k, v = _tokens(g, B, T, Hc, d, dtype), _tokens(g, B, T, Hc, d, dtype)
    c = nlp.kv_cache.QuantKVCache(B, Hc, d, room, ctx='cuda', layout=layout)
    kk = torch.full((B, room, Hc, d), math.nan if poison else 0.0).to(dtype)
    vv = kk.clone()
    for b in range(B):
        kk[b, :int(lengths[b])] = k[b, :int(lengths[b])]
        vv[b, :int(lengths[b])] = v[b, :int(lengths[b])]
    c.set_length(room)
    c.write(_to_layout(kk.cuda(), layout), _to_layout(vv.cuda(), layout))
    c.set_length(torch.as_tensor(lengths).int().cuda())
    qk, ks, km = ref.quantise(k)
    qv, vs, vm = ref.quantise(v)
    return c, qk, qv, (ks.max().item(), km.abs().max().item(), qv.abs().max().item())


def _check(got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    err = (got - want).abs().max().item()
    assert err <= tol, 'error {} > {}'.format(err, tol)


CASES = [
    # B, cached heads, share, d, Lq, T, causal, bias, mask
    (1, 1, 1, 64, 1, 1, True, None, False),
    (2, 3, 1, 64, 1, 31, True, None, False),
    (2, 2, 1, 64, 1, 129, True, 'table', False),
    (3, 2, 1, 64, 1, 700, True, 'edge', True),
    (2, 2, 4, 64, 1, 515, True, None, False),
    (2, 1, 2, 128, 1, 1030, True, None, False),
    (2, 2, 1, 128, 7, 333, True, 'table', False),
    (1, 2, 3, 80, 5, 260, True, 'edge', False),
    (2, 2, 1, 64, 8, 256, False, None, False),
    (2, 2, 1, 64, 16, 64, False, None, True),
    (1, 2, 1, 64, 37, 200, True, 'table', False),
    (1, 1, 5, 33, 9, 77, True, 'edge', True),
    (2, 1, 1, 8, 2, 45, False, 'edge', False),
    (1, 1, 1, 1, 3, 50, True, None, False),
]


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('B,Hc,share,d,Lq,T,causal,bias,masked', CASES)
def test_attention(nlp, dtype, B, Hc, share, d, Lq, T, causal, bias, masked):
    g = _gen(T * 7 + d + Lq)
    H = Hc * share
    lengths = torch.randint(max(1, T // 2), T + 1, (B,), generator=g)
    lengths[0] = T
    c, k, v, size = _filled(nlp, g, B, Hc, d, T, T + 5, lengths, dtype)
    q = torch.randn(B, Lq, H, d, generator=g).to(dtype)
    kw, rkw = {}, {}
    if bias == 'table':
        rkw['table'] = torch.randn(H, 50, generator=g).to(dtype)
        kw['edge_table'] = rkw['table'].cuda()
    if bias == 'edge':
        e = torch.randn(1, H, 1 if d == 8 else Lq, T, generator=g).to(dtype)
        rkw['edge'], kw['edge_scores'] = e, e.cuda()
    if masked:
        m = torch.rand(B, Lq, T, generator=g) < 0.7
        m[0, 0] = False                                     # a row that sees nothing
        rkw['mask'], kw['mask'] = m, m.cuda()
    got = nlp.attention_cell.multi_head_dot_attn_cached(q.cuda(), c, causal=causal, **kw)
    want = ref.attention(q, k, v, lengths, share, causal, temperature=math.sqrt(d), **rkw)
    tol = ref.attention_tolerance(q, *size, T, math.sqrt(d), dtype)
    _check(got.reshape(B, Lq, H, d), want, tol)
    if masked:
        assert (got.reshape(B, Lq, H, d)[0, 0] == 0).all()


@pytest.mark.parametrize('layout', ['NTK', 'NKT', 'TNK'])
def test_attention_layouts(nlp, layout):
    B, H, d, Lq, T = 2, 3, 64, 2, 90
    g = _gen(4)
    lengths = torch.tensor([90, 51])
    c, k, v, size = _filled(nlp, g, B, H, d, T, T, lengths, BF16, layout=layout)
    q = torch.randn(B, Lq, H, d, generator=g).to(BF16)
    qd = _to_layout(q.cuda(), layout).contiguous()
    got = nlp.attention_cell.multi_head_dot_attn_cached(qd, c)
    if layout == 'TNK':
        got = got.transpose(0, 1)
    want = ref.attention(q, k, v, lengths, temperature=8.0)
    _check(got.reshape(B, Lq, H, d), want, ref.attention_tolerance(q, *size, T, 8.0, BF16))


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_attention_ragged_queries_and_empty_rows(nlp, dtype):
    B, H, d, Lq, T = 6, 2, 64, 4, 40
    g = _gen(6)
    lengths = torch.tensor([0, 1, 2, 40, 17, 33])
    ql = torch.tensor([4, 1, 4, 0, 2, 4])
    c, k, v, size = _filled(nlp, g, B, H, d, T, T, lengths, dtype)
    q = torch.randn(B, Lq, H, d, generator=g).to(dtype)
    for causal in (True, False):
        got = nlp.attention_cell.multi_head_dot_attn_cached(
            q.cuda(), c, causal=causal, query_length=ql.cuda(), scaled=False)
        want = ref.attention(q, k, v, lengths, causal=causal, query_length=ql)
        _check(got.reshape(B, Lq, H, d), want, ref.attention_tolerance(q, *size, T, 1.0, dtype))
        assert (got[0] == 0).all() and (got[3] == 0).all() and (got[4, 2:] == 0).all()
    assert nlp.attention_cell.multi_head_dot_attn_cached(q[:, :0].cuda(), c).shape == (B, 0, H * d)


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('Lq,share', [(5, 1), (3, 1), (19, 1), (2, 17)])
def test_attention_biases_that_end_an_allocation(nlp, dtype, Lq, share):
    """Bias and mask lie at the end of their memory: queries that fill a tile of rows in part read
    nothing behind them."""
    B, T, d = 2, 720, 64
    g = _gen(Lq)
    c, k, v, size = _filled(nlp, g, B, 1, d, T, T, [T, 300], dtype)
    q = torch.randn(B, Lq, share, d, generator=g).to(dtype)
    e = torch.randn(B, share, Lq, T, generator=g).to(dtype)
    m = torch.rand(B, Lq, T, generator=g) < 0.8
    room = 32 << 20                                        # (an allocation of its own)
    ends = []
    for x in (e, m):
        own = torch.zeros(room // x.element_size(), dtype=x.dtype, device='cuda')
        own[-x.numel():] = x.reshape(-1).cuda()
        ends.append(own[-x.numel():].view(x.shape))
    got = nlp.attention_cell.multi_head_dot_attn_cached(q.cuda(), c, edge_scores=ends[0],
                                                        mask=ends[1])
    want = ref.attention(q, k, v, [T, 300], share, edge=e, mask=m, temperature=8.0)
    _check(got.reshape(B, Lq, share, d), want, ref.attention_tolerance(q, *size, T, 8.0, dtype))


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_attention_extreme_biases(nlp, dtype):
    """-inf and the type's lowest number as masks, in part of a row and all over it; what masked
    places hold cannot matter."""
    B, H, d, Lq, T = 1, 2, 64, 5, 150
    g = _gen(8)
    c, k, v, size = _filled(nlp, g, B, H, d, T, T, [T], dtype)
    q = torch.randn(B, Lq, H, d, generator=g).to(dtype)
    e = torch.randn(1, 1, Lq, T, generator=g).to(dtype)
    e[0, 0, 0] = -math.inf                       # nothing left: zeros
    e[0, 0, 1] = torch.finfo(dtype).min          # all the lowest: equal weights
    e[0, 0, 2, 10:] = torch.finfo(dtype).min
    e[0, 0, 3, :140] = -math.inf
    m = torch.ones(1, Lq, T, dtype=torch.bool)
    m[0, 4, 100:] = False
    e[0, 0, 4, 100:120] = math.nan               # behind the mask
    e[0, 0, 4, 120:] = math.inf
    got = nlp.attention_cell.multi_head_dot_attn_cached(
        q.cuda(), c, causal=False, edge_scores=e.cuda(), mask=m.cuda(), scaled=False)
    e2 = torch.where(m[:, None], e, torch.zeros_like(e))
    want = ref.attention(q, k, v, [T], causal=False, edge=e2, mask=m)
    tol = ref.attention_tolerance(q, *size, T, 1.0, dtype)
    got = got.reshape(B, Lq, H, d)
    assert (got[0, 0] == 0).all()
    _check(got, want, tol)


def test_attention_far_from_the_start(nlp):
    """Codes beyond 2^32 bytes from the array's start, lengths of the last layer and sequence."""
    B, H, d, T = 1, 2, 128, 256
    slots = (2 ** 32 // (H * d // 2)) // 32 * 32 + 4096
    g = _gen(11)
    c = nlp.kv_cache.QuantKVCache(B, H, d, slots, ctx='cuda')
    k, v = _tokens(g, B, T, H, d, BF16), _tokens(g, B, T, H, d, BF16)
    c.set_length(slots)
    c.write(k.cuda(), v.cuda())                  # the last 256 slots of both heads
    gk, _ = c.read(T, start=torch.tensor([slots - T]).cuda())
    exact, ks, km = ref.quantise(k)
    assert ((gk.cpu().double() - exact).abs() <= exact.abs() * 2.0 ** -24).all()
    m = torch.zeros(1, 1, slots, dtype=torch.bool, device='cuda')
    m[:, :, -T:] = True
    q = torch.randn(B, 1, H, d, generator=g).to(BF16)
    got = nlp.attention_cell.multi_head_dot_attn_cached(q.cuda(), c, mask=m)
    qv = ref.quantise(v)[0]
    want = ref.attention(q, exact, qv, [T], temperature=math.sqrt(d))
    tol = ref.attention_tolerance(q, ks.max().item(), km.abs().max().item(), qv.abs().max().item(),
                                  slots / 64, math.sqrt(d), BF16)
    _check(got.reshape(B, 1, H, d), want, tol)


def test_attention_does_not_depend_on_the_hint(nlp):
    """The number of workgroups follows a hint; a row's result is right for any."""
    g = _gen(12)
    c, k, v, size = _filled(nlp, g, 1, 1, 64, 3000, 3000, [3000], F32)
    q = torch.randn(1, 1, 1, 64, generator=g)
    want = ref.attention(q, k, v, [3000], temperature=8.0)
    tol = ref.attention_tolerance(q, *size, 3000, 8.0, F32)
    for bound in (1, 600, 3000):
        c._bound = bound
        _check(nlp.attention_cell.multi_head_dot_attn_cached(q.cuda(), c).reshape(1, 1, 1, 64),
               want, tol)


def test_repeated_calls_agree(nlp):
    g = _gen(13)
    c, _, _, _ = _filled(nlp, g, 2, 4, 64, 2000, 2000, [2000, 900], BF16)
    q = torch.randn(2, 3, 4, 64, generator=g).to(BF16).cuda()
    first = nlp.attention_cell.multi_head_dot_attn_cached(q, c)
    for _ in range(3):
        assert torch.equal(nlp.attention_cell.multi_head_dot_attn_cached(q, c), first)


def test_captured_steps(nlp):
    """A decoding step captured once and replayed follows the lengths on the device; two graphs of
    one cache and eager calls in between share nothing but the cache."""
    B, H, d, room = 2, 3, 64, 40
    g = _gen(14)
    x = [torch.randn(3, B, 1, H, d, generator=g).to(BF16).cuda() for _ in range(12)]
    eager = nlp.kv_cache.QuantKVCache(B, H, d, room, ctx='cuda')
    want = []
    for q, k, v in x:
        eager.extend(1)
        eager.write(k, v)
        want.append(nlp.attention_cell.multi_head_dot_attn_cached(q, eager))
    c = nlp.kv_cache.QuantKVCache(B, H, d, room, ctx='cuda')
    feed = torch.zeros_like(x[0])
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            c.extend(1)
            c.write(feed[1], feed[2])
            out = nlp.attention_cell.multi_head_dot_attn_cached(feed[0], c)
        graphs.append(graph)
        outs.append(out)
    c.reset()
    for i, step in enumerate(x):
        feed.copy_(step)
        if i % 3 == 2:
            c.extend(1)
            c.write(feed[1], feed[2])
            got = nlp.attention_cell.multi_head_dot_attn_cached(feed[0], c)
        else:
            graphs[i % 2].replay()
            got = outs[i % 2]
        torch.cuda.synchronize()
        assert torch.equal(got, want[i])


def test_lengths_that_replays_moved(nlp):
    """After a graph's replays the host does not know the lengths: extend looks, and refuses what
    does not fit; replays beyond the buffer store nothing and leave the rest as it was."""
    B, H, d, room = 2, 2, 64, 32
    c = nlp.kv_cache.QuantKVCache(B, H, d, room, ctx='cuda')
    k = torch.randn(B, 1, H, d, generator=_gen(16)).to(BF16).cuda()
    q = torch.ones(B, 1, H, d, dtype=BF16).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.extend(1)
        c.write(k, k)
        out = nlp.attention_cell.multi_head_dot_attn_cached(q, c)
    c.reset()
    c.extend(2)
    c.write(torch.cat([k, -k], 1), torch.cat([k, -k], 1))
    for _ in range(28):
        graph.replay()
    assert c.length.tolist() == [30, 30]
    with pytest.raises(ValueError, match='33 tokens'):
        c.extend(3)
    assert c.length.tolist() == [30, 30]
    c.extend(2)
    c.write(torch.cat([k, k], 1), torch.cat([k, k], 1))
    with pytest.raises(ValueError, match='33 tokens'):
        c.extend(1)
    before = [x.clone() for x in c.read()]
    want = nlp.attention_cell.multi_head_dot_attn_cached(q, c)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(c.read(), before))
        assert torch.equal(out, want)


def test_another_stream(nlp):
    g = _gen(15)
    c, _, _, _ = _filled(nlp, g, 2, 2, 64, 1500, 1500, [1500, 700], BF16)
    q = torch.randn(2, 1, 2, 64, generator=g).to(BF16).cuda()
    want = nlp.attention_cell.multi_head_dot_attn_cached(q, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = nlp.attention_cell.multi_head_dot_attn_cached(q, c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------------ selection
def _check_select(nlp, x, s, f, **kw):
    rkw = dict(kw)
    if 'eos_id' in rkw:
        rkw['eos'] = rkw.pop('eos_id')
    if 'length_base' in rkw:
        rkw['base'] = rkw.pop('length_base')
    if isinstance(rkw.get('step'), torch.Tensor):
        rkw['step'] = int(rkw['step'])
    got = nlp.sequence_sampler.beam_search_select(x, s, f, **kw)
    ws, wp, wt, wf = ref.select(x, s, f, **rkw)
    assert torch.equal(got[1].cpu().long(), wp) and torch.equal(got[2].cpu().long(), wt)
    assert torch.equal(got[3].cpu(), wf)
    gs = got[0].cpu().double()
    inf = ws == -math.inf
    assert torch.equal(gs == -math.inf, inf)
    # a sum of V float32 exponentials in 64-bit parts: a logsumexp off by a few half steps of the
    # largest term; the score itself is rounded once
    scale = ws[~inf].abs() + 20.0
    assert ((gs[~inf] - ws[~inf]).abs() <= scale * 2.0 ** -24 * 8).all()
    return got


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('N,K,V', [(1, 1, 1), (1, 1, 50), (2, 4, 1000), (3, 5, 4096), (2, 8, 32128),
                                   (1, 32, 4100), (4, 3, 9999), (1, 16, 70001), (2, 24, 40),
                                   (1, 32, 2)])
def test_select(nlp, dtype, N, K, V):
    g = _gen(N + K * 10 + V)
    x = (3 * torch.randn(N, K, V, generator=g)).to(dtype).cuda()
    s = -torch.rand(N, K, generator=g).cuda() * 5
    f = (torch.rand(N, K, generator=g) < 0.3).cuda()
    _check_select(nlp, x, s, f, eos_id=min(3, V - 1), step=4, alpha=0.7, length_base=5)
    _check_select(nlp, x, s, None, temperature=0.6)


def test_select_ties_and_constant_rows(nlp):
    N, K, V = 2, 4, 9000
    s = torch.tensor([[-1.0, -1.0, -2.0, -3.0]] * N).cuda()
    x = torch.zeros(N, K, V).cuda()                       # every candidate of a beam ties
    got = _check_select(nlp, x, s, None)
    assert got[2].tolist() == [[0, 1, 2, 3]] * N and got[1].tolist() == [[0] * 4] * N
    x = torch.randint(0, 4, (N, K, V), generator=_gen(1)).float().cuda()
    _check_select(nlp, x, s, None)
    x[0, 0] = -math.inf                                    # a row without a candidate
    x[0, 1, ::2] = -math.inf
    x[1] = -math.inf
    _check_select(nlp, x, s, None)
    x = torch.full((1, 4, V), -math.inf).cuda()            # masked but for two tokens
    x[:, :, 77] = 1.0
    x[:, :, 8000] = 2.0
    _check_select(nlp, x, torch.tensor([[0.0, -math.inf, -math.inf, -math.inf]]).cuda(), None)
    _check_select(nlp, x, torch.tensor([[0.0, -1e18, -1e30, -math.inf]]).cuda(), None)
    x = torch.tensor([0.0, -0.0] * 300).reshape(1, 1, 600).repeat(1, 4, 1).cuda()
    _check_select(nlp, x, torch.tensor([[0.0, 0.0, 0.0, 0.0]]).cuda(), None)


def test_select_masked_places(nlp):
    """NaN and infinities; what finished beams hold is not read."""
    N, K, V = 2, 3, 5000
    g = _gen(3)
    x = torch.randn(N, K, V, generator=g)
    s = -torch.rand(N, K, generator=g)
    f = torch.tensor([[False, True, False], [True, True, True]])
    x[0, 0, 10:20] = math.nan
    x[0, 2, 5] = math.inf
    x[0, 2, 4000] = math.inf
    clean = x.clone()
    x[0, 1] = math.nan
    x[1] = math.inf
    got = _check_select(nlp, x.cuda(), s.cuda(), f.cuda())
    other = nlp.sequence_sampler.beam_search_select(clean.cuda(), s.cuda(), f.cuda())
    assert all(torch.equal(a, b) for a, b in zip(got, other))
    assert got[3][1].all() and (got[2][1] == -1).all()


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('low', [-1e4, -1e9, 'lowest'])
def test_select_masks_of_low_values(nlp, dtype, low):
    """Masks that are numbers: over all of a chunk of the vocabulary, over all of a row."""
    low = torch.finfo(dtype).min if low == 'lowest' else low
    N, K, V = 2, 4, 20000
    g = _gen(8)
    x = torch.randn(N, K, V, generator=g)
    x[0, :, 3000:] = low                                   # whole chunks, and the end of one
    x[1, 0] = low                                          # all of a beam: its tokens tie
    x[1, 1, :19000] = low
    s = -torch.rand(N, K, generator=g)
    s[1, 0] = 6.0                                          # (log 20000 = 9.9: among the best)
    for temperature in (1.0, 0.01, 30.0):
        _check_select(nlp, x.to(dtype).cuda(), s.cuda(), None, temperature=temperature)


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('N,K,V', [(2, 16, 40000), (1, 32, 9000), (3, 8, 250112), (2, 5, 4099)])
def test_select_ties_that_overfill_the_lists(nlp, dtype, N, K, V):
    """Masks but for a few tokens, constant rows, two values, dead and finished beams among them."""
    g = _gen(K)
    s = -torch.rand(N, K, generator=g)
    dead = s.clone()
    dead[:, 1:] = -math.inf
    base = torch.randn(N, K, V, generator=g)
    masked = base.clone()
    masked[:, :, 100:] = -math.inf
    few = torch.full_like(base, -math.inf)
    few[:, :, V // 2] = 1.0
    few[:, :, V - 1] = 2.0
    two = (base > 1.0).float()
    most = torch.where(base < 3.0, torch.zeros_like(base), base)
    f = torch.rand(N, K, generator=g) < 0.4
    for x in (masked, few, two, most, torch.full_like(base, -3.0)):
        x = x.to(dtype).cuda()
        for scores in (s, dead):
            _check_select(nlp, x, scores.cuda(), None)
            _check_select(nlp, x, scores.cuda(), f.cuda(), eos_id=V // 2)
    _check_select(nlp, base.to(dtype).cuda(), dead.cuda(), None)
    close = (1.0 + 1e-6 * base).float()                    # values that differ in their last bits
    if dtype == F32:
        _check_select(nlp, close.cuda(), s.cuda(), None)


def test_select_large_logits(nlp):
    """Logits whose product with the temperature leaves float32's precise range: the differences
    count."""
    g = _gen(9)
    steps = torch.randint(0, 12, (2, 3, 9000), generator=g).float()
    s = -torch.rand(2, 3, generator=g).cuda()
    for x in (1e9 + 64 * steps, -1e9 + 64 * steps, 3e38 + 1e37 * (steps / 4 - 1), 40000 + steps):
        for temperature in (1.0, 100.0):
            _check_select(nlp, x.cuda(), s, None, temperature=temperature)


def test_select_step_on_the_device_out_of_range(nlp):
    """lp is not a number: scores -inf, and candidates that exist (of a beam, only its K best logits
    become candidates; they tie here, to the lowest index)."""
    x = torch.randn(1, 3, 700, generator=_gen(10)).cuda()
    s = -torch.rand(1, 3, generator=_gen(11)).cuda()
    step = torch.tensor([-50], dtype=torch.int32).cuda()
    sc, parents, tokens, done = nlp.sequence_sampler.beam_search_select(x, s, step=step, alpha=0.5)
    assert (sc == -math.inf).all() and parents.tolist() == [[0, 0, 0]]
    assert tokens.tolist() == [sorted(x[0, 0].topk(3).indices.tolist())] and not done.any()


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('V', [300, 9000, 9003])
@pytest.mark.parametrize('normalize', [False, True])
def test_select_nan_and_infinities(nlp, dtype, V, normalize):
    """In a few places, in most of a row, in all of a chunk and of a row; of both signs."""
    N, K = 2, 5
    g = _gen(V)
    x = torch.randn(N, K, V, generator=g)
    x[0, 0, ::3] = math.nan
    x[0, 1, 4:] = math.nan
    x[0, 2] = -math.nan
    x[0, 3, : V // 2] = -math.inf
    x[1, 0, V // 2:] = math.nan
    x[1, 0, 7] = math.inf
    x[1, 1, 5] = -math.nan
    x[1, 2, 1:] = -math.inf
    x[1, 2, 11] = math.nan
    s = -torch.rand(N, K, generator=g)
    _check_select(nlp, x.to(dtype).cuda(), s.cuda(), None, normalize=normalize)


def test_select_strides_log_probabilities_and_device_step(nlp):
    N, K, V = 2, 3, 777
    g = _gen(5)
    wide = torch.randn(N * K, V + 23, generator=g).cuda()
    s = -torch.rand(N, K, generator=g).cuda()
    x = wide[:, 5:5 + V]                                   # rows of a wider tensor, misaligned
    a = nlp.sequence_sampler.beam_search_select(x, s)
    b = nlp.sequence_sampler.beam_search_select(x.reshape(N, K, V).contiguous(), s)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    logp = torch.log_softmax(x.double(), -1).float().reshape(N, K, V)
    _check_select(nlp, logp, s, None, normalize=False)
    for idtype in (torch.int32, torch.int64):
        step = torch.tensor([9], dtype=idtype).cuda()
        a = _check_select(nlp, x.reshape(N, K, V), s, None, step=step, alpha=1.0)
        b = nlp.sequence_sampler.beam_search_select(x, s, step=9, alpha=1.0)
        assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])


def test_select_captured(nlp):
    N, K, V = 2, 4, 6000
    g = _gen(6)
    xs = [torch.randn(N, K, V, generator=g).cuda() for _ in range(4)]
    s = -torch.rand(N, K, generator=g).cuda()
    x, step = xs[0].clone(), torch.tensor([1], dtype=torch.int32).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = nlp.sequence_sampler.beam_search_select(x, s, step=step, alpha=0.9)
    for i, xi in enumerate(xs):
        x.copy_(xi)
        step.fill_(i + 1)
        graph.replay()
        torch.cuda.synchronize()
        want = nlp.sequence_sampler.beam_search_select(xi, s, step=i + 1, alpha=0.9)
        assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))
        assert torch.allclose(got[0], want[0], rtol=0, atol=1e-6)


# ------------------------------------------------------------------------------------ reordering
@pytest.mark.parametrize('N,K', [(1, 1), (2, 4), (3, 5), (1, 20), (2, 32)])
@pytest.mark.parametrize('in_place', [False, True])
def test_reorder_states(nlp, N, K, in_place):
    g = _gen(N * 40 + K)
    rows = N * K
    states = [(torch.randn(rows, 3, 4, 64, generator=g).to(BF16).cuda(),
               torch.randn(5, rows, 7, generator=g).cuda()),
              (torch.randint(-9, 9, (rows, 33), generator=g, dtype=torch.int8).cuda(),
               torch.randn(2, rows, 3, 8, generator=g).to(BF16).cuda()),
              (torch.randn(rows, 70001, generator=g).cuda(), None)]
    axes = [(0, 1), (0, 1), (0, 0)]
    parents = torch.randint(0, K, (N, K), generator=g)
    at = (torch.arange(N)[:, None] * K + parents).reshape(-1).cuda()
    want = [tuple(None if t is None else t.index_select(a, at) for t, a in zip(p, ax))
            for p, ax in zip(states, axes)]
    for idtype in (torch.int32, torch.int64):
        p = parents.to(idtype).cuda()
        mine = [tuple(None if t is None else t.clone() for t in x) for x in states]
        got = nlp.sequence_sampler.reorder_states(mine, p, axes, out=mine if in_place else None)
        for gp, wp, sp in zip(got, want, mine):
            for a, b, s in zip(gp, wp, sp):
                assert (a is None) if b is None else torch.equal(a, b)
                assert b is None or (a.data_ptr() == s.data_ptr()) == in_place


def test_reorder_many_tensors_into_given_ones(nlp):
    g = _gen(2)
    states = [torch.randn(6, 1 + i, 16, generator=g).cuda() for i in range(40)]
    out = [torch.empty_like(s) for s in states]
    p = torch.tensor([[2, 2, 0], [0, 1, 1]]).cuda()
    got = nlp.sequence_sampler.reorder_states(states, p, out=out)
    at = torch.tensor([2, 2, 0, 3, 4, 4]).cuda()
    for a, o, s in zip(got, out, states):
        assert a.data_ptr() == o.data_ptr() and torch.equal(a, s[at])
    empty = [torch.zeros(6, 0, 4).cuda(), torch.zeros(6, 3).cuda()]
    assert nlp.sequence_sampler.reorder_states(empty, p)[0].shape == (6, 0, 4)


@pytest.mark.parametrize('d,N,K', [(64, 2, 4), (100, 1, 7)])
def test_reorder_cache(nlp, d, N, K):
    B, H, T = N * K, 2, 70
    g = _gen(d)
    k, v = _tokens(g, B, T, H, d, F32), _tokens(g, B, T, H, d, F32)
    c = nlp.kv_cache.QuantKVCache(B, H, d, T, num_layers=3, ctx='cuda')
    lengths = torch.randint(0, T + 1, (B,), generator=g)
    c.set_length(T)
    for layer in range(3):
        c.write(k.cuda() + layer, v.cuda() - layer, layer)
    c.set_length(lengths.cuda())
    before = [c.read(layer=i) for i in range(3)]
    parents = torch.randint(0, K, (N, K), generator=g)
    at = (torch.arange(N)[:, None] * K + parents).reshape(-1)
    nlp.sequence_sampler.reorder_states([c], parents.cuda())
    assert torch.equal(c.length.cpu().long(), lengths[at])
    for i in range(3):
        for a, b in zip(c.read(layer=i), before[i]):
            assert torch.equal(a.cpu(), b.cpu()[at])
