"""Host side of the decoding operators: struct layout, refusals at the C entries (all before any
launch) and in the Python wrappers, and the reference format's own invariants.  No GPU."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from tests import decode_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def nlp():
    import gluonnlp_amd
    return gluonnlp_amd


@pytest.fixture(scope='module')
def lib():
    from gluonnlp_amd import _lib
    return _lib.load()


def test_structs_match_the_header(tmp_path):
    from gluonnlp_amd import _lib
    structs = {'gnlp_kv4_cache': _lib.Kv4Cache, 'gnlp_kv4_attn_desc': _lib.Kv4AttnDesc,
               'gnlp_beam_desc': _lib.BeamDesc, 'gnlp_state': _lib.State}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "gluonnlp_amd.h"',
             'int main(void) {']
    for c, cls in structs.items():
        lines.append('printf("%s %zu\\n", "{0}", sizeof({0}));'.format(c))
        for f, _ in cls._fields_:
            lines.append('printf("%s.%s %zu\\n", "{0}", "{1}", offsetof({0}, {1}));'.format(c, f))
    src, exe = tmp_path / 'abi.c', tmp_path / 'abi'
    src.write_text('\n'.join(lines + ['return 0; }']))
    subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(exe)])
    got = dict(l.split() for l in subprocess.check_output([str(exe)]).decode().split('\n') if l)
    for c, cls in structs.items():
        assert int(got[c]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[c + '.' + f]) == getattr(cls, f).offset, (c, f)


# a pointer that no call may follow: every call below is refused before a launch
P = 1 << 20


def _cache(_lib, **kw):
    c = _lib.Kv4Cache()
    c.B, c.H, c.slots, c.d = 2, 2, 64, 64
    c.k_codes = c.v_codes = c.k_par = c.v_par = P
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize('bad', [dict(d=0), dict(d=129), dict(slots=33), dict(slots=2 ** 30),
                                 dict(B=-1), dict(B=70000), dict(k_codes=None), dict(v_par=P + 8)])
def test_bad_caches_are_refused(lib, bad):
    from gluonnlp_amd import _lib
    c = _cache(_lib, **bad)
    st = _lib.I64x3(1, 1, 1)
    for fn in (lib.gnlp_kv4_write, lib.gnlp_kv4_read):
        assert fn(ctypes.byref(c), P, P, _lib.BF16, 4, st, st, P, _lib.I32, None, 0, None) < 0
    d = _lib.Kv4AttnDesc()
    d.Lq, d.share, d.length = 1, 1, P
    assert lib.gnlp_kv4_attn(P, P, ctypes.byref(c), ctypes.byref(d), _lib.BF16, None, 0, None) < 0
    assert lib.gnlp_last_error()


def test_bad_cache_calls_are_refused(lib):
    from gluonnlp_amd import _lib
    c, st = _cache(_lib), _lib.I64x3(1, 1, 1)
    w = lib.gnlp_kv4_write
    assert w(None, P, P, _lib.BF16, 4, st, st, P, _lib.I32, None, 0, None) < 0
    assert w(ctypes.byref(c), None, P, _lib.BF16, 4, st, st, P, _lib.I32, None, 0, None) < 0
    assert w(ctypes.byref(c), P, P, 7, 4, st, st, P, _lib.I32, None, 0, None) < 0
    assert w(ctypes.byref(c), P, P, _lib.BF16, -1, st, st, P, _lib.I32, None, 0, None) < 0
    assert w(ctypes.byref(c), P, P, _lib.BF16, 4, st, st, P, 9, None, 0, None) < 0
    assert w(ctypes.byref(c), P, P, _lib.BF16, 0, st, st, P, _lib.I32, None, 0, None) == 0


def test_bad_attention_calls_are_refused(lib):
    from gluonnlp_amd import _lib

    def rc(ws=None, nws=0, q=P, **kw):
        c, d = _cache(_lib), _lib.Kv4AttnDesc()
        d.Lq, d.share, d.length = 1, 1, P
        for k, v in kw.items():
            setattr(d, k, v) if hasattr(d, k) else setattr(c, k, v)
        return lib.gnlp_kv4_attn(P, q, ctypes.byref(c), ctypes.byref(d), _lib.BF16, ws, nws, None)
    assert rc(Lq=-1) < 0
    assert rc(share=0) < 0
    assert rc(length=None) < 0
    assert rc(q=None) < 0
    assert rc(edge_scores=P, edge_table=P, table_len=4, Lm=4) < 0
    assert rc(edge_table=P, table_len=0) < 0
    assert rc(mask=P, Lm=-1) < 0
    assert rc(length_dtype=5) < 0
    assert rc(Lq=1 << 25) < 0
    assert rc(slots=1 << 20) < 0                    # several workgroups a sequence, no workspace
    assert rc(slots=1 << 20, ws=P + 4, nws=1 << 30) < 0
    assert rc(Lq=0) == 0


def test_bad_selections_are_refused(lib):
    from gluonnlp_amd import _lib

    def rc(ws=P, nws=1 << 30, scores=P, **kw):
        d = _lib.BeamDesc()
        d.N, d.K, d.V, d.row_stride, d.normalize, d.eos, d.step = 2, 4, 100, 100, 1, -1, 1
        d.temperature, d.alpha, d.length_base = 1.0, 0.0, 4.0
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.gnlp_beam_select(P, P, P, P, P, _lib.F32, scores, None, ctypes.byref(d), ws, nws,
                                    None)
    for bad in (dict(K=0), dict(K=33), dict(V=0), dict(V=2 ** 31), dict(row_stride=99), dict(N=-1),
                dict(N=20000), dict(temperature=0.0), dict(temperature=math.inf),
                dict(alpha=math.nan), dict(length_base=-1.0), dict(step=-3), dict(scores=None),
                dict(ws=None), dict(nws=16), dict(ws=P + 4), dict(step_dev=P, step_dtype=4)):
        assert rc(**bad) < 0, bad
    assert rc(N=0) == 0


def test_selections_out_of_range_are_refused(lib):
    from gluonnlp_amd import _lib

    def rc(out=1 << 20, out_finished=1 << 21, scores=1 << 22, finished=1 << 23, **kw):
        d = _lib.BeamDesc()
        d.N, d.K, d.V, d.row_stride, d.normalize, d.eos, d.step = 2, 4, 100, 100, 1, -1, 1
        d.temperature, d.alpha, d.length_base = 1.0, 0.0, 4.0
        for k, v in kw.items():
            setattr(d, k, v)
        # (no workspace: a call that gets that far ends there)
        return lib.gnlp_beam_select(out, P, P, out_finished, P, _lib.F32, scores, finished,
                                    ctypes.byref(d), None, 0, None), lib.gnlp_last_error()
    assert b'workspace' in rc()[1]
    for bad in (dict(temperature=1e-31), dict(temperature=1e31), dict(temperature=math.nan),
                dict(alpha=1e6, step=50), dict(alpha=-1e6, step=50)):
        code, why = rc(**bad)
        assert code < 0 and b'range' in why or b'temperature' in why, bad
    for bad in (dict(out=(1 << 22) + 28), dict(out_finished=1 << 23)):
        code, why = rc(**bad)
        assert code < 0 and b'alias' in why, bad


def test_states_whose_rows_overlap_are_refused(lib):
    from gluonnlp_amd import _lib

    def rc(in_place=True, **kw):
        s = _lib.State()
        s.src, s.dst = 1 << 40, (1 << 40) if in_place else 1 << 41
        s.outer, s.outer_stride, s.row_stride = 3, 8 * 128, 128
        s.nseg, s.seg_stride, s.seg_bytes = 2, 64, 64
        for k, v in kw.items():
            setattr(s, k, v)
        return lib.gnlp_reorder_states(ctypes.byref(s), 1, 2, 4, P, _lib.I32, None, 0, None), \
            lib.gnlp_last_error()
    for bad in (dict(row_stride=0), dict(row_stride=100), dict(seg_stride=32), dict(outer_stride=0),
                dict(outer_stride=8 * 128 - 16), dict(outer_stride=1 << 62)):
        for in_place in (True, False):
            code, why = rc(in_place, **bad)
            assert code < 0 and b'strides' in why, bad


def test_bad_reorderings_are_refused(lib):
    from gluonnlp_amd import _lib

    def rc(n=1, N=2, K=4, code=_lib.I32, parents=P, **kw):
        arr = (_lib.State * 2)()
        for i, s in enumerate(arr):
            s.src, s.dst = P, 2 * P
            s.outer, s.row_stride, s.nseg, s.seg_bytes = 1, 64, 1, 64
        for k, v in kw.items():
            setattr(arr[0], k, v)
        return lib.gnlp_reorder_states(arr, n, N, K, parents, code, None, 0, None)
    assert rc(K=0) < 0
    assert rc(code=3) < 0
    assert rc(parents=None) < 0
    assert rc(src=None) < 0
    assert rc(outer=-1) < 0
    assert rc(n=2, dst=P) < 0                       # one in place, one not
    assert rc(dst=P, K=33) < 0                      # in place beyond 32 beams
    assert rc(slots_per_unit=8, unit_bytes=0) < 0
    assert rc(N=2 ** 29, K=8) < 0
    assert rc(n=0) == 0 and rc(N=0) == 0 and rc(seg_bytes=0) == 0


def test_wrappers_refuse(nlp):
    cache = nlp.kv_cache.QuantKVCache(2, 2, 64, 32, ctx='cpu')
    x = torch.zeros(2, 1, 2, 64)
    with pytest.raises(RuntimeError, match='MI355X'):
        cache.read(1)
    with pytest.raises(RuntimeError, match='MI355X'):
        nlp.sequence_sampler.beam_search_select(torch.zeros(2, 3, 5), torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match='MI355X'):
        nlp.sequence_sampler.reorder_states(x, torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match='does not match'):
        cache.write(torch.zeros(2, 1, 3, 64), x)
    with pytest.raises(IndexError):
        cache.layer_desc(1)
    for bad in (dict(head_units=0), dict(head_units=129), dict(batch_size=0), dict(max_length=0),
                dict(num_heads=0), dict(num_layers=0)):
        kw = dict(batch_size=1, num_heads=1, head_units=8, max_length=4, ctx='cpu')
        with pytest.raises(ValueError):
            nlp.kv_cache.QuantKVCache(**dict(kw, **bad))
    with pytest.raises(NotImplementedError):
        nlp.kv_cache.QuantKVCache(1, 1, 8, 4, ctx='cpu', layout='TKN')


def test_lengths_are_counted(nlp):
    c = nlp.kv_cache.QuantKVCache(2, 1, 8, 10, ctx='cpu')
    c.extend(4)
    c.extend(3)
    with pytest.raises(ValueError, match='do not fit'):
        c.extend(4)
    c.extend(3)
    assert c.length.tolist() == [10, 10]
    with pytest.raises(ValueError):
        c.extend(11)
    with pytest.raises(ValueError):
        c.set_length(11)
    c.set_length(2)
    assert c.length.tolist() == [2, 2]
    c.reset()
    assert c.length.tolist() == [0, 0]


@pytest.mark.parametrize('d', [1, 33, 64, 100, 128])
def test_reference_format_error(d):
    """A value is off by at most half a scale, plus what rounding the scale (15 codes of it, 2^-8
    relative) and the minimum (2^-8 of it) to bfloat16 can add."""
    x = torch.randn(50, d, generator=torch.Generator().manual_seed(d)) * 3 + 1
    v, s, m = ref.quantise(x)
    assert ((v - x).abs() <= s * (0.5 + 15 * 2.0 ** -8) + m.abs() * 2.0 ** -8 + 1e-6).all()
