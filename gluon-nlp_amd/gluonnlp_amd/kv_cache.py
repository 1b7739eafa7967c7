"""Key / value cache of incremental decoding, held in 4 bits.

The decoders' own states are float tensors that grow by concatenation (reference
models/transformer.py:607-734, models/t5.py:374-490).  ``QuantKVCache`` keeps the same keys and
values in 72 bytes a token and head of 64 channels where bfloat16 takes 256, in buffers that do not
move: a decoding step neither allocates nor copies the past, and can be captured in a graph.
``attention_cell.multi_head_dot_attn_cached`` attends over it.

The format (include/gluonnlp_amd.h): 64 channels of a token and head share a scale and a minimum in
bfloat16, a value is ``code * scale + minimum`` with a code of 0 .. 15; the error of a value is at
most half a scale, (max - min) / 30, plus the roundings of scale and minimum to bfloat16.
"""
import ctypes
import struct

import torch

from . import _lib
from . import _tensor as T

__all__ = ['QuantKVCache', 'QuantDecoderStates']

_TIME = {'NKT': 2, 'NTK': 1, 'TNK': 0}
_PERM = {'NKT': (0, 1, 2), 'NTK': (0, 2, 1), 'TNK': (1, 2, 0)}
_pack3 = struct.Struct('3q').pack
_DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16}


class QuantKVCache:
    """Keys and values of ``num_layers`` attention layers, ``max_length`` tokens of ``batch_size``
    sequences, ``num_heads`` cached heads of ``head_units`` (1 .. 128) channels.

    A step: ``cache.extend(n)`` counts the n new tokens of every sequence in, then each layer
    stores them with ``cache.write(key, value, layer)`` and attends.  All layers share ``length``,
    a device int32 vector (batch_size,) of the tokens held: nothing is read back to the host, and a
    captured graph replays with the lengths of its time.  ``layout`` is that of the keys and values
    ('NTK', 'NKT' or 'TNK' as in ``multi_head_dot_attn``).

    ``extend`` refuses tokens beyond ``max_length``; the replays of a graph cannot: there, tokens
    beyond the buffer (``max_length`` rounded up to 32) are not stored.  Once a graph has captured a
    change of the lengths, an ``extend`` outside of it reads them back first.  Two writes, or a write and a
    reading call, on different streams have to be ordered by the caller, like any two uses of a
    tensor."""

    def __init__(self, batch_size, num_heads, head_units, max_length, num_layers=1, ctx=None,
                 layout='NTK'):
        if layout not in _PERM:
            raise NotImplementedError('layout="{}" is not supported! We only support layout = '
                                      '"NKT", "NTK", and "TNK".'.format(layout))
        for name, v, lo, hi in (('batch_size', batch_size, 1, 65535),
                                ('num_heads', num_heads, 1, 65535),
                                ('head_units', head_units, 1, 128),
                                ('max_length', max_length, 1, 2 ** 30 - 32),
                                ('num_layers', num_layers, 1, 65535)):
            if not lo <= int(v) <= hi:
                raise ValueError('{}={} is outside [{}, {}]'.format(name, v, lo, hi))
        self.batch_size, self.num_heads, self.head_units = batch_size, num_heads, head_units
        self.max_length, self.num_layers, self.layout = max_length, num_layers, layout
        dev = torch.device('cuda' if ctx is None else ctx)
        if dev.type == 'cuda' and dev.index is None:
            dev = torch.device('cuda', torch.cuda.current_device())
        self.device = dev
        self._slots = slots = (max_length + 31) // 32 * 32
        self._padded = padded = 64 if head_units <= 64 else 128
        groups = padded // 64
        lead = (num_layers, batch_size, num_heads)
        self._k_codes = torch.zeros(lead + (slots, padded // 2), dtype=torch.uint8, device=dev)
        self._v_codes = torch.zeros(lead + (slots // 8, padded), dtype=torch.int32, device=dev)
        self._k_par = torch.zeros(lead + (groups, slots), dtype=torch.int32, device=dev)
        self._v_par = torch.zeros(lead + (groups, slots), dtype=torch.int32, device=dev)
        self._length = torch.zeros(batch_size, dtype=torch.int32, device=dev)
        self._bound = 0            # no sequence holds more tokens, as far as the host knows
        self._replays = False      # a graph's replays may change the lengths behind its back
        self._desc = []
        for i in range(num_layers):
            c = _lib.Kv4Cache()
            c.B, c.H, c.slots, c.d = batch_size, num_heads, slots, head_units
            c.k_codes, c.v_codes = self._k_codes[i].data_ptr(), self._v_codes[i].data_ptr()
            c.k_par, c.v_par = self._k_par[i].data_ptr(), self._v_par[i].data_ptr()
            self._desc.append(c)
        self._refs = [ctypes.addressof(c) for c in self._desc]
        self._length_ptr = self._length.data_ptr()

    def __repr__(self):
        return '{}(batch_size={}, num_heads={}, head_units={}, max_length={}, num_layers={}, ' \
               'layout="{}")'.format(self.__class__.__name__, self.batch_size, self.num_heads,
                                     self.head_units, self.max_length, self.num_layers, self.layout)

    @property
    def length(self):
        """(batch_size,) int32 on the device: the tokens held (written by the calls below only)."""
        return self._length

    def layer_desc(self, layer):
        """Address of the layer's gnlp_kv4_cache."""
        if not 0 <= layer < self.num_layers:
            raise IndexError('layer {} of {}'.format(layer, self.num_layers))
        return self._refs[layer]

    def _lengths(self, v, name):
        """A (batch_size,) device vector of whole numbers."""
        if type(v) is not torch.Tensor:
            v = T.as_tensor(v)
        if v.dtype not in (torch.int32, torch.int64):
            raise TypeError('{} must be int32 or int64, got {}'.format(name, v.dtype))
        if v.dim() != 1 or v.shape[0] != self.batch_size:
            raise ValueError('{} {} != (batch_size,) = ({},)'.format(name, tuple(v.shape),
                                                                     self.batch_size))
        T.device_index(self.length, v)
        return v if v.is_contiguous() else v.contiguous()

    # ---- lengths ----
    def _capturing(self):
        if self.device.type != 'cuda' or not torch.cuda.is_current_stream_capturing():
            return False
        self._replays = True
        return True

    def reset(self):
        """Forget all tokens."""
        self._capturing()
        self.length.zero_()
        self._bound = 0

    def set_length(self, length):
        """Set the number of tokens held, an int or a (batch_size,) vector (int32 / int64; its values
        stay on the device and are not looked at)."""
        self._capturing()
        if isinstance(length, int):
            if not 0 <= length <= self.max_length:
                raise ValueError('length={} is outside [0, {}]'.format(length, self.max_length))
            self.length.fill_(length)
            self._bound = length
        else:
            self.length.copy_(self._lengths(length, 'length'))
            self._bound = self.max_length

    def extend(self, n, new_length=None):
        """Count in n new tokens of every sequence (``new_length``: its own number of each, at most
        n).  They are stored by the ``write`` calls that follow."""
        if n < 0 or n > self.max_length:
            raise ValueError('n={} is outside [0, max_length={}]'.format(n, self.max_length))
        if new_length is not None:
            new_length = self._lengths(new_length, 'new_length')
        if self._capturing():
            self._bound = self.max_length      # (the replays go on from lengths of their own)
        elif self._replays or self._bound + n > self.max_length:
            # the bound is loose after ragged steps and unknown after replays: look (the one place
            # that waits for the device)
            self._bound = max(0, int(self.length.max()))
            grown = self._bound + n if new_length is None else \
                int((self.length + new_length.clamp(0, n)).max())
            if grown > self.max_length:
                raise ValueError('{} tokens do not fit max_length={}'.format(grown,
                                                                            self.max_length))
        if new_length is None:
            self.length.add_(n)
        else:
            self.length.add_(new_length.clamp(0, n))
        self._bound = min(self._bound + n, self.max_length)

    # ---- tokens ----
    def _tokens(self, x, name):
        """-> (tensor with contiguous channels, its packed (b, h, t) strides)"""
        if type(x) is not torch.Tensor:
            x = T.as_tensor(x)
        p, shape = _PERM[self.layout], x.shape
        if len(shape) != 4 or shape[p[0]] != self.batch_size or shape[p[1]] != self.num_heads \
                or shape[3] != self.head_units:
            raise ValueError('{} {} does not match {}'.format(name, tuple(shape), self))
        st = x.stride()
        if st[3] != 1 and shape[3] != 1:
            x = x.contiguous()
            st = x.stride()
        if x.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError('a 4-bit cache has no gradient: decode under torch.no_grad()')
        return x, _pack3(st[p[0]], st[p[1]], st[p[2]])

    def write(self, key, value, layer=0, new_length=None):
        """Store the last tokens counted in: key / value (batch_size, n, num_heads, head_units) in
        the cache's layout go to the last n of the ``length`` tokens of each sequence.  With
        ``new_length`` (batch_size,), sequence b stores its first new_length[b] tokens as its last
        new_length[b] (the others, padding, are not read).  Other tokens keep their values."""
        k, ks = self._tokens(key, 'key')
        v, vs = self._tokens(value, 'value')
        dev = T.device_index(self.length, k, v)
        if k.dtype != v.dtype or k.shape != v.shape:
            raise ValueError('key and value must share shape and dtype')
        n = k.shape[_TIME[self.layout]]
        nl, code = None, 0
        if new_length is not None:
            new_length = self._lengths(new_length, 'new_length')
            nl = new_length.data_ptr()
            code = _lib.I64 if new_length.dtype == torch.int64 else _lib.I32
        elif n > self._bound and not self._replays:
            raise ValueError('write of {} tokens, {} are counted in: call extend() first'
                             .format(n, self._bound))
        T.launch(dev, _lib.load().gnlp_kv4_write, self.layer_desc(layer), k.data_ptr(),
                 v.data_ptr(), T.code(k), n, ks, vs, self._length_ptr, _lib.I32, nl, code)

    def read(self, n=None, start=None, layer=0, dtype='float32'):
        """The values held: (key, value) of n tokens (default: max_length) from ``start``
        (batch_size,) on (default 0), in the cache's layout; zeros where no token is held."""
        n = self.max_length if n is None else int(n)
        if n < 0:
            raise ValueError('n={} is negative'.format(n))
        dev = T.device_index(self.length)
        st, code = None, 0
        if start is not None:
            start = self._lengths(start, 'start')
            st = start.data_ptr()
            code = _lib.I64 if start.dtype == torch.int64 else _lib.I32
        B, H, d = self.batch_size, self.num_heads, self.head_units
        if self.layout == 'NTK':
            shape, strides = (B, n, H, d), _pack3(n * H * d, d, H * d)
        elif self.layout == 'NKT':
            shape, strides = (B, H, n, d), _pack3(H * n * d, n * d, d)
        else:
            shape, strides = (n, B, H, d), _pack3(H * d, d, B * H * d)
        key = self._length.new_empty(shape, dtype=_DTYPES.get(dtype) or T.torch_dtype(dtype))
        value = torch.empty_like(key)
        T.launch(dev, _lib.load().gnlp_kv4_read, self.layer_desc(layer), key.data_ptr(),
                 value.data_ptr(), T.code(key), n, strides, strides, self._length_ptr, _lib.I32, st,
                 code)
        return key, value

    def reorder(self, parents):
        """Beam search: sequence n K + k goes on from sequence n K + parents[n, k]; ``parents``
        (items, K) whole numbers in [0, K), K <= 32.  In place, all layers in one launch; only the
        tokens held are moved."""
        self.check_reorder(parents)
        self._move(parents)

    def check_reorder(self, parents):
        """The errors of ``reorder``, before anything moves -> the caches that it moves."""
        from .sequence_sampler import check_parents
        p, N, K = check_parents(parents, self.batch_size)
        T.device_index(self.length, p)
        if K > 32:
            raise ValueError('beam size {} > 32'.format(K))
        return [self]

    def _move(self, parents):
        from .sequence_sampler import check_parents, launch_reorder
        p, N, K = check_parents(parents, self.batch_size)
        dev = T.device_index(self.length, p)
        flat = []
        L, B, H, S = self.num_layers, self.batch_size, self.num_heads, self._slots
        groups = self._padded // 64
        for t, nseg, per, unit in ((self._k_codes, H, 1, self._padded // 2),
                                   (self._v_codes, H, 8, self._padded * 4),
                                   (self._k_par, H * groups, 1, 4),
                                   (self._v_par, H * groups, 1, 4)):
            seg = S // per * unit
            row = nseg * seg
            flat += [t.data_ptr(), t.data_ptr(), L, B * row, row, nseg, seg, seg, per, unit]
        launch_reorder(dev, flat, N, K, p, self.length)
        # (a launch of its own: the one above reads the lengths)
        at = self.length.data_ptr()
        launch_reorder(dev, [at, at, 1, 4 * B, 4, 1, 4, 4, 0, 0], N, K, p, None)


class QuantDecoderStates:
    """States of ``T5Decoder.incremental_decode`` / ``TransformerDecoder.incremental_decode`` with
    keys and values in 4 bits (made by the decoders' ``init_quant_states``): ``self_cache`` grows by
    a token a step; ``memory_cache`` holds the memory's projections, written once, one sequence an
    item -- the beams of an item (consecutive rows) attend over it as the queries of one call.
    ``bias_table``: T5's position bias by distance.  Projections and table are those of the weights
    at the time the states were made.  A step does not change its shapes: it can be captured in a
    graph and replayed."""

    def __init__(self, self_cache, memory_cache, bias_table=None):
        if self_cache.batch_size % memory_cache.batch_size:
            raise ValueError('{} rows do not share {} memories evenly'.format(
                self_cache.batch_size, memory_cache.batch_size))
        self.self_cache, self.memory_cache, self.bias_table = self_cache, memory_cache, bias_table

    @property
    def length(self):
        return self.self_cache.length

    def begin(self, decoder, x):
        """Count a token in for a step of ``decoder`` on x; a call that asks for gradients is
        refused before."""
        if torch.is_grad_enabled() and (x.requires_grad or
                                        any(p.requires_grad for p in decoder.parameters())):
            raise NotImplementedError('a 4-bit cache has no gradient: decode under torch.no_grad()')
        if x.numel() != self.self_cache.batch_size * x.shape[-1]:
            raise ValueError('a step of {} does not fit states of {} rows'.format(
                tuple(x.shape), self.self_cache.batch_size))
        self.self_cache.extend(1)

    def reorder(self, parents):
        """Beam search: row n K + k goes on from row n K + parents[n, k].  The memory stays: the
        beams of an item share it."""
        for c in self.check_reorder(parents):
            c._move(parents)

    def check_reorder(self, parents):
        """The errors of ``reorder``, before anything moves -> the caches that it moves."""
        if self.memory_cache.batch_size not in (parents.shape[0], self.self_cache.batch_size):
            raise ValueError('{} items, the states hold {} memories'.format(
                parents.shape[0], self.memory_cache.batch_size))
        moved = [self.self_cache]
        if self.memory_cache.batch_size != parents.shape[0]:
            moved.append(self.memory_cache)
        for c in moved:
            c.check_reorder(parents)
        return moved

    def memory_queries(self, q):
        """(rows, 1, H, d) or (1, rows, H, d) -> (memories, beams, H, d)."""
        return q.reshape(self.memory_cache.batch_size, -1, q.shape[2], q.shape[3])


def quant_decoder_states(mem, mem_valid_length, projections, num_heads, head_units, max_length,
                         beam_size, layout, bias_table=None):
    """The states of a decoder; ``projections``: per layer the Dense layers of the memory's keys and
    values.  mem: (items, Lm, C) / (Lm, items, C)."""
    m = T.as_tensor(mem)
    axis = 1 if layout == 'NT' else 0
    items, Lm = m.shape[1 - axis], m.shape[axis]
    kv = 'NTK' if layout == 'NT' else 'TNK'
    n = len(projections)
    with torch.no_grad():
        memory = QuantKVCache(items, num_heads, head_units, Lm, n, m.device, kv)
        memory.set_length(Lm)
        for i, (key, value) in enumerate(projections):
            memory.write(*(T.as_tensor(p(m)).reshape(m.shape[0], m.shape[1], num_heads, head_units)
                           for p in (key, value)), layer=i)
        if mem_valid_length is not None:
            # (as the float states' mask takes them: any number, more than Lm is all of it; the
            # buffer has a few more slots)
            memory.set_length(T.valid_length_arg(mem_valid_length)[0].clamp(0, Lm))
        rows = QuantKVCache(items * beam_size, num_heads, head_units, max_length, n, m.device, kv)
    return QuantDecoderStates(rows, memory, bias_table)
