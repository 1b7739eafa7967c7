"""Beam search on the device: the selection of one step, and the reordering of the decoding states
that follows it (what the reference's sequence_sampler.py builds from log_softmax, topk and take)."""
import array
import ctypes
import functools
import struct
import warnings

import torch

from . import _lib
from . import _tensor as T
from .kv_cache import QuantDecoderStates, QuantKVCache

__all__ = ['beam_search_select', 'reorder_states', 'BeamSearchSampler']

MAX_BEAMS = 32


_BEAM_DESC = struct.Struct('7qPq3d')     # gnlp_beam_desc


@functools.lru_cache(maxsize=1024)
def _select_workspace(N, K, V):
    d = _lib.BeamDesc()
    d.N, d.K, d.V = N, K, V
    return _lib.load().gnlp_beam_select_workspace_bytes(ctypes.byref(d))


def _row_stride(shape, stride):
    """Elements between the rows of logits (N, K, V) or (rows, V); 0 where they are not V neighbouring
    elements each, at one distance.  The stride of an axis of one element says nothing: a transposed
    or sliced view keeps whatever it was, and ``contiguous`` leaves it."""
    V = shape[-1]
    if V > 1 and stride[-1] != 1:
        return 0
    axes = [(n, st) for n, st in zip(shape[:-1], stride) if n != 1]
    if not axes:
        return V
    if len(axes) == 2 and axes[0][1] != axes[1][0] * axes[1][1]:
        return 0
    return axes[-1][1]


def beam_search_select(outputs, scores, finished=None, *, eos_id=None, step=1, alpha=0.0,
                       length_base=None, temperature=1.0, normalize=True):
    """One step of a beam search over N items of K beams (K <= 32).

    outputs (N, K, V) or (N * K, V), float32 / bfloat16 logits (``normalize=False``:
    log-probabilities); scores (N, K) float32; finished (N, K) bool or None.  A candidate, token v
    of an unfinished beam k, scores

        (scores[k] * lp(step - 1) + z[k, v] - logsumexp(z[k])) / lp(step),  z = outputs / temperature
        lp(s) = ((length_base + s) / (length_base + 1)) ** alpha            (length_base: default K)

    (the default of ``length_base`` changes with the beams; ``BeamSearchSampler`` gives 5, whatever
    they are), a finished beam is its own only candidate, with its score.  Returns the K best of each
    item, best first, ties to the lowest k * V + v and finished beams last:

        scores (N, K) float32, parents (N, K) int32, tokens (N, K) int32 (-1: was finished),
        finished (N, K) bool (the parent was, or the token is ``eos_id``)

    NaN outputs count as -inf, +inf as the largest float.  A beam whose score is not above -1e15 is
    dead (the start of a search: scores [0, -inf, ...]); its candidates count as -inf.  The outputs
    of finished beams are not read.  ``step`` may be a device integer tensor of one element (a
    captured step then follows it).  Candidates are compared in 64 bits (the exponentials of a
    logsumexp are summed in 32 bits within 4096 or 8192 logits, in 64 over them)."""
    x, s, f = T.as_tensor(outputs), T.as_tensor(scores), T.as_tensor(finished)
    dev = T.device_index(x, s, f)
    if s.dim() != 2 or s.dtype != torch.float32:
        raise ValueError('scores must be (items, beams) float32, got {} {}'.format(
            tuple(s.shape), s.dtype))
    N, K = s.shape
    if not 1 <= K <= MAX_BEAMS:
        raise ValueError('beam size {} is outside [1, {}]'.format(K, MAX_BEAMS))
    shape = x.shape
    if shape[:-1] not in ((N, K), (N * K,)) or shape[-1] < 1:
        raise ValueError('outputs {} do not match scores {}'.format(tuple(shape), tuple(s.shape)))
    if (x.requires_grad or s.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError('the selection has no gradient: search under torch.no_grad()')
    V = shape[-1]
    row_stride = V if x.is_contiguous() else _row_stride(shape, x.stride())
    if row_stride < V:
        x, row_stride = x.contiguous(), V
    if not s.is_contiguous():
        s = s.contiguous()
    fp = None
    if f is not None:
        if f.shape != s.shape:
            raise ValueError('finished {} does not match scores {}'.format(tuple(f.shape),
                                                                           tuple(s.shape)))
        if f.dtype != torch.bool:
            f = f != 0
        if not f.is_contiguous():
            f = f.contiguous()
        fp = f.data_ptr()
    step_ptr, step_code = 0, 0
    if isinstance(step, torch.Tensor):
        T.device_index(x, step)
        if step.numel() != 1 or step.dtype not in (torch.int32, torch.int64):
            raise ValueError('step must hold one int32 / int64')
        step_ptr = step.data_ptr()
        step_code = _lib.I64 if step.dtype == torch.int64 else _lib.I32
        step = 0
    desc = _BEAM_DESC.pack(N, K, V, row_stride, bool(normalize),
                           -1 if eos_id is None else int(eos_id), step, step_ptr, step_code,
                           temperature, alpha, K if length_base is None else length_base)
    out_scores = torch.empty_like(s)
    parents, tokens = s.new_empty((2, N, K), dtype=torch.int32).unbind(0)
    out_finished = s.new_empty((N, K), dtype=torch.bool)
    nws = _select_workspace(N, K, V)
    ws = s.new_empty(nws, dtype=torch.uint8)
    T.launch(dev, _lib.load().gnlp_beam_select, out_scores.data_ptr(), parents.data_ptr(),
             tokens.data_ptr(), out_finished.data_ptr(), x.data_ptr(), T.code(x), s.data_ptr(), fp,
             desc, ws.data_ptr(), nws)
    if type(outputs) is torch.Tensor:
        return out_scores, parents, tokens, out_finished
    return tuple(T.like_caller(o, outputs) for o in (out_scores, parents, tokens, out_finished))


def check_parents(parents, rows):
    p = T.as_tensor(parents)
    if p.dim() != 2 or p.dtype not in (torch.int32, torch.int64):
        raise ValueError('parents must be (items, beams) int32 / int64, got {} {}'.format(
            tuple(p.shape), p.dtype))
    N, K = p.shape
    if rows is not None and N * K != rows:
        raise ValueError('parents {} do not match {} rows'.format(tuple(p.shape), rows))
    return p if p.is_contiguous() else p.contiguous(), N, K


def launch_reorder(dev, flat, N, K, parents, length):
    """flat: the fields of one gnlp_state (include/gluonnlp_amd.h) after the other."""
    buf = array.array('q', flat)
    T.launch(dev, _lib.load().gnlp_reorder_states, buf.buffer_info()[0], len(flat) // 10, N, K,
             parents.data_ptr(), _lib.I64 if parents.dtype == torch.int64 else _lib.I32,
             None if length is None else length.data_ptr(), _lib.I32)


def reorder_states(states, parents, batch_axis=0, out=None):
    """Reorder decoding states after a selection: row n K + k along the batch axis of every tensor
    becomes its row n K + parents[n, k] (parents (N, K), values in [0, K); others are clamped).

    states: a tensor, a ``QuantKVCache``, ``QuantDecoderStates``, None, or nested lists / tuples of
    them, as ``incremental_decode`` returns them; ``batch_axis``: one int, or axes nested like the states
    (a decoder's ``state_batch_axis``).  Returns the same structure: new tensors, or the tensors of
    ``out`` (nested like the states, contiguous, no overlap with the states), or, with
    ``out=states``, the states themselves, rewritten in place (K <= 32; each tensor once).  Caches
    are always reordered in place.  Up to 32 tensors move in one launch."""
    p, N, K = check_parents(parents, None)
    in_place = out is states
    if in_place and K > MAX_BEAMS:
        raise ValueError('in place: beam size {} > {}'.format(K, MAX_BEAMS))
    dev = T.device_index(p)
    rows, grad = N * K, torch.is_grad_enabled()
    flat, sources, caches, written = [], [], [], []
    last = (None, None, None)              # (shape, dtype, axis) of the state before, and its rows
    tail = None

    def one(s, axis, o):
        nonlocal last, tail
        t = s if type(s) is torch.Tensor else T.as_tensor(s)
        if t.get_device() != dev:
            T.require_device(p, t)
        if grad and t.requires_grad:
            raise NotImplementedError('reordering has no gradient: decode under torch.no_grad()')
        shape, dtype = t.shape, t.dtype
        if last[0] != shape or last[1] is not dtype or last[2] is not axis:
            if type(axis) is not int or not 0 <= axis < len(shape) or shape[axis] != rows:
                raise ValueError('state {}: axis {} does not hold {} x {} rows'.format(
                    tuple(shape), axis, N, K))
            last, tail, n = (shape, dtype, axis), None, t.numel()
            if n:
                outer = 1
                for i in range(axis):
                    outer *= shape[i]
                row = n // (outer * rows) * t.element_size()
                tail = (outer, row * rows, row, 1, row, row, 0, 0)
        if not t.is_contiguous():
            if in_place:
                raise ValueError('in place: the states must be contiguous')
            t = t.contiguous()
            sources.append(t)              # (it has to live until the launch)
        if in_place:
            d = t
        elif o is None:
            d = torch.empty_like(t)
        else:
            d = o if type(o) is torch.Tensor else T.as_tensor(o)
            if d.shape != shape or d.dtype is not dtype or not d.is_contiguous() or \
                    d.get_device() != dev:
                raise ValueError('out {} {} does not fit the state {} {}'.format(
                    tuple(d.shape), d.dtype, tuple(shape), dtype))
        if o is not None or in_place:
            written.append(d)
        if tail is not None:
            flat.append(t.data_ptr())
            flat.append(d.data_ptr())
            flat.extend(tail)
        return d if type(s) is torch.Tensor else T.like_caller(d, s)

    def walk(s, axis, o):
        if isinstance(s, torch.Tensor):
            return one(s, axis, o)
        if s is None:
            return None
        if isinstance(s, (QuantKVCache, QuantDecoderStates)):
            # (refused before anything moves; each cache once, also where states and their cache come)
            caches.extend(c for c in s.check_reorder(p) if not any(c is x for x in caches))
            return s
        if isinstance(s, (list, tuple)):
            n = len(s)
            axes = axis if isinstance(axis, (list, tuple)) else (axis,) * n
            outs = o if isinstance(o, (list, tuple)) else (o,) * n
            if len(axes) != n or len(outs) != n or (o is not None and outs is not o):
                raise ValueError('batch_axis / out are not nested like the states')
            r = []
            for x, ax, ox in zip(s, axes, outs):
                if type(x) is not torch.Tensor:
                    r.append(walk(x, ax, ox))
                    continue
                # (states are mostly alike: one that is like the one before needs no more checks)
                d = x if in_place else ox
                if tail is None or type(d) is not torch.Tensor or ax is not last[2] or \
                        x.shape != last[0] or x.dtype is not last[1] or x.get_device() != dev or \
                        not x.is_contiguous() or grad and x.requires_grad or d is not x and (
                            d.shape != last[0] or d.dtype is not last[1] or
                            d.get_device() != dev or not d.is_contiguous()):
                    r.append(one(x, ax, ox))
                    continue
                flat.extend((x.data_ptr(), d.data_ptr()) + tail)
                written.append(d)
                r.append(d)
            return r if isinstance(s, list) else tuple(r)
        return one(s, axis, o)

    result = walk(states, batch_axis, None if in_place else out)
    if flat:
        launch_reorder(dev, flat, N, K, p, None)
        if written:       # (what is kept for a tensor as it was -- a memory's projections, what autograd
            torch.autograd.graph.increment_version(written)     # saved -- shall see that it changed)
    for c in caches:
        c._move(p)
    return result


class BeamSearchSampler:
    """Beam search with a step decoder (the reference's sequence_sampler.BeamSearchSampler).

    decoder(step_input (N * K,), states) -> (outputs (N * K, V), states): logits (or, with
    ``normalize=False``, log-probabilities) of the next token, and the states after the step;
    the states hold N * K rows along ``state_batch_axis``.  A candidate's score is its
    log-probability sum over ((length_base + length) / (length_base + 1)) ** alpha.

    ``from_logits`` is the earlier name of ``normalize`` and means the same (true: the outputs are
    unnormalised); elsewhere the name says the opposite, that the outputs are log-probabilities
    already, so giving it warns."""

    def __init__(self, beam_size, decoder, eos_id, alpha=1.0, length_base=5, max_length=100,
                 temperature=1.0, normalize=True, state_batch_axis=0, early_return=True, *,
                 from_logits=None):
        if from_logits is not None:
            warnings.warn('BeamSearchSampler: from_logits={0} means normalize={0} here (true: the '
                          'decoder gives unnormalised logits); give normalize'.format(from_logits),
                          FutureWarning, stacklevel=2)
            normalize = from_logits
        if not 1 <= beam_size <= MAX_BEAMS:
            raise ValueError('beam size {} is outside [1, {}]'.format(beam_size, MAX_BEAMS))
        if max_length < 1:
            raise ValueError('max_length={} must be positive'.format(max_length))
        self._beam_size, self._decoder, self._eos_id = beam_size, decoder, eos_id
        self._alpha, self._length_base, self._max_length = alpha, length_base, max_length
        self._temperature, self._normalize = temperature, normalize
        self._axis, self._early_return = state_batch_axis, early_return

    def __call__(self, inputs, states):
        """inputs (N,): the first token of each item.  Returns samples (N, K, T) int32 -- the first
        token, the tokens found, then -1 --, scores (N, K), best first, and valid_length (N, K)
        (the first token and the end of sentence counted)."""
        first = T.as_tensor(inputs)
        N, K = first.shape[0], self._beam_size
        T.require_device(first)
        with torch.no_grad():
            samples = torch.full((N * K, self._max_length + 1), -1, dtype=torch.int32,
                                 device=first.device)
            step_input = first.to(torch.int32).repeat_interleave(K)
            samples[:, 0] = step_input
            scores = torch.full((N, K), -float('inf'), dtype=torch.float32, device=first.device)
            scores[:, 0] = 0.0
            finished = None
            pad = 0 if self._eos_id is None else int(self._eos_id)
            steps = 0
            for step in range(1, self._max_length + 1):
                outputs, states = self._decoder(step_input, states)
                scores, parents, tokens, finished = beam_search_select(
                    outputs, scores, finished, eos_id=self._eos_id, step=step, alpha=self._alpha,
                    length_base=self._length_base, temperature=self._temperature,
                    normalize=self._normalize)
                steps = step
                reorder_states(samples, parents, out=samples)
                samples[:, step] = tokens.reshape(-1)
                if step == self._max_length or self._early_return and bool(finished.all()):
                    break
                states = reorder_states(states, parents, batch_axis=self._axis)
                # (a finished beam is decoded on, from the end of sentence; nothing reads it)
                step_input = torch.where(tokens < 0, pad, tokens).reshape(-1)
        samples = samples[:, :steps + 1].reshape(N, K, steps + 1)
        valid_length = (samples >= 0).sum(-1).to(torch.int32)
        return tuple(T.like_caller(o, inputs) for o in (samples, scores, valid_length))

