"""Beam search on the device: the selection of one step, and the reordering of the decoding states
that follows it (what the reference's sequence_sampler.py builds from log_softmax, topk and take)."""
import array
import ctypes

import torch

from . import _lib
from . import _tensor as T
from .autograd import wants_grad
from .kv_cache import QuantKVCache

__all__ = ['beam_search_select', 'reorder_states']

MAX_BEAMS = 32


def beam_search_select(outputs, scores, finished=None, *, eos_id=None, step=1, alpha=0.0,
                       length_base=None, temperature=1.0, normalize=True):
    """One step of a beam search over N items of K beams (K <= 32).

    outputs (N, K, V) or (N * K, V), float32 / bfloat16 logits (``normalize=False``:
    log-probabilities); scores (N, K) float32; finished (N, K) bool or None.  A candidate, token v
    of an unfinished beam k, scores

        (scores[k] * lp(step - 1) + z[k, v] - logsumexp(z[k])) / lp(step),  z = outputs / temperature
        lp(s) = ((length_base + s) / (length_base + 1)) ** alpha            (length_base: default K)

    a finished beam is its own only candidate, with its score.  Returns the K best of each item,
    best first, ties to the lowest k * V + v and finished beams last:

        scores (N, K) float32, parents (N, K) int32, tokens (N, K) int32 (-1: was finished),
        finished (N, K) bool (the parent was, or the token is ``eos_id``)

    NaN outputs count as -inf, +inf as the largest float.  A beam whose score is not above -1e15 is
    dead (the start of a search: scores [0, -inf, ...]); its candidates count as -inf.  The outputs
    of finished beams are not read.  ``step`` may be a device integer tensor of one element (a
    captured step then follows it).  Candidates are compared in 64 bits."""
    x, s, f = T.as_tensor(outputs), T.as_tensor(scores), T.as_tensor(finished)
    dev = T.require_device(x, s, f)
    if s.dim() != 2 or s.dtype != torch.float32:
        raise ValueError('scores must be (items, beams) float32, got {} {}'.format(
            tuple(s.shape), s.dtype))
    N, K = s.shape
    if not 1 <= K <= MAX_BEAMS:
        raise ValueError('beam size {} is outside [1, {}]'.format(K, MAX_BEAMS))
    if x.dim() not in (2, 3) or x.shape[:-1] not in ((N, K), (N * K,)) or x.shape[-1] < 1:
        raise ValueError('outputs {} do not match scores {}'.format(tuple(x.shape), tuple(s.shape)))
    if wants_grad(x, s):
        raise NotImplementedError('the selection has no gradient: search under torch.no_grad()')
    V = x.shape[-1]
    if x.stride(-1) != 1 and V > 1 or x.dim() == 3 and x.stride(0) != K * x.stride(1) \
            or x.stride(-2) < V:
        x = x.contiguous()
    if not s.is_contiguous():
        s = s.contiguous()
    if f is not None:
        if f.shape != s.shape:
            raise ValueError('finished {} does not match scores {}'.format(tuple(f.shape),
                                                                           tuple(s.shape)))
        if f.dtype != torch.bool:
            f = f != 0
        if not f.is_contiguous():
            f = f.contiguous()
    d = _lib.BeamDesc()
    d.N, d.K, d.V, d.row_stride = N, K, V, x.stride(-2)
    d.normalize, d.eos = bool(normalize), -1 if eos_id is None else int(eos_id)
    d.temperature, d.alpha = temperature, alpha
    d.length_base = K if length_base is None else length_base
    if isinstance(step, torch.Tensor):
        T.require_device(x, step)
        if step.numel() != 1 or step.dtype not in (torch.int32, torch.int64):
            raise ValueError('step must hold one int32 / int64')
        d.step_dev = step.data_ptr()
        d.step_dtype = _lib.I64 if step.dtype == torch.int64 else _lib.I32
    else:
        d.step = step
    lib = _lib.load()
    out_scores = torch.empty((N, K), dtype=torch.float32, device=dev)
    parents, tokens = torch.empty((2, N, K), dtype=torch.int32, device=dev).unbind(0)
    out_finished = torch.empty((N, K), dtype=torch.bool, device=dev)
    nws = lib.gnlp_beam_select_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(nws, dtype=torch.uint8, device=dev)
    T.launch(dev, lib.gnlp_beam_select, out_scores.data_ptr(), parents.data_ptr(),
             tokens.data_ptr(), out_finished.data_ptr(), x.data_ptr(), T.code(x), s.data_ptr(),
             T.ptr(f), ctypes.byref(d), ws.data_ptr(), nws)
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
    T.launch(dev, _lib.load().gnlp_reorder_states,
             ctypes.cast(buf.buffer_info()[0], ctypes.POINTER(_lib.State)), len(flat) // 10, N, K,
             parents.data_ptr(), _lib.I64 if parents.dtype == torch.int64 else _lib.I32,
             T.ptr(length), _lib.I32)


def reorder_states(states, parents, batch_axis=0, out=None):
    """Reorder decoding states after a selection: row n K + k along the batch axis of every tensor
    becomes its row n K + parents[n, k] (parents (N, K), values in [0, K); others are clamped).

    states: a tensor, a ``QuantKVCache``, None, or nested lists / tuples of them, as
    ``incremental_decode`` returns them; ``batch_axis``: one int, or axes nested like the states
    (a decoder's ``state_batch_axis``).  Returns the same structure: new tensors, or the tensors of
    ``out`` (nested like the states, contiguous, no overlap with the states), or, with
    ``out=states``, the states themselves, rewritten in place (K <= 32; each tensor once).  Caches
    are always reordered in place.  Up to 32 tensors move in one launch."""
    p, N, K = check_parents(parents, None)
    in_place = out is states
    if in_place and K > MAX_BEAMS:
        raise ValueError('in place: beam size {} > {}'.format(K, MAX_BEAMS))
    flat, sources, caches = [], [], []
    dev = T.require_device(p)

    def walk(s, axis, o):
        if s is None:
            return None
        if isinstance(s, QuantKVCache):
            if s not in caches:
                caches.append(s)
            return s
        if isinstance(s, (list, tuple)):
            n = len(s)
            axes = axis if isinstance(axis, (list, tuple)) else [axis] * n
            outs = o if isinstance(o, (list, tuple)) else [o] * n
            if len(axes) != n or len(outs) != n or (o is not None and outs is not o):
                raise ValueError('batch_axis / out are not nested like the states')
            return type(s)([walk(*x) for x in zip(s, axes, outs)])
        t = T.as_tensor(s)
        T.require_device(p, t)
        if wants_grad(t):
            raise NotImplementedError('reordering has no gradient: decode under torch.no_grad()')
        if not isinstance(axis, int) or not 0 <= axis < t.dim() or t.shape[axis] != N * K:
            raise ValueError('state {}: axis {} does not hold {} x {} rows'.format(
                tuple(t.shape), axis, N, K))
        if in_place:
            if not t.is_contiguous():
                raise ValueError('in place: the states must be contiguous')
            d = t
        else:
            t = t.contiguous()
            if o is None:
                d = torch.empty_like(t)
            else:
                d = T.as_tensor(o)
                if d.shape != t.shape or d.dtype != t.dtype or not d.is_contiguous():
                    raise ValueError('out {} {} does not fit the state {} {}'.format(
                        tuple(d.shape), d.dtype, tuple(t.shape), t.dtype))
                T.require_device(p, d)
        row = t.stride(axis) * t.element_size() if t.numel() else 0
        outer = t.numel() // (N * K * t.stride(axis)) if row else 0
        flat.extend((t.data_ptr(), d.data_ptr(), outer, row * N * K, row, 1, row, row, 0, 0))
        sources.append(t)      # (a contiguous copy has to live until the launch)
        return T.like_caller(d, s)

    result = walk(states, batch_axis, None if in_place else out)
    if flat:
        # no destination may be read, or written twice
        spans = sorted((flat[i + w], flat[i + 2] * flat[i + 3], w)
                       for i in range(0, len(flat), 10) for w in ((1,) if in_place else (0, 1)))
        end = last = 0
        for at, size, w in spans:
            if size and at < end and (w or last):
                raise ValueError('states and out overlap')
            if at + size > end:
                end, last = at + size, w
        launch_reorder(dev, flat, N, K, p, None)
    for c in caches:
        c.reorder(p)
    return result
