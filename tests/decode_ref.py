"""Plain evaluations of the decoding operators in 64 bits (the choice of a 4-bit code is defined in
32 bits), for tests/test_gpu_decode.py.  On the CPU, with torch; no code of the package."""
import math

import torch

GROUP = 64


def quantise(x):
    """x (..., d) -> (values in float64, scale, minimum per channel): the 4-bit format."""
    x = x.detach().cpu().float()
    vals, scales, mins = [], [], []
    for c in range(0, x.shape[-1], GROUP):
        part = x[..., c:c + GROUP]
        lo, hi = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
        bad = ~torch.isfinite(part).all(-1, keepdim=True)
        s = ((hi - lo) * torch.tensor(1.0 / 15, dtype=torch.float32)).bfloat16().float()
        m = lo.bfloat16().float()
        bad = bad | ~torch.isfinite(s) | ~torch.isfinite(m)
        flat = s < 2.0 ** -126
        s = torch.where(flat, torch.zeros_like(s), s)
        code = torch.round((part - m) / torch.where(flat, torch.ones_like(s), s)).clamp(0, 15)
        code = torch.where(flat | bad, torch.zeros_like(code), code)
        s = torch.where(bad, torch.full_like(s, math.nan), s)
        m = torch.where(bad, torch.full_like(m, math.nan), m)
        vals.append(code.double() * s.double() + m.double())
        scales.append(s.expand_as(part))
        mins.append(m.expand_as(part))
    return torch.cat(vals, -1), torch.cat(scales, -1), torch.cat(mins, -1)


def attention(q, k, v, lengths, share=1, causal=True, edge=None, table=None, mask=None,
              query_length=None, temperature=1.0):
    """q (B, Lq, H, d); k, v (B, T, Hc, d) float64 -> (B, Lq, H, d) float64."""
    q = q.detach().cpu().double()
    B, Lq, H, d = q.shape
    T = k.shape[1]
    out = torch.zeros(B, Lq, H, d, dtype=torch.float64)
    reach = T
    if edge is not None:
        e = edge.detach().cpu().double()
        reach = min(reach, e.shape[-1]) if e.shape[-1] != 1 else reach
        e = torch.broadcast_to(e, (B, H, Lq, e.shape[-1] if e.shape[-1] != 1 else T))
    if mask is not None:
        m = mask.cpu()
        reach = min(reach, m.shape[-1]) if m.shape[-1] != 1 else reach
        m = torch.broadcast_to(m, (B, Lq, m.shape[-1] if m.shape[-1] != 1 else T))
    for b in range(B):
        n = int(lengths[b])
        ql = Lq if query_length is None else max(0, min(Lq, int(query_length[b])))
        for i in range(ql):
            pos = n - ql + i
            end = max(0, min(pos + 1 if causal else n, reach, T))
            if end == 0:
                continue
            for h in range(H):
                s = k[b, :end, h // share] @ q[b, i, h]
                if edge is not None:
                    s = s + e[b, h, i, :end]
                if table is not None:
                    R = table.shape[1]
                    at = (R - 1 - (pos - torch.arange(end))).clamp(0, R - 1)
                    s = s + table[h].detach().cpu().double()[at]
                s = s / temperature
                if mask is not None:
                    s = torch.where(m[b, i, :end] != 0, s, torch.full_like(s, -math.inf))
                if s.max() == -math.inf:
                    continue
                w = torch.exp(s - s.max())
                on = w > 0
                out[b, i, h] = (w[on, None] * v[b, :end, h // share][on]).sum(0) / w.sum()
    return out


def attention_tolerance(q, ks, km, vabs, T, temperature, dtype):
    """How far an evaluation as the kernel's may be from attention(): per element, from the data.
    A score is s (A - 16 Q) + m Q with A = sum q (16 + n), a sum of d products that the matrix core
    adds 32 at a time (d / 32 + 32 roundings at most, each half a step of at most sum|q| 31 s), then
    6 more operations on numbers of that size; with e = its error / temperature a weight is off by
    2 e + 8 half steps relative (exp2, its argument: |score| < 100 adds 100 half steps), and a
    result by twice that of the largest value.  Values add T / 32 + 64 half steps of 31 / 7.5 times
    the largest value; bf16 outputs half a step, and the two bf16 parts of a weight 2^-16."""
    half = 2.0 ** -24
    d = q.shape[-1]
    size = (q.detach().cpu().double().abs().amax(1, keepdim=True).amax(2, keepdim=True) *
            torch.ones(1, 1, 1, d, dtype=torch.float64)).sum(-1).max().item()
    e = (d / 32 + 32 + 6) * half * size * (31 * ks + km) / temperature
    tol = 2 * (2 * e + 108 * half) * vabs + (T / 32 + 64) * half * 5 * vabs
    if dtype == torch.bfloat16:
        tol += (2.0 ** -8 + 2 * 2.0 ** -16) * vabs
    return tol


def select(outputs, scores, finished, eos=None, step=1, alpha=0.0, base=None, temperature=1.0,
           normalize=True):
    x = outputs.detach().cpu().double()
    N, K = scores.shape
    V = x.shape[-1]
    x = x.reshape(N, K, V)
    big = torch.finfo(torch.float32).max
    x = torch.nan_to_num(x, nan=-math.inf, posinf=big, neginf=-math.inf)
    z = x / temperature
    base = K if base is None else base
    before, after = (((base + s) / (base + 1.0)) ** alpha for s in (step - 1, step))
    prev = scores.detach().cpu().double()
    fin = torch.zeros(N, K, dtype=torch.bool) if finished is None else finished.cpu()
    if normalize:      # the maximum first: a log-probability keeps its digits beside huge logits
        top = z.amax(-1, keepdim=True)
        safe = torch.where(top == -math.inf, torch.zeros_like(top), top)
        total = torch.exp(z - safe).sum(-1, keepdim=True)
        logp = z - safe - torch.log(torch.where(total == 0, torch.ones_like(total), total))
    else:
        logp = z
    live = prev > -1e15
    cand = torch.where(z == -math.inf, z, (prev[..., None] * before + logp) / after)
    cand = torch.where(live[..., None], cand, torch.full_like(cand, -math.inf))
    out = []
    for n in range(N):
        rows = []
        for k in range(K):
            if not fin[n, k]:
                best = torch.sort(cand[n, k], descending=True, stable=True)
                rows += [(-s.item(), k * V + i.item()) for s, i in
                         zip(best.values[:K], best.indices[:K])]
            else:
                rows.append((-prev[n, k].item() if live[n, k] else math.inf, K * V + k))
        rows.sort()
        out.append(rows[:K])
    s = torch.tensor([[-r[0] for r in rows] for rows in out], dtype=torch.float64)
    at = torch.tensor([[r[1] for r in rows] for rows in out])
    was = at >= K * V
    parents = torch.where(was, at - K * V, at // V)
    tokens = torch.where(was, torch.full_like(at, -1), at % V)
    done = was | (tokens == eos if eos is not None else torch.zeros_like(was))
    return s, parents, tokens, done
