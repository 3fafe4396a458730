"""Plain 64-bit statements (CPU, one row at a time) of ops.top_logits, ops.top_distill and ops.verify_draft."""
import math

import torch


def _rows(t):
    return t.detach().cpu().double().reshape(-1, t.shape[-1])


def top(logits, k, temp):
    """-> index [R, k], lse [R]"""
    index, lse = [], []
    for x in _rows(logits):
        index.append(torch.sort(x, descending=True, stable=True).indices[:k])     # NaN first, equal ones in their order
        lse.append(torch.logsumexp(x / temp, 0))
    return torch.stack(index), torch.stack(lse)


def distill(logits, values, index, lse, temp, tail, g):
    """-> loss [R], gradient [R, V], a scale for the gradient's error [R, V] (the sum of the magnitudes it is a difference of)"""
    x, t = _rows(logits), _rows(values)
    index, g = index.cpu().reshape(-1, index.shape[-1]), g.detach().cpu().double().reshape(-1)
    V = x.shape[1]
    losses, grads, scales = [], [], []
    for r in range(x.shape[0]):
        slots = [j for j in range(index.shape[1]) if 0 <= index[r, j] < V and t[r, j] != -math.inf]
        if not slots:
            losses.append(torch.zeros((), dtype=torch.float64)); grads.append(torch.zeros(V, dtype=torch.float64)); scales.append(torch.zeros(V, dtype=torch.float64))
            continue
        at, tj = index[r, slots], (t[r, slots] - (0 if tail else t[r, slots].max())) / temp
        c = lse.cpu().double().reshape(-1)[r] if tail else torch.logsumexp(tj, 0)
        p = (tj - c).exp()
        z = (x[r] - x[r].max()) / temp                        # +inf or nothing but -inf: NaN, as for a NaN
        logq = z - z.exp().sum().log()
        q = logq.exp()
        loss = torch.where(p != 0, p * ((tj - c) - logq[at]), 0.0).sum()
        rest = torch.ones(V, dtype=torch.bool)
        rest[at] = False
        mass, bucket = p.sum(), 0.0                           # of all the terms of the loss; what the rest bucket takes from q
        if tail:
            pr, log_qr = max(0.0, 1.0 - p.sum().item()), torch.logsumexp(logq[rest], 0) if rest.any() else torch.tensor(-math.inf).double()
            if pr > 0 and log_qr > -math.inf:
                loss = loss + pr * (math.log(pr) - log_qr)
                mass = mass + pr
                bucket = pr * (logq[rest] - log_qr).exp()
        dz, size = mass * q, mass * q                         # log q_v = z_v - logsumexp(z), in every term: q_v times their mass
        dz[rest] -= bucket
        size[rest] += bucket
        for j, v in enumerate(at.tolist()):
            dz[v] -= p[j]
            size[v] += p[j]
        losses.append(loss)
        grads.append(dz * g[r] / temp if g[r] != 0 else torch.zeros(V, dtype=torch.float64))
        scales.append(size * g[r].abs() / temp)
    return torch.stack(losses), torch.stack(grads), torch.stack(scales)


def _probs(x, temp):
    """softmax, or None where the row has no distribution"""
    z = x.detach().cpu().double() / temp
    if torch.isnan(z).any() or (z == math.inf).any() or (z == -math.inf).all():
        return None
    return torch.softmax(z, 0)


def verify(target, tokens, u, E, draft, lengths, temp):
    B, N, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    out, accepted = torch.full((B, N + 1), -1), torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        n = N if lengths is None else min(N, max(0, int(lengths[b])))
        i, q = 0, None
        while i < n:
            d = int(tokens[b, i])
            p = _probs(target[b, i], temp)
            if draft is None:
                q = torch.zeros(V, dtype=torch.float64)
                if 0 <= d < V:
                    q[d] = 1
            else:
                q = _probs(draft[b, i], temp)
                q = torch.zeros(V, dtype=torch.float64) if q is None else q
            if p is None or not 0 <= d < V or not q[d] > 0 or not float(u[b, i]) * q[d] < p[d]:
                break
            out[b, i] = d
            i, q = i + 1, None
        accepted[b] = i
        p = _probs(target[b, i], temp)
        if p is None:
            continue
        w = p if q is None else (p - q).clamp(min=0)
        if not (w > 0).any():
            w = p
        score = torch.where(w > 0, w / E[b].detach().cpu().double(), 0.0)
        out[b, i] = int((score == score.max()).nonzero()[0])
    return out, accepted
