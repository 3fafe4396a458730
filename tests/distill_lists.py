"""Teachers' lists for ops.top_distill whose probabilities, with the rest bucket, add up to more or less than one, and the loss written
out in 64 bits so that autograd can differentiate it."""
import math

import torch

KINDS = ["fits", "rounded", "twice", "lowered lse", "everything, less", "everything, more", "no rest, less", "nothing at all"]


def lists(kind, dtype, V, R=4, K=20, temp=1.3):
    """-> logits [R, V] (dtype), values [R, K], index [R, K], lse [R], temp; on the CPU"""
    gen = torch.Generator().manual_seed(KINDS.index(kind) + 7)
    if kind.startswith("everything") or kind == "nothing at all":
        V = K
    x = (torch.randn(R, V, generator=gen) * 2.5).to(dtype)
    t = x.float() + torch.randn(R, V, generator=gen)
    if kind == "rounded":                                          # a teacher sure of its first token, its list kept in bf16
        t[:, 3] = torch.tensor([16.21, 17.93, 21.94, 19.19])[:R] * temp
    values, index = t.topk(K, 1)
    lse = torch.logsumexp(t.double() / temp, 1).float()
    if kind == "rounded":
        values = values.to(torch.bfloat16)
        values[:, 0] = torch.tensor([16.25, 18.0, 22.0, 19.25])[:R] * temp          # rounded up
    elif kind == "twice":                                          # the likeliest id in two slots: its mass counts twice
        index[:, 7], values[:, 7] = index[:, 0], values[:, 0]
        lse -= 0.2
    elif kind == "lowered lse":
        lse -= 0.9
    elif kind == "everything, less":
        lse += 0.25
    elif kind == "everything, more":
        lse -= 0.25
    elif kind == "no rest, less":                                  # the student rules out all that the list does not name
        rest = torch.ones(R, V, dtype=torch.bool).scatter(1, index, False)
        x[rest] = -math.inf
        lse += 0.3
    elif kind == "nothing at all":                                 # no mass in the list, no token outside it
        lse += 1e4
    return x, values, index, lse, temp


def loss64(z, values, index, lse, temp, tail):
    """-> loss [R], the mass of its terms [R]; z double"""
    V, losses, masses = z.shape[1], [], []
    for r in range(z.shape[0]):
        used = [j for j in range(index.shape[1]) if 0 <= index[r, j] < V and values[r, j] > -math.inf]
        at, t = index[r, used], values[r, used].double() / temp
        logq = torch.log_softmax(z[r] / temp, 0)
        logp = t - (lse[r].double() if tail else torch.logsumexp(t, 0))
        p = logp.exp()
        loss, mass = (p * (logp - logq[at])).sum(), p.sum().item()
        named = torch.zeros(V, dtype=torch.bool)
        named[at] = True
        if tail and mass < 1 and (z[r][~named] > -math.inf).any():
            loss = loss + (1 - mass) * (math.log(1 - mass) - torch.logsumexp(logq[~named], 0))
            mass = 1.0
        losses.append(loss)
        masses.append(mass)
    return torch.stack(losses), torch.tensor(masses, dtype=torch.float64)
