"""The vocabulary-row operators of distillation and draft verification, with real sizes and their plain forms.

  top      the k largest logits of every row, their token ids and the row's log-sum-exp: what a teacher hands over
  distill  a student's loss against a teacher's top logits, forward and backward (one training pass: loss and gradient)
  verify   drafted tokens against a target's probabilities, from given random numbers (speculative sampling)

`own` False: every operator from elementary torch operations.  `own` True: nast_amd's kernels."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # a teacher at decode time: a handful of sentences, latency only
        dict(name="top_8x32000_f32_k16", op="top", rows=8, vocab=32000, k=16, dtype="f32", temp=1.0, masked=0),
        # the generator's own shape (512 sentences of 32 tokens, 9600 words) as a teacher over a whole batch
        dict(name="top_16384x9600_f32_k32", op="top", rows=16384, vocab=9600, k=32, dtype="f32", temp=2.0, masked=0),
        # an odd vocabulary: rows start at every alignment
        dict(name="top_1021x50021_f16_k100", op="top", rows=1021, vocab=50021, k=100, dtype="f16", temp=1.0, masked=21),
        # a large teacher that writes its top logits for a training set
        dict(name="top_2048x131072_bf16_k64", op="top", rows=2048, vocab=131072, k=64, dtype="bf16", temp=1.0, masked=72),
        # a student's step on one small batch
        dict(name="distill_33x9600_f32_k8", op="distill", rows=33, vocab=9600, k=8, dtype="f32", temp=1.0, tail=False, ragged=False, masked=0),
        # the generator's own shape as a student, teacher mass outside the list in a bucket of its own
        dict(name="distill_16384x9600_f32_k32_tail", op="distill", rows=16384, vocab=9600, k=32, dtype="f32", temp=2.0, tail=True,
             ragged=False, masked=0),
        # an odd vocabulary, lists of unequal length (a teacher that kept a nucleus), some rows without a list
        dict(name="distill_1021x50021_f16_k20_ragged", op="distill", rows=1021, vocab=50021, k=20, dtype="f16", temp=1.0, tail=True,
             ragged=True, masked=21),
        # a large student's step
        dict(name="distill_4096x131072_bf16_k64", op="distill", rows=4096, vocab=131072, k=64, dtype="bf16", temp=1.0, tail=False,
             ragged=False, masked=72),
        # serving one user: latency only
        dict(name="verify_1x4_32000_bf16", op="verify", seqs=1, drafts=4, vocab=32000, dtype="bf16", temp=1.0, noise=0.6, greedy=False,
             ragged=False, cut=0.0),
        # the generator's output as a draft: its most likely word at every one of 32 positions, no probabilities with it
        dict(name="verify_128x32_9600_f32_greedy", op="verify", seqs=128, drafts=32, vocab=9600, dtype="f32", temp=0.7, noise=0.6,
             greedy=True, ragged=True, cut=0.0),
        # serving a middling batch, improbable words cut off on both sides
        dict(name="verify_48x5_50021_f16", op="verify", seqs=48, drafts=5, vocab=50021, dtype="f16", temp=0.8, noise=0.6, greedy=False,
             ragged=True, cut=8.0),
        # serving a full batch of a large vocabulary
        dict(name="verify_256x8_131072_bf16", op="verify", seqs=256, drafts=8, vocab=131072, dtype="bf16", temp=1.0, noise=0.6,
             greedy=False, ragged=False, cut=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["top", "distill", "verify"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    vocab = _log_int(rng, 1000, 200000)
    temp = round(rng.uniform(0.5, 3.0), 2)
    if op == "verify":
        drafts = rng.randint(1, 32)
        most = min(512, (1 << 30) // (2 * (drafts + 1) * vocab * SIZE[dtype]))
        return dict(op=op, seqs=_log_int(rng, 1, max(1, most)), drafts=drafts, vocab=vocab, dtype=dtype, temp=temp,
                    noise=round(rng.uniform(0.2, 1.2), 2), greedy=rng.random() < 0.3, ragged=rng.random() < 0.5,
                    cut=rng.choice([0.0, 0.0, 8.0]))
    most = min(20000, (512 << 20) // (vocab * SIZE[dtype]))
    case = dict(op=op, rows=_log_int(rng, 1, most), vocab=vocab, k=_log_int(rng, 1, 256), dtype=dtype, temp=temp,
                masked=rng.choice([0, 0, rng.randint(1, 200)]))
    if op == "distill":
        case.update(tail=rng.random() < 0.5, ragged=rng.random() < 0.5)
    return case


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _logits(gen, rows, vocab):
    """Language-model-like rows in float32: a word frequency shared by all rows, context on top, a few likely words each."""
    x = torch.randn(rows, vocab, generator=gen, device="cuda").mul_(1.5)
    x += torch.randn(vocab, generator=gen, device="cuda") * 1.5
    quarter = vocab // 4                # one likely word in each quarter: the four of a row differ
    at = torch.randint(0, quarter, (rows, 4), generator=gen, device="cuda") + torch.arange(4, device="cuda") * quarter
    x.scatter_(1, at, torch.rand(rows, 4, generator=gen, device="cuda") * 12.0 + 2.0)
    return x


def _masked(x, n):
    """The last n ids are padding of the vocabulary: no probability (one id at least stays)."""
    if n:
        x[:, max(1, x.shape[1] - n):] = -math.inf
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, vocab = DTYPES[case["dtype"]], case["vocab"]
    state = {"case": case}
    if case["op"] == "top":
        state["logits"] = _masked(_logits(gen, case["rows"], vocab), case["masked"]).to(dtype)
    elif case["op"] == "distill":
        rows, k = case["rows"], case["k"]
        teacher = _masked(_logits(gen, rows, vocab), case["masked"])
        student = _masked(teacher + torch.randn(rows, vocab, generator=gen, device="cuda") * 0.8, case["masked"])
        state["lse"] = torch.logsumexp(teacher / case["temp"], 1)
        state["values"], state["index"] = torch.topk(teacher, k, dim=1)
        del teacher
        if case["ragged"]:              # a list ends where the teacher's ended: -1 in the slots behind
            n = torch.randint(0, k + 1, (rows, 1), generator=gen, device="cuda")
            state["index"] = state["index"].masked_fill(torch.arange(k, device="cuda") >= n, -1)
        state["values"] = state["values"].to(dtype)
        state["logits"] = student.to(dtype).requires_grad_()
        # a mean over the rows; half precision trains with a scaled loss, or small gradients leave its range
        state["grad_loss"] = torch.rand(rows, generator=gen, device="cuda") * (64.0 if case["dtype"] == "f16" else 1.0 / rows)
    else:
        seqs, n, t = case["seqs"], case["drafts"], case["temp"]
        target = _logits(gen, seqs * (n + 1), vocab).view(seqs, n + 1, vocab)
        drafter = target[:, :n] + torch.randn(seqs, n, vocab, generator=gen, device="cuda") * case["noise"]
        if case["cut"]:
            target.masked_fill_(target < target.amax(-1, keepdim=True) - case["cut"], -math.inf)
            drafter.masked_fill_(drafter < drafter.amax(-1, keepdim=True) - case["cut"], -math.inf)
        state["target"], drafter = target.to(dtype), drafter.to(dtype)
        del target
        if case["greedy"]:
            state["tokens"], state["draft"] = drafter.argmax(-1), None
        else:                           # the drafter draws from its own probabilities
            q = (drafter.float() / t).softmax(-1)
            state["tokens"] = q.div_(torch.empty_like(q).exponential_(generator=gen)).argmax(-1)
            state["draft"] = drafter
        state["lengths"] = torch.randint(0, n + 1, (seqs,), generator=gen, device="cuda") if case["ragged"] else None
        state["u"] = torch.rand(seqs, n, generator=gen, device="cuda")
        state["noise"] = torch.empty(seqs, vocab, device="cuda").exponential_(generator=gen)
    return state


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _plain_top(x, k, temp):
    # one integer key per element, ordered by value and then by the lower id, so that no two are equal
    x = x.float() + 0.0
    bits = x.view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -2147483648 - bits - 1, bits)
    key = order * (1 << 31) + ((1 << 31) - 1 - torch.arange(x.shape[1], device=x.device))
    key = torch.topk(key, k, dim=1).values
    index = (1 << 31) - 1 - key.remainder(1 << 31)
    z = x / temp
    m = z.amax(1, keepdim=True)
    m = torch.where(m.isfinite(), m, 0.0)
    lse = (m + (z - m).exp().sum(1, keepdim=True).log()).squeeze(1)
    return x.gather(1, index), index, lse


def _plain_distill(x, values, index, lse_t, temp, tail, g):
    # in 64 bits: the loss is a small difference of sums over the whole vocabulary
    vocab = x.shape[1]
    z = x.detach().double() / temp
    used = (index >= 0) & (index < vocab)
    some = used.any(1)
    at = index.clamp(0, vocab - 1)
    t = torch.where(used, values.double() / temp, -math.inf)
    if not tail:
        top = t.amax(1, keepdim=True)
        top = torch.where(top.isfinite(), top, 0.0)
        lse_t = (top + (t - top).exp().sum(1, keepdim=True).log()).squeeze(1)
    logp = t - torch.where(some, lse_t, 0.0).unsqueeze(1)
    p = logp.exp()
    m = z.amax(1, keepdim=True)
    e = (z - m).exp()
    s = e.sum(1, keepdim=True)
    logq = z.gather(1, at) - m - s.log()
    dz = e / s
    loss = torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    if tail:
        inside = torch.zeros_like(z).scatter_add_(1, at, used.double()) > 0
        p_rest = (1.0 - p.sum(1, keepdim=True)).clamp(min=0.0)
        q_rest = torch.where(inside, 0.0, e).sum(1, keepdim=True) / s
        loss = loss + torch.where(p_rest > 0, p_rest * (p_rest.log() - q_rest.log()), 0.0).squeeze(1)
        ratio = torch.where(q_rest > 0, p_rest / q_rest, 0.0)
        dz = torch.where(inside, dz, dz * (1.0 - ratio))
    dz = dz.scatter_add_(1, at, torch.where(used, -p, 0.0)) * (g / temp).unsqueeze(1)
    return torch.where(some, loss, 0.0).float(), torch.where(some.unsqueeze(1), dz, 0.0).to(x.dtype)


def _log_probs(x, temp):
    z = x.double() / temp
    m = z.amax(-1, keepdim=True)
    return z.sub_(m).sub_(z.exp().sum(-1, keepdim=True).log())


def _plain_verify(target, tokens, u, noise, draft, lengths, temp):
    # in 64 bits: an accepted token hangs on which side of a border a number falls
    seqs, n, vocab = target.shape[0], target.shape[1] - 1, target.shape[2]
    logp = _log_probs(target, temp)
    at = tokens.unsqueeze(-1)
    lp = logp[:, :n].gather(2, at).squeeze(2)
    if draft is None:
        lq = torch.zeros_like(lp)
    else:
        logq = _log_probs(draft, temp)
        lq = logq.gather(2, at).squeeze(2)
    ok = (u.double() < (lp - lq).exp()) & (lq > -math.inf)
    place = torch.arange(n, device=target.device)
    length = torch.full((seqs,), n, device=target.device) if lengths is None else lengths
    ok &= place < length.unsqueeze(1)
    accepted = ok.long().cumprod(1).sum(1)
    row = torch.arange(seqs, device=target.device)
    p = logp[row, accepted].exp()
    at_draft = accepted.clamp(max=max(n - 1, 0))
    if draft is None:
        q = torch.zeros_like(p).scatter_(1, tokens[row, at_draft].unsqueeze(1), 1.0)
    else:
        q = logq[row, at_draft].exp()
    rest = (p - torch.where((accepted < length).unsqueeze(1), q, 0.0)).clamp(min=0.0)
    rest = torch.where(rest.amax(1, keepdim=True) > 0, rest, p)
    score = rest / noise.double()
    best = score.amax(1, keepdim=True)
    ids = torch.arange(vocab, device=target.device)
    new = torch.where(score == best, ids, vocab).amin(1)
    out = torch.where(place < accepted.unsqueeze(1), tokens, -1)
    out = torch.cat((out, torch.full((seqs, 1), -1, device=out.device)), 1)
    return out.scatter(1, accepted.unsqueeze(1), new.unsqueeze(1)), accepted


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "top":
        x, k = state["logits"], case["k"]
        if own:
            from nast_amd import ops
            top = ops.top_logits(x, k, case["temp"])
            return {"values": top.values, "index": top.index, "lse": top.lse}
        values, index, lse = _plain_top(x, k, case["temp"])
        return {"values": values.to(x.dtype), "index": index, "lse": lse}
    if case["op"] == "distill":
        x, g, lse = state["logits"], state["grad_loss"], state["lse"] if case["tail"] else None
        if own:
            from nast_amd import ops
            top = ops.TopLogits(state["values"], state["index"], lse, case["temp"])
            loss = ops.top_distill(x, top, case["temp"], tail=case["tail"])
            return {"loss": loss.detach(), "grad": torch.autograd.grad(loss, x, g)[0]}
        loss, grad = _plain_distill(x, state["values"], state["index"], lse, case["temp"], case["tail"], g)
        return {"loss": loss, "grad": grad}
    arguments = state["target"], state["tokens"], state["u"], state["noise"], state["draft"], state["lengths"], case["temp"]
    if own:
        from nast_amd import ops
        tokens, accepted = ops.verify_draft(*arguments)
    else:
        tokens, accepted = _plain_verify(*arguments)
    return {"tokens": tokens, "accepted": accepted}


def work(case):
    vocab, size = case["vocab"], SIZE[case["dtype"]]
    if case["op"] == "top":
        # every logit once; an exponential and a comparison each
        return {"bytes": case["rows"] * (vocab * size + case["k"] * (size + 8) + 4), "flops": 4.0 * case["rows"] * vocab}
    if case["op"] == "distill":
        # the logits and the list read once, the gradient written once
        return {"bytes": case["rows"] * (2 * vocab * size + case["k"] * (size + 8) + 12), "flops": 8.0 * case["rows"] * vocab}
    # the rows behind a rejected token need not be read.  A draft drawn from logits that are `noise` away is accepted with probability
    # erfc(noise / temp / sqrt(8)); the most likely word of such rows with about 0.6
    a = 0.6 if case["greedy"] else math.erfc(case["noise"] / case["temp"] / math.sqrt(8.0))
    lengths = range(case["drafts"] + 1) if case["ragged"] else [case["drafts"]]
    target = sum(sum(a ** i for i in range(n + 1)) for n in lengths) / len(lengths)
    draft = 0.0 if case["greedy"] else sum(sum(a ** i for i in range(n)) for n in lengths) / len(lengths)
    return {"bytes": case["seqs"] * vocab * ((target + draft) * size + 4.0), "flops": case["seqs"] * vocab * (4.0 * (target + draft) + 4.0)}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_distill(state):
    """By blocks of rows: probabilities of student and teacher over the whole vocabulary, differences of their logarithms."""
    case, x = state["case"], state["logits"].detach()
    losses, grads = [], []
    step = max(1, (1 << 27) // case["vocab"])
    for r in range(0, case["rows"], step):
        index, t = state["index"][r:r + step], state["values"][r:r + step].double() / case["temp"]
        z = (x[r:r + step].double() / case["temp"]).requires_grad_()
        good = (index >= 0) & (index < case["vocab"])
        logq = torch.log_softmax(z, 1)
        t = torch.where(good, t, torch.full_like(t, -math.inf))
        empty = ~good.any(1)
        if case["tail"]:
            p = (t - state["lse"][r:r + step].double().unsqueeze(1)).exp()
        else:
            p = torch.softmax(torch.where(empty.unsqueeze(1), torch.zeros_like(t), t), 1) * good
        loss = (torch.xlogy(p, p) - torch.where(p > 0, p * logq.gather(1, index.clamp(0, case["vocab"] - 1)), 0.0)).sum(1)
        if case["tail"]:
            rest = (1.0 - p.sum(1)).clamp(min=0.0)
            mask = torch.zeros_like(logq, dtype=torch.bool)
            row = torch.arange(index.shape[0], device=x.device).unsqueeze(1).expand_as(index)
            mask[row[good], index[good]] = True
            log_rest = torch.logsumexp(logq.masked_fill(mask, -math.inf), 1)
            loss = loss + torch.where(rest > 0, torch.xlogy(rest, rest) - rest * log_rest, 0.0)
        loss = torch.where(empty, 0.0, loss)
        # d loss / d logits = d loss / d z / temp
        (grad,) = torch.autograd.grad((loss * state["grad_loss"][r:r + step].double()).sum(), z)
        losses.append(loss.detach())
        grads.append(grad / case["temp"])
    return {"loss": torch.cat(losses), "grad": torch.cat(grads)}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "verify":
        return None                     # whole numbers only
    if case["op"] == "distill":
        return _exact_distill(state)
    x, k = state["logits"], case["k"]
    lse, values = [], []
    step = max(1, (1 << 27) // case["vocab"])
    for r in range(0, case["rows"], step):
        z = x[r:r + step].double()
        lse.append(torch.logsumexp(z / case["temp"], 1))
        values.append(torch.sort(z, 1, descending=True).values[:, :k])
    return {"values": torch.cat(values), "index": None, "lse": torch.cat(lse)}
