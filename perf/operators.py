"""Losses over vocabulary logits, forward and backward: what is measured, and their plain forms.

Four operators of training and scoring a language model from its logits [rows, vocab]:

  token_logprobs     log-probability of one given token a row (and its gradient)
  policy_loss        clipped policy loss with a KL term to a reference and an entropy bonus
  preference_loss    logistic loss of paired log ratios over packed sequences
  distillation_loss  KL divergence from a teacher's top logits

A case's "op" names the operator.  ``run`` takes one pass through it: the plain form in elementary torch
operations, or, where ``own`` is true, the calls a user makes of kdn_b200.
"""

import math
import os
import sys

import torch

own = False

IGNORE = -100
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # scoring the one token that a decode step has just produced: latency alone
        dict(name="logprobs-one-token", op="token_logprobs", grad=False, rows=1, vocab=32000, dtype="bf16",
             layout="packed", index="int64", masked=0, temperature=1.0),
        # the reference policy's scores of a packed batch of prompts and answers (prompts masked)
        dict(name="logprobs-batch", op="token_logprobs", grad=False, rows=8192, vocab=32000, dtype="bf16",
             layout="packed", index="int64", masked=1024, temperature=1.0),
        # a training step on fp32 logits of an odd vocabulary, rows that start at no 16-byte boundary
        dict(name="logprobs-train-odd", op="token_logprobs", grad=True, rows=1999, vocab=50021, dtype="fp32",
             layout="packed", index="int32", masked=100, temperature=0.7),
        # a policy step on a handful of tokens
        dict(name="policy-few", op="policy_loss", rows=32, vocab=32000, dtype="bf16", layout="packed",
             index="int64", masked=4, temperature=1.0, weights=False, reference=True, kl=0.05, entropy=0.0),
        # an ordinary micro-batch of a policy update
        dict(name="policy-batch", op="policy_loss", rows=4096, vocab=32000, dtype="bf16", layout="packed",
             index="int64", masked=512, temperature=1.0, weights=True, reference=True, kl=0.05, entropy=0.0),
        # the largest: a long micro-batch over a large vocabulary, with an entropy bonus
        dict(name="policy-largest", op="policy_loss", rows=8192, vocab=131072, dtype="bf16", layout="packed",
             index="int64", masked=1024, temperature=0.9, weights=True, reference=True, kl=0.02, entropy=0.01),
        # two short pairs
        dict(name="preference-few", op="preference_loss", rows=96, vocab=32000, dtype="bf16", layout="packed",
             index="int64", masked=16, temperature=1.0, pairs=2, reference=True, average=False, beta=0.1,
             smoothing=0.0),
        # an ordinary micro-batch of pairs
        dict(name="preference-batch", op="preference_loss", rows=8192, vocab=32000, dtype="bf16",
             layout="packed", index="int64", masked=2048, temperature=1.0, pairs=16, reference=True, average=False,
             beta=0.1, smoothing=0.0),
        # without a reference, by the mean over a sequence's tokens; fp32 logits of an odd vocabulary whose rows
        # the projection has padded to 16 bytes
        dict(name="preference-odd", op="preference_loss", rows=1531, vocab=20011, dtype="fp32", layout="padded",
             index="int32", masked=200, temperature=1.0, pairs=5, reference=False, average=True, beta=2.0,
             smoothing=0.1),
        # distilling a few tokens
        dict(name="distill-few", op="distillation_loss", rows=16, vocab=32000, dtype="bf16", layout="packed",
             index="int64", masked=0, temperature=1.0, top=32, tail=False, weights=False),
        # an ordinary micro-batch, softened logits, the teacher renormalised over its top entries
        dict(name="distill-batch", op="distillation_loss", rows=4096, vocab=32000, dtype="bf16", layout="packed",
             index="int64", masked=256, temperature=2.0, top=64, tail=False, weights=True),
        # fp32 logits over a large vocabulary, the rest of the teacher's mass as one more class
        dict(name="distill-tail-large", op="distillation_loss", rows=4096, vocab=131072, dtype="fp32",
             layout="packed", index="int32", masked=256, temperature=1.0, top=128, tail=True, weights=True),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["token_logprobs", "policy_loss", "preference_loss", "distillation_loss"])
    dtype = rng.choice(["bf16", "fp32"])
    vocab = spread(200, 131072)
    if rng.random() < 0.4:
        vocab = max(200, vocab // 64 * 64)
    most = (1 << 29) if dtype == "bf16" else (1 << 28)
    rows = spread(1, max(1, min(16384, most // vocab)))
    case = dict(op=op, rows=rows, vocab=vocab, dtype=dtype, layout=rng.choice(["packed", "packed", "padded"]),
                index=rng.choice(["int64", "int32"]), masked=int(rows * rng.choice([0.0, 0.0, 0.1, 0.5])),
                temperature=rng.choice([1.0, 1.0, 0.7, 2.0]))
    if op == "token_logprobs":
        case.update(grad=rng.random() < 0.5)
    elif op == "policy_loss":
        case.update(weights=rng.random() < 0.5, reference=rng.random() < 0.7, kl=rng.choice([0.02, 0.1]),
                    entropy=rng.choice([0.0, 0.0, 0.01]))
        if not case["reference"]:
            case["kl"] = 0.0
    elif op == "preference_loss":
        least = -(-rows // 512)
        case.update(pairs=spread(least, max(least, min(64, rows))), reference=rng.random() < 0.7,
                    smoothing=rng.choice([0.0, 0.1]))
        case.update(average=not case["reference"], beta=rng.choice([0.1, 0.3] if case["reference"] else [1.0, 2.0]))
    else:
        case.update(top=spread(1, 256), tail=rng.random() < 0.5, weights=rng.random() < 0.5)
        case["top"] = min(case["top"], vocab // 2)
    return case


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    n, V, op, T = case["rows"], case["vocab"], case["op"], case["temperature"]
    dtype = _DTYPES[case["dtype"]]
    index = torch.int64 if case["index"] == "int64" else torch.int32
    dev = "cuda"

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    # logits as a language model's head leaves them: a broad bulk, and a few tokens that stand out of it
    per16 = 16 // torch.empty((), dtype=dtype).element_size()
    width = -(-V // per16) * per16 if case["layout"] == "padded" else V
    logits = torch.randn(n, width, generator=g, device=dev, dtype=dtype).mul_(2.0)[:, :V]
    state = dict(case, logits=logits)

    order = torch.argsort(rand(n))
    ignored = torch.zeros(n, dtype=torch.bool, device=dev)
    ignored[order[:case["masked"]]] = True
    live = max(1, n - case["masked"])

    if op == "distillation_loss":
        K = case["top"]
        lo = torch.arange(K, device=dev) * V // K
        hi = torch.arange(1, K + 1, device=dev) * V // K
        ids = lo + torch.floor(rand(n, K) * (hi - lo)).long().clamp_(max=V)
        ids = torch.minimum(ids, hi - 1)
        ids = torch.gather(ids, 1, torch.argsort(rand(n, K), dim=1))  # distinct, in no order
        teacher = torch.sort(6.0 + 2.5 * randn(n, K), dim=1, descending=True).values
        logits.scatter_(1, ids, (teacher + randn(n, K)).to(dtype))
        state["teacher_logits"] = teacher
        state["teacher_ids"] = torch.where(ignored[:, None], -1, ids).to(index)
        state["teacher_lse"] = None
        if case["tail"]:  # the top entries hold 70 to 98 of 100 parts of the teacher's mass
            state["teacher_lse"] = _lse(teacher / T) - torch.log(0.7 + 0.28 * rand(n))
        state["weights"] = (0.5 + rand(n)) / live if case["weights"] else None
        return state

    labels = torch.floor(rand(n) * V).long().clamp_(max=V - 1)
    likely = rand(n) < 0.7
    bumped = torch.where(likely, 8.0 + randn(n), 2.0 * randn(n))
    logits[torch.arange(n, device=dev), labels] = bumped.to(dtype)
    state["labels"] = torch.where(ignored, IGNORE, labels).to(index)
    if op == "token_logprobs":
        if case["grad"]:
            state["dlogps"] = randn(n) / live
            logits.requires_grad_()
        return state

    step = max(1, (1 << 26) // V)
    logp = torch.cat([(logits[i:i + step].float() / T).gather(1, labels[i:i + step, None])[:, 0]
                      - _lse(logits[i:i + step].float() / T) for i in range(0, n, step)])
    if op == "policy_loss":
        # the sampling policy is a few updates old: probability ratios around one, some of them clipped.
        # The gradient jumps where a ratio meets the edge of its clip, so none lies nearer to it than 1e-3.
        ratio = torch.exp(0.25 * randn(n))
        for edge in (0.8, 1.2):
            ratio = torch.where((ratio - edge).abs() < 1e-3, torch.full_like(ratio, edge + 2e-3), ratio)
        state["old_logps"] = logp - torch.log(ratio)
        state["advantages"] = 0.5 + randn(n)
        state["ref_logps"] = logp + 0.3 * randn(n) if case["reference"] else None
        state["weights"] = (0.5 + rand(n)) / live if case["weights"] else None
    else:
        cuts = torch.sort(torch.floor(rand(2 * case["pairs"] - 1) * (n + 1)).long().clamp_(max=n)).values
        state["cu_seqlens"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), n)])
        state["ref_logps"] = logp + 0.2 * randn(n) if case["reference"] else None
    return state


def _lse(x):
    m = x.amax(-1)
    return m + torch.log(torch.exp(x - m[..., None]).sum(-1))


# ------------------------------------------------------------------------------------------------- a pass
def _kdn():
    if "kdn_b200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "kernel-deltanet_b200"))
        import kdn_b200  # noqa: F401
    return sys.modules["kdn_b200"]


def run(s):
    if own:
        return _OWN[s["op"]](_kdn(), s)
    with torch.no_grad():
        return _PLAIN[s["op"]](s)


def _own_token_logprobs(kdn, s):
    logps = kdn.token_logprobs(s["logits"], s["labels"], temperature=s["temperature"], ignore_index=IGNORE)
    if not s["grad"]:
        return {"logps": logps}
    (dlogits,) = torch.autograd.grad(logps, s["logits"], s["dlogps"])
    return {"logps": logps, "dlogits": dlogits}


def _own_policy_loss(kdn, s):
    loss, logps, entropy, dlogits = kdn.policy_loss_and_grad(
        s["logits"], s["labels"], s["old_logps"], s["advantages"], ref_logps=s["ref_logps"], weights=s["weights"],
        clip_low=0.2, clip_high=0.2, kl_coef=s["kl"], entropy_coef=s["entropy"], temperature=s["temperature"],
        ignore_index=IGNORE)
    return {"loss": loss, "logps": logps, "entropy": entropy, "dlogits": dlogits}


def _own_preference_loss(kdn, s):
    loss, log_ratios, logps, dlogits = kdn.preference_loss_and_grad(
        s["logits"], s["labels"], s["cu_seqlens"], ref_logps=s["ref_logps"], beta=s["beta"],
        label_smoothing=s["smoothing"], length_normalised=s["average"], temperature=s["temperature"],
        ignore_index=IGNORE)
    return {"loss": loss, "log_ratios": log_ratios, "logps": logps, "dlogits": dlogits}


def _own_distillation_loss(kdn, s):
    loss, divergence, dlogits = kdn.distillation_loss_and_grad(
        s["logits"], s["teacher_logits"], s["teacher_ids"], teacher_lse=s["teacher_lse"], weights=s["weights"],
        temperature=s["temperature"])
    return {"loss": loss, "divergence": divergence, "dlogits": dlogits}


_OWN = {"token_logprobs": _own_token_logprobs, "policy_loss": _own_policy_loss,
        "preference_loss": _own_preference_loss, "distillation_loss": _own_distillation_loss}


# The plain forms.  x = logits / T, lse = log sum exp x, log q = x - lse; a row whose label is IGNORE (or whose
# first teacher id is negative) counts for nothing and has a zero gradient.
def _stats(s):
    x = s["logits"].float() / s["temperature"]
    lse = _lse(x)
    y = s["labels"].long()
    live = y != IGNORE
    y = torch.where(live, y, 0)
    logps = torch.where(live, x.gather(1, y[:, None])[:, 0] - lse, 0.0)
    return x, lse, y, live, logps


def _through_logps(s, x, lse, y, live, dlogps):
    """d/dlogits of sum_t dlogps_t logp_t: dlogps_t (1[j = y_t] - q_tj) / T."""
    c = torch.where(live, dlogps, 0.0) / s["temperature"]
    d = torch.exp(x - lse[:, None]) * -c[:, None]
    d.scatter_add_(1, y[:, None], c[:, None])
    return torch.where(live[:, None], d, 0.0)


def _plain_token_logprobs(s):
    x, lse, y, live, logps = _stats(s)
    if not s["grad"]:
        return {"logps": logps}
    return {"logps": logps, "dlogits": _through_logps(s, x, lse, y, live, s["dlogps"]).to(s["logits"].dtype)}


def _plain_policy_loss(s):
    x, lse, y, live, logps = _stats(s)
    logq = x - lse[:, None]
    q = torch.exp(logq)
    entropy = torch.where(live, -(q * logq).sum(-1), 0.0)
    w = s["weights"] if s["weights"] is not None else 1.0 / live.sum().clamp(min=1)
    w = torch.where(live, w, 0.0)
    a, ratio = s["advantages"], torch.exp(logps - s["old_logps"])
    clipped = torch.clamp(ratio, 0.8, 1.2)
    free = ratio * a <= clipped * a
    term = -torch.where(free, ratio * a, clipped * a) - s["entropy"] * entropy
    slope = -torch.where(free, ratio * a, 0.0)
    if s["ref_logps"] is not None:
        gap = s["ref_logps"] - logps
        term = term + s["kl"] * (torch.expm1(gap) - gap)
        slope = slope - s["kl"] * torch.expm1(gap)
    loss = torch.where(live, w * term, 0.0).sum()
    d = _through_logps(s, x, lse, y, live, w * slope)
    if s["entropy"]:
        c = w * s["entropy"] / s["temperature"]
        d = d + torch.where(live[:, None], q * (logq + entropy[:, None]), 0.0) * c[:, None]
    return {"loss": loss, "logps": logps, "entropy": entropy, "dlogits": d.to(s["logits"].dtype)}


def _plain_preference_loss(s):
    x, lse, y, live, logps = _stats(s)
    cu, at = s["cu_seqlens"], torch.arange(x.shape[0], device=x.device)
    gap = logps - torch.where(live, s["ref_logps"], 0.0) if s["ref_logps"] is not None else logps
    member = ((at >= cu[:-1, None]) & (at < cu[1:, None])).float()
    size = (member * live).sum(-1).clamp(min=1.0) if s["average"] else torch.ones_like(cu[1:], dtype=torch.float32)
    log_ratios = (member * gap).sum(-1) / size
    h = s["beta"] * (log_ratios[0::2] - log_ratios[1::2])
    eps, pairs = s["smoothing"], s["pairs"]

    def log_sigmoid(v):
        return torch.clamp(v, max=0.0) - torch.log1p(torch.exp(-v.abs()))

    loss = -((1 - eps) * log_sigmoid(h) + eps * log_sigmoid(-h)).sum() / pairs
    dh = (torch.exp(log_sigmoid(h)) - (1 - eps)) * s["beta"] / pairs
    dlogps = (member * (torch.stack([dh, -dh], 1).reshape(-1) / size)[:, None]).sum(0)
    return {"loss": loss, "log_ratios": log_ratios, "logps": logps,
            "dlogits": _through_logps(s, x, lse, y, live, dlogps).to(s["logits"].dtype)}


def _plain_distillation_loss(s):
    T = s["temperature"]
    x = s["logits"].float() / T
    ids = s["teacher_ids"].long()
    live = ids[:, 0] >= 0
    ids = ids.clamp(min=0)
    t = s["teacher_logits"].float() / T
    w = s["weights"] if s["weights"] is not None else (1.0 / live.sum().clamp(min=1)).expand(live.shape)
    w = torch.where(live, w, 0.0)
    logp = t - (_lse(t) if s["teacher_lse"] is None else s["teacher_lse"])[:, None]
    p = torch.exp(logp)
    lse = _lse(x)
    q = torch.exp(x - lse[:, None])
    logq_top = x.gather(1, ids) - lse[:, None]
    divergence = (p * (logp - logq_top)).sum(-1)
    if s["teacher_lse"] is None:
        d = q.scatter_add(1, ids, -p)
    else:
        p_rest = torch.clamp(1.0 - p.sum(-1), min=0.0)
        rest = torch.exp(x - lse[:, None]).scatter(1, ids, 0.0)
        q_rest = rest.sum(-1)
        divergence = divergence + p_rest * torch.log(p_rest / q_rest)
        d = q.scatter_add(1, ids, -p) - rest * (p_rest / q_rest)[:, None]
    divergence = torch.where(live, divergence, 0.0)
    d = torch.where(live[:, None], d * (w * T)[:, None], 0.0)
    return {"loss": T * T * (w * divergence).sum(), "divergence": divergence, "dlogits": d.to(s["logits"].dtype)}


_PLAIN = {"token_logprobs": _plain_token_logprobs, "policy_loss": _plain_policy_loss,
          "preference_loss": _plain_preference_loss, "distillation_loss": _plain_distillation_loss}


# ------------------------------------------------------------------------------------------------- floors
def work(case):
    """Live rows are read once; every row of the gradient is written once.  Per element: scale and exponent,
    sum, and for the gradient exponent and product again."""
    n, V, live = case["rows"], case["vocab"], case["rows"] - case["masked"]
    size, idx = (2 if case["dtype"] == "bf16" else 4), (8 if case["index"] == "int64" else 4)
    grad = case.get("grad", True)
    per_row = 4 + idx + (4 if grad else 0)
    if case["op"] == "policy_loss":
        per_row = idx + 16 + 4 * bool(case["weights"]) + 4 * bool(case["reference"])
    elif case["op"] == "preference_loss":
        per_row = idx + 4 + 4 * bool(case["reference"])
    elif case["op"] == "distillation_loss":
        per_row = case["top"] * (4 + idx) + 4 + 4 * bool(case["tail"]) + 4 * bool(case["weights"])
    return {"bytes": live * V * size + (n * V * size if grad else 0) + n * per_row,
            "flops": live * V * (4 + (4 if grad else 0))}


# ------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time; gradients by differentiating them."""
    s = prepare(case, seed)
    n, V, T, op = case["rows"], case["vocab"], case["temperature"], case["op"]
    logits = s["logits"].detach()
    step = max(1, (1 << 27) // V)
    blocks = [slice(i, min(n, i + step)) for i in range(0, n, step)]
    d = torch.empty(n, V, dtype=torch.float64, device="cuda") if case.get("grad", True) else None

    def wide(name, b):
        return s[name][b].double() if s.get(name) is not None else None

    def log_q(b):
        z = logits[b].double().requires_grad_()
        return z, torch.log_softmax(z / T, dim=-1)

    def picked(lq, b):
        y = s["labels"][b].long()
        return torch.where(y == IGNORE, 0.0, lq.gather(1, y.clamp(min=0)[:, None])[:, 0])

    if op == "distillation_loss":
        live = s["teacher_ids"][:, 0] >= 0
        share = wide("weights", slice(None)) if s["weights"] is not None else 1.0 / live.double().sum().clamp(min=1)
        share = torch.where(live, share, 0.0)
        found, total = [], 0.0
        for b in blocks:
            z, lq = log_q(b)
            at = s["teacher_ids"][b].long().clamp(min=0)
            t = wide("teacher_logits", b) / T
            if s["teacher_lse"] is None:
                lp = torch.log_softmax(t, dim=-1)
                kl = (lp.exp() * (lp - lq.gather(1, at))).sum(-1)
            else:
                lp = t - wide("teacher_lse", b)[:, None]
                rest = torch.clamp(1.0 - lp.exp().sum(-1), min=0.0)
                lq_rest = torch.logsumexp(lq.scatter(1, at, float("-inf")), dim=-1)
                kl = (lp.exp() * (lp - lq.gather(1, at))).sum(-1) + torch.xlogy(rest, rest) - rest * lq_rest
            kl = torch.where(live[b], kl, 0.0)
            loss = T * T * (share[b] * kl).sum()
            (d[b],) = torch.autograd.grad(loss, z)
            found.append(kl.detach())
            total = total + loss.detach()
        return {"loss": total, "divergence": torch.cat(found), "dlogits": d}

    if op == "token_logprobs":
        found = []
        for b in blocks:
            z, lq = log_q(b)
            lp = picked(lq, b)
            if d is not None:
                (d[b],) = torch.autograd.grad(lp, z, wide("dlogps", b))
            found.append(lp.detach())
        return {"logps": torch.cat(found)} if d is None else {"logps": torch.cat(found), "dlogits": d}

    live = s["labels"] != IGNORE
    if op == "policy_loss":
        share = wide("weights", slice(None)) if s["weights"] is not None else 1.0 / live.double().sum().clamp(min=1)
        share = torch.where(live, share, 0.0)
        found, spread, total = [], [], 0.0
        for b in blocks:
            z, lq = log_q(b)
            lp = picked(lq, b)
            h = torch.where(live[b], torch.special.entr(lq.exp()).sum(-1), 0.0)
            r, a = torch.exp(lp - wide("old_logps", b)), wide("advantages", b)
            each = -torch.minimum(r * a, torch.clamp(r, 0.8, 1.2) * a) - case["entropy"] * h
            if s["ref_logps"] is not None:
                u = wide("ref_logps", b) - lp
                each = each + case["kl"] * (torch.exp(u) - u - 1.0)
            loss = torch.where(live[b], share[b] * each, 0.0).sum()
            (d[b],) = torch.autograd.grad(loss, z)
            found.append(lp.detach())
            spread.append(h.detach())
            total = total + loss.detach()
        return {"loss": total, "logps": torch.cat(found), "entropy": torch.cat(spread), "dlogits": d}

    found = []
    for b in blocks:
        with torch.no_grad():
            found.append(picked(log_q(b)[1], b))
    lp = torch.cat(found).requires_grad_()
    gap = lp - torch.where(live, wide("ref_logps", slice(None)), 0.0) if s["ref_logps"] is not None else lp
    cu = s["cu_seqlens"].tolist()
    spans = [slice(cu[i], cu[i + 1]) for i in range(2 * case["pairs"])]
    ratios = torch.stack([gap[b].sum() / (live[b].sum().clamp(min=1) if case["average"] else 1) for b in spans])
    h = case["beta"] * (ratios[0::2] - ratios[1::2])
    eps = case["smoothing"]
    ls = torch.nn.functional.logsigmoid
    loss = -((1 - eps) * ls(h) + eps * ls(-h)).mean()
    (up,) = torch.autograd.grad(loss, lp)
    for b in blocks:
        z, lq = log_q(b)
        (d[b],) = torch.autograd.grad(picked(lq, b), z, up[b])
    return {"loss": loss.detach(), "log_ratios": ratios.detach(), "logps": lp.detach(), "dlogits": d}
