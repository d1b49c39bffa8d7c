"""The streaming kernel of the losses over logits, at length: many rows for every CTA (or cluster), so that its queue of
32 rows, its 13 chunks, 8 buffers and 6 teachers' buffers are used again and again, requests of two rows and a short last
one, runs of ignored rows, rows that start at every place within 16 bytes (their ends are written into the ring by plain
stores, the slots then copied over), clusters of 2, 4 and 8.  Every element of every output against float64 on the GPU, in
blocks of rows.

Tolerances.  X = (row's largest - smallest logit) / T.  An exponent (z - m) / T carries 2^-24 of its size from each of its
two roundings; the base-2 exponential 2^-22; the sum, its logarithm (one unit of 2^-20) and the rounding of a result below
32 (2^-20) together 2^-19: a log-probability is within 2^-23 X + 2^-19.  Its roundings go to both sides, so that over the
rows their root mean square is below 2^-20 x 1.5, and the mean below 2^-22 (the exponential's own, which may be one-sided)
and three standard errors.  A gradient is a sum of a few terms, each a product of exponentials and of a coefficient that
carries the log-probability's error: within rho = 2 (2^-23 X + 2^-19) of the sum of their sizes, and half a unit of bf16,
2^-8 of the value.  What is left of the teacher, 1 - P, is within delta = 2^-19 absolutely (entries of |t / T - lse| below
20, each within 2^-20 of itself, and their sum)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

# rows, vocabulary, type, first element, distance of rows beyond V, temperature
SHAPES = [
    (5001, 16411, torch.bfloat16, 1, 0, 1.0),   # one CTA a row, 34 rows each, requests of two rows
    (3000, 33001, torch.float32, 0, 0, 0.7),    # the longest share, nine chunks
    (1500, 80003, torch.bfloat16, 3, 2, 1.0),   # clusters of two, 20 rows each
    (1200, 80003, torch.float32, 1, 0, 1.0),    # of four, 32 rows each
    (400, 300007, torch.bfloat16, 0, 0, 2.0),   # of eight, 22 rows each
    (5000, 16416, torch.bfloat16, 0, 0, 1.0),   # whole vectors throughout
]


def _logits(n, V, dtype, first, gap):
    """The view ends with its allocation: nothing may be read behind it."""
    g = torch.Generator(device="cuda").manual_seed(V + n)
    flat = torch.empty(first + n * (V + gap) - gap, device="cuda", dtype=dtype).normal_(0.0, 3.0, generator=g)
    return flat.as_strided((n, V), (V + gap, 1), first)


def _dead(n, rng):
    dead = rng.random(n) < 0.1
    dead[n // 3:n // 3 + min(200, n // 8)] = True
    dead[[0, n - 1]] = False
    return dead


def _blocks(n, V):
    step = max(1, (1 << 24) // V)
    return [slice(i, min(n, i + step)) for i in range(0, n, step)]


def _check_logps(got, want, live, X):
    d = (got.double() - want)[live]
    bound = 2.0 ** -23 * X[live] + 2.0 ** -19
    assert bool((d.abs() <= bound).all()), float((d.abs() / bound).max())
    rms = float(d.square().mean().sqrt())
    assert rms <= 1.5 * 2.0 ** -20
    assert abs(float(d.mean())) <= 2.0 ** -22 + 3 * rms / int(live.sum()) ** 0.5
    assert not got[~live].any()


def _check_grad(got, ref, size, rho, b):
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    bad = (got.double() - ref).abs() > size * rho + ref.abs() * half + 1e-37
    assert not bool(bad.any()), (b.start, bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), ref[bad][:4].tolist())


@pytest.mark.parametrize("n,V,dtype,first,gap,T", SHAPES)
@pytest.mark.parametrize("entropy_coef", [0.0, 0.01])
def test_policy_loss_at_length(n, V, dtype, first, gap, T, entropy_coef):
    import kdn_b200 as kdn

    rng = np.random.default_rng(n)
    z = _logits(n, V, dtype, first, gap)
    g = torch.Generator(device="cuda").manual_seed(7)
    dead = torch.from_numpy(_dead(n, rng)).cuda()
    y = torch.randint(V, (n,), device="cuda", generator=g)
    live = ~dead
    logp, X = torch.empty(n, dtype=torch.float64, device="cuda"), torch.empty(n, dtype=torch.float64, device="cuda")
    H = torch.empty_like(logp)
    for b in _blocks(n, V):
        x = z[b].double() / T
        lq = torch.log_softmax(x, -1)
        logp[b] = lq.gather(1, y[b, None])[:, 0]
        H[b] = -(lq.exp() * lq).sum(-1)
        X[b] = x.amax(-1) - x.amin(-1)
    ratio = torch.exp(0.3 * torch.randn(n, device="cuda", generator=g, dtype=torch.float64))
    for edge in (0.8, 1.2):  # the gradient jumps there
        ratio = torch.where((ratio - edge).abs() < 1e-3, edge + 2e-3, ratio)
    old = (logp - ratio.log()).float()
    adv = torch.randn(n, device="cuda", generator=g)
    ref = (logp + 0.3 * torch.randn(n, device="cuda", generator=g, dtype=torch.float64)).float()
    labels = torch.where(dead, -100, y)
    kw = dict(ref_logps=ref, kl_coef=0.05, entropy_coef=entropy_coef, temperature=T)
    loss, logps, ent, d = kdn.policy_loss_and_grad(z, labels, old, adv, **kw)
    plain = kdn.policy_loss(z, labels, old, adv, **kw)
    assert torch.equal(plain[0], loss) and torch.equal(plain[1], logps) and torch.equal(plain[2], ent)
    again = kdn.policy_loss_and_grad(z, labels, old, adv, **kw)
    assert torch.equal(again[0], loss) and torch.equal(again[3], d)
    _check_logps(logps, logp, live, X)
    eps = 2.0 ** -23 * X + 2.0 ** -19
    assert bool(((ent.double() - H).abs()[live] <= (eps * (2 + np.log(V)))[live]).all()) and not ent[dead].any()
    w, a, r = 1.0 / int(live.sum()), adv.double(), torch.exp(logp - old.double())
    gap_ = ref.double() - logp
    clipped = r.clamp(0.8, 1.2) * a
    each = -torch.minimum(r * a, clipped) + 0.05 * (torch.expm1(gap_) - gap_) - entropy_coef * H
    slope = torch.where(r * a <= clipped, -r * a, 0.0)
    kl = -0.05 * torch.expm1(gap_)
    size = (r * a).abs() + 0.05 * gap_.exp()
    assert abs(float(loss) - w * float(each[live].sum())) <= w * float(
        ((size + 0.05 + entropy_coef * (2 + np.log(V))) * eps * 2)[live].sum()) + 2.0 ** -23 * abs(float(loss))
    for b in _blocks(n, V):
        lq = torch.log_softmax(z[b].double() / T, -1)
        q = lq.exp()
        at = torch.zeros_like(q).scatter_(1, y[b, None], 1.0)
        c, e = ((slope + kl) * w / T)[b, None], entropy_coef * w / T
        want = c * (at - q) + e * q * (lq + H[b, None])
        parts = ((size * w / T)[b, None] * (at + q) + e * q * (lq.abs() + H[b, None] + 1.0))
        want, parts = (torch.where(live[b, None], t, 0.0) for t in (want, parts))
        _check_grad(d[b], want, parts, 2 * eps[b, None], b)


@pytest.mark.parametrize("n,V,dtype,first,gap,T", SHAPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("K", [33, 128])
def test_distillation_loss_at_length(n, V, dtype, first, gap, T, tail, K):
    import kdn_b200 as kdn

    rng = np.random.default_rng(n + K)
    z = _logits(n, V, dtype, first, gap)
    g = torch.Generator(device="cuda").manual_seed(9)
    dead = torch.from_numpy(_dead(n, rng)).cuda()
    live = ~dead
    lo = torch.arange(K, device="cuda") * V // K
    hi = torch.arange(1, K + 1, device="cuda") * V // K
    ids = lo + (torch.rand(n, K, device="cuda", generator=g) * (hi - lo)).long()
    ids[:, 0], ids[:, K - 1] = 0, V - 1  # the row's ends
    ids = ids.gather(1, torch.argsort(torch.rand(n, K, device="cuda", generator=g), 1))
    t = 2.0 * torch.randn(n, K, device="cuda", generator=g)
    lse = (torch.logsumexp(t.double() / T, -1) - torch.log(0.6 + 0.3 * torch.rand(n, device="cuda", generator=g))).float()
    w = (0.5 + torch.rand(n, device="cuda", generator=g)) / n
    given = torch.where(dead[:, None], -1, ids)
    kw = dict(teacher_lse=lse if tail else None, weights=w, temperature=T)
    loss, kl, d = kdn.distillation_loss_and_grad(z, t, given, **kw)
    plain = kdn.distillation_loss(z, t, given, **kw)
    assert torch.equal(plain[0], loss) and torch.equal(plain[1], kl)
    again = kdn.distillation_loss_and_grad(z, t, given, **kw)
    assert torch.equal(again[0], loss) and torch.equal(again[2], d)
    assert not kl[dead].any()
    delta, total = 2.0 ** -19, torch.zeros((), dtype=torch.float64, device="cuda")
    for b in _blocks(n, V):
        x = z[b].double() / T
        X = (x.amax(-1) - x.amin(-1))[:, None]
        eps = 2.0 ** -23 * X + 2.0 ** -19
        lq = torch.log_softmax(x, -1)
        lp = torch.log_softmax(t[b].double() / T, -1) if not tail else t[b].double() / T - lse[b, None].double()
        p, at = lp.exp(), lq.gather(1, ids[b])
        want = (p * (lp - at)).sum(-1)
        P = p.sum(-1, keepdim=True)
        bound = 2 * eps[:, 0] + 2 * delta
        c = (w[b, None].double() * T)
        q = lq.exp()
        grad, parts = c * q, c * q
        if tail:
            rest = 1.0 - P
            log_rest = torch.logsumexp(lq.scatter(1, ids[b], -float("inf")), -1, keepdim=True)
            want = want + (rest * (rest.log() - log_rest))[:, 0]
            bound = bound + delta * (rest.log() - log_rest).abs()[:, 0]
            other = c * rest * (lq - log_rest).exp()
            grad, parts = grad - other, parts + other * (1 + delta / rest / eps)
        atids = c * (at.exp() - p)
        grad, parts = grad.scatter(1, ids[b], atids), parts.scatter(1, ids[b], c * (at.exp() + p * (1 + delta / eps)))
        ok = live[b]
        assert bool(((kl[b].double() - want).abs() <= bound)[ok].all())
        total += (w[b].double() * want)[ok].sum()
        grad, parts = (torch.where(ok[:, None], v, 0.0) for v in (grad, parts))
        _check_grad(d[b], grad, parts, 2 * eps, b)
    assert abs(float(loss) - T * T * float(total)) <= 2.0 ** -16 * T * T
