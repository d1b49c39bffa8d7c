"""Losses over vocabulary logits at the edges of their inputs, against the float64 oracle (oracle/losses.py): values that
are not finite, masses far below a row's largest, labels outside the vocabulary, ids given twice.  The register kernels
and the streaming kernel are reached by the number of rows (streamed: two rows an SM, more than 32 KiB each)."""

import numpy as np
import pytest
import torch

from oracle import losses as oracle

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


def _logits(n, V, dtype, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(n, V, generator=g, device="cuda")).to(dtype)


def _np(t):
    return t.detach().double().cpu().numpy()


def _cuda(*arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


def _device_error():
    import ctypes

    from kdn_b200 import _lib

    code = ctypes.c_int(0)
    assert _lib.load().kdn_device_error(_lib.stream_handle(torch.device("cuda:0")), ctypes.byref(code)) == 0
    return code.value


# ------------------------------------------------------------------------------------------------- NaN in an input
def test_oracle_passes_a_nan_on():
    z, y = np.zeros((3, 4)), np.array([0, 1, -100])
    for bad in ("old", "adv"):
        f = dict(old=np.full(3, -1.0), adv=np.ones(3))
        f[bad][:] = np.nan
        loss, logps, H, d = oracle.policy_loss(z, y, f["old"], f["adv"])
        assert np.isnan(loss) and np.isnan(d[:2]).all() and (d[2] == 0).all()


@gpu
@pytest.mark.parametrize("n,V", [(6, 300), (300, 700), (2, 131072), (300, 16411), (300, 80003)])
@pytest.mark.parametrize("name", ["old_logps", "advantages", "ref_logps"])
@pytest.mark.parametrize("entropy", [0.0, 0.01])
def test_a_nan_in_a_policy_input_reaches_loss_and_gradient(n, V, name, entropy):
    """In a row that counts; in rows that do not (ignored, of weight zero) it changes nothing."""
    import kdn_b200 as kdn

    rng = np.random.default_rng(n + V)
    z = _logits(n, V, torch.bfloat16, seed=V)
    y = rng.integers(0, V, n)
    w = (0.5 + rng.random(n).astype(np.float32)) / n
    dead = 1 % n
    if n > 2:
        y[2], w[dead] = -100, 0.0
    yd, wd = _cuda(y, w)
    logp = kdn.token_logprobs(z, yd)
    given = dict(old_logps=logp - 0.1, advantages=torch.full_like(logp, 1.5), ref_logps=logp + 0.1)
    call = lambda f, **kw: f(z, yd, given["old_logps"], given["advantages"], ref_logps=given["ref_logps"], kl_coef=0.1,
                             entropy_coef=entropy, **kw)
    clean = call(kdn.policy_loss_and_grad, weights=wd)
    if n > 2:
        given[name][[dead, 2]] = float("nan")
        again = call(kdn.policy_loss_and_grad, weights=wd)
        assert torch.equal(again[0], clean[0]) and torch.equal(again[3], clean[3])
    at = n - 1
    given[name][at] = float("nan")
    for weights in (wd, None):
        loss, logps, H, d = call(kdn.policy_loss_and_grad, weights=weights)
        assert torch.isnan(loss)
        assert torch.isnan(d[at]).all()
        assert torch.equal(logps, clean[1]) and torch.equal(H, clean[2])
        if weights is not None:
            assert torch.equal(d[:at], clean[3][:at])
        assert torch.isnan(call(kdn.policy_loss, weights=weights)[0])
        want = oracle.policy_loss(_np(z[at:]), y[at:], _np(given["old_logps"][at:]), _np(given["advantages"][at:]),
                                  _np(given["ref_logps"][at:]), kl_coef=0.1, entropy_coef=entropy)
        assert np.isnan(want[0]) and np.isnan(want[3]).all()


@gpu
def test_a_ratio_that_overflows_times_no_advantage_is_nothing():
    import kdn_b200 as kdn

    z, y = _logits(4, 300, torch.float32), np.array([3, 5, 7, 9])
    yd, = _cuda(y)
    adv = np.array([0.0, 1.0, 0.0, -0.0], np.float32)
    old = _np(kdn.token_logprobs(z, yd)).astype(np.float32) - np.array([200, 200, 0, 100], np.float32)
    o, a = _cuda(old, adv)
    loss, _, _, d = kdn.policy_loss_and_grad(z, yd, o, a)
    want = oracle.policy_loss(_np(z), y, old, adv)
    assert abs(want[0] + 1.2 / 4) < 1e-6 and abs(float(loss) - want[0]) < 1e-6  # the one clipped ratio, 1 + 0.2
    assert not want[3].any() and not d.any()


# -------------------------------------------------------------------------------- a student's mass far below its top
def _rest_reference(z, T, t, ids, lse):
    """One row in float64, in logarithms throughout: the divergence, p and q at the ids, p_r and log q_r of what is
    left, log q outside relative to q_r."""
    lq = z / T - np.logaddexp.reduce(z / T)
    p = np.exp(t / T - lse)
    outside = np.ones(z.size, bool)
    outside[ids] = False
    p_r, log_qr = max(0.0, 1.0 - p.sum()), np.logaddexp.reduce(lq[outside])
    kl = (p * (t / T - lse - lq[ids])).sum() + (p_r * (np.log(p_r) - log_qr) if p_r > 0 else 0.0)
    return kl, p, np.exp(lq[ids]), p_r, log_qr, outside, lq - log_qr


def test_oracle_of_a_far_rest():
    rng = np.random.default_rng(0)
    n, V, K = 4, 30, 5
    z = rng.standard_normal((n, V))
    ids = np.stack([rng.permutation(V)[:K] for _ in range(n)])
    for r, drop in enumerate((5.0, 300.0, 1e4, 1e6)):
        outside = np.ones(V, bool)
        outside[ids[r]] = False
        z[r, outside] -= drop
    t = rng.standard_normal((n, K))
    lse = np.logaddexp.reduce(t, axis=1) + 0.3
    loss, kl, d = oracle.distillation_loss(z, t, ids, lse)
    for r in range(n):
        want, p, q, p_r, log_qr, outside, rel = _rest_reference(z[r], 1.0, t[r], ids[r], lse[r])
        assert abs(kl[r] - want) <= 1e-12 * abs(want)
        total = p.sum() + p_r
        assert np.allclose(d[r][outside] * n, total * np.exp(rel[outside] + log_qr) - p_r * np.exp(rel[outside]), 1e-11, 0)
        # the divergence moves by -p_r softmax of the outside along them, however far they lie
        step = np.where(outside, rng.standard_normal(V), 0.0)
        f = lambda h: oracle.distillation_loss(z[r:r + 1] + h * step, t[r:r + 1], ids[r:r + 1], lse[r:r + 1])[1][0]
        h = 1e-4
        assert abs((f(h) - f(-h)) / (2 * h) - (d[r] * n * step).sum()) <= 1e-6 + 1e-15 * abs(want) / h


@gpu
@pytest.mark.parametrize("drop", [20.0, 60.0, 86.5, 87.2, 87.8, 100.0, 1e4])
@pytest.mark.parametrize("n,V,K,dtype,T", [
    (9, 50, 40, torch.float32, 1.0), (5, 700, 6, torch.bfloat16, 1.0), (7, 4099, 64, torch.float32, 0.5),
    (2, 131072, 300, torch.bfloat16, 1.0), (300, 16411, 40, torch.bfloat16, 1.0), (300, 8200, 128, torch.float32, 2.0),
    (297, 80003, 33, torch.float32, 1.0)])
def test_a_rest_far_below_the_ids(n, V, K, dtype, T, drop):
    """Finite logits outside the teacher's ids, however far below the row's largest (peaked rows, small temperatures,
    finite masks): the divergence is finite, and the gradient outside is -w T p_r softmax(outside).  Rows 0 and 1: one
    entry outside is left, and none, where the divergence is infinite and the gradient outside zero.

    Tolerances: exponents (z - m) / T and t / T - lse carry 2^-23 of their size, exponentials and sums 2^-17 in all (see
    test_losses.py).  p_r is one minus a sum of p: delta absolutely, and log(p_r / q_r) multiplies it."""
    import kdn_b200 as kdn

    rng = np.random.default_rng(n + V + K)
    ids = np.stack([rng.permutation(V)[:K] for _ in range(n)])
    z = _logits(n, V, torch.float32, seed=V, scale=2.0)
    top = torch.full((n, V), -drop * T, device="cuda")
    idd, = _cuda(ids)
    top.scatter_(1, idd, 3.0)
    z = (z + top).to(dtype)
    z.scatter_(1, idd, (torch.randn(n, K, device="cuda", generator=torch.Generator("cuda").manual_seed(1))).to(dtype))
    one = (ids[0, 0] + 1) % V
    while one in ids[0]:
        one = (one + 1) % V
    keep = torch.zeros(2, V, dtype=torch.bool, device="cuda").scatter_(1, idd[:2], True)
    keep[0, one] = True
    z[:2] = torch.where(keep, z[:2], -float("inf"))
    t = np.sort(2.0 * rng.standard_normal((n, K)), axis=1)[:, ::-1].astype(np.float32).copy()
    lse = (np.logaddexp.reduce(t.astype(np.float64) / T, axis=1) - np.log(0.6 + 0.3 * rng.random(n))).astype(np.float32)
    w = ((0.5 + rng.random(n)) / n).astype(np.float32)
    td, ld, wd = _cuda(t, lse, w)
    loss, kl, d = kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld, weights=wd, temperature=T)
    plain = kdn.distillation_loss(z, td, idd, teacher_lse=ld, weights=wd, temperature=T)
    assert torch.equal(plain[0], loss) and torch.equal(plain[1], kl) and float(loss) == float("inf")
    got, g = _np(kl), _np(d)
    assert got[1] == np.inf and np.isfinite(g[1]).all()
    outside = np.ones(V, bool)
    outside[ids[1]] = False
    assert (g[1][outside] == 0).all()
    delta = 2.0 ** -23 * (np.abs(t).max() / T + 20) + 2.0 ** -17
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    rows = range(n) if n < 50 else [0, *range(2, n, 13), n - 1]
    for r in rows:
        if r == 1:
            continue
        zr = _np(z[r])
        want, p, q, p_r, log_qr, out, rel = _rest_reference(zr, T, t[r].astype(np.float64), ids[r], float(lse[r]))
        X = 2.0 ** -23 * (zr.max() - zr[np.isfinite(zr)].min()) / T + 2.0 ** -17
        assert abs(got[r] - want) <= 2 * X + delta * (abs(np.log(p_r) - log_qr) + 2)
        c, total = float(w[r]) * T, p.sum() + p_r
        ref = c * (total * np.exp(rel[out] + log_qr) - p_r * np.exp(rel[out]))
        part = c * (total * np.exp(rel[out] + log_qr) + p_r * np.exp(rel[out]))
        fin = rel[out][np.isfinite(rel[out])]
        share = 4 * (2.0 ** -23 * (fin.max() - fin.min()) + 2.0 ** -17 + delta / p_r)
        assert (np.abs(g[r][out] - ref) <= part * share + np.abs(ref) * half + 1e-37).all()
        ref = c * (q * total - p)
        assert (np.abs(g[r][ids[r]] - ref) <= 4 * c * (q + p) * (X + delta) + np.abs(ref) * half + 1e-37).all()


@gpu
@pytest.mark.parametrize("n,V,dtype", [(5, 700, torch.float32), (3, 131072, torch.bfloat16), (300, 16411, torch.bfloat16)])
def test_a_teacher_without_a_rest_and_a_student_with_a_mask(n, V, dtype):
    """All of the teacher's mass lies in its entries (one minus its sum is rounding alone) and the student's other logits
    are masked, by -inf or by the type's lowest value: the divergence is that over the entries."""
    import kdn_b200 as kdn

    K = 40
    rng = np.random.default_rng(V)
    ids = np.stack([rng.permutation(V)[:K] for _ in range(n)])
    idd, = _cuda(ids)
    for mask in (-float("inf"), torch.finfo(dtype).min, -1e30):
        z = torch.full((n, V), mask, device="cuda").to(dtype)
        z.scatter_(1, idd, _logits(n, K, dtype, seed=5, scale=2.0))
        t = (2.0 * rng.standard_normal((n, K))).astype(np.float32)
        lse = np.logaddexp.reduce(t.astype(np.float64), axis=1).astype(np.float32)
        td, ld = _cuda(t, lse)
        loss, kl, d = kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld)
        want = oracle.distillation_loss(np.take_along_axis(_np(z), ids, 1), t, np.tile(np.arange(K), (n, 1)))
        assert np.abs(_np(kl) - want[1]).max() <= 2.0 ** -16
        # p_r, at most 2^-20, is left out
        g = np.take_along_axis(_np(d), ids, 1)
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
        assert (np.abs(g - want[2]) <= 2.0 ** -16 / n + half * np.abs(want[2])).all()
        assert torch.equal(d.scatter(1, idd, 0.0), torch.zeros_like(d))


# ------------------------------------------------------------------------------------ labels outside the vocabulary
@gpu
@pytest.mark.parametrize("n,V", [(9, 300), (700, 300), (300, 16411)])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_labels_outside_the_vocabulary_count_as_ignored_ones(n, V, index):
    """In the mean over the rows that count and in a sequence's length, too: equal bits."""
    import kdn_b200 as kdn

    rng = np.random.default_rng(n)
    z = _logits(n, V, torch.bfloat16, seed=1)
    wrong, right = (torch.from_numpy(rng.integers(0, V, n)).cuda().to(index) for _ in range(2))
    wrong[1::4], wrong[2::4], wrong[3::8] = V, -7, -100
    right = torch.where((wrong < 0) | (wrong >= V), -100, wrong)
    old = kdn.token_logprobs(z, right) - 0.1
    adv = torch.ones_like(old)
    assert _device_error() == 0
    for call in (lambda y: kdn.policy_loss_and_grad(z, y, old, adv),
                 lambda y: kdn.policy_loss(z, y, old, adv),
                 lambda y: kdn.preference_loss_and_grad(z, y, torch.tensor([0, n // 3, n], device="cuda"), old + 0.3,
                                                        beta=0.5, length_normalised=True)):
        want = call(right)
        assert _device_error() == 0
        got = call(wrong)
        assert _device_error() == 1
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    some = int((right >= 0).sum())
    loss, _, _, d = kdn.policy_loss_and_grad(z, wrong, old, adv, clip_high=1e9)
    assert _device_error() == 1
    assert abs(float(loss) + np.exp(0.1)) < 1e-4  # every ratio is e^0.1: so is their mean, over `some` of n rows
    assert 0 < some < n


# ------------------------------------------------------------------------------------------------- ids given twice
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,K", [(64, 4100, 128), (64, 4100, 200), (3, 131072, 1024), (300, 16411, 128)])
def test_an_id_given_twice_gives_equal_bits(n, V, K, dtype):
    """Whatever warps its entries belong to: 3 and 100, 7 and 40, 9 and the last."""
    import kdn_b200 as kdn

    rng = np.random.default_rng(K)
    z = _logits(n, V, dtype, seed=3)
    ids = np.stack([rng.permutation(V)[:K] for _ in range(n)])
    ids[:, 100], ids[:, 40], ids[:, -1] = ids[:, 3], ids[:, 7], ids[:, 9]
    t = (2.0 * rng.standard_normal((n, K))).astype(np.float32)
    lse = (np.logaddexp.reduce(t.astype(np.float64), axis=1) + 0.2).astype(np.float32)
    td, idd, ld = _cuda(t, ids, lse)
    want = kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld)
    ref = oracle.distillation_loss(_np(z), t, ids, lse)
    assert np.abs(_np(want[1]) - ref[1]).max() <= 30 * (2.0 ** -17 + 2.0 ** -23 * 60)
    for _ in range(100):
        got = kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


# ------------------------------------------------------------------------------------------------- autograd's surface
@gpu
def test_forward_mode_is_refused():
    """A tangent of the logits is not dropped."""
    import torch.autograd.forward_ad as fwad

    import kdn_b200 as kdn

    z, y, f = _logits(4, 33, torch.float32), torch.arange(4, device="cuda"), torch.zeros(4, device="cuda")
    cu, ids = torch.tensor([0, 2, 4], device="cuda"), torch.arange(8, device="cuda").view(4, 2)
    st = torch.ones(4, 2, device="cuda")
    calls = [lambda x: kdn.token_logprobs(x, y), lambda x: kdn.token_logprobs_backward(x, y, st, f),
             lambda x: kdn.policy_loss(x, y, f, f), lambda x: kdn.policy_loss_and_grad(x, y, f, f),
             lambda x: kdn.preference_loss(x, y, cu), lambda x: kdn.preference_loss_and_grad(x, y, cu),
             lambda x: kdn.distillation_loss(x, z[:, :2], ids), lambda x: kdn.distillation_loss_and_grad(x, z[:, :2], ids)]
    for call in calls:
        call(z)
        with fwad.dual_level():
            call(z)
            for x in (z, z.detach().requires_grad_()):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(fwad.make_dual(x, torch.ones_like(z)))


@gpu
@pytest.mark.parametrize("grad", [False, True])
def test_outputs_of_a_call_are_tensors_of_their_own(grad):
    """Writing to one in place does not invalidate a graph that has kept another."""
    import kdn_b200 as kdn

    n = 6
    z = _logits(n, 33, torch.float32).requires_grad_(grad)
    y, f = torch.arange(n, device="cuda"), torch.zeros(n, device="cuda")
    cu, ids = torch.tensor([0, 2, n], device="cuda"), torch.arange(2 * n, device="cuda").view(n, 2)
    for call in (lambda: kdn.policy_loss(z, y, f, f), lambda: kdn.preference_loss(z, y, cu),
                 lambda: kdn.distillation_loss(z, z.detach()[:, :2].contiguous(), ids),
                 lambda: kdn.policy_loss_and_grad(z.detach(), y, f, f)):
        count = len(call())
        for kept in range(count):
            for written in range(count):
                if written == kept:
                    continue
                out = [o.detach() if o.requires_grad else o for o in call()]
                w = torch.ones_like(out[kept]).requires_grad_()
                kept_value = out[kept].clone()
                loss = (w * out[kept]).sum()
                out[written].mul_(2.0)
                loss.backward()
                assert torch.equal(w.grad, kept_value)


# ------------------------------------------------------------------------------------------- the rest of the teacher
@gpu
@pytest.mark.parametrize("n,V,K,dtype", [(5, 700, 6, torch.float32), (40, 4099, 200, torch.bfloat16),
                                         (300, 16411, 64, torch.bfloat16), (300, 8200, 20, torch.float32)])
@pytest.mark.parametrize("T", [1.0, 0.7, 2.0])
@pytest.mark.parametrize("offset", [0.0, 1000.0])
def test_the_rest_of_the_teacher_is_as_exact_as_its_inputs(n, V, K, dtype, T, offset):
    """t / T - lse of two numbers however large: its error is that of the difference.  With entries of |t / T - lse| below
    16 for all but 2^-20 of the mass, each rounded twice (2^-21 each), an exponential of 2^-22 and a sum of up to 256, 1 - P
    is within delta = 2^-19; log(p_r / q_r) multiplies it."""
    import kdn_b200 as kdn

    rng = np.random.default_rng(K)
    z = _logits(n, V, dtype, seed=11, scale=0.5)
    ids = np.stack([rng.permutation(V)[:K] for _ in range(n)])
    t = (T * rng.standard_normal((n, K)) + offset).astype(np.float32)
    lse = (np.logaddexp.reduce(t.astype(np.float64) / T, axis=1) - np.log(0.6 + 0.3 * rng.random(n))).astype(np.float32)
    td, idd, ld = _cuda(t, ids, lse)
    _, kl, d = kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld, weights=torch.ones(n, device="cuda"),
                                              temperature=T)
    zz, got, g, delta = _np(z), _np(kl), _np(d), 2.0 ** -19
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    for r in range(0, n, max(1, n // 25)):
        want, p, q, p_r, log_qr, out, rel = _rest_reference(zz[r], T, t[r].astype(np.float64), ids[r], float(lse[r]))
        eps = 2.0 ** -23 * (zz[r].max() - zz[r].min()) / T + 2.0 ** -19
        assert abs(got[r] - want) <= 2 * eps + delta * (abs(np.log(p_r) - log_qr) + 2)
        ref = T * (q * (p.sum() + p_r) - p)
        assert (np.abs(g[r][ids[r]] - ref) <= T * (2 * eps * q + 2 * delta * (p + q)) + np.abs(ref) * half).all()
        ref = T * np.exp(rel[out]) * ((p.sum() + p_r) * np.exp(log_qr) - p_r)
        size = T * np.exp(rel[out]) * ((p.sum() + p_r) * np.exp(log_qr) + p_r)
        assert (np.abs(g[r][out] - ref) <= size * (2 * eps + 2 * delta / p_r) + np.abs(ref) * half + 1e-37).all()
